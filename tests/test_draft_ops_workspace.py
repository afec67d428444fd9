"""CPU: what the operators over drafted tokens ask for as workspace."""
import math
import os
import random
import subprocess
import sys

import pytest

from sili__new_amd import device as dev
from tests.test_draft_ops_host import attend, changed, linear

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

EMPTY_LINEAR = [dict(tokens=0), dict(w__n_out=0), dict(w__n_in=0), dict(tokens=0, w__n_out=0), dict(tokens=0, w__n_in=0), dict(tokens=20, w__n_out=0),
                dict(tokens=20, w__n_in=0)]
EMPTY_TREES = [dict(tokens=0), dict(requests=0), dict(max_new=0), dict(max_len=0), dict(table_width=0), dict(cache__n_pages=0)]


def test_an_empty_call_needs_none():
    """In a process of its own: a division by zero would end it."""
    code = ("from tests.test_draft_ops_workspace import *\n"
            "for kw in EMPTY_LINEAR:\n"
            "    for dtype in (dev.F32, dev.BF16, dev.F16): assert dev.fp4_linear_workspace(changed(linear, dtype=dtype, **kw)) == 0, kw\n"
            "for kw in EMPTY_TREES:\n"
            "    for dtype in (dev.F32, dev.BF16, dev.F16): assert dev.kv4_attend_tree_workspace(changed(attend, dtype=dtype, **kw)) == 0, kw\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr)


def few(tokens, n_out, n_in, group=128, dtype=dev.BF16):
    """The bytes of a call with those weights."""
    return dev.fp4_linear_workspace(changed(linear, tokens=tokens, dtype=dtype, w__n_out=n_out, w__n_in=n_in, w__group=group, w__codes_stride=n_in // 2,
                                            w__scales_stride=n_in // group))


def test_waves_share_outputs_only_where_a_block_holds_all_of_x():
    """4 rows of x (tokens times parts) at most: a block either holds all their inputs, and needs no workspace, or the inputs go
    to blocks that are joined, as many as 5 rows' do."""
    for dtype, parts in ((dev.BF16, 1), (dev.F16, 2), (dev.F32, 3)):
        for group in (32, 128):
            for tokens in range(1, 4 // parts + 1):
                for n_in in range(1024, 16385, 1024):
                    need = few(tokens, 1500, n_in, group, dtype)
                    if need:
                        assert need // tokens == few(5, 1500, n_in, group, dev.BF16) // 5, (dtype, group, tokens, n_in)
                    else:  # 112 KiB hold them beside 8 waves' codes and scales
                        assert tokens * parts * n_in * 2 <= (112 << 10) - 8 * 16 * (36 + 256 // group) * 4


@pytest.mark.parametrize("dtype", [dev.F32, dev.BF16, dev.F16])
@pytest.mark.parametrize("group", [32, 128])
def test_more_tokens_never_need_less(dtype, group):
    """A buffer for the most tokens does for fewer, which may split the inputs where those do not."""
    counts = list(range(0, 400)) + [511, 512, 513, 1000, 4096, 5000, 16384, 16385, 70000, (1 << 31) - 1]
    for n_out in (1, 16, 127, 129, 1000, 1500, 5120, 8192, 16384, 32768, 33000, 65536, 131071):
        for n_in in (group, 128, 640, 1024, 5120, 11264, 12288, 16384, 32768):
            sizes = [few(t, n_out, n_in, group, dtype) for t in counts]
            assert sizes == sorted(sizes), (n_out, n_in)
            assert sizes[-1] <= max(sizes[16], 32 << 20)  # of more than 16 tokens 512 blocks split at most


@pytest.mark.parametrize("dtype", [dev.F32, dev.BF16, dev.F16])
@pytest.mark.parametrize("window", [0, 1, 1000])
def test_smaller_trees_never_need_more(dtype, window):
    """A buffer for the largest step does for every step of fewer requests, tokens or keys."""
    rng = random.Random(window)
    log = lambda n: int(math.exp(rng.uniform(0, math.log(n + 1))))  # noqa: E731
    split = 0
    for _ in range(300):
        kv, group, d = rng.choice([1, 2, 5, 8, 40]), rng.choice([1, 2, 5, 16]), rng.choice([64, 128, 256])

        def need(r, n, t, length):
            return dev.kv4_attend_tree_workspace(changed(attend, dtype=dtype, window=window, cache__kv_heads=kv, q_heads=kv * group, cache__head_dim=d,
                                                         cache__n_pages=1 << 17, table_width=1 << 13, requests=r, max_new=n, tokens=t, max_len=length))

        r, n, length = log(256), log(64), log(131072)
        largest = need(r, n, r * n, length)
        for _ in range(20):
            fewer, less, shorter = rng.randint(1, r), rng.randint(1, n), rng.choice([length, log(length)])
            bytes_ = need(fewer, less, rng.randint(1, fewer * less), shorter)
            assert bytes_ <= largest, (kv, group, d, r, n, length, fewer, less, shorter)
            split += bytes_ > 0
        assert largest <= 20 << 20
    assert split > 300 or window == 1
