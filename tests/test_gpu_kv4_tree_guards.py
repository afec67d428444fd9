"""GPU: attention of drafted tokens with starts and lengths of any value, its
outputs inside larger buffers: which rows are written, with what, and that nothing
else is.

Tolerances as in test_gpu_kv4_tree_parts.py."""
import numpy as np
import pytest
import torch

from tests import block_ref as ref
from tests.test_gpu_kv4 import filled, np64, queries, strided
from tests.test_gpu_kv4_tree import attend
from sili__new_amd import device as dev

pytestmark = pytest.mark.gpu

MARGIN, MOST = 80, 2 ** 31 - 1


def owned(start, r, tokens, max_new):
    """Request r's first row, its tokens by q_start, and how many rows it computes."""
    first, upto = start[r], start[r + 1]
    if first < 0 or upto <= first:
        return 0, 0, 0
    return first, upto - first, max(0, min(upto - first, max_new, tokens - first))


def keys_of(mask, new, length, window, cap):
    """The keys below cap that a token sees, whatever the lengths: exact integers, nothing of their size."""
    length = max(length, 0)
    base, bits = length - new, [j for j in range(min(new, 64)) if mask >> j & 1]
    begin = base + len(bits) - window if window else 0
    drafted = bits[-window:] if window else bits
    return [k for k in range(cap) if begin <= k < base] + [base + j for j in drafted if 0 <= base + j < cap]


@pytest.mark.parametrize("dtype,group", [(torch.float32, 1), (torch.bfloat16, 2), (torch.bfloat16, 20), (torch.float16, 5)])
@pytest.mark.parametrize("start,lens", [([0, 70, 74], [300, 90]), ([0, 4, MOST], [100, 90]), ([-1, 4, 6], [100, 90]), ([3, 1, 6], [100, 90]),
                                        ([0, 4, 6], [-7, MOST]), ([0, 4, 6], [MOST, -2 ** 31]), ([0, 0, 6], [12, 3]), ([2, 4, 5], [0, 1]),
                                        ([6, 6, 6], [50, 50]), ([5, MOST, 6], [90, 90]), ([-2 ** 31, MOST, 5], [60, 70]), ([0, 3, 6], [111, 96])])
def test_rows_written_and_rows_left(hip, start, lens, dtype, group):
    heads, d, page = 2, 64, 16
    host, gpu, table = filled(np.array([112, 96]), heads, page, d, 7)
    t = 76 if start[1] == 70 else 6
    rng = np.random.default_rng(t + group)
    masks = [int(m) | 1 << i % 64 for i, m in enumerate(rng.integers(0, 2 ** 63, t))]
    hq = heads * group
    q = queries(t, hq, d, dtype, 4)
    for window in (0, 3, 30):
        for max_new in (64, 3):
            wide = torch.full((t + 2 * MARGIN, hq, d), 7.0, device="cuda").to(dtype)
            sums = torch.full((t + 2 * MARGIN, hq), 7.0, device="cuda")
            s = attend(gpu, q, masks, [0, t], [1], table[:1], max_new=1)  # the buffers of a call; its sizes and values follow
            a = s["args"]
            i32 = lambda v: torch.from_numpy(np.array(v, np.int64).astype(np.int32)).cuda()  # noqa: E731
            keep = dict(start=i32(start), lens=i32(lens), table=i32(table))
            a.q_start, a.kv_lens, a.block_table, a.table_width = *(keep[k].data_ptr() for k in ("start", "lens", "table")), table.shape[1]
            a.requests, a.max_new, a.max_len, a.window = 2, max_new, MOST, window
            a.out, a.out_token_stride, a.out_head_stride = strided(wide[MARGIN:])
            a.lse = sums[MARGIN:].data_ptr()
            a.workspace_bytes = dev.kv4_attend_tree_workspace(a)
            work = torch.full((a.workspace_bytes + 4096,), 255, dtype=torch.uint8, device="cuda")
            a.workspace = work.data_ptr()
            torch.cuda.synchronize()
            dev.kv4_attend_tree(a, s["masks"].data_ptr())
            torch.cuda.synchronize()
            assert bool((work[a.workspace_bytes:] == 255).all())
            out, lse = np64(wide), np64(sums)
            left = np.ones(t + 2 * MARGIN, bool)
            for r in range(2):
                first, new, n = owned(start, r, t, max_new)
                cap = min(max(lens[r], 0), table.shape[1] * page)
                for i in range(n):
                    row = MARGIN + first + i
                    left[row] = False
                    keys = np.array(keys_of(masks[first + i], new, lens[r], window, cap), int)
                    held = table[r, keys // page]
                    keys, held = keys[held >= 0], held[held >= 0]
                    for h in range(hq):
                        if not len(keys):
                            assert np.isneginf(lse[row, h]) and not out[row, h].any()
                            continue
                        kk, vv = (ref.kv4_values(host, name, held, h // group, keys % page) for name in "kv")
                        x = np64(q[first + i, h])
                        score = kk @ x * d ** -0.5
                        p = np.exp(score - score.max())
                        want, size = p @ vv / p.sum(), p @ np.abs(vv) / p.sum()
                        reach = (np.abs(kk) @ np.abs(x)).max() * d ** -0.5
                        tol = (2 * reach * 2.0 ** -16 + 2.0 ** -15) * size
                        assert np.all(np.abs(out[row, h] - want) <= tol + ref.rounding(str(dtype)[6:], np.abs(want) + tol)), (window, max_new, r, i, h)
                        total = score.max() + np.log(p.sum())
                        assert abs(lse[row, h] - total) <= reach * 2.0 ** -16 + 2.0 ** -20 * (1 + abs(total))
            assert (out[left] == 7).all() and (lse[left] == 7).all()


def test_in_place_and_columns_of_one_buffer(hip):
    """out on q itself, beside it in one row, and with heads before tokens."""
    host, gpu, table = filled(np.array([300, 90]), 2, 16, 64, 3)
    start, lens, t, hq, d = [0, 40, 47], np.array([300, 90]), 47, 10, 64
    masks = [2 ** (i % 40 + 1) - 1 for i in range(40)] + [2 ** (i + 1) - 1 for i in range(7)]
    for dtype in (torch.float32, torch.bfloat16):
        q = queries(t, hq, d, dtype, 5)
        want = attend(gpu, q, masks, start, lens, table)
        mine = q.clone()
        s = attend(gpu, mine, masks, start, lens, table, out=mine)
        assert torch.equal(mine, want["out"]) and torch.equal(s["lse"], want["lse"])
        both = torch.zeros(t, 2 * hq * d, device="cuda").to(dtype)
        both[:, :hq * d] = q.reshape(t, -1)
        attend(gpu, both[:, :hq * d].view(t, hq, d), masks, start, lens, table, out=both[:, hq * d:].view(t, hq, d))
        assert torch.equal(both[:, hq * d:].reshape(t, hq, d), want["out"]) and torch.equal(both[:, :hq * d].reshape(t, hq, d), q)
        turned = torch.zeros(hq, 2 * t, d, device="cuda").to(dtype)
        turned[:, :t] = q.transpose(0, 1)
        attend(gpu, turned[:, :t].transpose(0, 1), masks, start, lens, table, out=turned[:, t:].transpose(0, 1))
        assert torch.equal(turned[:, t:].transpose(0, 1), want["out"])
