"""GPU: bf16 parts in attention of drafted tokens: q in three (fp32), two (f16) or
one (bf16), a softmax weight in three (fp32) or two, however many rows a request
has.

Tolerances, before any run.  Where all that the parts before hold cancels, as for
sili_kv4_attend: products, cancelling sums and scales (powers of two) are exact in
float32, so 2^-20 of the row for exp2, the sum over the keys and the division, and
one rounding to the type; a lost part is an error of the whole value.  Random
values: a score is off by at most 2^-16 of the sum of its terms' magnitudes
(float32 sums of up to 256 terms), its weight by twice that, relative; a weight's
second part is rounded at 2^-16 of it, its exp2 and the sums over up to a few
hundred keys leave as much again, so 2^-15 of the sum of the weighted values'
magnitudes in every type; the output is rounded once."""
import numpy as np
import pytest
import torch

from tests import block_ref, draft_ref as ref
from tests.test_gpu_kv4 import filled, new_cache, np64, queries, starts
from tests.test_gpu_kv4_parts import bf16, last_part
from tests.test_gpu_kv4_tree import attend, tree_masks

pytestmark = pytest.mark.gpu

TYPES = [(torch.float32, 3), (torch.float16, 2), (torch.bfloat16, 2)]
# rows of a request: up to a tile's parts, a tile, and two, four and more of them
ROWS = [(1, 3), (4, 2), (16, 1), (1, 16), (1, 17), (3, 11), (5, 13), (2, 64)]


@pytest.mark.parametrize("dtype,parts", TYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group,new", ROWS)
@pytest.mark.parametrize("context", [64, 3000])
def test_the_last_part_of_the_weights(hip, dtype, parts, d, group, new, context):
    """Scores of zero: every weight is its key's scale. Two keys, one cached and one drafted, that only differ in its
    last part and their sign."""
    heads, n, page = 2, context + new, 16
    pages = -(-n // page)
    host, _ = new_cache(pages, heads, page, d)
    rng = np.random.default_rng(group + new)
    table = rng.permutation(pages)[None]
    x, without = last_part(parts, heads, d)
    sign = rng.choice([0, 8], (heads, d))  # code 6 or -6
    for h in range(heads):
        for at, scale, code in zip((rng.integers(context), context), (x[h], without[h]), (7 + sign[h], 15 - sign[h])):
            p = table[0, at // page]
            host["v"][p, h, at % page // 16, :, at % 16] = (code[0::2] | code[1::2] << 4).astype(np.uint8)
            host["v_scale"][p, h, at % page] = scale
    masks = [1 | 1 << i for i in range(new)]
    q = torch.zeros(new, heads * group, d, device="cuda").to(dtype)
    s = attend({k: torch.from_numpy(v).cuda() for k, v in host.items()}, q, masks, starts([new]), np.array([n]), table)
    want, lse, _, _ = ref.attend_tree(host, np64(q), masks, starts([new]), [n], table, 1.0)
    assert np.all(np.abs(want) > 0)
    err = np.abs(np64(s["out"]) - want)
    assert np.all(err <= 2.0 ** -20 * np.abs(want) + block_ref.rounding(str(dtype)[6:], want))
    assert np.all(np.abs(np64(s["lse"]) - lse) <= 2.0 ** -20 * (1 + lse))


@pytest.mark.parametrize("dtype,parts", TYPES[:2])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group,new", ROWS)
def test_the_last_part_of_q(hip, dtype, parts, d, group, new):
    """q's earlier parts meet their opposites in channels of the same level: the scores hold the last part alone."""
    heads, context, page = 2, 40, 16
    n = context + new
    pages = -(-n // page)
    host, _ = new_cache(pages, heads, page, d)
    rng = np.random.default_rng(d + group + new)
    table = rng.permutation(pages)[None]
    j = np.arange(n)
    level = rng.choice([0.5, 1, 1.5, 2, 3, 4, 6, -0.5, -1, -1.5, -3, -6], (n, heads))
    codes = np.searchsorted(block_ref.LEVELS[:8], np.abs(level)) + 8 * (level < 0)
    slots = table[0, j // page] * page + j % page
    block_ref.kv4_store(host, slots, np.zeros((n, heads, d)), rng.normal(size=(n, heads, d)))
    host["k"][table[0, j // page], :, j % page] = (codes * 17).astype(np.uint8)[..., None]
    host["k_scale"][table[0, j // page], :, j % page] = rng.choice([0.5, 1.0, 2.0], (n, heads))
    x, without = last_part(parts, (new, heads * group), d)
    q = np.zeros((new, heads * group, d))
    for t in range(new):
        for h in range(heads * group):
            a = bf16(x[t, h])
            q[t, h, rng.permutation(d)[:3]] = x[t, h], -a, a - without[t, h]
    q = torch.from_numpy(q).cuda().to(dtype)
    masks, scale = tree_masks(rng, [new]), 2.0 ** (18 if parts == 3 else 8)
    s = attend({k: torch.from_numpy(v).cuda() for k, v in host.items()}, q, masks, starts([new]), np.array([n]), table, scale=scale)
    want, lse, size, _ = ref.attend_tree(host, np64(q), masks, starts([new]), [n], table, scale)
    most = np.abs(lse).max() + np.log(n)  # the largest score
    tol = (4 * 2.0 ** -22 * most + 2.0 ** -20) * size
    assert np.all(np.abs(np64(s["out"]) - want) <= tol + block_ref.rounding(str(dtype)[6:], np.abs(want) + tol))
    assert np.all(np.abs(np64(s["lse"]) - lse) <= 2.0 ** -20 * (1 + most))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group,new", ROWS)
@pytest.mark.parametrize("window", [0, 50])
def test_random_values_with_all_parts(hip, dtype, d, group, new, window):
    new = np.array([new, 1, max(1, new // 2)])
    lens = new + np.array([70, 0, 333])
    host, gpu, table = filled(lens, 2, 16, d, d + group)
    masks = tree_masks(np.random.default_rng(d + group), new)
    q = queries(int(new.sum()), 2 * group, d, dtype, 3)
    s = attend(gpu, q, masks, starts(new), lens, table, window)
    want, _, size, reach = ref.attend_tree(host, np64(q), masks, starts(new), lens, table, d ** -0.5, window)
    tol = (2 * reach * 2.0 ** -16 + 2.0 ** -15)[..., None] * size
    assert np.all(np.abs(np64(s["out"]) - want) <= tol + block_ref.rounding(str(dtype)[6:], np.abs(want) + tol))


@pytest.mark.parametrize("window", [0, 4100])
@pytest.mark.parametrize("longest", [4095, 4096, 4500])
@pytest.mark.parametrize("most", [64, 9])
def test_many_long_trees(hip, most, longest, window):
    """About the sizes from which a wave takes two tiles of rows: 32 requests of up to 1024 rows over 2 kv heads; requests without
    tokens, whose last tile of a pair is empty, of one token; a hidden page."""
    rng = np.random.default_rng(most + longest)
    new = rng.integers(1, 4, 32)
    new[[0, 1, 2, 3, 4]] = 5, 0, 1, most, min(most, 17)
    lens = new + rng.integers(0, 60, 32)
    lens[0], lens[3], lens[5] = longest, 300, longest - 1
    host, gpu, table = filled(lens, 2, 32, 128, 6)
    table = table.copy()
    table[0, 5], table[3, 1] = -1, len(host["k"])
    masks = tree_masks(rng, new)
    q = queries(int(new.sum()), 32, 128, torch.bfloat16, 4)
    s = attend(gpu, q, masks, starts(new), lens, table, window)
    want, lse, size, reach = ref.attend_tree(host, np64(q), masks, starts(new), lens, table, 128 ** -0.5, window)
    tol = (2 * reach * 2.0 ** -16 + 2.0 ** -15)[..., None] * size
    assert np.all(np.abs(np64(s["out"]) - want) <= tol + block_ref.rounding("bfloat16", np.abs(want) + tol))
    assert np.all(np.abs(np64(s["lse"]) - lse) <= reach * 2.0 ** -16 + 2.0 ** -20 * (1 + np.abs(lse)))
    again = attend(gpu, q, masks, starts(new), lens, table, window)
    assert torch.equal(s["out"], again["out"]) and torch.equal(s["lse"], again["lse"])
