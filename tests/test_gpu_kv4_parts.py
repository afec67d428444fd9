"""GPU: attention's bf16 parts.  fp32 queries and weights enter in three, f16
queries and the weights of f16 and bf16 in two; here all that the parts before
hold cancels, so a row is decided by its last part alone.

Tolerances, before any run.  The products, the sums that cancel and the scales
(powers of two) are exact in float32, so a score carries the rounding of scale *
log2(e) and of one product, 2^-22 in all, and its weight twice that; exp2, the
sum over the keys and the division add less than 2^-20 of the weights; one
rounding to the type.  A lost part is an error of the whole value."""
import numpy as np
import pytest
import torch

from tests import block_ref as ref
from tests.test_gpu_kv4 import attend, new_cache, np64

pytestmark = pytest.mark.gpu


def bf16(x):
    return torch.from_numpy(np.asarray(x, np.float32)).to(torch.bfloat16).double().numpy()


def last_part(parts, shape, seed):
    """Values whose last bf16 part is about 2^-9 (two) or 2^-18 (three) of them: -> x, x without it."""
    rng = np.random.default_rng(seed)
    a = bf16(1.02 + 0.95 * rng.random(shape))  # above 1, so that x lies in a's binade
    sign = rng.choice([-1.0, 1.0], shape)
    if parts == 2:
        return a + sign * 2.0 ** -9, a  # f16 holds it
    b = bf16(sign * 2.0 ** -9 * (1 + rng.random(shape) / 4))
    x = a + b + rng.choice([-1.0, 1.0], shape) * 2.0 ** -19
    assert (x.astype(np.float32) == x).all() and (bf16(x) == a).all() and (bf16(x - a) == b).all()
    return x, a + b


def close(s, host, start, lens, table, scale):
    want, lse, size, _ = ref.attend(host, np64(s["q"]), start, lens, table, scale, 1, 0)
    dtype = str(s["q"].dtype)[6:]
    most = np.abs(lse).max() + np.log(lens.max())  # the largest score
    tol = (4 * 2.0 ** -22 * most + 2.0 ** -20) * size
    assert np.all(np.abs(np64(s["out"]) - want) <= tol + ref.rounding(dtype, np.abs(want) + tol))
    assert np.all(np.abs(np64(s["lse"]) - lse) <= 2.0 ** -20 * (1 + most))
    return want


@pytest.mark.parametrize("dtype,parts", [(torch.float32, 3), (torch.float16, 2)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group,new", [(1, 1), (4, 1), (7, 1), (16, 1), (1, 4), (2, 30)])
def test_the_last_part_of_q(hip, dtype, parts, d, group, new):
    heads, n, page = 2, 45, 16
    rng = np.random.default_rng(d + group)
    host, _ = new_cache(3, heads, page, d)
    table = np.array([[2, 0, 1]])
    j = np.arange(n)
    # a key is one level in all its channels, at a scale that is a power of two
    level = rng.choice([0.5, 1, 1.5, 2, 3, 4, 6, -0.5, -1, -1.5, -3, -6], (n, heads))
    codes = np.searchsorted(ref.LEVELS[:8], np.abs(level)) + 8 * (level < 0)
    host["k"][table[0, j // page], :, j % page] = (codes * 17).astype(np.uint8)[..., None]
    host["k_scale"][table[0, j // page], :, j % page] = rng.choice([0.5, 1.0, 2.0], (n, heads))
    values, _ = new_cache(3, heads, page, d)
    ref.kv4_store(values, table[0, j // page] * page + j % page, np.zeros((n, heads, d)), rng.normal(size=(n, heads, d)))
    host["v"], host["v_scale"] = values["v"], values["v_scale"]
    x, without = last_part(parts, (new, heads * group), d)
    q = np.zeros((new, heads * group, d))
    for t in range(new):
        for h in range(heads * group):
            c = rng.permutation(d)[:3]
            a = bf16(x[t, h])
            q[t, h, c] = x[t, h], -a, a - without[t, h]
    q = torch.from_numpy(q).cuda().to(dtype)
    start, lens, scale = np.array([0, new]), np.array([n]), 2.0 ** (18 if parts == 3 else 8)
    s = attend({k: torch.from_numpy(v).cuda() for k, v in host.items()}, q, start, lens, table, scale=scale)
    want = close(s, host, start, lens, table, scale)
    # without the last part all scores would be equal
    flat, _, size, _ = ref.attend(host, np.zeros(q.shape), start, lens, table, scale, 1, 0)
    assert np.median(np.abs(want - flat) / (size + 1e-300)) > 2.0 ** -5


@pytest.mark.parametrize("dtype,parts", [(torch.float32, 3), (torch.float16, 2), (torch.bfloat16, 2)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("group,new", [(1, 1), (4, 1), (7, 1), (16, 1), (1, 4), (2, 30)])
def test_the_last_part_of_the_weights(hip, dtype, parts, d, group, new):
    """Scores of zero: every weight is its key's scale. Two keys that only differ in its last part and their sign."""
    heads, n, page = 3, 64 + new, 16
    host, _ = new_cache(6, heads, page, d)
    table = np.array([[5, 2, 0, 1, 4, 3]])
    x, without = last_part(parts, heads, d)
    rng = np.random.default_rng(group)
    sign = rng.choice([0, 8], (heads, d))  # code 6 or -6
    for h in range(heads):
        for at, scale, code in zip(rng.permutation(n - new)[:2], (x[h], without[h]), (7 + sign[h], 15 - sign[h])):
            p = table[0, at // page]
            host["v"][p, h, at % page // 16, :, at % 16] = (code[0::2] | code[1::2] << 4).astype(np.uint8)
            host["v_scale"][p, h, at % page] = scale
    q = torch.zeros(new, heads * group, d, device="cuda").to(dtype)
    start, lens = np.array([0, new]), np.array([n])
    s = attend({k: torch.from_numpy(v).cuda() for k, v in host.items()}, q, start, lens, table)
    want, lse, _, _ = ref.attend(host, np64(q), start, lens, table, 1.0, 1, 0)
    assert np.all(np.abs(want) > 0)
    err = np.abs(np64(s["out"]) - want)
    assert np.all(err <= 2.0 ** -20 * np.abs(want) + ref.rounding(str(dtype)[6:], want))
    assert np.all(np.abs(np64(s["lse"]) - lse) <= 2.0 ** -20 * (1 + lse))
