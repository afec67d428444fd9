"""GPU: long chunks whose query heads share kv heads, beside short requests of the
same batch, and scales of any sign."""
import numpy as np
import pytest
import torch

from tests.test_gpu_kv4 import attend, check, filled, queries, starts

pytestmark = pytest.mark.gpu


def batch(group):
    """Requests about the edge between few rows and many (256), in one call of 512 blocks or more."""
    edge = 256 // group
    new = np.array([300, 257, edge, edge + 1, 1, 280])
    return new, np.array([300, 700, 90, 411, 64, 270])


@pytest.mark.parametrize("heads,group,causal,window,page", [(8, 5, 1, 0, 16), (8, 5, 1, 70, 32), (8, 3, 0, 0, 48), (16, 2, 1, 300, 16), (3, 16, 1, 0, 16)])
def test_long_chunks(hip, heads, group, causal, window, page):
    new, lens = batch(group)
    host, gpu, table = filled(lens, heads, page, 128, page + group)
    table = table.copy()
    table[1, 2], table[5, 1] = -1, len(host["k"]) + 5
    t, hq = int(new.sum()), heads * group
    q = queries(t, hq, 128, torch.bfloat16, 3)
    s = attend(gpu, q, starts(new), lens, table, causal, window)
    check(host, s, starts(new), lens, table, causal, window)
    # q out of a fused projection at an odd offset, out with gaps, heads before tokens
    wide = torch.zeros(t, hq + 3, 130, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:hq + 1, 1:129] = q
    out = torch.full((hq, t, 136), 3.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    a = attend(gpu, wide[:, 1:hq + 1, 1:129], starts(new), lens, table, causal, window, out=out[..., :128])
    assert torch.equal(a["out"], s["out"]) and torch.equal(a["lse"], s["lse"]) and float((out[..., 128:].float() - 3).abs().max()) == 0


@pytest.mark.parametrize("scale", [0.0, -0.07, -1.0])
def test_scales_of_long_chunks(hip, scale):
    new, lens = batch(3)
    host, gpu, table = filled(lens, 8, 16, 128, 2)
    q = queries(int(new.sum()), 24, 128, torch.bfloat16, 5, 1.0)
    check(host, attend(gpu, q, starts(new), lens, table, scale=scale), starts(new), lens, table, scale=scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [0.0, -0.125, -2.0])
@pytest.mark.parametrize("d,group", [(64, 1), (128, 5), (256, 16)])
def test_scales(hip, dtype, scale, d, group):
    new, lens = np.array([1, 7, 2]), np.array([900, 60, 1])
    host, gpu, table = filled(lens, 2, 16, d, 2)
    q = queries(10, 2 * group, d, dtype, 5, 0.5)
    for window in (0, 33):
        s = attend(gpu, q, starts(new), lens, table, window=window, scale=scale)
        check(host, s, starts(new), lens, table, window=window, scale=scale)
