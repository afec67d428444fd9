"""GPU: outputs that are columns of the matrix that holds an input."""
import pytest
import torch

from sili__new_amd import device as dev
from tests.test_gpu_fp4_linear import BF16, F16, F32, check as check_linear, linear, random_weights, weights
from tests.test_gpu_logits import case, check as check_logits, constrain, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens", [1, 2, 8, 20, 130])
@pytest.mark.parametrize("first", [True, False])
def test_fp4_linear(hip, tokens, dtype, first):
    n_out, n_in, group = 200, 512, 64
    codes, scales = random_weights(n_out, n_in, group, F32, tokens)
    both = torch.full((tokens, n_in + n_out), 3.0, device="cuda").to(dtype)
    x, y = (both[:, :n_in], both[:, n_in:]) if first else (both[:, n_out:], both[:, :n_out])
    x.copy_(torch.randn(tokens, n_in, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda"))
    kept = x.clone()
    check_linear(linear(weights(codes, scales, group), x, dtype, y=y), codes, scales, group)
    assert torch.equal(x, kept)


def test_fp4_codes_beside_scales(hip):
    """A row's codes, then its scales, in one allocation."""
    n_out, n_in, group = 70, 256, 32
    rows = torch.randn(n_out, n_in, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    both = torch.zeros(n_out, n_in // 2 + 32, dtype=torch.uint8, device="cuda")
    codes, scales = both[:, :n_in // 2], both.view(F32)[:, n_in // 8:]
    apart = torch.zeros(n_out, n_in // 2, dtype=torch.uint8, device="cuda"), torch.zeros(n_out, n_in // group, device="cuda")
    torch.cuda.synchronize()
    for c, s in ((codes, scales), apart):
        dev.fp4_pack(dev.Fp4Pack(w=weights(c, s, group, n_in), dtype=dev.F32, rows=rows.data_ptr(), row_stride=n_in))
    torch.cuda.synchronize()
    assert torch.equal(codes, apart[0]) and torch.equal(scales, apart[1]) and bool(apart[0].any())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [513, 3000])
def test_logits_constrain(hip, vocab, dtype):
    rng, kw = case(3, [3, 1, 9], vocab, 60)
    z = logits(rng, 13, vocab, dtype)
    both = torch.full((13, 2 * vocab), 3.0, device="cuda").to(dtype)
    both[:, vocab:] = z
    t = constrain(both[:, vocab:], out=both[:, :vocab], **kw)
    check_logits(t, z, left=None, **kw)
    assert torch.equal(both[:, vocab:], z)
    turned = torch.full((13, vocab), 3.0, device="cuda").to(dtype)
    a = t["args"]
    a.out, a.out_stride = turned[12:].data_ptr(), -vocab  # the last row first
    torch.cuda.synchronize()
    dev.logits_constrain(a)
    torch.cuda.synchronize()
    assert torch.equal(turned.flip(0), both[:, :vocab])
