"""GPU: 4-bit weights about the sizes from which a call is cut another way.

Tolerances as in test_gpu_fp4_linear.py."""
import pytest
import torch

from sili__new_amd import device as dev
from tests import block_ref
from tests.test_gpu_fp4_linear import BF16, F16, F32, check, linear, random_weights, weights

pytestmark = pytest.mark.gpu


def run(n_out, n_in, group, tokens, dtype):
    codes, scales = random_weights(n_out, n_in, group, BF16, n_out + tokens)
    x = torch.randn(tokens, n_in, generator=torch.Generator(device="cuda").manual_seed(n_in), device="cuda").to(dtype)
    s = linear(weights(codes, scales, group), x, F32)
    check(s, codes, scales, group)
    assert torch.equal(s["y"], linear(weights(codes, scales, group), x, F32)["y"])


@pytest.mark.parametrize("dtype,tokens", [(BF16, 3), (BF16, 4), (F16, 1), (F16, 2), (F32, 1)])
@pytest.mark.parametrize("n_in", [11264, 11520, 15104, 15360, 16384, 16640])
def test_a_few_rows_of_x_that_a_block_holds_or_not(hip, n_in, dtype, tokens):
    for n_out, group in ((300, 128), (5120, 32)):
        run(n_out, n_in, group, tokens, dtype)


@pytest.mark.parametrize("tokens", [64, 65, 128, 129, 192, 193, 256])
@pytest.mark.parametrize("n_out,n_in,group", [(65408, 2048, 128), (65409, 2048, 64), (131000, 992, 32), (260, 349952, 128), (2049, 65600, 64)])
def test_tiles_of_tokens_in_pairs(hip, n_out, n_in, group, tokens):
    """About 8192 steps of 128 outputs, 128 tokens and 128 inputs; the products in 64 bits on the GPU."""
    codes, scales = random_weights(n_out, n_in, group, BF16, n_out + tokens)
    x = torch.randn(tokens, n_in, generator=torch.Generator(device="cuda").manual_seed(n_in), device="cuda").to(BF16)
    s = linear(weights(codes, scales, group), x, F32)
    levels = torch.from_numpy(block_ref.LEVELS).cuda()
    w = torch.stack([levels[(codes & 15).long()], levels[(codes >> 4).long()]], -1).view(n_out, n_in // group, group) * scales.double()[..., None]
    w = w.view(n_out, n_in).t().contiguous()
    want, size = x.double() @ w, x.double().abs() @ w.abs()
    tol = 2.0 ** -18 * size
    assert bool(((s["y"].double() - want).abs() <= tol + 2.0 ** -24 * (want.abs() + tol)).all())


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("tokens", [65, 128, 200])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_more_tokens_than_a_tile(hip, group, tokens, dtype):
    for n_out, n_in in ((70000, 256), (700, 3200)):
        run(n_out, n_in, group, tokens, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n_out,n_in", [(1000, 4096), (5120, 1024), (300, 16384)])
def test_one_workspace_for_every_step(hip, n_out, n_in, dtype):
    """A server's: asked for once, for the most tokens that a step may have."""
    group, most = 64, 700
    codes, scales = random_weights(n_out, n_in, group, BF16, 3)
    x = torch.randn(most, n_in, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    s = linear(weights(codes, scales, group), x, F32)
    a, y = s["args"], s["y"]
    check(s, codes, scales, group)
    for tokens in (1, 2, 5, 16, 17, 32, 33, 64, 65, 128, 129, 300, 699):
        y.fill_(7)
        a.tokens = tokens
        torch.cuda.synchronize()
        dev.fp4_linear(a)
        torch.cuda.synchronize()
        assert bool((s["work"][a.workspace_bytes:] == 255).all()) and bool((y[tokens:] == 7).all())
        check(dict(x=x[:tokens], y=y[:tokens]), codes, scales, group)


def test_a_call_that_is_not_split_needs_none(hip):
    """Enough blocks to fill the GPU: no workspace, though fewer tokens would need one."""
    codes, scales = random_weights(5120, 1024, 64, BF16, 3)
    s = linear(weights(codes, scales, 64), torch.randn(1000, 1024, device="cuda").to(BF16), F32)
    a, want = s["args"], s["y"].clone()
    assert a.workspace_bytes > 0
    a.workspace, a.workspace_bytes = None, 0
    s["y"].fill_(7)
    torch.cuda.synchronize()
    dev.fp4_linear(a)
    torch.cuda.synchronize()
    assert torch.equal(s["y"], want)
