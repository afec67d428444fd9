"""GPU: dense weights in 4 bits, packed exactly, and their products against 64 bits.

Tolerance, before any run: codes are exact and x enters with all its bits, so
what is left are float32 sums: of a group's products on the matrix cores, its
scale, and the sums over groups, waves and splits.  With n terms one after another
they are off by at most n 2^-24 of the sum of the terms' magnitudes, and far less
in a tree; 2^-18 of it allows 64 roundings in one direction, and the output is
rounded once."""
import numpy as np
import pytest
import torch

from sili__new_amd import device as dev
from tests import block_ref, draft_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def name_of(dtype):
    return str(dtype)[6:]


def weights(codes, scales, group, n_in=None):
    """A descriptor of codes [n_out, >= n_in / 2] and scales [n_out, ...] on the GPU."""
    return dev.Fp4Weights(codes=codes.data_ptr(), scales=scales.data_ptr(), n_out=codes.shape[0], n_in=2 * codes.shape[1] if n_in is None else n_in,
                          group=group, codes_stride=codes.stride(0), scales_stride=scales.stride(0), scale_dtype=dev.DTYPES[name_of(scales.dtype)])


def random_weights(n_out, n_in, group, scale_dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (n_out, n_in // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = (0.01 * torch.exp(torch.randn(n_out, n_in // group, generator=gen, device="cuda"))).to(scale_dtype)
    return codes, scales


def linear(w, x, out_dtype, y=None, stream=None):
    t = x.shape[0]
    s = dict(x=x, y=torch.full((t, w.n_out), 7.0, device="cuda").to(out_dtype) if y is None else y)
    a = dev.Fp4Linear(w=w, dtype=dev.DTYPES[name_of(x.dtype)], out_dtype=dev.DTYPES[name_of(out_dtype)], tokens=t, x=x.data_ptr(),
                      x_stride=x.stride(0), y=s["y"].data_ptr(), y_stride=s["y"].stride(0))
    need = dev.fp4_linear_workspace(a)
    s["work"] = torch.full((need + 16,), 255, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = s["work"].data_ptr(), need
    torch.cuda.synchronize()
    dev.fp4_linear(a, stream)
    torch.cuda.synchronize()
    assert bool((s["work"][need:] == 255).all())
    s["args"] = a
    return s


def check(s, codes, scales, group):
    w = ref.fp4_weights(codes.cpu().numpy(), scales.float().cpu().numpy(), group)
    x = s["x"].double().cpu().numpy()
    want, size = x @ w.T, np.abs(x) @ np.abs(w).T
    dtype = name_of(s["y"].dtype)
    tol = 2.0 ** -18 * size
    err = np.abs(s["y"].double().cpu().numpy() - want)
    tol = tol + block_ref.rounding(dtype, np.abs(want) + tol)
    assert np.all(err <= tol), (np.max(err / tol), np.argwhere(~(err <= tol))[:3])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("scale_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_packing_is_exact(hip, group, scale_dtype, dtype):
    gen = torch.Generator(device="cuda").manual_seed(group)
    n, k = 37, 3 * 128 + group
    x = (torch.randn(n, k, generator=gen, device="cuda") * torch.exp(3 * torch.randn(n, 1, generator=gen, device="cuda"))).to(dtype)
    x[0, :16] = torch.tensor([6, -6, .25, -.25, .75, -.75, 1.25, 1.75, 2.5, -2.5, 3.5, 5, -5, 0.0, -0.0, .2499], device="cuda").to(dtype)
    x[0, 16:group] = 0
    x[1] = 0
    x[2, 3], x[3, 5], x[4, k - 1] = float("nan"), float("inf"), float("-inf")
    x[5] = (x[5].float() * 1e-30).to(dtype)
    x[6] = 6e4 if dtype == F16 else 3e38
    codes = torch.full((n, k // 2 + 32), 255, dtype=torch.uint8, device="cuda")
    scales = torch.full((n, k // group + 3), 7.0, device="cuda").to(scale_dtype)
    a = dev.Fp4Pack(w=weights(codes, scales, group, k), dtype=dev.DTYPES[name_of(dtype)], rows=x.data_ptr(), row_stride=x.stride(0))
    torch.cuda.synchronize()
    dev.fp4_pack(a)
    torch.cuda.synchronize()
    want_codes, want_scales = ref.fp4_pack(x.float().cpu().numpy(), group, name_of(scale_dtype))
    got = scales.float().cpu().numpy()
    assert np.array_equal(got[:, :k // group], want_scales, equal_nan=True) and (got[:, k // group:] == 7).all()
    assert np.array_equal(codes.cpu().numpy()[:, :k // 2], want_codes) and bool((codes[:, k // 2:] == 255).all())


def test_rows_packed_from_an_odd_offset(hip):
    base = torch.randn(9 * 131 + 1, device="cuda").to(BF16)
    x = base[1:].view(9, 131)[:, 2:130]
    codes, scales = torch.zeros(9, 64, dtype=torch.uint8, device="cuda"), torch.zeros(9, 4, device="cuda")
    torch.cuda.synchronize()
    dev.fp4_pack(dev.Fp4Pack(w=weights(codes, scales, 32), dtype=dev.BF16, rows=x.data_ptr(), row_stride=131))
    torch.cuda.synchronize()
    want_codes, want_scales = ref.fp4_pack(x.float().cpu().numpy(), 32, "float32")
    assert np.array_equal(codes.cpu().numpy(), want_codes) and np.array_equal(scales.cpu().numpy(), want_scales)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 9, 16, 17, 31, 33, 64, 70, 130])
def test_tokens(hip, tokens, group, dtype):
    """About every edge of tiles of tokens; outputs and inputs that fill no tile."""
    n_out, n_in = 150, 5 * 128 + group
    scale_dtype = [F32, BF16, F16][(tokens + group // 32) % 3]
    codes, scales = random_weights(n_out, n_in, group, scale_dtype, tokens)
    gen = torch.Generator(device="cuda").manual_seed(tokens + 1)
    x = torch.randn(tokens, n_in, generator=gen, device="cuda").to(dtype)
    for out in {dtype, F32}:
        check(linear(weights(codes, scales, group), x, out), codes, scales, group)


@pytest.mark.parametrize("n_out,n_in,group,tokens", [(1, 32, 32, 1), (15, 64, 64, 2), (16, 96, 32, 7), (17, 128, 128, 1), (64, 160, 32, 40), (129, 192, 64, 1),
                                                     (1000, 512, 32, 5), (300, 8192, 128, 1), (33, 32768, 32, 3), (5, 16384, 64, 100), (4100, 1024, 64, 12),
                                                     (1030, 2048, 128, 33), (2000, 384, 128, 200), (260, 4096, 32, 256)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_sizes(hip, n_out, n_in, group, tokens, dtype):
    codes, scales = random_weights(n_out, n_in, group, F32, n_out)
    gen = torch.Generator(device="cuda").manual_seed(n_in)
    x = torch.randn(tokens, n_in, generator=gen, device="cuda").to(dtype)
    s = linear(weights(codes, scales, group), x, F32)
    check(s, codes, scales, group)
    again = linear(weights(codes, scales, group), x, F32)
    assert torch.equal(s["y"], again["y"])


@pytest.mark.parametrize("n_out,n_in,group,tokens", [(131071, 96, 32, 3), (131071, 64, 64, 16), (110000, 256, 128, 1), (40, 16384, 64, 1), (1500, 16384, 128, 1),
                                                     (20, 32768, 128, 16), (300, 6144 - 32, 32, 11), (33000, 640, 64, 9), (8200, 1280, 32, 4)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_few_tokens_over_many_outputs_and_inputs(hip, n_out, n_in, group, tokens, dtype):
    """Blocks that go on to other outputs, waves that share outputs, inputs that LDS does not hold at once."""
    codes, scales = random_weights(n_out, n_in, group, F32, n_out)
    gen = torch.Generator(device="cuda").manual_seed(n_in)
    x = torch.randn(tokens, n_in, generator=gen, device="cuda").to(dtype)
    s = linear(weights(codes, scales, group), x, F32)
    check(s, codes, scales, group)
    assert torch.equal(s["y"], linear(weights(codes, scales, group), x, F32)["y"])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens", [1, 6, 50, 140])
def test_strides(hip, tokens, dtype):
    """Rows of everything with gaps, x at an odd offset; the gaps of y stay."""
    n_out, n_in, group = 90, 320, 64
    codes = torch.full((n_out, 256), 255, dtype=torch.uint8, device="cuda")
    scales = torch.full((n_out, 9), float("nan"), device="cuda")
    c, sc = random_weights(n_out, n_in, group, F32, 5)
    codes[:, 32:192], scales[:, 1:6] = c, sc
    wide = torch.full((tokens * 353 + 1,), float("nan"), device="cuda").to(dtype)
    x = wide[1:].view(tokens, 353)[:, 3:323]
    x.copy_(torch.randn(tokens, n_in, device="cuda"))
    y = torch.full((tokens, 97), 3.0, device="cuda").to(BF16)
    s = linear(weights(codes[:, 32:192], scales[:, 1:6], group), x, BF16, y=y[:, 2:92])
    check(s, c, sc, group)
    assert float((y[:, :2].float() - 3).abs().max()) == 0 and float((y[:, 92:].float() - 3).abs().max()) == 0


def test_no_inputs_give_zeros(hip):
    codes, scales = random_weights(20, 32, 32, F32, 1)
    for tokens in (1, 40, 200):
        s = linear(weights(codes, scales, 32, 0), torch.randn(tokens, 32, device="cuda"), F32)
        assert not s["y"].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("tokens", [1, 3, 7, 20, 140])
def test_what_is_not_finite_stays_in_its_row_and_output(hip, tokens, dtype):
    n_out, n_in, group = 40, 640, 32
    codes, scales = random_weights(n_out, n_in, group, F32, 3)
    x = torch.randn(tokens, n_in, device="cuda").to(dtype)
    bad = tokens // 2
    x[bad, 600], x[bad, 7] = float("inf"), float("nan")
    y = linear(weights(codes, scales, group), x, F32)["y"]
    fine = torch.isfinite(y).all(1).cpu().numpy()
    assert not torch.isfinite(y[bad]).any() and np.array_equal(fine, np.arange(tokens) != bad)
    x[bad] = 1
    scales[11, 4] = float("nan")
    y = linear(weights(codes, scales, group), x, F32)["y"]
    nan = torch.isnan(y)
    assert bool(nan[:, 11].all()) and int(nan.sum()) == tokens


@pytest.mark.parametrize("dtype,top", [(F32, 3.4e38), (BF16, 3e38), (F16, 65504.0), (F32, 1e-30), (F16, 6e-8)])
@pytest.mark.parametrize("tokens", [2, 9])
def test_the_largest_and_smallest_values(hip, tokens, dtype, top):
    """Parts of the largest finite value are finite; of the smallest nothing that counts is lost."""
    n_out, n_in, group = 24, 256, 64
    codes, scales = random_weights(n_out, n_in, group, F32, 4)
    codes &= 0x99  # 0 and a half, so that a group's sum is finite
    scales *= 2.0 ** -20
    x = torch.zeros(tokens, n_in, device="cuda")
    x[:, ::64] = top
    s = linear(weights(codes, scales, group), x.to(dtype), F32)
    assert torch.isfinite(s["y"]).all()
    check(s, codes, scales, group)


def test_zero_minus_counts_as_zero(hip):
    codes = torch.full((20, 64), 0x88, dtype=torch.uint8, device="cuda")
    scales = torch.ones(20, 4, device="cuda")
    assert not linear(weights(codes, scales, 32), torch.randn(3, 128, device="cuda"), F32)["y"].any()


def test_offsets_past_32_bits(hip):
    """Rows of codes and of x that lie more than 4 GiB apart."""
    n_out, n_in, group = 130, 256, 32
    gap = 36 << 20
    codes = torch.zeros(n_out, gap, dtype=torch.uint8, device="cuda")
    c, sc = random_weights(n_out, n_in, group, F32, 9)
    codes[:, :n_in // 2] = c
    x = torch.zeros(40, 30 << 20, device="cuda")
    small = torch.randn(40, n_in, device="cuda")
    x[:, :n_in] = small
    s = linear(weights(codes, sc, group, n_in), x[:, :n_in], F32)
    near = linear(weights(c, sc, group), small, F32)
    assert torch.equal(s["y"], near["y"])
    check(near, c, sc, group)


@pytest.mark.parametrize("tokens", [1, 3, 20])
def test_replayed_in_two_graphs_with_workspaces_of_their_own(hip, tokens):
    n_out, n_in, group = 80, 8192, 128
    codes, scales = random_weights(n_out, n_in, group, BF16, 2)
    st = torch.cuda.Stream()
    w = weights(codes, scales, group)
    calls = [linear(w, torch.randn(tokens, n_in, device="cuda"), F32, stream=st.cuda_stream) for _ in range(2)]
    graphs = []
    for s in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            dev.fp4_linear(s["args"], st.cuda_stream)
        graphs.append(g)
    for _ in range(3):
        for s in calls:
            s["x"].normal_()
            s["y"].fill_(7)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s in calls:
            check(s, codes, scales, group)
            assert torch.equal(s["y"], linear(w, s["x"], F32)["y"])


def test_two_calls_at_once_on_streams_of_their_own(hip):
    """Split calls of few and of many tokens, with a workspace each, in turn on two streams."""
    n_out, n_in, group = 80, 8192, 64
    codes, scales = random_weights(n_out, n_in, group, F32, 4)
    w = weights(codes, scales, group)
    calls = [(linear(w, torch.randn(tokens, n_in, device="cuda").to(dtype), F32), torch.cuda.Stream())
             for tokens, dtype in ((8, BF16), (100, F16), (3, F32), (40, F32))]
    want = [s["y"].clone() for s, _ in calls]
    for s, _ in calls:
        check(s, codes, scales, group)
        s["y"].fill_(7)
    torch.cuda.synchronize()
    for _ in range(5):
        for s, st in calls:
            dev.fp4_linear(s["args"], st.cuda_stream)
    torch.cuda.synchronize()
    for (s, _), y in zip(calls, want):
        assert torch.equal(s["y"], y)
