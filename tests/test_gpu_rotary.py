"""GPU: rotary positions against complex rotations in 64 bits, and their
gradient against the transposed rotation and differences.

Tolerance: a rotated channel is two products and a sum of float32, sines and
cosines within 2^-22, an angle within 2 pi 2^-32: 2^-21 of |x1| + |x2| in all,
and one rounding to the type."""
import numpy as np
import pytest
import torch

from sili__new_amd import device as dev
from tests import block_ref as ref

pytestmark = pytest.mark.gpu


def strided(t):
    return t.data_ptr(), t.stride(0), t.stride(1)


def turn(q, k, pos, steps, rot, layout, inverse=0, scale=1.0, out=None, stream=None):
    qo, ko = out or (torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty_like(k, memory_format=torch.contiguous_format))
    p = torch.from_numpy(np.asarray(pos, np.int32)).cuda()
    s = torch.from_numpy(np.ascontiguousarray(steps).view(np.int64)).cuda()
    torch.cuda.synchronize()
    a = dev.Rotary(dtype=dev.DTYPES[str(q.dtype)[6:]], tokens=q.shape[0], head_dim=q.shape[2], rot_dim=rot, layout=layout, inverse=inverse,
                   scale=scale, positions=p.data_ptr(), phase_steps=s.data_ptr(), q_heads=q.shape[1], k_heads=k.shape[1])
    a.q, a.q_token_stride, a.q_head_stride = strided(q)
    a.k, a.k_token_stride, a.k_head_stride = strided(k)
    a.q_out, a.q_out_token_stride, a.q_out_head_stride = strided(qo)
    a.k_out, a.k_out_token_stride, a.k_out_head_stride = strided(ko)
    dev.rotary(a, stream)
    torch.cuda.synchronize()
    return qo, ko


def near(got, x, pos, steps, rot, layout, inverse, scale):
    x = x.double().cpu().numpy()
    half = layout == dev.ROTARY_HALF
    want = ref.rotary(x, pos, steps, rot, half, inverse, scale)
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
    size = np.zeros_like(x)
    size[..., a] = size[..., b] = scale * (np.abs(x[..., a]) + np.abs(x[..., b]))
    dtype = str(got.dtype)[6:]
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.all(err <= 2.0 ** -21 * size + ref.rounding(dtype, np.abs(want) + 2.0 ** -21 * size))
    # what is not rotated is copied
    assert np.array_equal(got.double().cpu().numpy()[..., rot:], x[..., rot:])


SHAPES = [(1, 1, 0, 2, 2), (1, 40, 40, 128, 128), (3, 5, 1, 64, 32), (17, 8, 2, 80, 40), (5, 3, 3, 10, 6), (33, 4, 1, 256, 64),
          (130, 7, 7, 96, 94), (2, 2, 1, 64, 0), (600, 12, 4, 128, 128), (9, 3, 1, 7, 6)]


@pytest.mark.parametrize("layout", [dev.ROTARY_HALF, dev.ROTARY_INTERLEAVED])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,hq,hk,d,rot", SHAPES)
def test_matches_complex_rotation(hip, t, hq, hk, d, rot, dtype, layout):
    gen = torch.Generator(device="cuda").manual_seed(t * 131 + d)
    qkv = torch.randn(t, (hq + 2 * hk) * d, generator=gen, device="cuda").to(dtype)
    q, k = qkv[:, :hq * d].view(t, hq, d), qkv[:, hq * d:(hq + hk) * d].view(t, hk, d)
    rng = np.random.default_rng(d)
    pos = rng.integers(0, 1 << 20, t)
    pos[0] = 2 ** 31 - 1 if t > 1 else 12345
    pos[-1] = -7
    steps, scale = dev.rotary_steps(rot, 10000.0, dev.ROTARY_BANDS, 4.0, 4096.0)
    for inverse in (0, 1):
        qo, ko = turn(q, k, pos, steps, rot, layout, inverse, scale)
        near(qo, q, pos, steps, rot, layout, inverse, scale)
        near(ko, k, pos, steps, rot, layout, inverse, scale)


@pytest.mark.parametrize("layout", [dev.ROTARY_HALF, dev.ROTARY_INTERLEAVED])
def test_strides_alignment_and_in_place(hip, layout):
    """Heads before tokens, an odd offset, an output with gaps, and in place."""
    t, h, d, rot = 21, 6, 64, 48
    gen = torch.Generator(device="cuda").manual_seed(5)
    steps, scale = dev.rotary_steps(rot)
    pos = np.arange(t) * 977
    heads_first = torch.randn(h, t, d, generator=gen, device="cuda").transpose(0, 1)
    odd = torch.randn(t * h * 67 + 3, generator=gen, device="cuda")[3:3 + t * h * 67].view(t, h, 67)[..., 1:65]
    out = (torch.full((t, h, 80), 9.0, device="cuda")[..., :d], torch.full((t, h, 81), 9.0, device="cuda")[..., 1:d + 1])
    q, k = turn(heads_first, odd, pos, steps, rot, layout, out=out)
    near(q, heads_first, pos, steps, rot, layout, 0, scale)
    near(k, odd, pos, steps, rot, layout, 0, scale)
    # the gaps are not written
    assert float(out[0]._base[..., d:].min()) == 9.0 and float(out[1]._base[..., 0].min()) == 9.0
    a, b = heads_first.contiguous(), odd.contiguous()
    turn(a, b, pos, steps, rot, layout, out=(a, b))
    assert torch.equal(a, q) and torch.equal(b, k)


def test_inverse_is_the_gradient(hip):
    """<turn(x), g> = <x, inverse(g)>, and differences of the loss along a direction."""
    t, h, d = 6, 3, 32
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, g, dx = (torch.randn(t, h, d, generator=gen, device="cuda") for _ in range(3))
    none = x[:, :0]
    steps, _ = dev.rotary_steps(d)
    pos = np.arange(t) * 31 + 5

    def loss(z):
        return (turn(z, none, pos, steps, d, dev.ROTARY_HALF, scale=1.25)[0].double() * g.double()).sum()

    back = turn(g, none, pos, steps, d, dev.ROTARY_HALF, inverse=1, scale=1.25)[0].double()
    want = float((back * dx.double()).sum())
    # linear: a difference at any step is exact to the outputs' rounding
    size = float((g.double().abs() * 2.5 * (x.double().abs() + dx.double().abs()).amax()).sum())
    assert abs(float(loss(x + dx) - loss(x - dx)) / 2 - want) <= 2.0 ** -20 * size


def test_on_another_stream_and_in_a_graph(hip):
    t, h, d = 40, 4, 64
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k = (torch.randn(t, h, d, generator=gen, device="cuda") for _ in range(2))
    steps, scale = dev.rotary_steps(d)
    pos = np.arange(t)
    st = torch.cuda.Stream()
    qo, ko = turn(q, k, pos, steps, d, dev.ROTARY_HALF, stream=st.cuda_stream)
    near(qo, q, pos, steps, d, dev.ROTARY_HALF, 0, scale)
    p = torch.from_numpy(pos.astype(np.int32)).cuda()
    s = torch.from_numpy(steps.view(np.int64)).cuda()
    a = dev.Rotary(dtype=dev.F32, tokens=t, head_dim=d, rot_dim=d, scale=1.0, positions=p.data_ptr(), phase_steps=s.data_ptr(), q_heads=h)
    a.q, a.q_token_stride, a.q_head_stride = strided(q)
    a.q_out, a.q_out_token_stride, a.q_out_head_stride = strided(qo)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        dev.rotary(a, st.cuda_stream)
    for k in range(3):
        p += 11
        q.mul_(1.5)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        near(qo, q, pos + 11 * (k + 1), steps, d, dev.ROTARY_HALF, 0, scale)
