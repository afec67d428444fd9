"""GPU: the norms around a block with gate and residual scale, forward and
backward, against their formulas in 64 bits.

Tolerances, before any run: a mean of n float32 terms in the kernels' trees
(at most n / 64 terms in a row, then a tree) is within E(n) = (n / 64 + 32)
2^-24 of the sum of its terms' magnitudes; every output carries a few such
errors of its own terms, and one rounding to the type."""
import numpy as np
import pytest
import torch

from sili__new_amd import device as dev
from tests import block_ref as ref

pytestmark = pytest.mark.gpu
EPS = 1e-5


def e(n):
    return (n / 64 + 32) * 2.0 ** -24


def p(t):
    return None if t is None else t.data_ptr()


def row(t):
    return (None, 0) if t is None else (t.data_ptr(), t.stride(0) if t.dim() == 2 else 0)


def np64(t):
    return None if t is None else t.double().cpu().numpy()


def scene(t, n, dtype, gate, post, pre, x, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return dict(u=rand(t, n).to(dtype), x=(2 * rand(t, n)).to(dtype) if x else None, dy=rand(t, n).to(dtype), dh=rand(t, n).to(dtype),
                gate=None if gate == "none" else (rand(n) if gate == "channel" else rand(t, n)).to(dtype),
                w_post=1 + 0.3 * rand(n) if post else None, w_pre=1 + 0.3 * rand(n) if pre else None)


def args(s, a_u=0.4, a_x=0.9):
    u = s["u"]
    a = dev.BlockNorm(dtype=dev.DTYPES[str(u.dtype)[6:]], tokens=u.shape[0], width=u.shape[1], u_scale=a_u, x_scale=a_x, eps=EPS,
                      w_post=p(s["w_post"]), w_pre=p(s["w_pre"]))
    a.u, a.u_stride = row(u)
    a.x, a.x_stride = row(s["x"])
    a.gate, a.gate_stride = row(s["gate"])
    return a


def forward(s, out=None, stream=None):
    t, n = s["u"].shape
    o = out or dict(y=torch.empty_like(s["u"]), h=torch.empty_like(s["u"]))
    o["r1"], o["r2"] = torch.zeros(t, device="cuda"), torch.zeros(t, device="cuda")
    a = args(s)
    a.y, a.y_stride = row(o["y"])
    a.h, a.h_stride = row(o["h"])
    a.rstd_post, a.rstd_pre = p(o["r1"]), p(o["r2"])
    torch.cuda.synchronize()
    dev.block_norm_forward(a, stream)
    torch.cuda.synchronize()
    o["args"] = a
    return o


def check_forward(s, o):
    t, n = s["u"].shape
    dtype = str(s["u"].dtype)[6:]
    want = ref.norm_forward(*(np64(s[k]) for k in ("u", "x", "gate", "w_post", "w_pre")), 0.4, 0.9, EPS)
    tol = (e(n) + 2.0 ** -21) * np.abs(want["part"]) + 2.0 ** -22 * np.abs(want["y"] - want["part"])
    err = np.abs(np64(o["y"]) - want["y"])
    assert np.all(err <= tol + ref.rounding(dtype, np.abs(want["y"]) + tol))
    if s["w_post"] is not None:
        assert np.all(np.abs(np64(o["r1"]) - want["r1"]) <= (e(n) + 2.0 ** -21) * want["r1"])
    if s["w_pre"] is not None:
        # y's error, relative in the norm
        rel = 2 * e(n) + 2.0 ** -19
        assert np.all(np.abs(np64(o["r2"]) - want["r2"]) <= rel * want["r2"])
        scale = want["r2"][:, None] * np.abs(np64(s["w_pre"]))
        tol = tol * scale + rel * np.abs(want["h"])
        assert np.all(np.abs(np64(o["h"]) - want["h"]) <= tol + ref.rounding(dtype, np.abs(want["h"]) + tol))


def backward(s, y, r1, r2, dy=True, dh=True, stream=None):
    t, n = s["u"].shape
    o = dict(du=torch.empty_like(s["u"]), dx=torch.empty_like(s["u"]), dw_pre=torch.full((n,), 5.0, device="cuda"))
    a = args(s)
    a.y, a.y_stride = row(y)
    a.rstd_post, a.rstd_pre = p(r1), p(r2)
    g = dev.BlockNormGrad()
    g.dy, g.dy_stride = row(s["dy"] if dy else None)
    g.dh, g.dh_stride = row(s["dh"] if dh else None)
    g.du, g.du_stride = row(o["du"])
    g.dx, g.dx_stride = row(o["dx"])
    if s["w_pre"] is not None:
        g.dw_pre = p(o["dw_pre"])
    if s["w_post"] is not None:
        o["dw_post"] = torch.full((n,), 5.0, device="cuda")
        g.dw_post = p(o["dw_post"])
    if s["gate"] is not None:
        o["dgate"] = torch.full((n,), 5.0, device="cuda") if s["gate"].dim() == 1 else torch.empty_like(s["u"])
        g.dgate, g.dgate_stride = row(o["dgate"])
    need = dev.block_norm_workspace(a)
    o["work"] = torch.full((need,), 255, dtype=torch.uint8, device="cuda")  # NaNs
    g.workspace, g.workspace_bytes = p(o["work"]), need
    torch.cuda.synchronize()
    dev.block_norm_backward(a, g, stream)
    torch.cuda.synchronize()
    o["args"] = (a, g)
    return o


def check_backward(s, o, y, r1, r2, dy=True, dh=True):
    t, n = s["u"].shape
    dtype = str(s["u"].dtype)[6:]
    want = ref.norm_backward(np64(s["u"]), np64(y), *(np64(s[k]) for k in ("gate", "w_post", "w_pre")), 0.4, 0.9, np64(r1), np64(r2),
                             np64(s["dy"]) if dy else None, np64(s["dh"]) if dh else None)
    if s["w_pre"] is not None and not dh:
        want["dw_pre"] = (np.zeros(n), np.zeros(n))
    for name, (w, size) in want.items():
        got = np64(o[name])
        summed = name.startswith("dw") or (name == "dgate" and w.ndim == 1)
        tol = (4 * e(n) + 2.0 ** -20 + (e(64 * t) if summed else 0)) * size
        if not summed:
            tol = tol + ref.rounding(dtype, np.abs(w) + tol)
        assert np.all(np.abs(got - w) <= tol), (name, np.max(np.abs(got - w) / (tol + 1e-300)))


def kept(s):
    """What a forward pass keeps, exact: y, r1, r2."""
    f = ref.norm_forward(*(np64(s[k]) for k in ("u", "x", "gate", "w_post", "w_pre")), 0.4, 0.9, EPS)
    y = torch.from_numpy(f["y"]).cuda().to(s["u"].dtype)
    r2 = 1 / np.sqrt((np64(y) ** 2).mean(-1) + EPS)
    return y, torch.from_numpy(f["r1"]).float().cuda(), torch.from_numpy(r2).float().cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,n", [(1, 1), (3, 7), (5, 64), (2, 255), (9, 320), (1, 1000), (4, 2816), (3, 5120), (2, 8192), (2, 20001), (1, 32768)])
@pytest.mark.parametrize("gate,post,pre,x", [("channel", True, True, True), ("token", True, True, False), ("none", False, True, True),
                                             ("none", True, False, True), ("token", False, False, True)])
def test_forward_and_backward(hip, t, n, dtype, gate, post, pre, x):
    s = scene(t, n, dtype, gate, post, pre, x, t * 7 + n)
    check_forward(s, forward(s))
    k = kept(s)
    check_backward(s, backward(s, *k), *k) if pre else check_backward(s, backward(s, *k, dh=False), *k, dh=False)


@pytest.mark.parametrize("t,n,dtype", [(1025, 96, torch.float32), (700, 640, torch.bfloat16), (3000, 33, torch.float16), (513, 2048, torch.float32)])
@pytest.mark.parametrize("dy,dh", [(True, True), (False, True), (True, False)])
def test_many_rows(hip, t, n, dtype, dy, dh):
    s = scene(t, n, dtype, "channel", True, True, True, n)
    check_forward(s, forward(s))
    k = kept(s)
    o = backward(s, *k, dy=dy, dh=dh)
    check_backward(s, o, *k, dy=dy, dh=dh)
    again = backward(s, *k, dy=dy, dh=dh)
    for name in ("du", "dx", "dgate", "dw_post", "dw_pre"):
        assert torch.equal(o[name], again[name]), name


def test_strides_and_in_place(hip):
    """Rows with gaps at odd offsets; y over x and h over u."""
    t, n = 6, 330
    base = scene(t, n, torch.float32, "token", True, True, True, 3)
    s = dict(base)
    for name, pad, off in (("u", 400, 1), ("x", 337, 3), ("gate", 352, 16)):
        wide = torch.zeros(t, pad, device="cuda")
        s[name] = wide[:, off:off + n]
        s[name].copy_(base[name])
    o = forward(s, dict(y=torch.zeros(t, 345, device="cuda")[:, 2:n + 2], h=torch.zeros(t, 352, device="cuda")[:, :n]))
    check_forward(base, o)
    assert float(o["y"]._base[:, n + 2:].abs().max()) == 0.0 and float(o["h"]._base[:, n:].abs().max()) == 0.0
    plain = forward(base)
    u, x = base["u"].clone(), base["x"].clone()
    over = forward(dict(base, u=u, x=x), dict(y=x, h=u))
    assert torch.equal(over["y"], plain["y"]) and torch.equal(over["h"], plain["h"])


def test_gradients_against_differences(hip):
    """The forward pass's change along a direction, by central differences of
    step 1/64 (error of second order: 2^-12 of third derivatives of order one;
    outputs rounded at 2^-23)."""
    t, n = 4, 48
    s = scene(t, n, torch.float32, "channel", True, True, True, 9)
    f = forward(s)
    o = backward(s, f["y"], f["r1"], f["r2"])
    d = scene(t, n, torch.float32, "channel", True, True, True, 10)

    def loss(sign):
        moved = dict(s)
        for name in ("u", "x", "gate", "w_post", "w_pre"):
            moved[name] = s[name] + sign / 64 * d[name]
        q = forward(moved)
        return float((q["y"].double() * s["dy"].double() + q["h"].double() * s["dh"].double()).sum())

    got = (loss(1) - loss(-1)) * 32
    want = sum(float((o[g].double() * d[name].double()).sum())
               for g, name in (("du", "u"), ("dx", "x"), ("dgate", "gate"), ("dw_post", "w_post"), ("dw_pre", "w_pre")))
    size = sum(float((o[g].double() * d[name].double()).abs().sum())
               for g, name in (("du", "u"), ("dx", "x"), ("dgate", "gate"), ("dw_post", "w_post"), ("dw_pre", "w_pre")))
    assert abs(got - want) <= 2.0 ** -10 * size


def test_zero_rows_and_infinities(hip):
    """A row of zeros norms to zeros; one with an infinity or a NaN stays in its own row."""
    s = scene(4, 256, torch.float32, "channel", True, True, True, 4)
    s["u"][1], s["x"][1] = 0, 0
    s["u"][2, 5] = float("inf")
    s["x"][3, 7] = float("nan")
    o = forward(s)
    assert float(o["y"][1].abs().max()) == 0 and float(o["h"][1].abs().max()) == 0
    assert torch.isfinite(o["h"][:2]).all() and torch.isnan(o["h"][3]).all()
    one = {k: (v[:1] if v is not None and v.dim() == 2 else v) for k, v in s.items()}
    assert torch.equal(forward(one)["h"], o["h"][:1])


def test_no_tokens_give_zero_weight_gradients(hip):
    s = scene(1, 40, torch.bfloat16, "channel", True, True, True, 4)
    s = {k: (v[:0] if v is not None and v.dim() == 2 else v) for k, v in s.items()}
    z = torch.zeros(0, device="cuda")
    o = backward(s, s["u"], z, z)
    for name in ("dgate", "dw_post", "dw_pre"):
        assert float(o[name].abs().max()) == 0.0


def test_in_a_graph(hip):
    s = scene(20, 512, torch.bfloat16, "channel", True, True, True, 6)
    st = torch.cuda.Stream()
    f = forward(s, stream=st.cuda_stream)
    o = backward(s, f["y"], f["r1"], f["r2"], stream=st.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        dev.block_norm_forward(f["args"], st.cuda_stream)
        dev.block_norm_backward(*o["args"], st.cuda_stream)
    for k in range(3):
        s["u"].mul_(0.5)
        s["dh"].add_(0.25)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check_forward(s, f)
        eager = backward(s, f["y"], f["r1"], f["r2"])
        for name in ("du", "dx", "dgate", "dw_post", "dw_pre"):
            assert torch.equal(o[name], eager[name]), (k, name)
