"""GPU: the 4-bit cache (rows written, read back) exactly, and attention over it
against softmax attention in 64 bits on the stored values.

Tolerances, before any run.  A score is off by at most 2^-16 of the sum of its
terms' magnitudes (float32: parts of 16 bits, and float32 sums of up to 256
terms; bf16 and f16: the sums alone, no more), so a softmax weight by twice
that, relative; weights are multiplied with 8 significant bits (bf16, f16: 2^-8
each) or 16 (float32), and the output is rounded once."""
import numpy as np
import pytest
import torch

from sili__new_amd import device as dev
from tests import block_ref as ref

pytestmark = pytest.mark.gpu


def np64(t):
    return t.double().cpu().numpy()


def strided(t):
    return t.data_ptr(), t.stride(0), t.stride(1)


def new_cache(pages, heads, page, d, fill=0):
    """Arrays of a cache in host and device memory; `fill`: the bytes of what is
    never written (255: codes of any kind under NaN scales)."""
    shapes = dict(k=(pages, heads, page, d // 2), v=(pages, heads, page // 16, d // 2, 16), k_scale=(pages, heads, page), v_scale=(pages, heads, page))
    c = {}
    for name, shape in shapes.items():
        c[name] = np.full(shape, fill, np.uint8) if name in "kv" else np.full(shape, np.nan if fill else 0, np.float32)
    return c, {k: torch.from_numpy(v).cuda() for k, v in c.items()}


def desc(t):
    pages, heads, page, half = t["k"].shape
    return dev.Kv4Cache(k=t["k"].data_ptr(), v=t["v"].data_ptr(), k_scale=t["k_scale"].data_ptr(), v_scale=t["v_scale"].data_ptr(),
                        n_pages=pages, kv_heads=heads, head_dim=2 * half, page_size=page)


def rows(call, cache, k, v, slots, stream=None):
    s = torch.from_numpy(np.asarray(slots, np.int32)).cuda()
    a = dev.Kv4Rows(cache=cache, dtype=dev.DTYPES[str(k.dtype)[6:]], tokens=len(slots), slots=s.data_ptr())
    a.k, a.k_token_stride, a.k_head_stride = strided(k)
    a.v, a.v_token_stride, a.v_head_stride = strided(v)
    torch.cuda.synchronize()
    call(a, stream)
    torch.cuda.synchronize()
    return a


# ---- rows ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,heads,d,page", [(1, 1, 64, 16), (1, 40, 128, 16), (5, 3, 128, 32), (33, 2, 256, 48), (70, 8, 64, 128), (257, 1, 128, 16)])
def test_append_and_read(hip, t, heads, d, page, dtype):
    gen = torch.Generator(device="cuda").manual_seed(t + d)
    kv = torch.randn(t, 2 * heads * d, generator=gen, device="cuda") * torch.exp(2 * torch.randn(t, 1, generator=gen, device="cuda"))
    kv = kv.to(dtype)
    k, v = kv[:, :heads * d].view(t, heads, d), kv[:, heads * d:].view(t, heads, d)
    # equal magnitudes, ties and signed zeros
    k[0, 0, :16] = torch.tensor([6, -6, .25, -.25, .75, -.75, 1.25, 1.75, 2.5, -2.5, 3.5, 5, -5, 0.0, -0.0, .2499], device="cuda").to(dtype)
    k[0, 0, 16:] = 0
    v[0, 0] = 0
    pages = -(-t // page) + 2
    host, gpu = new_cache(pages, heads, page, d, fill=255)
    slots = np.random.default_rng(t).permutation(pages * page)[:t]
    if t > 4:
        slots[3], slots[4] = -1, pages * page  # padding
    rows(dev.kv4_append, desc(gpu), k, v, slots)
    ref.kv4_store(host, slots, k.float().cpu().numpy(), v.float().cpu().numpy())
    for name in host:
        assert np.array_equal(gpu[name].cpu().numpy().view(np.uint8), host[name].view(np.uint8)), name
    for out in (torch.float32, dtype):
        ko, vo = (torch.full((t, heads, d), 7.0, device="cuda").to(out) for _ in range(2))
        rows(dev.kv4_read, desc(gpu), ko, vo, slots)
        for name, got in (("k", ko), ("v", vo)):
            for i, slot in enumerate(slots):
                p, at = divmod(int(slot), page)
                held = 0 <= slot < pages * page
                want = np.stack([ref.kv4_values(host, name, np.array([p]), h, np.array([at]))[0] for h in range(heads)]) if held else np.zeros((heads, d))
                want = torch.from_numpy(want.astype(np.float32)).to(out)
                assert torch.equal(got[i].cpu(), want), (name, i)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append_of_what_is_not_finite_or_tiny(hip, dtype):
    d, page = 64, 16
    k = torch.randn(6, 1, d, device="cuda").to(dtype)
    k[0, 0, 3], k[1, 0, 5], k[2, 0, 63] = float("nan"), float("inf"), float("-inf")
    k[3] *= 1e-38
    k[4] = 2.0 ** -120
    k[5] = 3e38
    host, gpu = new_cache(1, 1, page, d)
    rows(dev.kv4_append, desc(gpu), k, k, np.arange(6))
    ref.kv4_store(host, np.arange(6), k.float().cpu().numpy(), k.float().cpu().numpy())
    assert np.isnan(host["k_scale"][0, 0, :3]).all() and host["k_scale"][0, 0, 3] == 0 and host["k_scale"][0, 0, 4] > 0
    for name in host:
        assert np.array_equal(gpu[name].cpu().numpy().view(np.uint8), host[name].view(np.uint8)), name


def test_rows_with_strides(hip):
    """Heads before tokens, an odd element offset."""
    t, heads, d, page = 19, 3, 64, 16
    gen = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn(heads, t, d, generator=gen, device="cuda").transpose(0, 1)
    v = torch.randn(t * heads * 67 + 1, generator=gen, device="cuda")[1:].view(t, heads, 67)[..., 2:66]
    host, gpu = new_cache(2, heads, page, d)
    slots = np.arange(t) + 5
    rows(dev.kv4_append, desc(gpu), k, v, slots)
    ref.kv4_store(host, slots, k.cpu().numpy(), v.cpu().numpy())
    for name in host:
        assert np.array_equal(gpu[name].cpu().numpy(), host[name]), name
    ko, vo = torch.zeros(heads, t, d, device="cuda").transpose(0, 1), torch.zeros(t, heads, 67, device="cuda")[..., 2:66]
    rows(dev.kv4_read, desc(gpu), ko, vo, slots)
    k2, v2 = torch.zeros(t, heads, d, device="cuda"), torch.zeros(t, heads, d, device="cuda")
    rows(dev.kv4_read, desc(gpu), k2, v2, slots)
    assert torch.equal(ko, k2) and torch.equal(vo, v2) and float(k2.abs().max()) > 0


# ---- attention -------------------------------------------------------------------------

def filled(lens, heads, page, d, seed, spare=2, fill=255):
    """A cache whose requests' tokens are stored, in pages of no order; all else
    is `fill`.  -> host arrays, device arrays, table."""
    rng = np.random.default_rng(seed)
    need = [-(-int(n) // page) for n in lens]
    pages = sum(need) + spare
    perm = rng.permutation(pages)
    table = np.full((len(lens), max(need + [1])), -1)
    host, _ = new_cache(pages, heads, page, d, fill)
    at = 0
    for r, n in enumerate(lens):
        table[r, :need[r]] = perm[at:at + need[r]]
        at += need[r]
        j = np.arange(n)
        if n:
            x = rng.normal(size=(2, n, heads, d)).astype(np.float32)
            ref.kv4_store(host, table[r, j // page] * page + j % page, x[0], x[1])
    return host, {k: torch.from_numpy(v).cuda() for k, v in host.items()}, table


def attend(gpu, q, q_start, lens, table, causal=1, window=0, scale=None, max_new=None, max_len=None, out=None, lse=True, stream=None):
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
    t, hq, d = q.shape
    s = dict(start=i32(q_start), lens=i32(lens), table=i32(table), out=torch.full((t, hq, d), 7.0, device="cuda").to(q.dtype) if out is None else out,
             lse=torch.full((t, hq), 7.0, device="cuda") if lse else None)
    a = dev.Kv4Attend(cache=desc(gpu), dtype=dev.DTYPES[str(q.dtype)[6:]], causal=causal, requests=len(lens), tokens=t, q_heads=hq,
                      q_start=s["start"].data_ptr(), kv_lens=s["lens"].data_ptr(), block_table=s["table"].data_ptr(), table_width=table.shape[1],
                      max_new=int(np.max(np.diff(q_start))) if max_new is None else max_new, max_len=int(np.max(lens)) if max_len is None else max_len,
                      window=window, scale=d ** -0.5 if scale is None else scale, lse=s["lse"].data_ptr() if lse else None)
    a.q, a.q_token_stride, a.q_head_stride = strided(q)
    a.out, a.out_token_stride, a.out_head_stride = strided(s["out"])
    need = dev.kv4_attend_workspace(a)
    s["work"] = torch.full((need + 16,), 255, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = s["work"].data_ptr(), need
    torch.cuda.synchronize()
    dev.kv4_attend(a, stream)
    torch.cuda.synchronize()
    s["args"], s["q"] = a, q
    return s


def check(host, s, q_start, lens, table, causal=1, window=0, scale=None, max_len=None):
    q = s["q"]
    dtype = str(q.dtype)[6:]
    want, lse, size, reach = ref.attend(host, np64(q), q_start, lens, table, q.shape[2] ** -0.5 if scale is None else scale, causal, window, max_len)
    score = reach * (2.0 ** -16)
    weights = 2.0 ** -15 if dtype == "float32" else 2.0 ** -8
    tol = (2 * score + weights)[..., None] * size
    got = np64(s["out"])
    err = np.abs(got - want)
    assert np.all(err <= tol + ref.rounding(dtype, np.abs(want) + tol)), (np.max(err), np.argwhere(~(err <= tol + ref.rounding(dtype, np.abs(want) + tol)))[:3])
    if s["lse"] is not None:
        g = np64(s["lse"])
        assert np.array_equal(np.isneginf(g), np.isneginf(lse))
        fine = np.isfinite(lse)
        assert np.all(np.abs(g[fine] - lse[fine]) <= score[fine] + 2.0 ** -20 * (1 + np.abs(lse[fine])))
    empty = np.isneginf(lse)
    assert not np.any(got[empty])


def queries(t, hq, d, dtype, seed, amp=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (amp * torch.randn(t, hq, d, generator=gen, device="cuda")).to(dtype)


def starts(new):
    return np.concatenate([[0], np.cumsum(new)])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 5), (1, 16), (3, 2), (1, 40)])
def test_decode(hip, d, heads, group, dtype):
    """One token a request, lengths about every edge of pages and tiles."""
    lens = np.array([1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 200, 0, 255, 256, 257])
    host, gpu, table = filled(lens, heads, 16 if d < 256 else 32, d, d + group)
    q = queries(len(lens), heads * group, d, dtype, d)
    start = np.arange(len(lens) + 1)
    check(host, attend(gpu, q, start, lens, table), start, lens, table)


@pytest.mark.parametrize("page", [16, 48, 128])
@pytest.mark.parametrize("group", [1, 4])
@pytest.mark.parametrize("window", [0, 1, 64, 100, 1000])
def test_long_axis_is_split_and_joined(hip, page, group, window):
    lens = np.array([5000, 3, 2777, 1024])
    host, gpu, table = filled(lens, 2, page, 64, page + group)
    q = queries(4, 2 * group, 64, torch.float32, 5)
    start = np.arange(5)
    s = attend(gpu, q, start, lens, table, window=window)
    check(host, s, start, lens, table, window=window)
    again = attend(gpu, q, start, lens, table, window=window)
    assert torch.equal(s["out"], again["out"]) and torch.equal(s["lse"], again["lse"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,heads,group,page", [(128, 1, 1, 16), (64, 2, 3, 32), (128, 2, 5, 16), (256, 1, 2, 64), (128, 1, 17, 16)])
@pytest.mark.parametrize("causal,window", [(1, 0), (0, 0), (1, 33), (1, 300)])
def test_chunks(hip, d, heads, group, page, dtype, causal, window):
    """Several query tokens a request, ragged: none, one, a few, many."""
    new = np.array([3, 0, 1, 70, 17, 130])
    lens = np.array([9, 40, 300, 70, 200, 419])
    host, gpu, table = filled(lens, heads, page, d, d + group + page)
    q = queries(int(new.sum()), heads * group, d, dtype, 3)
    check(host, attend(gpu, q, starts(new), lens, table, causal, window), starts(new), lens, table, causal, window)


@pytest.mark.parametrize("causal,window,page", [(1, 0, 16), (0, 0, 48), (1, 70, 32)])
def test_a_batch_of_long_chunks(hip, causal, window, page):
    """Enough rows for blocks of 128 of them: chunks beside single tokens and
    requests without any, lengths about the edges of steps, hidden pages."""
    new = np.array([257, 300, 1, 0, 259, 320, 257, 2, 258, 299, 511, 257])
    lens = np.array([257, 411, 700, 64, 320, 250, 513, 40, 385, 300, 600, 1000])
    heads = 16
    host, gpu, table = filled(lens, heads, page, 128, page)
    table = table.copy()
    table[5, 1], table[8, 0] = -1, len(host["k"]) + 3
    q = queries(int(new.sum()), heads, 128, torch.bfloat16, 3)
    s = attend(gpu, q, starts(new), lens, table, causal, window)
    check(host, s, starts(new), lens, table, causal, window)
    # strides, and a NaN scale that only the rows that see it meet
    wide = torch.zeros(q.shape[0], heads + 1, 131, dtype=torch.bfloat16, device="cuda")
    wide[:, :heads, 1:129] = q
    out = torch.full((q.shape[0], heads, 132), 3.0, dtype=torch.bfloat16, device="cuda")
    t = attend(gpu, wide[:, :heads, 1:129], starts(new), lens, table, causal, window, out=out[..., :128])
    assert torch.equal(t["out"], s["out"]) and torch.equal(t["lse"], s["lse"]) and float((out[..., 128:].float() - 3).abs().max()) == 0
    bad, r = 280, 1
    gpu["v_scale"][table[r, bad // page], :, bad % page] = float("nan")
    got = np.isnan(np64(attend(gpu, q, starts(new), lens, table, causal, window)["out"])).all(-1)
    pos = lens[r] - new[r] + np.arange(new[r])
    sees = (pos >= bad) & ((pos - window < bad) | (window == 0)) if causal else np.ones(new[r], bool)
    want = np.zeros(q.shape[0], bool)
    want[starts(new)[r]:starts(new)[r + 1]] = sees
    assert np.array_equal(got, np.repeat(want[:, None], heads, 1))


def test_rows_without_keys(hip):
    """More new tokens than keys: the first queries see nothing; a request without keys."""
    new, lens = np.array([5, 2, 4]), np.array([2, 0, 4])
    host, gpu, table = filled(lens, 1, 16, 128, 1)
    for dtype in (torch.float32, torch.bfloat16):
        q = queries(11, 4, 128, dtype, 2)
        s = attend(gpu, q, starts(new), lens, table)
        check(host, s, starts(new), lens, table)
        assert np.isneginf(np64(s["lse"])[:3]).all() and np.isfinite(np64(s["lse"])[3:5]).all() and np.isneginf(np64(s["lse"])[5:7]).all()


def test_bounds_and_pages_outside_the_cache(hip):
    """max_len below a length hides the keys past it, max_new the queries past
    it; a table entry outside the cache hides its page."""
    lens, new = np.array([100, 90]), np.array([4, 2])
    host, gpu, table = filled(lens, 2, 16, 64, 7)
    q = queries(6, 2, 64, torch.float32, 4)
    s = attend(gpu, q, starts(new), lens, table, max_len=70)
    check(host, s, starts(new), lens, table, max_len=70)
    s = attend(gpu, q, starts(new), lens, table, max_new=2)
    assert float((s["out"][2:4] - 7.0).abs().max()) == 0 and float((s["lse"][2:4] - 7.0).abs().max()) == 0
    hidden = table.copy()
    hidden[0, 2], hidden[1, 0], hidden[1, 3] = -1, len(host["k"]), 2 ** 31 - 1
    check(host, attend(gpu, q, starts(new), lens, hidden), starts(new), lens, hidden)
    check(host, attend(gpu, q, starts(new), lens, table[:, :3]), starts(new), lens, table[:, :3])


@pytest.mark.parametrize("heads,requests,window", [(1, 3, 0), (8, 40, 0), (4, 3, 50), (8, 40, 130)])
def test_bounds_that_bound_nothing(hip, heads, requests, window):
    """The largest max_len and max_new: the table's width and the batch bound the work."""
    rng = np.random.default_rng(requests + window)
    new = rng.integers(1, 4, requests)
    lens = new + rng.integers(0, 900, requests)
    host, gpu, table = filled(lens, heads, 16, 128, 5)
    for dtype in (torch.float32, torch.bfloat16):
        q = queries(int(new.sum()), 2 * heads, 128, dtype, 4)
        s = attend(gpu, q, starts(new), lens, table, 1, window, max_new=(1 << 30) - 1, max_len=(1 << 31) - 1)
        check(host, s, starts(new), lens, table, 1, window)


def test_tokens_of_no_request_are_left_alone(hip):
    """Padding before the first and past the last request's tokens."""
    lens = np.array([20, 33])
    host, gpu, table = filled(lens, 1, 16, 64, 7)
    q = queries(6, 1, 64, torch.bfloat16, 4)
    start = np.array([1, 2, 4])
    s = attend(gpu, q, start, lens, table)
    check(host, dict(s, out=s["out"][1:4], lse=s["lse"][1:4], q=q[1:4]), start - 1, lens, table)
    for t in (0, 4, 5):
        assert float((s["out"][t].float() - 7.0).abs().max()) == 0 and float((s["lse"][t] - 7.0).abs().max()) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(hip, dtype):
    """q out of a fused projection, out with gaps, odd element offsets."""
    lens, new = np.array([50, 70, 8]), np.array([1, 9, 2])
    host, gpu, table = filled(lens, 2, 16, 128, 11)
    base = queries(12, 11, 128, dtype, 3).reshape(-1)
    q = base[1:1 + 12 * 8 * 129 + 0].view(12, 8, 129)[:, 1:5, :128]
    out = torch.full((12, 4, 131), 3.0, device="cuda").to(dtype)
    s = attend(gpu, q, starts(new), lens, table, out=out[..., 1:129])
    check(host, s, starts(new), lens, table)
    assert float((out[..., 0].float() - 3).abs().max()) == 0 and float((out[..., 129:].float() - 3).abs().max()) == 0


@pytest.mark.parametrize("n,new", [(40, 1), (700, 1), (90, 60)])
def test_nan_keys_reach_the_rows_that_see_them_only(hip, n, new):
    lens = np.array([n, n])
    host, gpu, table = filled(lens, 1, 16, 64, 2)
    bad = n - 2
    gpu["v_scale"][table[0, bad // 16], 0, bad % 16] = float("nan")
    q = queries(2 * new, 2, 64, torch.float32, 8)
    s = attend(gpu, q, starts([new, new]), lens, table)
    got = np.isnan(np64(s["out"])).all(-1)
    sees = np.concatenate([np.arange(n - new, n) >= bad, np.zeros(new, bool)])
    assert np.array_equal(got, np.repeat(sees[:, None], 2, 1)) and np.array_equal(np.isnan(np64(s["out"])).any(-1), got)
    gpu["k_scale"][table[1, 0], 0, 3] = float("nan")
    s = attend(gpu, q, starts([new, new]), lens, table)
    assert np.isnan(np64(s["out"])[new:]).all()


@pytest.mark.parametrize("amp", [0.0, 1e-20, 300.0, 1e6])
def test_scores_of_any_size(hip, amp):
    """Rows of equal scores, and rows that one key takes whole."""
    lens, new = np.array([130, 90]), np.array([1, 5])
    host, gpu, table = filled(lens, 1, 16, 128, 6)
    for dtype in (torch.float32, torch.bfloat16):
        q = queries(6, 3, 128, dtype, 1, amp)
        s = attend(gpu, q, starts(new), lens, table)
        if amp <= 1:
            check(host, s, starts(new), lens, table)
        else:
            # a score's error is a factor here; compare where one key leads by more than it
            want, lse, size, reach = ref.attend(host, np64(q), starts(new), lens, table, 128 ** -0.5, 1, 0)
            assert np.all(np.abs(np64(s["lse"]) - lse) <= 2.0 ** -15 * (reach + np.abs(lse)))
            assert torch.isfinite(s["out"].float()).all()


def test_offsets_past_32_bits(hip):
    """A cache whose code arrays pass 4 GiB: pages at its far end."""
    heads, page, d = 64, 128, 256
    pages = (5 << 30) // (heads * page * d // 2)
    t = dict(k=torch.zeros(pages, heads, page, d // 2, dtype=torch.uint8, device="cuda"),
             v=torch.zeros(pages, heads, page // 16, d // 2, 16, dtype=torch.uint8, device="cuda"),
             k_scale=torch.zeros(pages, heads, page, device="cuda"), v_scale=torch.zeros(pages, heads, page, device="cuda"))
    n = 2 * page - 3
    gen = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(n, heads, d, generator=gen, device="cuda") for _ in range(2))
    table = np.array([[pages - 1, pages - 2]])
    j = np.arange(n)
    slots = table[0, j // page] * page + j % page
    rows(dev.kv4_append, desc(t), k, v, slots)
    small = {name: a[pages - 2:].contiguous() for name, a in t.items()}
    host = {name: a.cpu().numpy() for name, a in small.items()}
    want, _ = new_cache(2, heads, page, d)
    ref.kv4_store(want, slots - (pages - 2) * page, k.cpu().numpy(), v.cpu().numpy())
    for name in host:
        assert np.array_equal(host[name], want[name]), name
    q = queries(2, heads, d, torch.bfloat16, 4)
    s = attend(t, q, np.array([0, 2]), np.array([n]), table)
    near = attend(small, q, np.array([0, 2]), np.array([n]), table - (pages - 2))
    assert torch.equal(s["out"], near["out"]) and torch.equal(s["lse"], near["lse"])
    check(host, near, np.array([0, 2]), np.array([n]), table - (pages - 2))


def test_in_a_graph_and_on_another_stream(hip):
    """A decode step of three requests replayed as their lengths grow."""
    lens = np.array([700, 31, 90])
    host, gpu, table = filled(lens + 8, 2, 16, 64, 13)
    q = queries(3, 4, 64, torch.float32, 3)
    st = torch.cuda.Stream()
    start = np.arange(4)
    s = attend(gpu, q, start, lens, table, max_len=708, stream=st.cuda_stream)
    check(host, s, start, lens, table)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        dev.kv4_attend(s["args"], st.cuda_stream)
    for step in range(1, 4):
        s["lens"] += 2
        q.mul_(0.75)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(host, s, start, lens + 2 * step, table)
        eager = attend(gpu, q, start, lens + 2 * step, table, max_len=708)
        assert torch.equal(eager["out"], s["out"])


def test_no_lse_wanted(hip):
    lens = np.array([900, 12])
    host, gpu, table = filled(lens, 1, 16, 64, 5)
    q = queries(2, 1, 64, torch.float16, 3)
    check(host, attend(gpu, q, np.arange(3), lens, table, lse=False), np.arange(3), lens, table)
