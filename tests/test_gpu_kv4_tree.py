"""GPU: attention of drafted tokens over the 4-bit cache against softmax
attention in 64 bits on the stored values.

Tolerances as for sili_kv4_attend, which shares its products: a score is off by
at most 2^-16 of the sum of its terms' magnitudes (float32: three bf16 parts are
24 bits; the rest is for float32 sums of up to 256 terms), so a weight by twice
that, relative; a weight enters with 16 bits or more (bf16, f16: 8, where one
part may do: 2^-8 each), and the output is rounded once."""
import numpy as np
import pytest
import torch

from sili__new_amd import device as dev
from tests import block_ref, draft_ref as ref
from tests.test_gpu_kv4 import attend as attend_causal, desc, filled, np64, queries, starts, strided

pytestmark = pytest.mark.gpu


def attend(gpu, q, masks, q_start, lens, table, window=0, scale=None, max_new=None, max_len=None, out=None, lse=True, stream=None):
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
    t, hq, d = q.shape
    s = dict(start=i32(q_start), lens=i32(lens), table=i32(table), masks=torch.from_numpy(np.array([int(m) for m in masks], np.uint64).view(np.int64)).cuda(),
             out=torch.full((t, hq, d), 7.0, device="cuda").to(q.dtype) if out is None else out,
             lse=torch.full((t, hq), 7.0, device="cuda") if lse else None)
    a = dev.Kv4Attend(cache=desc(gpu), dtype=dev.DTYPES[str(q.dtype)[6:]], causal=1, requests=len(lens), tokens=t, q_heads=hq,
                      q_start=s["start"].data_ptr(), kv_lens=s["lens"].data_ptr(), block_table=s["table"].data_ptr(), table_width=table.shape[1],
                      max_new=int(min(64, np.max(np.diff(q_start)))) if max_new is None else max_new,
                      max_len=int(np.max(lens)) if max_len is None else max_len,
                      window=window, scale=d ** -0.5 if scale is None else scale, lse=s["lse"].data_ptr() if lse else None)
    a.q, a.q_token_stride, a.q_head_stride = strided(q)
    a.out, a.out_token_stride, a.out_head_stride = strided(s["out"])
    need = dev.kv4_attend_tree_workspace(a)
    s["work"] = torch.full((need + 16,), 255, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = s["work"].data_ptr(), need
    torch.cuda.synchronize()
    dev.kv4_attend_tree(a, s["masks"].data_ptr(), stream)
    torch.cuda.synchronize()
    assert bool((s["work"][need:] == 255).all())
    s["args"], s["q"] = a, q
    return s


def check(host, s, masks, q_start, lens, table, window=0, scale=None, max_len=None, rows=None):
    """rows: those that are compared (all)."""
    q = s["q"]
    dtype = str(q.dtype)[6:]
    rows = np.arange(q.shape[0]) if rows is None else rows
    want, lse, size, reach = (x[rows] for x in ref.attend_tree(host, np64(q), masks, q_start, lens, table,
                                                               q.shape[2] ** -0.5 if scale is None else scale, window, max_len))
    score = reach * 2.0 ** -16
    weights = 2.0 ** -15 if dtype == "float32" else 2.0 ** -8
    tol = (2 * score + weights)[..., None] * size
    got = np64(s["out"])[rows]
    tol = tol + block_ref.rounding(dtype, np.abs(want) + tol)
    err = np.abs(got - want)
    assert np.all(err <= tol), (np.max(err), np.argwhere(~(err <= tol))[:3])
    if s["lse"] is not None:
        g = np64(s["lse"])[rows]
        assert np.array_equal(np.isneginf(g), np.isneginf(lse))
        fine = np.isfinite(lse)
        assert np.all(np.abs(g[fine] - lse[fine]) <= score[fine] + 2.0 ** -20 * (1 + np.abs(lse[fine])))
    assert not np.any(got[np.isneginf(lse)])


def tree_masks(rng, new):
    parents = np.concatenate([[int(rng.integers(max(-1, i - 5), i)) if i else -1 for i in range(n)] for n in new] + [np.zeros(0, int)]).astype(int)
    return ref.draft_tree(parents, starts(new), [0] * len(new))[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads,group,page", [(1, 1, 16), (2, 5, 48), (1, 16, 32), (3, 2, 128)])
def test_trees(hip, d, heads, group, page, dtype):
    """Trees of one token to 64, contexts about the edges of steps of 64 keys."""
    new = np.array([1, 64, 3, 0, 17, 64, 2, 31])
    lens = np.array([1, 64, 66, 40, 64 + 17, 191, 300, 129])
    host, gpu, table = filled(lens, heads, page, d, d + group + page)
    masks = tree_masks(np.random.default_rng(d + group), new)
    q = queries(int(new.sum()), heads * group, d, dtype, 3)
    check(host, attend(gpu, q, masks, starts(new), lens, table), masks, starts(new), lens, table)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window", [1, 2, 5, 33, 64, 100, 300, 2 ** 31 - 1])
def test_windows(hip, window, dtype):
    """A window that ends in the context, at its end, among the drafted tokens."""
    new = np.array([40, 5, 64, 1, 9])
    lens = np.array([340, 69, 64, 1, 265])
    host, gpu, table = filled(lens, 2, 16, 64, 7)
    masks = tree_masks(np.random.default_rng(window), new)
    q = queries(int(new.sum()), 6, 64, dtype, 3)
    check(host, attend(gpu, q, masks, starts(new), lens, table, window), masks, starts(new), lens, table, window)


@pytest.mark.parametrize("window", [0, 700])
@pytest.mark.parametrize("dtype,group,d", [(torch.float32, 1, 128), (torch.bfloat16, 5, 128), (torch.float16, 2, 64), (torch.bfloat16, 1, 256),
                                           (torch.bfloat16, 12, 128)])
def test_a_long_axis_is_split_and_joined(hip, window, dtype, group, d):
    new = np.array([13, 64, 1])
    lens = np.array([9001, 2777, 5056])
    host, gpu, table = filled(lens, 2, 16, d, 3)
    masks = tree_masks(np.random.default_rng(5), new)
    q = queries(int(new.sum()), 2 * group, d, dtype, 5)
    s = attend(gpu, q, masks, starts(new), lens, table, window)
    check(host, s, masks, starts(new), lens, table, window)
    again = attend(gpu, q, masks, starts(new), lens, table, window)
    assert torch.equal(s["out"], again["out"]) and torch.equal(s["lse"], again["lse"])


@pytest.mark.parametrize("dtype,d", [(torch.float32, 128), (torch.bfloat16, 256), (torch.float16, 64)])
@pytest.mark.parametrize("longest", [1280, 1281, 2600])
def test_many_blocks_over_contexts_about_a_split(hip, longest, dtype, d):
    """128 and 120 (request, kv head) pairs of one tile of rows: whole, and split from one length on."""
    rng = np.random.default_rng(longest)
    for requests in (16, 15):
        new = rng.integers(1, 8, requests)
        lens = rng.integers(8, longest + 1, requests)
        lens[3], lens[4] = longest, longest - 1
        host, gpu, table = filled(lens, 8, 16, d, 5)
        masks = tree_masks(rng, new)
        q = queries(int(new.sum()), 16, d, dtype, 3)
        for window in (0, 1217):
            check(host, attend(gpu, q, masks, starts(new), lens, table, window), masks, starts(new), lens, table, window)


def test_two_calls_at_once_on_streams_of_their_own(hip):
    """Split calls with a workspace each, in turn on two streams, against the same calls one after another."""
    rng = np.random.default_rng(6)
    new, lens = np.array([13, 64, 1]), np.array([9001, 2777, 5056])
    host, gpu, table = filled(lens, 2, 16, 128, 3)
    calls = []
    for seed in (5, 6):
        masks = tree_masks(rng, new)
        q = queries(int(new.sum()), 10, 128, torch.bfloat16, seed)
        calls.append((attend(gpu, q, masks, starts(new), lens, table), torch.cuda.Stream()))
    want = [(s["out"].clone(), s["lse"].clone()) for s, _ in calls]
    for s, _ in calls:
        s["out"].fill_(7)
        s["lse"].fill_(7)
    torch.cuda.synchronize()
    for _ in range(5):
        for s, st in calls:
            dev.kv4_attend_tree(s["args"], s["masks"].data_ptr(), st.cuda_stream)
    torch.cuda.synchronize()
    for (s, _), (out, lse) in zip(calls, want):
        assert torch.equal(s["out"], out) and torch.equal(s["lse"], lse)


def test_many_requests_of_large_trees(hip):
    """Enough blocks of many rows to fill the GPU, requests without tokens and of one among them; hidden pages."""
    rng = np.random.default_rng(8)
    new = rng.integers(48, 65, 40)
    new[[3, 17]], new[[5, 30]] = 0, 1
    lens = new + rng.integers(0, 400, 40)
    lens[7], lens[9] = new[7], new[9] + 64
    host, gpu, table = filled(lens, 8, 16, 128, 4)
    table = table.copy()
    table[11, 1], table[12, 0], table[13, 0] = -1, len(host["k"]), 2 ** 31 - 1
    masks = tree_masks(rng, new)
    for dtype in (torch.bfloat16, torch.float16):
        q = queries(int(new.sum()), 40, 128, dtype, 3)
        for window in (0, 90):
            check(host, attend(gpu, q, masks, starts(new), lens, table, window), masks, starts(new), lens, table, window)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks_of_any_kind(hip, dtype):
    """No bits (the context alone, or nothing), all bits, bits past the request's tokens, no own bit."""
    rng = np.random.default_rng(2)
    new = np.array([6, 4, 64, 3])
    lens = np.array([70, 4, 150, 10])
    full = 2 ** 64 - 1
    masks = [0, full, 1 << 5, 1 << 63, 0b101010, full - 1] + [0, 0b1000, full << 4 & full, 0b0110] + [int(m) for m in rng.integers(0, 2 ** 63, 64)] + [1 << 2, 0, 7]
    host, gpu, table = filled(lens, 2, 16, 128, 9)
    q = queries(int(new.sum()), 4, 128, dtype, 3)
    for window in (0, 3):
        s = attend(gpu, q, masks, starts(new), lens, table, window)
        check(host, s, masks, starts(new), lens, table, window)
        lse = np64(s["lse"])
        assert np.isneginf(lse[[6, 8]]).all() and np.isfinite(lse[:6]).all()


def test_a_chain_is_the_causal_mask(hip):
    new, lens = np.array([9, 64, 1]), np.array([200, 64, 31])
    host, gpu, table = filled(lens, 2, 16, 128, 1)
    masks = [2 ** (i + 1) - 1 for n in new for i in range(n)]
    for dtype in (torch.float32, torch.bfloat16):
        for window in (0, 20):
            q = queries(int(new.sum()), 6, 128, dtype, 2)
            s = attend(gpu, q, masks, starts(new), lens, table, window)
            c = attend_causal(gpu, q, starts(new), lens, table, window=window)
            check(host, s, masks, starts(new), lens, table, window)
            check(host, dict(c, q=q), masks, starts(new), lens, table, window)


def test_more_tokens_than_keys(hip):
    """The first new tokens lie before the first key."""
    new, lens = np.array([5, 2, 4]), np.array([2, 0, 4])
    host, gpu, table = filled(lens, 1, 16, 64, 1)
    masks = tree_masks(np.random.default_rng(1), new)
    # key base + j exists from j = 3 on in the first request
    want = [m >> 3 & 0b11 for m in masks[:5]]
    for dtype in (torch.float32, torch.bfloat16):
        s = attend(gpu, queries(11, 2, 64, dtype, 2), masks, starts(new), lens, table)
        lse = np64(s["lse"])
        assert np.array_equal(np.isneginf(lse[:5, 0]), np.array(want) == 0) and np.isneginf(lse[5:7]).all() and np.isfinite(lse[7:]).all()
        assert not np64(s["out"])[np.isneginf(lse)].any()
        check(host, s, masks, starts(new), lens, table, rows=np.arange(7, 11))


def test_bounds_and_pages_outside_the_cache(hip):
    lens, new = np.array([100, 90]), np.array([4, 20])
    host, gpu, table = filled(lens, 2, 16, 64, 7)
    masks = tree_masks(np.random.default_rng(3), new)
    q = queries(24, 2, 64, torch.float32, 4)
    s = attend(gpu, q, masks, starts(new), lens, table, max_len=80)
    check(host, s, masks, starts(new), lens, table, max_len=80)
    s = attend(gpu, q, masks, starts(new), lens, table, max_len=(1 << 31) - 1, max_new=64)
    check(host, s, masks, starts(new), lens, table)
    s = attend(gpu, q, masks, starts(new), lens, table, max_new=2)
    left = np.r_[2:4, 6:24]
    assert float((s["out"][left] - 7.0).abs().max()) == 0 and float((s["lse"][left] - 7.0).abs().max()) == 0
    check(host, s, masks, starts(new), lens, table, rows=np.array([0, 1, 4, 5]))
    hidden = table.copy()
    hidden[0, 2], hidden[0, 6], hidden[1, 0], hidden[1, 5] = -1, -5, len(host["k"]), 2 ** 31 - 1
    check(host, attend(gpu, q, masks, starts(new), lens, hidden), masks, starts(new), lens, hidden)
    check(host, attend(gpu, q, masks, starts(new), lens, table[:, :5]), masks, starts(new), lens, table[:, :5])


@pytest.mark.parametrize("start,lens", [([0, 70, 74], [300, 90]), ([0, 4, 2 ** 31 - 1], [100, 90]), ([-1, 4, 6], [100, 90]), ([3, 1, 6], [100, 90]),
                                        ([0, 4, 6], [-7, 2 ** 31 - 1]), ([0, 4, 6], [2 ** 31 - 1, -2 ** 31])])
def test_starts_and_lengths_of_any_value_stay_within_the_buffers(hip, start, lens):
    """What is in bounds is computed or left alone; nothing else is touched."""
    _, gpu, table = filled(np.array([100, 90]), 1, 16, 64, 7)
    t = 76 if start[1] == 70 else 6
    masks = [1] * t
    for window in (0, 30):
        s = attend(gpu, queries(t, 2, 64, torch.bfloat16, 4), masks, np.array(start), np.array(lens), table, window, max_new=64, max_len=2 ** 31 - 1)
        out = np64(s["out"])
        assert (np.isfinite(out) | np.isnan(out)).all()
        if start[1] == 70:  # of 70 new tokens the first 64
            assert (out[64:70] == 7).all() and not (out[63] == 7).any() and not (out[70] == 7).any()


def test_strides_and_padding(hip):
    lens, new = np.array([50, 70, 8]), np.array([1, 9, 2])
    host, gpu, table = filled(lens, 2, 16, 128, 11)
    start = starts(new) + 1  # a row before the first request's, two past the last's
    masks = [0] + tree_masks(np.random.default_rng(3), new) + [2 ** 64 - 1] * 2
    for dtype in (torch.float32, torch.bfloat16):
        base = queries(15, 11, 128, dtype, 3).reshape(-1)
        q = base[1:1 + 15 * 8 * 129].view(15, 8, 129)[:, 1:5, :128]
        out = torch.full((15, 4, 131), 3.0, device="cuda").to(dtype)
        s = attend(gpu, q, masks, start, lens, table, out=out[..., 1:129], max_new=9)
        check(host, s, masks, start, lens, table, rows=np.arange(1, 13))
        assert float((out[..., 0].float() - 3).abs().max()) == 0 and float((out[..., 129:].float() - 3).abs().max()) == 0
        for t in (0, 13, 14):
            assert float((out[t].float() - 3.0).abs().max()) == 0 and float((s["lse"][t] - 7.0).abs().max()) == 0


@pytest.mark.parametrize("many", [False, True])
def test_nan_keys_reach_the_rows_that_see_them_only(hip, many):
    """In the context all rows of the request; a drafted one its descendants."""
    new = np.array([30, 30] * (20 if many else 1))
    lens = np.array([200, 100] * (20 if many else 1))
    heads = 8 if many else 1
    _, gpu, table = filled(lens, heads, 16, 128, 2)
    masks = tree_masks(np.random.default_rng(6), new)
    bad = 200 - 30 + 4
    for name in ("v_scale", "k_scale"):
        gpu[name][table[0, bad // 16], :, bad % 16] = float("nan")
    gpu["v_scale"][table[1, 1], :, 5] = float("nan")
    q = queries(int(new.sum()), heads * 9, 128, torch.bfloat16, 8)
    out = np64(attend(gpu, q, masks, starts(new), lens, table)["out"])
    got = np.isnan(out).all((-1, -2))
    assert np.array_equal(got, np.isnan(out).any((-1, -2)))
    assert np.array_equal(got[:30], np.array([m >> 4 & 1 == 1 for m in masks[:30]])) and got[30:60].all() and not got[60:].any()


def test_replayed_with_other_trees_on_another_stream(hip):
    new = np.array([12, 7, 30])
    lens = np.array([700, 31, 90])
    host, gpu, table = filled(lens + 8, 2, 16, 64, 13)
    rng = np.random.default_rng(1)
    masks = tree_masks(rng, new)
    q = queries(49, 4, 64, torch.float32, 3)
    st = torch.cuda.Stream()
    s = attend(gpu, q, masks, starts(new), lens, table, max_len=708, stream=st.cuda_stream)
    check(host, s, masks, starts(new), lens, table)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        dev.kv4_attend_tree(s["args"], s["masks"].data_ptr(), st.cuda_stream)
    for step in range(1, 4):
        s["lens"] += 2
        masks = tree_masks(rng, new)
        s["masks"].copy_(torch.from_numpy(np.array(masks, np.uint64).view(np.int64)))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(host, s, masks, starts(new), lens + 2 * step, table)
        eager = attend(gpu, q, masks, starts(new), lens + 2 * step, table, max_len=708)
        assert torch.equal(eager["out"], s["out"])
