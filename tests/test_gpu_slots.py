"""GPU: block tables, slot maps and positions from request lengths, equal to a
loop over the requests in Python."""
import numpy as np
import pytest
import torch

from sili__new_amd import device as dev
from tests import block_ref as ref

pytestmark = pytest.mark.gpu


def build(old, new, page, free, table, max_tokens, stream=None):
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
    n = len(old)
    t = dict(old=i32(old), new=i32(new), free=i32(free), block_table=i32(table))
    for name, size in (("q_start", n + 1), ("kv_lens", n), ("positions", max_tokens), ("slots", max_tokens), ("status", 2)):
        t[name] = torch.full((size,), -77, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    a = dev.RequestSlots(cached_lens=t["old"].data_ptr(), new_lens=t["new"].data_ptr(), requests=n, page_size=page,
                         free_pages=t["free"].data_ptr(), n_free=len(free), block_table=t["block_table"].data_ptr(),
                         table_width=np.asarray(table).shape[1], max_tokens=max_tokens, q_start=t["q_start"].data_ptr(),
                         kv_lens=t["kv_lens"].data_ptr(), positions=t["positions"].data_ptr(), slots=t["slots"].data_ptr(),
                         status=t["status"].data_ptr())
    dev.request_slots(a, stream)
    torch.cuda.synchronize()
    t["again"] = a
    return t


def same(got, want):
    for name, w in want.items():
        g = got[name].cpu().numpy()
        assert np.array_equal(g, w), (name, np.argwhere(g != w)[:4], g[g != w][:4], w[g != w][:4])


def scene(n, page, longest, chunk, seed, spare=4):
    rng = np.random.default_rng(seed)
    old = rng.integers(0, longest + 1, n)
    new = np.where(rng.random(n) < 0.5, rng.integers(0, 2, n), rng.integers(0, chunk + 1, n))
    have = -(-old // page)
    fresh = int((-(-(old + new) // page) - have).sum())
    width = -(-(longest + chunk) // page) + 1
    perm = rng.permutation(int(have.sum()) + fresh + spare)
    table = np.full((n, width), -1)
    at = 0
    for r in range(n):
        table[r, :have[r]] = perm[at:at + have[r]]
        at += have[r]
    return old, new, perm[at:], table, int(new.sum())


@pytest.mark.parametrize("n,page,longest,chunk", [(1, 16, 40, 1), (1, 1, 5, 9), (7, 16, 100, 40), (64, 16, 3000, 1), (63, 48, 500, 300),
                                                  (512, 32, 200, 5), (513, 16, 90, 50), (4096, 16, 64, 9), (4097, 16, 64, 9),
                                                  (9001, 32, 50, 3)])
@pytest.mark.parametrize("room", [0, 37])
def test_matches_a_loop(hip, n, page, longest, chunk, room):
    old, new, free, table, total = scene(n, page, longest, chunk, n + page)
    got = build(old, new, page, free, table, total + room)
    same(got, ref.request_slots(old, new, page, free, table, total + room))
    # the same call again, on the table it has written: the same
    dev.request_slots(got["again"])
    torch.cuda.synchronize()
    same(got, ref.request_slots(old, new, page, free, table, total + room))


@pytest.mark.parametrize("n", [5, 5000])
def test_what_does_not_fit_is_said(hip, n):
    old, new, free, table, total = scene(n, 16, 100, 60, 3)
    same(build(old, new, 16, free[:3], table, total), ref.request_slots(old, new, 16, free[:3], table, total))
    same(build(old, new, 16, free[:0], table, total), ref.request_slots(old, new, 16, free[:0], table, total))
    narrow = table[:, :3]
    same(build(old, new, 16, free, narrow, total), ref.request_slots(old, new, 16, free, narrow, total))
    same(build(old, new, 16, free, table, total // 2), ref.request_slots(old, new, 16, free, table, total // 2))
    bad = old.copy()
    bad[n // 2] = -5
    same(build(bad, new, 16, free, table, total), ref.request_slots(bad, new, 16, free, table, total))
    lost = np.where(table >= 0, -1, table)
    same(build(old, new, 16, free, lost, total), ref.request_slots(old, new, 16, free, lost, total))


def test_no_requests_and_no_tokens(hip):
    e = np.zeros(0, np.int32)
    got = build(e, e, 16, e, np.zeros((0, 4)), 5)
    same(got, dict(q_start=[0], status=[0, 0], slots=[-1] * 5, positions=[0] * 5))
    got = build([3, 0, 16], [0, 0, 0], 16, [9], np.full((3, 2), 1), 0)
    same(got, dict(q_start=[0, 0, 0, 0], kv_lens=[3, 0, 16], status=[0, 0]))


def test_slots_past_31_bits_are_refused_on_the_device(hip):
    got = build([0], [3], 1 << 20, [4000], np.full((1, 1), -1), 3)
    same(got, dict(slots=[-1] * 3, positions=[0, 1, 2], status=[1, dev.SLOTS_BAD_PAGE]))
    got = build([2 ** 31 - 2], [5], 1 << 30, [1], np.array([[0, 1]]), 6)
    same(got, dict(kv_lens=[2 ** 31 - 1], q_start=[0, 1], slots=[2 ** 31 - 2] + [-1] * 5, status=[0, dev.SLOTS_BAD_LENGTH]))


def test_in_a_graph_and_on_another_stream(hip):
    old, new, free, table, total = scene(33, 16, 300, 20, 8)
    want = ref.request_slots(old, new, 16, free, table, total + 5)
    st = torch.cuda.Stream()
    got = build(old, new, 16, free, table, total + 5, st.cuda_stream)
    same(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        dev.request_slots(got["again"], st.cuda_stream)
    for k in range(3):
        # a request grows between the replays, as a step does
        new2 = new.copy()
        new2[k] += k
        got["new"].copy_(torch.from_numpy(new2.astype(np.int32)))
        got["block_table"].copy_(torch.from_numpy(table.astype(np.int32)))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        same(got, ref.request_slots(old, new2, 16, free, table, total + 5))
