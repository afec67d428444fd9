"""GPU: ancestors and positions of drafted tokens, exactly."""
import numpy as np
import pytest
import torch

from sili__new_amd import device as dev
from tests import draft_ref as ref

pytestmark = pytest.mark.gpu


def call(parents, start, cached, max_new=64, tokens=None, stream=None):
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()  # noqa: E731
    n = len(parents)
    s = dict(parents=i32(parents), start=i32(start), cached=i32(cached), anc=torch.full((n,), -7, dtype=torch.int64, device="cuda"),
             pos=torch.full((n,), -9, dtype=torch.int32, device="cuda"))
    s["args"] = dev.DraftTree(parents=s["parents"].data_ptr(), q_start=s["start"].data_ptr(), cached_lens=s["cached"].data_ptr(),
                              requests=len(cached), tokens=n if tokens is None else tokens, max_new=max_new,
                              ancestors=s["anc"].data_ptr(), positions=s["pos"].data_ptr())
    torch.cuda.synchronize()
    dev.draft_tree(s["args"], stream)
    torch.cuda.synchronize()
    return s


def check(s, parents, start, cached, max_new=64, tokens=None):
    n = len(parents) if tokens is None else tokens
    anc, pos = ref.draft_tree(parents[:n], start, cached, max_new)
    anc, pos = anc + [None] * (len(parents) - n), pos + [None] * (len(parents) - n)
    got = s["anc"].cpu().numpy().view(np.uint64)
    assert [int(g) for g in got] == [2 ** 64 - 7 if a is None else a for a in anc]
    assert s["pos"].cpu().tolist() == [-9 if p is None else p for p in pos]


def trees(rng, new):
    return np.concatenate([[int(rng.integers(-1, i)) if i else -1 for i in range(n)] for n in new] + [np.zeros(0, int)]).astype(int)


@pytest.mark.parametrize("new", [[1], [64], [0, 3, 64, 1, 0, 17], [5] * 9, [64, 63, 33, 32, 31, 2]])
def test_random_trees(hip, new):
    rng = np.random.default_rng(sum(new))
    parents, start = trees(rng, new), np.concatenate([[0], np.cumsum(new)])
    cached = rng.integers(0, 5000, len(new))
    check(call(parents, start, cached), parents, start, cached)


def test_a_chain_and_a_star(hip):
    parents = np.concatenate([np.arange(64) - 1, np.full(64, -1), np.minimum(np.arange(64) - 1, 0)])
    start, cached = np.array([0, 64, 128, 192]), np.array([10, 0, 2 ** 31 - 3])
    s = call(parents, start, cached)
    check(s, parents, start, cached)
    assert s["pos"][:64].tolist() == list(range(10, 74)) and not s["pos"][64:128].any() and int(s["pos"][-1]) == 2 ** 31 - 2


def test_parents_and_lengths_of_any_value(hip):
    """What is no earlier token counts as none, a negative length as 0."""
    parents = np.array([-1, 1, 1, 7, -2 ** 31, 2 ** 31 - 1, 5, 3, 0, 0, 1, 2])
    start, cached = np.array([0, 8, 12]), np.array([-5, 2 ** 31 - 1])
    check(call(parents, start, cached), parents, start, cached)


@pytest.mark.parametrize("start", [[0, 5, 40], [2, 4, 9], [-3, 5, 9], [6, 2, 9], [0, 9, 2 ** 31 - 1], [2 ** 31 - 2, 2 ** 31 - 1, 2 ** 31 - 1],
                                   [-2 ** 31, 2 ** 31 - 1, 3]])
def test_starts_of_any_value_stay_within_the_batch(hip, start):
    rng = np.random.default_rng(1)
    parents, cached = trees(rng, [9, 3]), np.array([4, 11])
    check(call(parents, np.array(start), cached, tokens=9), parents, np.array(start), cached, tokens=9)


def test_tokens_past_max_new_are_left_alone(hip):
    new = [7, 2, 5]
    rng = np.random.default_rng(2)
    parents, start, cached = trees(rng, new), np.concatenate([[0], np.cumsum(new)]), np.array([4, 11, 0])
    check(call(parents, start, cached, max_new=3), parents, start, cached, max_new=3)


def test_replayed_with_other_trees(hip):
    new = [40, 3, 0, 64]
    rng = np.random.default_rng(3)
    start, cached = np.concatenate([[0], np.cumsum(new)]), rng.integers(0, 100, 4)
    st = torch.cuda.Stream()
    s = call(trees(rng, new), start, cached, stream=st.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        dev.draft_tree(s["args"], st.cuda_stream)
    for _ in range(3):
        parents = trees(rng, new)
        s["parents"].copy_(torch.from_numpy(parents.astype(np.int32)))
        s["cached"] += 3
        cached = cached + 3
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(s, parents, start, cached)
