"""GPU: steps of the folded stack (examples/folded_block.py) that it cannot take
are refused with nothing changed, and requests that rest in a step stay out of
its answers."""
import numpy as np
import pytest
import torch

from tests.test_gpu_folded_block import SIZES, example, near  # noqa: F401

pytestmark = pytest.mark.gpu


def test_refused_steps(hip, example):  # noqa: F811
    stack = example.Stack(**dict(SIZES, max_requests=3))
    stack.step([[1, 2], [3]])
    kept = list(stack.lens), list(stack.free), stack.table.clone()
    # more requests than the block table has rows, fewer than are served, none with tokens
    for tokens in ([[1]] * 4, [[1]], [], [[], []], [[], [], []]):
        with pytest.raises(ValueError):
            stack.step(tokens)
        assert (stack.lens, stack.free) == kept[:2] and torch.equal(stack.table, kept[2])
    # a step that does not fit leaves the requests as they were
    with pytest.raises(MemoryError):
        stack.step([[1] * 2000, [1], [1]])
    assert (stack.lens, stack.free) == kept[:2]
    h = stack.step([[4], [5], [6]])
    other = example.Stack(**dict(SIZES, max_requests=3))
    other.step([[1, 2], [3]])
    want = other.step([[4], [5], [6]])
    torch.cuda.synchronize()
    assert near(h.double().cpu().numpy(), want.double().cpu().numpy()) and stack.lens == [3, 2, 1]


def test_requests_that_rest(hip, example):  # noqa: F811
    stack = example.Stack(**SIZES)
    tokens = [[7, 8], [], [9], []]
    h = stack.step(tokens)
    picked = stack.next_tokens(h, tokens)
    assert [p is None for p in picked] == [False, True, False, True]
    with torch.cuda.stream(stack.stream):
        best = (h[torch.tensor([1, 1, 2, 2], device="cuda")] @ stack.out).argmax(1).tolist()
    assert [picked[0], picked[2]] == [best[0], best[2]]
    first = [[], [7, 8]]
    other = example.Stack(**SIZES)
    assert np.array_equal([p is None for p in other.next_tokens(other.step(first), first)], [True, False])
