"""GPU: steps of the folded stack (examples/folded_block.py) that it cannot take
are refused with nothing changed."""
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
