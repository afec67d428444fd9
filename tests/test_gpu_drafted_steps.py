"""GPU: the operators over drafted tokens as a served stack runs them together
(examples/folded_block.py): trees checked in one step give the tokens that the
stack gives one at a time, whatever the trees hold, and leave the cache as if it
had."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from tests import block_ref, draft_ref

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "folded_block.py")
SIZES = dict(hidden=192, heads=6, kv_heads=2, head_dim=64, mlp=320, blocks=2, pages=64, max_pages=20, vocabulary=300, head_bits=4, repetition=1.3,
             presence=0.2, frequency=0.1)


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("folded_block", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def prompts(seed):
    rng = np.random.default_rng(seed)
    return [rng.integers(300, size=n).tolist() for n in (30, 9, 17)]


def trees_of(known, rng):
    """Trees with the right continuation somewhere in them, cut at some depth, and wrong branches at every node."""
    def draft(past, token):
        right = next(k for k in known if k[:len(past) + 1] == past + [token])[len(past):][:int(rng.integers(1, 9))]
        tokens, parents, at = [token], [-1], 0
        for t in right[1:]:
            for _ in range(int(rng.integers(0, 3))):
                tokens.append(int((t + 1 + rng.integers(298)) % 300))
                parents.append(at)
                if rng.random() < 0.5:
                    tokens.append(int(rng.integers(300)))
                    parents.append(len(tokens) - 2)
            tokens.append(t)
            parents.append(at)
            at = len(tokens) - 1
        return tokens, parents
    return draft


def test_drafted_steps_give_the_tokens_of_single_steps(hip, example):
    start = prompts(4)
    plain = example.generate(example.Stack(**SIZES), start, 40, penalties=True)
    stack = example.Stack(**SIZES)
    out, calls = example.generate_drafted(stack, start, 24, trees_of(plain, np.random.default_rng(1)))
    for p, o, s in zip(plain, out, start):
        assert len(o) >= len(s) + 24 and o == p[:len(o)]
    assert calls < 24  # several tokens a step were right
    # the cache holds the tokens' own keys and values, the pages that are not needed are free again
    assert stack.lens == [len(o) for o in out]
    table = stack.table.cpu().numpy()
    held = [set(table[r, :-(-n // stack.page)].tolist()) for r, n in enumerate(stack.lens)]
    assert sum(len(h) for h in held) + len(stack.free) == 64 and set().union(*held, stack.free) == set(range(64))
    whole = example.Stack(**SIZES)
    whole.step(out)
    torch.cuda.synchronize()
    for b, c in zip(stack.blocks, whole.blocks):
        caches = [{k: t.cpu().numpy() for k, t in x["cache"].items()} for x in (b, c)]
        tables = [x.table.cpu().numpy() for x in (stack, whole)]
        for r, n in enumerate(stack.lens):
            j = np.arange(n)
            for name in "kv":
                for h in range(2):
                    got, want = (block_ref.kv4_values(x, name, t[r, j // 16], h, j % 16) for x, t in zip(caches, tables))
                    # a code next to a tie may fall either way
                    assert np.linalg.norm(got - want) <= 1e-2 * np.linalg.norm(want), (r, name, h)


def test_wrong_guesses_cost_nothing_but_the_step(hip, example):
    start = prompts(5)
    plain = example.generate(example.Stack(**SIZES), start, 12, penalties=True)
    rng = np.random.default_rng(2)
    wrong = lambda past, token: ([token] + rng.integers(300, size=20).tolist(), [-1] + [int(rng.integers(i)) for i in range(1, 21)])  # noqa: E731
    out, _ = example.generate_drafted(example.Stack(**SIZES), start, 8, wrong)
    for p, o in zip(plain, out):
        m = min(len(p), len(o))
        assert o[:m] == p[:m]


def test_lookup_drafts(hip, example):
    """The drafts of the example itself: what followed a token before."""
    assert example.lookup([5, 7, 8, 5, 9], 5) == ([5, 9, 7, 8, 5, 9], [-1, 0, 0, 2, 3, 4])
    start = [[3, 4, 5, 6] * 6, [7, 8] * 5]
    plain = example.generate(example.Stack(**SIZES), start, 14, penalties=True)
    out, _ = example.generate_drafted(example.Stack(**SIZES), start, 10)
    for p, o in zip(plain, out):
        m = min(len(p), len(o))
        assert o[:m] == p[:m]


def test_logits_of_the_packed_head(hip, example):
    stack = example.Stack(**SIZES)
    h = torch.randn(7, 192, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(stack.stream):
        z = stack.logits(h)
    torch.cuda.synchronize()
    codes, scales = draft_ref.fp4_pack(stack.out.t().contiguous().cpu().numpy(), 32, "float32")
    assert np.array_equal(stack.head[1].cpu().numpy(), codes) and np.array_equal(stack.head[2].cpu().numpy(), scales)
    w, x = draft_ref.fp4_weights(codes, scales, 32), h.double().cpu().numpy()
    assert np.all(np.abs(z.double().cpu().numpy() - x @ w.T) <= 2.0 ** -18 * (np.abs(x) @ np.abs(w).T))


def test_trees_that_are_none_are_refused(hip, example):
    stack = example.Stack(**SIZES)
    stack.step([[1, 2, 3]])
    for tree in (([1, 2], [-1, 1]), ([1, 2], [0, 0]), ([], []), ([1] * 65, [-1] + [0] * 64), ([1, 2], [-1]), ([1, 2], [-1, -1])):
        with pytest.raises(ValueError, match="tree"):
            stack.step_drafts([tree], [[1, 2, 3]])
    with pytest.raises(ValueError, match="trees"):
        stack.step_drafts([([1], [-1])] * 2, [[1, 2, 3]] * 2)
