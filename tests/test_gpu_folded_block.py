"""GPU: the operators between the layers as a served stack runs them together
(examples/folded_block.py): against a plain model in 64 bits, and a token at a
time against the whole prompt at once.

Tolerance: keys and values are quantised from float32 sums whose order differs,
so a code next to a tie may fall either way; one such code is an eighth of its
value at most, in one channel of one token.  1e-2 of a token's norm allows tens
of them; a wrong position, page, scale or mask is off by the norm itself."""
import importlib.util
import os

import numpy as np
import pytest
import torch

from sili__new_amd import device as dev
from tests import block_ref as ref

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "folded_block.py")
SIZES = dict(hidden=192, heads=6, kv_heads=2, head_dim=64, mlp=320, blocks=2, pages=64, max_pages=20, vocabulary=300)


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("folded_block", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def near(a, b):
    return np.all(np.linalg.norm(a - b, axis=-1) <= 1e-2 * np.linalg.norm(b, axis=-1))


def plain(stack, tokens):
    """One request's prompt through the stack in float64; stored keys and values are what the cache would hold."""
    np64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    dense = lambda layer: layer.forward_dense(np.eye(layer.n_inputs, dtype=np.float32)).astype(np.float64)  # noqa: E731
    x = np64(stack.embedding)[tokens]
    h = x / np.sqrt((x * x).mean(1, keepdims=True) + 1e-5) * np64(stack.w_first)
    t, d, g = len(tokens), stack.head_dim, stack.heads // stack.kv_heads
    steps, scale = dev.rotary_steps(d, 10000.0, dev.ROTARY_BANDS, 4.0, 4096)

    def stored(v):
        codes, s = ref.kv4_codes(v.astype(np.float32))
        return ref.LEVELS[codes] * s[..., None].astype(np.float64)

    def norm(half, u, x):
        f = ref.norm_forward(u, x, np64(half["gate"]), np64(half["w_post"]), np64(half["w_pre"]), 1.0, 1.0, 1e-5)
        return f["y"], f["h"]

    for b in stack.blocks:
        q, k, v = ((h @ dense(b[name])).reshape(t, -1, d) for name in "qkv")
        q = ref.rotary(q, np.arange(t), steps, d, True, False, scale)
        k, v = stored(ref.rotary(k, np.arange(t), steps, d, True, False, scale)), stored(v)
        s = np.einsum("thd,shd->hts", q, np.repeat(k, g, 1)) / np.sqrt(d)
        s = np.where(np.tril(np.ones((t, t), bool)), s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        o = np.einsum("hts,shd->thd", p / p.sum(-1, keepdims=True), np.repeat(v, g, 1)).reshape(t, -1)
        x, h = norm(b["halves"][0], o @ dense(b["o"]), x)
        a, u = h @ dense(b["gate"]), h @ dense(b["up"])
        x, h = norm(b["halves"][1], (a / (1 + np.exp(-a)) * u) @ dense(b["down"]), x)
    return h


def test_a_prompt_against_a_plain_model(hip, example):
    stack = example.Stack(**SIZES)
    tokens = np.random.default_rng(3).integers(300, size=75).tolist()
    h = stack.step([tokens])
    torch.cuda.synchronize()
    assert near(h.double().cpu().numpy(), plain(stack, tokens))


def test_token_by_token_is_the_prompt_at_once(hip, example):
    """Requests of unlike lengths, one that joins later; pages of no order."""
    rng = np.random.default_rng(4)
    prompts = [rng.integers(300, size=n).tolist() for n in (40, 9, 23)]
    step = example.Stack(**SIZES)
    step.free = rng.permutation(step.free).tolist()
    got = [[] for _ in prompts]

    def run(parts):
        h = step.step(parts)
        torch.cuda.synchronize()
        at = 0
        for r, p in enumerate(parts):
            got[r].append(h[at:at + len(p)].double().cpu().numpy())
            at += len(p)

    run([prompts[0][:17], prompts[1][:1]])
    run([prompts[0][17:18], prompts[1][1:2]])
    run([prompts[0][18:30], prompts[1][2:3], prompts[2][:20]])
    for i in range(3):
        run([prompts[0][30 + i:31 + i], prompts[1][3 + i:4 + i], prompts[2][20 + i:21 + i]])
    run([prompts[0][33:], prompts[1][6:], []])
    for r, p in enumerate(prompts):
        once = example.Stack(**SIZES)
        h = once.step([p])
        torch.cuda.synchronize()
        assert near(np.concatenate(got[r]), h.double().cpu().numpy()), r


def test_generate_and_a_full_cache(hip, example):
    stack = example.Stack(**SIZES)
    out = example.generate(stack, [[1, 2, 3], [4]], 5)
    assert [len(o) for o in out] == [8, 6] and all(0 <= t < 300 for o in out for t in o)
    assert out == example.generate(example.Stack(**SIZES), [[1, 2, 3], [4]], 5)
    with pytest.raises(MemoryError):
        stack.step([[1] * 400, [1]])
