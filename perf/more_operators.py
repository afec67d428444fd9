"""A decoding step over drafted tokens, as measurable cases.

draft    trees of drafted tokens: who descends from whom, and at which position, from each token's parent
tree     attention for such trees over the paged cache of 4-bit codes
linear   products with 4-bit weights and a scale a group of inputs: a vocabulary's logits, wide layers
logits   penalties for repeated tokens, biases and grammar masks on logits

A request brings up to 64 drafted tokens, one after another in the batch. Token i's parent is an earlier token of the
request, or -1: the request's last token in the cache. Bit j of ancestors[i] is set where j is i or one it descends from.
Token i sees the request's cached keys and those of its ancestors, under a window the last `window` of them.

Weights hold E2M1 codes [outputs][inputs / 2], the even input in the low nibble, and a scale a group of inputs.

A repeated token's logit z becomes z / repetition or, where it is negative, z * repetition; then frequency * (times it
occurred) and presence are taken off, biases are added, and what the row's mask does not allow becomes -infinity.
Times: in the request's history from counted_from on, and among the row's ancestors; repetition takes all of the history.
"""
from __future__ import annotations

import math
import zlib

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EDGES = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)
MOST_DRAFTED = 64


# ---- cases ------------------------------------------------------------------

def listed():
    return [
        # the bookkeeping of one step: a tree for each of the folded stack's 8 requests
        dict(name="draft_8x16", kind="draft", requests=8, nodes=16, longest=8192),
        # a full serving batch of the largest trees
        dict(name="draft_1024x64", kind="draft", requests=1024, nodes=64, longest=131072),
        # the folded stack checking 16 drafted tokens a request: a key head for every query head, float32 as the layers give it
        dict(name="tree_8x2048", kind="tree", requests=8, longest=2048, nodes=16, q_heads=40, kv_heads=40, head_dim=128, page=16, window=0,
             dtype="float32"),
        # a serving batch of ragged lengths, five query heads a key head
        dict(name="tree_64x8192", kind="tree", requests=64, longest=8192, nodes=32, q_heads=40, kv_heads=8, head_dim=128, page=32, window=0,
             dtype="bfloat16"),
        # one request with a long context and a small tree: one long axis
        dict(name="tree_1x131071", kind="tree", requests=1, longest=131071, nodes=13, q_heads=40, kv_heads=8, head_dim=128, page=16, window=0,
             dtype="bfloat16"),
        # small heads under a banded mask, odd trees: a latency-bound call
        dict(name="tree_24x3000_banded", kind="tree", requests=24, longest=3000, nodes=7, q_heads=15, kv_heads=5, head_dim=64, page=64,
             window=1024, dtype="float16"),
        # one token through a wide layer of the folded stack
        dict(name="linear_1x5120x32768", kind="linear", tokens=1, n_in=5120, n_out=32768, group=32, dtype="float32", scales="float32",
             out="float32"),
        # its token batch of 8, back to the hidden width
        dict(name="linear_8x32768x5120", kind="linear", tokens=8, n_in=32768, n_out=5120, group=64, dtype="bfloat16", scales="bfloat16",
             out="bfloat16"),
        # its token batch of 128 to the logits of a large vocabulary of odd size
        dict(name="linear_128x5120x131071", kind="linear", tokens=128, n_in=5120, n_out=131071, group=128, dtype="bfloat16", scales="bfloat16",
             out="float32"),
        # a few requests over a small vocabulary: the smallest call
        dict(name="logits_8x1000", kind="logits", requests=8, nodes=1, vocab=1000, longest=512, dtype="float32", bias="one", masks=4),
        # one request, a large vocabulary, a long history
        dict(name="logits_1x131071", kind="logits", requests=1, nodes=1, vocab=131071, longest=8192, dtype="float32", bias="one", masks=1),
        # every drafted token of a serving batch, biases of each request
        dict(name="logits_64x8x131071", kind="logits", requests=64, nodes=8, vocab=131071, longest=8192, dtype="bfloat16", bias="each", masks=16),
    ]


def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    kind = rng.choice(["draft", "tree", "tree", "tree", "tree", "linear", "linear", "linear", "linear", "logits", "logits", "logits"])
    if kind == "draft":
        return dict(kind=kind, requests=_log(rng, 1, 1024), nodes=_log(rng, 1, MOST_DRAFTED), longest=_log(rng, 64, 131072))
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if kind == "tree":
        d, page = rng.choice([64, 128, 128, 256]), rng.choice([16, 16, 32, 64, 128])
        kv_heads = rng.choice([1, 2, 5, 8])
        q_heads = kv_heads * rng.choice([1, 2, 3, 5, 8, 16] if kv_heads < 5 else [1, 2, 4, 5])
        requests, nodes = _log(rng, 1, 64), _log(rng, 1, MOST_DRAFTED)
        pairs = 64 * 32 * 40 * 8192 // 2 // (requests * nodes * q_heads)
        longest = nodes + _log(rng, 1, max(16, min(65536, pairs, 500_000 // requests * 8 // kv_heads * 64 // d)))
        return dict(kind=kind, requests=requests, longest=longest, nodes=nodes, q_heads=q_heads, kv_heads=kv_heads, head_dim=d, page=page,
                    window=rng.choice([0, 0, 0, 100, 1024, 4096]), dtype=dtype)
    if kind == "linear":
        group = rng.choice([32, 64, 128])
        n_in = group * _log(rng, 1, 32768 // group)
        n_out = _log(rng, 1, min(131071, 300_000_000 // n_in))
        return dict(kind=kind, tokens=_log(rng, 1, 256) if rng.random() < 0.5 else _log(rng, 1, 16), n_in=n_in, n_out=n_out, group=group,
                    dtype=dtype, scales=rng.choice(["float32", "bfloat16", "float16"]), out=rng.choice([dtype, "float32"]))
    vocab = _log(rng, 100, 200_000)
    requests = _log(rng, 1, min(256, 30_000_000 // vocab))
    return dict(kind=kind, requests=requests, nodes=_log(rng, 1, max(1, min(MOST_DRAFTED, 30_000_000 // vocab // requests))), vocab=vocab,
                longest=_log(rng, 1, 16384), dtype=dtype, bias=rng.choice(["none", "one", "each"]), masks=rng.choice([0, 1, 5, 32]))


def _rng(case, seed=None):
    text = repr(sorted((k, v) for k, v in case.items() if k != "name"))
    return np.random.RandomState(zlib.crc32(text.encode()) if seed is None else (zlib.crc32(text.encode()) ^ (int(seed) * 2654435761 + 1)) % (1 << 32))


def _new_tokens(case, rng):
    new = rng.randint(max(1, case["nodes"] * 3 // 4), case["nodes"] + 1, case["requests"])
    new[0] = case["nodes"]
    return new


def _drafts(case, seed=None):
    """Lengths in the cache, counts of drafted tokens, and each token's parent. The counts are part of the case, as is all
    of it without a seed."""
    n, longest, rng = case["requests"], case["longest"], _rng(case, seed)
    new = _new_tokens(case, _rng(case))
    total = rng.randint(longest // 4, longest + 1, n) if longest > 3 else np.full(n, longest)
    total[0] = longest
    # a token descends from one of the few before it, now and then from the cache's last one
    i = np.concatenate([np.arange(k) for k in new])
    back = rng.randint(1, 6, len(i))
    parents = np.where(rng.rand(len(i)) < 0.06, -1, np.maximum(i - back, -1))
    return np.maximum(total - new, 0), new, parents


def _masks_of(new, parents):
    """Ancestors as 64-bit masks, on the host."""
    out, at = [], 0
    for k in new:
        here = []
        for i in range(k):
            p = int(parents[at + i])
            here.append(1 << i | (here[p] if p >= 0 else 0))
        out += here
        at += k
    return np.array(out, np.uint64)


# ---- seeded inputs -----------------------------------------------------------

def _gen(seed, stream):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + stream) % (1 << 62))
    return g


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _i64(a):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.int64)).to(DEV)


def _pack(x):
    """[..., channels] float32 -> codes [..., channels / 2] (uint8) and scales [...]."""
    top = x.abs().amax(-1, keepdim=True)
    mag = torch.bucketize((x * (6.0 / top)).abs(), torch.tensor(EDGES, device=DEV), right=True).to(torch.uint8)
    code = mag | ((x < 0) & (mag > 0)).to(torch.uint8) << 3
    return code[..., 0::2] | code[..., 1::2] << 4, (top / 6.0)[..., 0]


def _cache(case, pages, gen):
    """A cache of that many pages, filled: keys and values ~N(0, 1), a few key
    channels of each head larger, as projections have them."""
    h, p, d = case["kv_heads"], case["page"], case["head_dim"]
    k, v = (torch.empty(pages, h, p, d // 2, dtype=torch.uint8, device=DEV) for _ in "kv")
    v = v.view(pages, h, p // 16, d // 2, 16)
    ks, vs = (torch.empty(pages, h, p, device=DEV) for _ in "kv")
    wide = 1.0 + 2.0 * (torch.rand(h, 1, d, generator=gen, device=DEV) < 0.03)
    step = max(1, (1 << 27) // (h * p * d))
    for i in range(0, pages, step):
        n = min(step, pages - i)
        k[i:i + n], ks[i:i + n] = _pack(_randn(gen, n, h, p, d) * wide)
        c, vs[i:i + n] = _pack(_randn(gen, n, h, p, d))
        v[i:i + n] = c.view(n, h, p // 16, 16, d // 2).transpose(3, 4)
    return dict(k=k, v=v, k_scale=ks, v_scale=vs)


def _table(lens, page, width, pages, gen):
    """A block table whose rows hold the pages of `lens` tokens each, in no order, -1 past them."""
    need = -(-lens // page)
    perm = torch.randperm(pages, generator=gen, device=DEV).int()
    start, at = _i32(np.cumsum(need) - need).long(), torch.arange(width, device=DEV)
    inside = at[None] < _i32(need)[:, None]
    return torch.where(inside, perm[(start[:, None] + at[None]).clamp(max=pages - 1)], -1).contiguous()


def _inputs(case, seed):
    kind, gen = case["kind"], _gen(seed, 1)
    if kind == "draft":
        old, new, parents = _drafts(case, seed)
        return dict(old=_i32(old), start=_i32(np.concatenate([[0], np.cumsum(new)])), parents=_i32(parents))
    dt = TYPES[case["dtype"]]
    if kind == "tree":
        old, new, parents = _drafts(case)  # lengths and trees are the case's own: any seed has the same
        lens, p = old + new, case["page"]
        s = dict(lens=_i32(lens), start=_i32(np.concatenate([[0], np.cumsum(new)])), longest=int(lens.max()),
                 ancestors=_i64(_masks_of(new, parents)))
        pages = int((-(-lens // p)).sum()) + 3
        s["table"] = _table(lens, p, -(-s["longest"] // p), pages, gen)
        s.update(_cache(case, pages, gen))
        s["q"] = (1.5 * _randn(gen, int(new.sum()), case["q_heads"], case["head_dim"])).to(dt)
        return s
    if kind == "linear":
        n, k, g = case["n_out"], case["n_in"], case["group"]
        codes = torch.empty(n, k // 2, dtype=torch.uint8, device=DEV)
        scales = torch.empty(n, k // g, dtype=TYPES[case["scales"]], device=DEV)
        step = max(1, (1 << 27) // k)
        for i in range(0, n, step):
            m = min(step, n - i)
            c, sc = _pack((_randn(gen, m, k) * k ** -0.5).view(m, k // g, g))
            codes[i:i + m], scales[i:i + m] = c.view(m, k // 2), sc.to(scales.dtype)
        return dict(codes=codes, scales=scales, x=_randn(gen, case["tokens"], k).to(dt))
    v, r, rng = case["vocab"], case["requests"], _rng(case, seed)
    shape = _rng(case)
    new = _new_tokens(case, shape)
    lens = shape.randint(case["longest"] // 2, case["longest"] + 1, r)
    lens[0] = case["longest"]
    rows = int(new.sum())
    # a few tokens are frequent, as in text
    words = lambda *n: np.minimum(v * rng.rand(*n) ** 6, v - 1).astype(np.int64)  # noqa: E731
    i = np.concatenate([np.arange(k) for k in new])
    parents = np.where(i == 0, -1, np.maximum(i - rng.randint(1, 6, rows), 0))
    s = dict(logits=(3.0 * _randn(gen, rows, v)).to(dt), start=_i32(np.concatenate([[0], np.cumsum(new)])), history=_i32(words(r, case["longest"])),
             lens=_i32(lens), counted_from=_i32((lens * rng.rand(r)).astype(np.int64)), tokens=_i32(words(rows)),
             ancestors=_i64(_masks_of(new, parents)), repetition=1.0 + torch.rand(r, generator=gen, device=DEV),
             presence=torch.rand(r, generator=gen, device=DEV), frequency=0.5 * torch.rand(r, generator=gen, device=DEV))
    s["bias"] = None if case["bias"] == "none" else _randn(gen, *([v] if case["bias"] == "one" else [r, v]))
    s["allow"] = s["allow_row"] = None
    if case["masks"]:
        # grammars that allow almost all, half, or a few of the tokens; some rows are free
        words32 = -(-v // 32)
        share = torch.tensor([0.95, 0.5, 0.01, 0.5, 0.1], device=DEV).repeat(7)[:case["masks"], None, None]
        bits = torch.rand(case["masks"], words32, 32, generator=gen, device=DEV) < share
        s["allow"] = (bits.long() << torch.arange(32, device=DEV)).sum(-1).to(torch.int32)
        s["allow_row"] = _i32(rng.randint(-1 if case["masks"] > 1 else 0, case["masks"], rows))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        s["call"] = _bind(s)
    torch.cuda.synchronize()
    return s


# ---- the framework's operators ---------------------------------------------------

def _bind(s):
    """The call of a case with its arguments, on buffers that live as long as the
    state: (function, arguments, outputs)."""
    from sili__new_amd import device as dev

    case, kind = s["case"], s["case"]["kind"]
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    empty = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device=DEV)  # noqa: E731
    if kind == "draft":
        n = len(s["parents"])
        out = dict(ancestors=empty(n, dtype=torch.int64), positions=empty(n, dtype=torch.int32))
        a = dev.DraftTree(parents=ptr(s["parents"]), q_start=ptr(s["start"]), cached_lens=ptr(s["old"]), requests=case["requests"], tokens=n,
                          max_new=case["nodes"], ancestors=ptr(out["ancestors"]), positions=ptr(out["positions"]))
        return dev.draft_tree, [a], out
    dt = dev.DTYPES[case["dtype"]]
    if kind == "tree":
        h, d = case["q_heads"], case["head_dim"]
        out = dict(out=torch.empty_like(s["q"]), lse=empty(s["q"].shape[0], h))
        cache = dev.Kv4Cache(k=ptr(s["k"]), v=ptr(s["v"]), k_scale=ptr(s["k_scale"]), v_scale=ptr(s["v_scale"]), n_pages=len(s["k"]),
                             kv_heads=case["kv_heads"], head_dim=d, page_size=case["page"])
        a = dev.Kv4Attend(cache=cache, dtype=dt, requests=case["requests"], tokens=s["q"].shape[0], q_heads=h, q_start=ptr(s["start"]),
                          kv_lens=ptr(s["lens"]), block_table=ptr(s["table"]), table_width=s["table"].shape[1], max_new=case["nodes"],
                          max_len=s["longest"], scale=d ** -0.5, causal=1, window=case["window"], lse=ptr(out["lse"]), q=ptr(s["q"]),
                          q_token_stride=h * d, q_head_stride=d, out=ptr(out["out"]), out_token_stride=h * d, out_head_stride=d)
        a.workspace_bytes = dev.kv4_attend_tree_workspace(a)
        s["work"] = empty(max(1, a.workspace_bytes), dtype=torch.uint8)
        a.workspace = ptr(s["work"])
        return dev.kv4_attend_tree, [a, ptr(s["ancestors"])], out
    if kind == "linear":
        t, k, n = case["tokens"], case["n_in"], case["n_out"]
        out = dict(y=empty(t, n, dtype=TYPES[case["out"]]))
        w = dev.Fp4Weights(codes=ptr(s["codes"]), scales=ptr(s["scales"]), scale_dtype=dev.DTYPES[case["scales"]], n_out=n, n_in=k,
                           group=case["group"], codes_stride=k // 2, scales_stride=k // case["group"])
        a = dev.Fp4Linear(w=w, dtype=dt, out_dtype=dev.DTYPES[case["out"]], tokens=t, x=ptr(s["x"]), x_stride=k, y=ptr(out["y"]), y_stride=n)
        a.workspace_bytes = dev.fp4_linear_workspace(a)
        s["work"] = empty(max(1, a.workspace_bytes), dtype=torch.uint8)
        a.workspace = ptr(s["work"])
        return dev.fp4_linear, [a], out
    rows, v = s["logits"].shape
    out = dict(logits=torch.empty_like(s["logits"]))
    a = dev.LogitsConstrain(dtype=dt, rows=rows, vocab=v, requests=case["requests"], logits=ptr(s["logits"]), logits_stride=v,
                            out=ptr(out["logits"]), out_stride=v, q_start=ptr(s["start"]), history=ptr(s["history"]),
                            history_lens=ptr(s["lens"]), history_stride=case["longest"], counted_from=ptr(s["counted_from"]),
                            tokens=ptr(s["tokens"]), ancestors=ptr(s["ancestors"]), repetition=ptr(s["repetition"]),
                            presence=ptr(s["presence"]), frequency=ptr(s["frequency"]), bias=ptr(s["bias"]),
                            bias_stride=v if case["bias"] == "each" else 0, allow=ptr(s["allow"]), allow_row=ptr(s["allow_row"]),
                            allow_stride=-(-v // 32), n_allow=case["masks"])
    return dev.logits_constrain, [a], out


# ---- the plain forms ---------------------------------------------------------------

def _requests_of(start, rows):
    """The request of each row, and the row's place in it."""
    t = torch.arange(rows, device=DEV)
    r = torch.searchsorted(start[1:].long(), t, right=True)
    return r, t - start.long()[r]


def _draft(s):
    parents, start = s["parents"].long(), s["start"].long()
    r, i = _requests_of(s["start"], len(parents))
    first = start[r]
    mask = torch.ones_like(i) << i
    up = torch.where(parents >= 0, first + parents, -1)
    # each round takes the masks of twice as many generations
    for _ in range(6):
        at = up.clamp(min=0)
        mask = torch.where(up >= 0, mask | mask[at], mask)
        up = torch.where(up >= 0, up[at], -1)
    depth = ((mask[:, None] >> torch.arange(MOST_DRAFTED, device=DEV)) & 1).sum(1)
    return dict(ancestors=mask, positions=(s["old"].long()[r] + depth - 1).int())


def _values(codes, scale):
    """codes [..., channels / 2] and scales [...] -> float32 [..., channels]."""
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=DEV)
    both = torch.stack([level.repeat(16), level.repeat_interleave(16)], 1)
    return both[codes.int()].flatten(-2) * scale.float()[..., None]


def _tree(s):
    case = s["case"]
    r, h, d, p = case["requests"], case["kv_heads"], case["head_dim"], case["page"]
    g, new, n = case["q_heads"] // h, case["nodes"], s["table"].shape[1] * p
    pages = s["table"].clamp(min=0).long()
    keys = _values(s["k"][pages], s["k_scale"][pages]).transpose(1, 2).reshape(r, h, n, d)
    lens, start = s["lens"].long(), s["start"].long()
    count = start[1:] - start[:-1]
    i = torch.arange(new, device=DEV)
    real = i[None] < count[:, None]
    token = (start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[token].view(r, new, h, g, d).permute(0, 2, 3, 1, 4).reshape(r, h, g * new, d)
    scores = torch.matmul(q * d ** -0.5, keys.transpose(2, 3).contiguous()).view(r, h, g, new, n)
    del keys
    # the cached keys, and of the drafted ones those of the row's ancestors
    old, j = (lens - count)[:, None], torch.arange(n, device=DEV)
    mask = s["ancestors"][token]
    at = j[None] - old
    bit = (mask[:, :, None] >> at.clamp(0, MOST_DRAFTED - 1)[:, None]) & 1
    drafted = ((at >= 0) & (at < MOST_DRAFTED) & (j[None] < lens[:, None]))[:, None]
    seen = (at < 0)[:, None] | drafted & (bit > 0)
    if case["window"]:
        # the last `window` of those: the keys from a row's last one back, counted
        seen &= seen.flip(-1).long().cumsum(-1).flip(-1) <= case["window"]
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    scores = scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    values = s["v"][pages].transpose(-1, -2).reshape(r, -1, h, p, d // 2)
    values = _values(values, s["v_scale"][pages]).transpose(1, 2).reshape(r, h, n, d)
    out = torch.matmul(scores.view(r, h, g * new, n), values).view(r, h, g, new, d)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 3, 1, 2, 4).reshape(r, new, h * g, d)
    lse = (top + torch.log(total))[..., 0].permute(0, 3, 1, 2).reshape(r, new, h * g)
    where = torch.where(real, token, s["q"].shape[0])
    full = torch.empty(s["q"].shape[0] + 1, h * g, d, dtype=s["q"].dtype, device=DEV)
    full_lse = torch.empty(s["q"].shape[0] + 1, h * g, device=DEV)
    full[where], full_lse[where] = out.to(s["q"].dtype), lse
    return dict(out=full[:-1], lse=full_lse[:-1])


def _linear(s):
    case = s["case"]
    n, k, g = case["n_out"], case["n_in"], case["group"]
    w = _values(s["codes"].view(n, k // g, g // 2), s["scales"]).view(n, k)
    return dict(y=torch.matmul(s["x"].float(), w.t()).to(TYPES[case["out"]]))


def _logits(s):
    case, v = s["case"], s["case"]["vocab"]
    r, i = _requests_of(s["start"], s["logits"].shape[0])
    at = torch.arange(case["longest"], device=DEV)[None]
    inside = at < s["lens"][:, None]
    recent = inside & (at >= s["counted_from"][:, None])
    ids, zero = s["history"].long(), torch.zeros(case["requests"], v, device=DEV)
    ever = zero.scatter_add(1, ids, inside.float())[r]
    times = zero.scatter_add(1, ids, recent.float())[r]
    bits = (s["ancestors"][:, None] >> torch.arange(MOST_DRAFTED, device=DEV)) & 1
    peers = s["start"].long()[r][:, None] + torch.arange(MOST_DRAFTED, device=DEV)
    drafted = s["tokens"].long()[peers.clamp(max=len(s["tokens"]) - 1)]
    times.scatter_add_(1, drafted, bits.float())
    z = s["logits"].float()
    rep = s["repetition"][r][:, None]
    z = torch.where(ever + times > 0, torch.where(z > 0, z / rep, z * rep), z)
    z = z - s["frequency"][r][:, None] * times - s["presence"][r][:, None] * (times > 0)
    if s["bias"] is not None:
        z = z + (s["bias"] if s["bias"].dim() == 1 else s["bias"][r])
    if s["allow"] is not None:
        words = s["allow"][s["allow_row"].long().clamp(min=0)]
        bit = (words[:, :, None] >> torch.arange(32, device=DEV)) & 1
        free = (s["allow_row"] < 0)[:, None]
        z = z.masked_fill(~(free | (bit.flatten(1)[:, :v] > 0)), -math.inf)
    return dict(logits=z.to(s["logits"].dtype))


PLAIN = {"draft": _draft, "tree": _tree, "linear": _linear, "logits": _logits}


def run(s):
    if own:
        call, args, out = s["call"]
        call(*args)
        return out
    return PLAIN[s["case"]["kind"]](s)


# ---- what a pass cannot do without -------------------------------------------------

def work(case):
    kind, r = case["kind"], case["requests"] if "requests" in case else 0
    if kind == "draft":
        old, new, _ = _drafts(case)
        t = int(new.sum())
        return dict(bytes=4.0 * t + 8.0 * (r + 1) + 12.0 * t, flops=0.0)
    b = BYTES[case["dtype"]]
    if kind == "tree":
        d, h, hq = case["head_dim"], case["kv_heads"], case["q_heads"]
        old, new, parents = _drafts(case)
        depth = [bin(int(m)).count("1") for m in _masks_of(new, parents)]
        w = case["window"] or 1 << 40
        context = np.repeat(old, new)
        pairs = sum(min(w, int(c) + k) for c, k in zip(context, depth))
        # no row reaches further back than the shallowest of its request
        keys, at = 0, 0
        for c, k in zip(old.tolist(), new.tolist()):
            keys += min(c, max(0, w - min(depth[at:at + k]))) + k
            at += k
        t = int(new.sum())
        return dict(bytes=keys * h * (d + 8.0) + 2.0 * b * t * hq * d + 4.0 * t * hq + 4.0 * keys / case["page"] + 8.0 * t, flops=4.0 * d * hq * pairs)
    if kind == "linear":
        t, k, n = case["tokens"], case["n_in"], case["n_out"]
        return dict(bytes=n * (k / 2.0 + k // case["group"] * BYTES[case["scales"]]) + float(t) * (k * b + n * BYTES[case["out"]]),
                    flops=2.0 * t * k * n)
    shape = _rng(case)
    new = _new_tokens(case, shape)
    lens = shape.randint(case["longest"] // 2, case["longest"] + 1, r)
    lens[0] = case["longest"]
    v, rows = case["vocab"], int(new.sum())
    bias = {"none": 0, "one": 4.0 * v, "each": 4.0 * v * r}[case["bias"]]
    return dict(bytes=2.0 * b * rows * v + bias + case["masks"] * v / 8.0 + 4.0 * int(lens.sum()) + 16.0 * rows + 20.0 * r, flops=6.0 * rows * v)


# ---- 64 bits -----------------------------------------------------------------------

def _exact_levels(codes):
    """E2M1 from its fields: sign, two exponent bits (bias 1), a mantissa bit."""
    c = codes.to(torch.int64)
    e, m = (c >> 1) & 3, (c & 1).double()
    mag = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2((e - 1).double()))
    return torch.where(c >= 8, -mag, mag)


def _exact_rows(codes, scale):
    """[..., D/2] bytes -> [..., D] float64."""
    out = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=DEV)
    out[..., 0::2], out[..., 1::2] = _exact_levels(codes & 15), _exact_levels(codes >> 4)
    return out * scale.double()[..., None]


def _exact_tree(case, s):
    h, d, p, w = case["kv_heads"], case["head_dim"], case["page"], case["window"]
    g = case["q_heads"] // h
    start, lens, table = s["start"].tolist(), s["lens"].tolist(), s["table"]
    masks = s["ancestors"].cpu().numpy().view(np.uint64)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device=DEV)
    for r in range(case["requests"]):
        a, b, n = start[r], start[r + 1], lens[r]
        hidden = np.zeros((b - a, n), bool)
        for t in range(a, b):
            mine = list(range(n - (b - a))) + [n - (b - a) + j for j in range(b - a) if int(masks[t]) >> j & 1]
            keep = np.zeros(n, bool)
            keep[mine[-w:] if w else mine] = True
            hidden[t - a] = ~keep
        hidden = torch.from_numpy(hidden).to(DEV)
        at = torch.arange(n, device=DEV)
        page, slot = table[r, at // p].long(), at % p
        for kh in range(h):
            keys = _exact_rows(s["k"][page, kh, slot], s["k_scale"][page, kh, slot])
            vals = _exact_rows(s["v"][page, kh, slot // 16, :, slot % 16], s["v_scale"][page, kh, slot])
            q = s["q"][a:b, kh * g:(kh + 1) * g].double()
            x = (q.reshape(-1, d) @ keys.T).view(b - a, g, n) / math.sqrt(d)
            x = x.masked_fill(hidden[:, None], -math.inf)
            z = torch.logsumexp(x, -1)
            weight = torch.exp(x - z[..., None])
            out[a:b, kh * g:(kh + 1) * g] = (weight.view(-1, n) @ vals).view(b - a, g, d)
            lse[a:b, kh * g:(kh + 1) * g] = z
    return dict(out=out, lse=lse)


def _exact_linear(case, s):
    n, k, g = case["n_out"], case["n_in"], case["group"]
    y = torch.empty(case["tokens"], n, dtype=torch.float64, device=DEV)
    x, step = s["x"].double(), max(1, (1 << 27) // k)
    for i in range(0, n, step):
        m = min(step, n - i)
        w = _exact_rows(s["codes"][i:i + m].view(m, k // g, g // 2), s["scales"][i:i + m]).view(m, k)
        y[:, i:i + m] = x @ w.T
    return dict(y=y)


def _exact_logits(case, s):
    v, start = case["vocab"], s["start"].tolist()
    z = s["logits"].double()
    masks = s["ancestors"].cpu().numpy().view(np.uint64)
    lens, since, picks = s["lens"].tolist(), s["counted_from"].tolist(), s["tokens"].tolist()
    for r in range(case["requests"]):
        before = torch.bincount(s["history"][r, :since[r]], minlength=v)
        after = torch.bincount(s["history"][r, since[r]:lens[r]], minlength=v)
        for t in range(start[r], start[r + 1]):
            path = [picks[start[r] + j] for j in range(start[r + 1] - start[r]) if int(masks[t]) >> j & 1]
            times = after + torch.bincount(torch.tensor(path, device=DEV), minlength=v)
            row, rep = z[t], s["repetition"][r].double()
            hit = (before + times) > 0
            row[hit] = torch.where(row[hit] < 0, row[hit] * rep, row[hit] / rep)
            row -= times * s["frequency"][r].double()
            row[times > 0] -= s["presence"][r].double()
            if s["bias"] is not None:
                row += s["bias"].double() if case["bias"] == "one" else s["bias"][r].double()
    if s["allow"] is not None:
        words = s["allow"].cpu().numpy().view(np.uint32)
        for t, m in enumerate(s["allow_row"].tolist()):
            if m >= 0:
                bits = np.unpackbits(words[m].view(np.uint8), bitorder="little")[:v]
                z[t, torch.from_numpy(bits == 0).to(DEV)] = -math.inf
    return dict(logits=z)


def exact(case, seed):
    if case["kind"] == "draft":
        return None  # whole numbers
    return {"tree": _exact_tree, "linear": _exact_linear, "logits": _exact_logits}[case["kind"]](case, _inputs(case, seed))
