"""A folded transformer stack served for several requests at once.

The linear layers are SparseLinearLayers on device buffers; what lies between
them is sili__new_amd.device: block tables and slots for the step's tokens,
rotary positions, keys and values written to a cache of 4-bit codes, attention
over it, and the norms around each half of a block with its gate and residual
scale.  A step takes any mix of prompts and single tokens:

    x, h = embedding, norm of it
    per block:  q, k, v = layers(h);  rotary;  append;  attend;  o = layer
                x, h = block_norm(o, x)
                d = down(silu(gate(h)) * up(h))
                x, h = block_norm(d, x)

Run it:  python examples/folded_block.py [--blocks 4] [--steps 16]
(the weights are random: the tokens mean nothing).
"""
from __future__ import annotations

import argparse
import ctypes as C
import os
import sys
import time

import numpy as np
import torch

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import sili__new_amd as sili
from sili__new_amd import device as dev

EPS = 1e-5


def sparse_layer(n_in, n_out, density, rng):
    """A layer with about `density` of its weights, ~N(0, 1 / sqrt(inputs of an output)), one scale a row."""
    keep = rng.random((n_in, n_out)) < density
    w = np.where(keep, rng.normal(0, (density * n_in) ** -0.5, (n_in, n_out)), 0).astype(np.float32)
    rows, cols = np.nonzero(keep)
    ptrs = np.concatenate([[0], np.cumsum(keep.sum(1))]).astype(np.int32)
    top = np.abs(w).max(1)
    scale = np.where(top > 0, top / 6, 1).astype(np.float32)
    layer = sili.SparseLinearLayer(n_in, n_out, len(cols))
    layer.load_weights(ptrs, cols.astype(np.int32), (w / scale[:, None])[rows, cols])
    layer.set_value_scales(scale)
    layer.forward_dense(np.zeros((1, n_in), np.float32))  # the scales go to the device with the layer's first call
    return layer


class Stack:
    """Blocks, a cache for each, and the requests they serve."""

    def __init__(self, hidden=512, heads=8, kv_heads=2, head_dim=64, mlp=1024, blocks=4, density=0.15, vocabulary=1000,
                 pages=256, page=16, max_requests=8, max_pages=64, context=4096, seed=0):
        rng = np.random.default_rng(seed)
        self.stream = torch.cuda.Stream()
        self.lib = C.CDLL(sili.LIB_PATH)
        self.lib.sili_last_error.restype = C.c_char_p
        self.lib.sili_forward_dense.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p]
        self.hidden, self.heads, self.kv_heads, self.head_dim, self.mlp = hidden, heads, kv_heads, head_dim, mlp
        self.page, self.max_pages = page, max_pages
        widths = dict(q=(hidden, heads * head_dim), k=(hidden, kv_heads * head_dim), v=(hidden, kv_heads * head_dim),
                      o=(heads * head_dim, hidden), gate=(hidden, mlp), up=(hidden, mlp), down=(mlp, hidden))
        with torch.cuda.stream(self.stream):
            near = lambda n, at=1.0: torch.from_numpy(rng.normal(at, 0.1, n).astype(np.float32)).cuda()  # noqa: E731
            self.embedding = torch.from_numpy(rng.normal(0, 1, (vocabulary, hidden)).astype(np.float32)).cuda()
            self.out = torch.from_numpy(rng.normal(0, 1, (hidden, vocabulary)).astype(np.float32)).cuda()
            self.blocks = []
            for _ in range(blocks):
                shape = (pages, kv_heads, page)
                b = {name: sparse_layer(n_in, n_out, density, rng) for name, (n_in, n_out) in widths.items()}
                # per half of the block: the norm after it, its gate; and the norm before the next half
                b["halves"] = [dict(w_post=near(hidden), w_pre=near(hidden), gate=near(hidden, 0.5)) for _ in range(2)]
                b["cache"] = dict(k=torch.zeros(*shape, head_dim // 2, dtype=torch.uint8, device="cuda"),
                                  v=torch.zeros(pages, kv_heads, page // 16, head_dim // 2, 16, dtype=torch.uint8, device="cuda"),
                                  k_scale=torch.zeros(shape, device="cuda"), v_scale=torch.zeros(shape, device="cuda"))
                self.blocks.append(b)
            self.w_first = near(hidden)
            steps, self.rotary_scale = dev.rotary_steps(head_dim, 10000.0, dev.ROTARY_BANDS, 4.0, context)
            self.steps = torch.from_numpy(steps.view(np.int64)).cuda()
            self.table = torch.full((max_requests, max_pages), -1, dtype=torch.int32, device="cuda")
        self.free = list(range(pages))
        self.lens = []  # of the requests, in the cache

    # ---- calls on device buffers, all on the stack's stream ----

    def linear(self, layer, x):
        y = torch.empty(x.shape[0], layer.n_outputs, device="cuda")
        if self.lib.sili_forward_dense(layer.handle, x.data_ptr(), x.shape[0], y.data_ptr(), self.stream.cuda_stream):
            raise RuntimeError(self.lib.sili_last_error().decode())
        return y

    def norm(self, half, u, x):
        y, h = torch.empty_like(x), torch.empty_like(x)
        n = x.shape[1]
        dev.block_norm_forward(dev.BlockNorm(
            dtype=dev.F32, tokens=x.shape[0], width=n, u=u.data_ptr(), u_stride=n, x=x.data_ptr(), x_stride=n, y=y.data_ptr(), y_stride=n,
            h=h.data_ptr(), h_stride=n, w_post=half["w_post"].data_ptr(), w_pre=half["w_pre"].data_ptr(), gate=half["gate"].data_ptr(),
            u_scale=1.0, x_scale=1.0, eps=EPS), self.stream.cuda_stream)
        return y, h

    def plan(self, new):
        """Pages, slots and positions of a step that brings new[r] tokens to request r."""
        i32 = lambda n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
        n, total = len(new), sum(new)
        lens = self.lens + [0] * (n - len(self.lens))
        old = torch.tensor(lens, dtype=torch.int32, device="cuda")
        fresh = torch.tensor(new, dtype=torch.int32, device="cuda")
        free = torch.tensor(self.free, dtype=torch.int32, device="cuda")
        p = dict(q_start=i32(n + 1), kv_lens=i32(n), positions=i32(total), slots=i32(total), status=i32(2))
        dev.request_slots(dev.RequestSlots(
            cached_lens=old.data_ptr(), new_lens=fresh.data_ptr(), requests=n, page_size=self.page, free_pages=free.data_ptr(),
            n_free=len(self.free), block_table=self.table.data_ptr(), table_width=self.max_pages, max_tokens=total,
            **{k: t.data_ptr() for k, t in p.items()}), self.stream.cuda_stream)
        taken, flags = p["status"].tolist()
        if flags:
            raise MemoryError(f"the cache or the block table is full (request_slots status {flags})")
        self.free = self.free[taken:]
        self.lens = [a + b for a, b in zip(lens, new)]
        p.update(tokens=total, requests=n, max_new=max(new), max_len=max(self.lens))
        return p

    def attention(self, b, h, p):
        t, d, st = p["tokens"], self.head_dim, self.stream.cuda_stream
        q, k, v = (self.linear(b[name], h) for name in "qkv")
        hq, hk = self.heads, self.kv_heads
        r = dev.Rotary(dtype=dev.F32, tokens=t, head_dim=d, rot_dim=d, layout=dev.ROTARY_HALF, scale=self.rotary_scale,
                       positions=p["positions"].data_ptr(), phase_steps=self.steps.data_ptr(), q_heads=hq, k_heads=hk)
        # in place
        r.q = r.q_out = q.data_ptr()
        r.k = r.k_out = k.data_ptr()
        r.q_token_stride = r.q_out_token_stride = hq * d
        r.k_token_stride = r.k_out_token_stride = hk * d
        r.q_head_stride = r.q_out_head_stride = r.k_head_stride = r.k_out_head_stride = d
        dev.rotary(r, st)
        c = b["cache"]
        cache = dev.Kv4Cache(**{name: c[name].data_ptr() for name in c}, n_pages=len(c["k"]), kv_heads=hk, head_dim=d, page_size=self.page)
        dev.kv4_append(dev.Kv4Rows(cache=cache, dtype=dev.F32, tokens=t, slots=p["slots"].data_ptr(), k=k.data_ptr(), v=v.data_ptr(),
                                   k_token_stride=hk * d, k_head_stride=d, v_token_stride=hk * d, v_head_stride=d), st)
        out = torch.empty_like(q)
        a = dev.Kv4Attend(cache=cache, dtype=dev.F32, causal=1, requests=p["requests"], tokens=t, q_heads=hq, q_start=p["q_start"].data_ptr(),
                          kv_lens=p["kv_lens"].data_ptr(), block_table=self.table.data_ptr(), table_width=self.max_pages,
                          max_new=p["max_new"], max_len=p["max_len"], scale=d ** -0.5, q=q.data_ptr(), q_token_stride=hq * d, q_head_stride=d,
                          out=out.data_ptr(), out_token_stride=hq * d, out_head_stride=d)
        a.workspace_bytes = dev.kv4_attend_workspace(a)
        work = torch.empty(max(1, a.workspace_bytes), dtype=torch.uint8, device="cuda")
        a.workspace = work.data_ptr()
        dev.kv4_attend(a, st)
        return self.linear(b["o"], out)

    def step(self, tokens):
        """tokens: a list of new tokens for each request (new requests at the end).
        -> the last hidden state of every token [tokens, hidden]."""
        if not len(self.lens) <= len(tokens) <= len(self.table):
            raise ValueError(f"{len(tokens)} lists of tokens: one for each of {len(self.lens)} requests, and {len(self.table)} requests at most")
        if not any(tokens):
            raise ValueError("a step without tokens")
        with torch.cuda.stream(self.stream):
            p = self.plan([len(t) for t in tokens])
            x = self.embedding[torch.tensor([i for t in tokens for i in t], device="cuda")]
            h = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * self.w_first
            for b in self.blocks:
                x, h = self.norm(b["halves"][0], self.attention(b, h, p), x)
                d = self.linear(b["down"], torch.nn.functional.silu(self.linear(b["gate"], h)) * self.linear(b["up"], h))
                x, h = self.norm(b["halves"][1], d, x)
            return h

    def next_tokens(self, h, tokens):
        """The most likely token after the last one of each request; None for one without tokens in this step."""
        with torch.cuda.stream(self.stream):
            last = torch.tensor(np.cumsum([len(t) for t in tokens]) - 1, device="cuda").clamp(min=0)
            picked = (h[last] @ self.out).argmax(1).tolist()
        return [p if t else None for p, t in zip(picked, tokens)]


def generate(stack, prompts, steps):
    """The prompts in one step, then a token a request and step."""
    tokens, out = [list(p) for p in prompts], [list(p) for p in prompts]
    for _ in range(steps):
        picked = stack.next_tokens(stack.step(tokens), tokens)
        for request, t in zip(out, picked):
            request.append(t)
        tokens = [[t] for t in picked]
    return out


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--blocks", type=int, default=4)
    ap.add_argument("--steps", type=int, default=16)
    a = ap.parse_args()
    stack = Stack(blocks=a.blocks)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(1000, size=n).tolist() for n in (37, 150, 1)]
    began = time.perf_counter()
    out = generate(stack, prompts, a.steps)
    torch.cuda.synchronize()
    for p, o in zip(prompts, out):
        print(f"{len(p)} tokens, then {o[len(p):]}")
    print(f"{a.steps} steps of {len(prompts)} requests in {time.perf_counter() - began:.3f} s")


if __name__ == "__main__":
    main()
