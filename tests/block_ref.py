"""Plain numpy forms, in 64 bits, of the operators between the layers, and what
their tests share."""
import numpy as np

# half the distance of 1 to the next value: 23, 7 and 10 fraction bits
HALF_ULP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 0.0, "bfloat16": 0.0, "float16": 2.0 ** -25}
LEVELS = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6])


def rounding(dtype, value):
    """Half a unit in the last place of `value` in `dtype`."""
    return HALF_ULP[dtype] * np.abs(value) + TINY[dtype]


# ---- request slots ---------------------------------------------------------------

def request_slots(old, new, page, free, table, max_tokens):
    table = np.array(table)
    q_start, kv, pos, slots, taken, flags = [0], [], [], [], 0, 0
    for r, (c, n) in enumerate(zip(old, new)):
        flags |= 8 if c < 0 or n < 0 else 0
        c, n = max(int(c), 0), max(int(n), 0)
        have, total = -(-c // page), -(-(c + n) // page)
        flags |= 2 if n and total > table.shape[1] else 0
        for at in range(have, total):
            p = -1
            if taken < len(free):
                p = int(free[taken])
                flags |= 16 if p < 0 else 0
            else:
                flags |= 1
            taken += 1
            if at < table.shape[1]:
                table[r, at] = p
        for i in range(n):
            at = (c + i) // page
            p = int(table[r, at]) if at < table.shape[1] else -1
            if at < have and p < 0 and at < table.shape[1]:
                flags |= 16
            pos.append(c + i)
            slots.append(p * page + (c + i) % page if p >= 0 else -1)
        kv.append(c + n)
        q_start.append(q_start[-1] + n)
    flags |= 4 if len(pos) > max_tokens else 0
    pad = max(0, max_tokens - len(pos))
    return dict(block_table=table, q_start=np.array(q_start), kv_lens=np.array(kv, int), status=np.array([min(taken, len(free)), flags]),
                positions=np.array(pos + [0] * pad, int)[:max_tokens], slots=np.array(slots + [-1] * pad, int)[:max_tokens])


# ---- rotary ------------------------------------------------------------------------

def rotary(x, pos, steps, rot, half, inverse, scale):
    """x [tokens, heads, head_dim]; steps: uint64 fractions of a turn."""
    x = np.array(x, np.float64)
    turns = (np.asarray(pos).astype(np.int64).view(np.uint64)[:, None] * np.asarray(steps)[None]).astype(np.uint64)
    angle = turns.astype(np.float64) / 2.0 ** 64 * 2 * np.pi * (-1 if inverse else 1)
    c, s = np.cos(angle)[:, None] * scale, np.sin(angle)[:, None] * scale
    a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if half else (slice(0, rot, 2), slice(1, rot, 2))
    x1, x2 = x[..., a].copy(), x[..., b].copy()
    x[..., a], x[..., b] = x1 * c - x2 * s, x2 * c + x1 * s
    return x


# ---- block norm --------------------------------------------------------------------

def norm_forward(u, x, gate, w_post, w_pre, u_scale, x_scale, eps):
    r1 = 1 / np.sqrt((u * u).mean(-1, keepdims=True) + eps)
    n = u * r1 * w_post if w_post is not None else u
    n = n * gate if gate is not None else n
    y = u_scale * n + (x_scale * x if x is not None else 0)
    r2 = 1 / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
    return dict(y=y, h=y * r2 * w_pre if w_pre is not None else None, r1=r1[:, 0], r2=r2[:, 0], part=u_scale * n)


def norm_backward(u, y, gate, w_post, w_pre, u_scale, x_scale, r1, r2, dy, dh):
    """The gradients, and `size`: for each the sum of its terms' magnitudes."""
    zero = np.zeros_like(u)
    dy = zero if dy is None else dy
    gy, size, out = dy, np.abs(dy), {}
    if dh is not None:
        yh, wd = y * r2[:, None], dh * w_pre
        gy = dy + r2[:, None] * (wd - yh * (wd * yh).mean(-1, keepdims=True))
        size = size + r2[:, None] * (np.abs(wd) + np.abs(yh) * np.abs(wd * yh).mean(-1, keepdims=True))
        out["dw_pre"] = ((dh * yh).sum(0), np.abs(dh * yh).sum(0))
    out["dx"] = (x_scale * gy, abs(x_scale) * size)
    uh = u * r1[:, None] if w_post is not None else u
    w = w_post if w_post is not None else 1.0
    g = gate if gate is not None else 1.0
    dn, dn_size = u_scale * gy * g, abs(u_scale) * size * np.abs(g)
    if gate is not None:
        dg, dg_size = u_scale * gy * uh * w, abs(u_scale) * size * np.abs(uh * w)
        out["dgate"] = (dg.sum(0), dg_size.sum(0)) if gate.ndim == 1 else (dg, dg_size)
    if w_post is None:
        out["du"] = (dn, dn_size)
        return out
    out["dw_post"] = ((dn * uh).sum(0), (dn_size * np.abs(uh)).sum(0))
    wd, wd_size = w * dn, np.abs(w) * dn_size
    out["du"] = (r1[:, None] * (wd - uh * (wd * uh).mean(-1, keepdims=True)),
                 r1[:, None] * (wd_size + np.abs(uh) * (wd_size * np.abs(uh)).mean(-1, keepdims=True)))
    return out


# ---- the 4-bit cache ---------------------------------------------------------------

def kv4_codes(x):
    """[..., D] float32 -> (codes [..., D], scale [...]), the arithmetic of the
    format in float32: the codes are equal, not near."""
    x = np.asarray(x, np.float32)
    top = np.abs(x).max(-1, keepdims=True)
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    zero = bad | (top < np.float32(2.0 ** -120))
    with np.errstate(all="ignore"):
        y = np.where(zero, np.float32(0), x * np.where(zero, np.float32(0), np.float32(6) * (np.float32(1) / top)))
    mag = np.searchsorted(np.float32([.25, .75, 1.25, 1.75, 2.5, 3.5, 5]), np.abs(y), side="right")
    scale = np.where(bad, np.float32(np.nan), np.where(zero, np.float32(0), top / np.float32(6)))
    return (mag + 8 * ((y < 0) & (mag > 0))).astype(np.uint8), scale[..., 0].astype(np.float32)


def kv4_store(cache, slots, k, v):
    """Rows k, v [tokens, heads, D] into the four arrays of a cache."""
    page_size = cache["k"].shape[2]
    for name, rows in (("k", k), ("v", v)):
        codes, scale = kv4_codes(rows)
        packed = codes[..., 0::2] | codes[..., 1::2] << 4
        for t, slot in enumerate(slots):
            if 0 <= slot < len(cache["k"]) * page_size:
                p, at = divmod(int(slot), page_size)
                if name == "k":
                    cache["k"][p, :, at] = packed[t]
                else:
                    cache["v"][p, :, at // 16, :, at % 16] = packed[t]
                cache[name + "_scale"][p, :, at] = scale[t]


def kv4_values(cache, name, page, head, at):
    """The values [n, D] of slots (page, at) of one head."""
    b = cache["k"][page, head, at] if name == "k" else cache["v"][page, head, at // 16, :, at % 16]
    out = np.empty((len(at), 2 * b.shape[-1]))
    out[:, 0::2], out[:, 1::2] = LEVELS[b & 15], LEVELS[b >> 4]
    return out * cache[name + "_scale"][page, head, at][:, None].astype(np.float64)


def attend(cache, q, q_start, kv_lens, table, scale, causal, window, max_len=None):
    """out, lse, and for the tolerances: sum p |v| and the largest sum |q k|
    among the keys of each row.  q [tokens, q_heads, D]."""
    n_pages, heads, page_size = cache["k"].shape[:3]
    tokens, q_heads, d = q.shape
    g = q_heads // heads
    out, size = np.zeros((tokens, q_heads, d)), np.zeros((tokens, q_heads, d))
    lse, reach = np.full((tokens, q_heads), -np.inf), np.zeros((tokens, q_heads))
    for r in range(len(kv_lens)):
        n = int(kv_lens[r])
        j = np.arange(min(n, table.shape[1] * page_size, n if max_len is None else max_len))
        page = table[r, j // page_size]
        j, page = j[(page >= 0) & (page < n_pages)], page[(page >= 0) & (page < n_pages)]
        for h in range(heads):
            kk, vv = (kv4_values(cache, name, page, h, j % page_size) for name in "kv")
            for t in range(q_start[r], q_start[r + 1]):
                pos = n - (q_start[r + 1] - t)
                seen = np.ones(len(j), bool)
                if causal:
                    seen = j <= pos
                    if window:
                        seen &= j > pos - window
                if not seen.any():
                    continue
                for qh in range(h * g, (h + 1) * g):
                    x = np.asarray(q[t, qh], np.float64)
                    with np.errstate(invalid="ignore"):
                        s = kk[seen] @ x * scale
                        m = s.max()
                        p = np.exp(s - m)
                        out[t, qh] = p @ vv[seen] / p.sum()
                        size[t, qh] = p @ np.abs(vv[seen]) / p.sum()
                        lse[t, qh] = m + np.log(p.sum())
                        reach[t, qh] = (np.abs(kk[seen]) @ np.abs(x)).max() * abs(scale)
    return out, lse, size, reach
