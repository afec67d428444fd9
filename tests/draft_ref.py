"""Plain numpy forms, in 64 bits, of the operators of a step over drafted tokens."""
import numpy as np

from tests import block_ref as ref


# ---- trees -----------------------------------------------------------------------

def draft_tree(parents, q_start, cached, max_new=64):
    """ancestors (python integers) and positions of the tokens of all requests; None where nothing is written."""
    anc, pos = [None] * len(parents), [None] * len(parents)
    for r, c in enumerate(cached):
        a, b = int(q_start[r]), int(q_start[r + 1])
        for i in range(min(b - max(a, 0), max_new, len(parents) - a) if a >= 0 and b >= a else 0):
            p = int(parents[a + i])
            anc[a + i] = 1 << i | (anc[a + p] if 0 <= p < i else 0)
            pos[a + i] = min(max(int(c), 0) + bin(anc[a + i]).count("1") - 1, 2 ** 31 - 1)
    return anc, pos


def tree_keys(mask, n, length, window):
    """The keys that a token with that mask sees, of a request with n new tokens among `length` keys."""
    base = length - n
    keys = list(range(max(base, 0))) + [base + j for j in range(min(n, 64)) if mask >> j & 1]
    keys = keys[-window:] if window else keys
    return [k for k in keys if 0 <= k < length]


def attend_tree(cache, q, masks, q_start, kv_lens, table, scale, window=0, max_len=None):
    """out, lse, and for the tolerances: sum p |v| and the largest sum |q k| of each row."""
    n_pages, heads, page_size = cache["k"].shape[:3]
    tokens, q_heads, d = q.shape
    g = q_heads // heads
    out, size = np.zeros((tokens, q_heads, d)), np.zeros((tokens, q_heads, d))
    lse, reach = np.full((tokens, q_heads), -np.inf), np.zeros((tokens, q_heads))
    for r in range(len(kv_lens)):
        n = int(kv_lens[r])
        most = min(n, table.shape[1] * page_size, n if max_len is None else max_len)
        for h in range(heads):
            j = np.arange(most)
            page = table[r, j // page_size]
            held = (page >= 0) & (page < n_pages)
            safe = np.where(held, page, 0)
            kk, vv = (ref.kv4_values(cache, name, safe, h, j % page_size) for name in "kv")
            for t in range(q_start[r], q_start[r + 1]):
                keys = np.array(tree_keys(int(masks[t]), int(q_start[r + 1] - q_start[r]), n, window), int)
                keys = keys[keys < most]
                keys = keys[held[keys]]
                if not len(keys):
                    continue
                for qh in range(h * g, (h + 1) * g):
                    x = np.asarray(q[t, qh], np.float64)
                    with np.errstate(invalid="ignore"):
                        s = kk[keys] @ x * scale
                        m = s.max()
                        p = np.exp(s - m)
                        out[t, qh] = p @ vv[keys] / p.sum()
                        size[t, qh] = p @ np.abs(vv[keys]) / p.sum()
                        lse[t, qh] = m + np.log(p.sum())
                        reach[t, qh] = (np.abs(kk[keys]) @ np.abs(x)).max() * abs(scale)
    return out, lse, size, reach


# ---- weights in 4 bits -----------------------------------------------------------

def round_to(x, dtype):
    """float32 values rounded to dtype ("float32", "bfloat16", "float16"), as float32."""
    x = np.asarray(x, np.float32)
    if dtype == "float32":
        return x
    if dtype == "float16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float32)
    b = x.view(np.uint32)
    r = ((b + 0x7FFF + (b >> 16 & 1)) & np.uint32(0xFFFF0000)).view(np.float32)
    return np.where(np.isnan(x), x, r)


def fp4_pack(x, group, scale_dtype):
    """[n_out, n_in] float32 -> (codes [n_out, n_in / 2] bytes, scales [n_out, n_in / group] float32): equal, not near."""
    x = np.asarray(x, np.float32)
    n, k = x.shape
    v = x.reshape(n, k // group, group)
    bad = ~np.isfinite(v).all(-1)
    with np.errstate(all="ignore"):
        scale = round_to(np.where(bad, np.float32(np.inf), np.abs(v).max(-1)) / np.float32(6), scale_dtype)
        finite = scale < np.inf
        zero = ~finite | (scale < np.float32(2.0 ** -120))
        inv = np.where(zero, np.float32(0), np.float32(1) / np.where(zero, np.float32(1), scale))
        y = np.where(zero[..., None], np.float32(0), v * inv[..., None])
    mag = np.searchsorted(np.float32([.25, .75, 1.25, 1.75, 2.5, 3.5, 5]), np.abs(y), side="right")
    code = (mag + 8 * ((y < 0) & (mag > 0))).astype(np.uint8).reshape(n, k)
    scale = np.where(finite, np.where(zero, np.float32(0), scale), np.float32(np.nan))
    return code[:, 0::2] | code[:, 1::2] << 4, scale.astype(np.float32)


def fp4_weights(codes, scales, group):
    """[n_out, n_in] float64."""
    n, half = codes.shape
    w = np.empty((n, 2 * half))
    w[:, 0::2], w[:, 1::2] = ref.LEVELS[codes & 15], ref.LEVELS[codes >> 4]
    return w * np.repeat(np.asarray(scales, np.float64), group, 1)


# ---- logits ----------------------------------------------------------------------

def logits(z, q_start=None, history=None, lens=None, since=None, tokens=None, masks=None, rep=None, freq=None, pres=None, bias=None,
           allow=None, allow_row=None, requests=None):
    """The constrained logits (float64), the sum of the terms' magnitudes, and which rows belong to a request.
    bias [vocab] or [requests, vocab]; allow [n, words] uint32."""
    z = np.array(z, np.float64)
    rows, vocab = z.shape
    size, mine = np.abs(z), np.zeros(rows, bool)
    for r in range(requests if requests is not None else (len(q_start) - 1 if q_start is not None else rows)):
        a, b = (int(q_start[r]), int(q_start[r + 1])) if q_start is not None else (r, r + 1)
        if a < 0 or b < a:
            continue
        past, counted = np.zeros(vocab, int), np.zeros(vocab, int)
        if history is not None:
            n = min(max(int(lens[r]), 0), history.shape[1])
            for i, v in enumerate(history[r, :n]):
                if 0 <= v < vocab:
                    past[v] += 1
                    counted[v] += since is None or i >= since[r]
        for t in range(a, min(b, rows)):
            mine[t] = True
            seen, times = past.copy(), counted.copy()
            if masks is not None:
                for j in range(min(b - a, 64, rows - a)):
                    v = int(tokens[a + j])
                    if int(masks[t]) >> j & 1 and 0 <= v < vocab:
                        seen[v] += 1
                        times[v] += 1
            x = z[t]
            if rep is not None:
                with np.errstate(all="ignore"):
                    x = np.where(seen > 0, np.where(x > 0, x / rep[r], x * rep[r]), x)
            size[t] = np.abs(x)
            off = (0 if freq is None else freq[r]) * times.astype(np.float64) + (0 if pres is None else pres[r]) * (times > 0)
            add = 0 if bias is None else np.asarray(bias[r] if np.ndim(bias) == 2 else bias, np.float64)
            x = x - off + add
            size[t] = size[t] + np.abs(off) + np.abs(add)
            if allow is not None:
                m = t if allow_row is None else int(allow_row[t])
                if 0 <= m < len(allow):
                    v = np.arange(vocab)
                    x = np.where(allow[m][v // 32] >> (v % 32).astype(np.uint32) & 1, x, -np.inf)
            z[t] = x
    return z, size, mine
