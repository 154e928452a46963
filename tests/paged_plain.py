"""Plain 64-bit forms of the paged serving operators (numpy), and builders of
small caches, for tests/test_paged*.py."""
import numpy as np


def plan(table, cached, new, free, bs, n_tokens):
    """paged_plan request by request; returns (table, q_start, seq_lens, positions, slots, counts)."""
    table = table.copy()
    width = table.shape[1]
    q_start, lens, f, t = [0], [], 0, 0
    pos = np.full(n_tokens, -1, np.int64)
    slot = np.full(n_tokens, -1, np.int64)
    for b, (c, n) in enumerate(zip(np.maximum(cached, 0), np.maximum(new, 0))):
        c = int(c)
        n = min(int(n), n_tokens - t)
        for j in range(-(-c // bs), min(-(-(c + n) // bs), width)):
            table[b, j] = free[f] if f < len(free) else -1
            f += 1
        for i in range(n):
            p = c + i
            pos[t + i] = p
            if p // bs < width and table[b, p // bs] >= 0:
                slot[t + i] = int(table[b, p // bs]) * bs + p % bs
        t += n
        q_start.append(t)
        lens.append(c + n)
    return table, np.array(q_start), np.array(lens, np.int64), pos, slot, np.array([min(f, len(free)), max(0, f - len(free))])


def norm_rope(x, w, cos, sin, eps):
    """One head row x [hd] in float64: norm (w None: skipped), then rotation by cos / sin [rot / 2]."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * w.astype(np.float64)
    h = cos.shape[-1]
    a, b = x[..., :h].copy(), x[..., h:2 * h].copy()
    y = x.copy()
    y[..., :h] = a * cos - b * sin
    y[..., h:2 * h] = a * sin + b * cos
    return y


def attend(q, kc, vc, table, q_start, lens, scale, window):
    """Returns (out, abs_out, abs_score, keys, sum_v) in float64: the result, sum p |v|, the largest
    scale * sum |q k|, the number of attended keys and sum |v|: what error bounds are made of."""
    T, H, hd = q.shape
    nb, KV, bs, _ = kc.shape
    out, ao = np.zeros((T, H, hd)), np.zeros((T, H, hd))
    asc, keys, sv = np.zeros((T, H, 1)), np.zeros((T, H, 1)), np.zeros((T, H, hd))
    q, kc, vc = (a.astype(np.float64) for a in (q, kc, vc))
    for b in range(len(lens)):
        n = q_start[b + 1] - q_start[b]
        for i in range(n):
            t = q_start[b] + i
            p = int(lens[b]) - n + i
            lo = max(0, p - window + 1) if window else 0
            js = [j for j in range(lo, min(p + 1, table.shape[1] * bs)) if 0 <= table[b, j // bs] < nb]
            if not js:
                continue
            pages = [table[b, j // bs] for j in js]
            rows = [j % bs for j in js]
            for h in range(H):
                g = h // (H // KV)
                k, v = kc[pages, g, rows], vc[pages, g, rows]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = (k @ q[t, h]) * scale
                    e = np.exp(s - s.max())
                    w = e / e.sum()
                    out[t, h] = w @ v
                    ao[t, h] = w @ np.abs(v)
                    asc[t, h] = abs(scale) * np.max(np.abs(k) @ np.abs(q[t, h]))
                keys[t, h] = len(js)
                sv[t, h] = np.abs(v).sum(0)
    return out, ao, asc, keys, sv


def sample(x, r, T, k=None, p=None, m=None):
    """One row of sample_rows in float64."""
    x = np.asarray(x, np.float32)
    n = len(x)
    if not T > 0:
        if np.isnan(x[0]) or not (x > -np.inf).any():
            return 0
        return int(np.nanargmax(np.where(np.isnan(x), -np.inf, x)))
    if not (x < np.inf).all() or not (x > -np.inf).any():
        return n - 1
    order = np.argsort(-x.astype(np.float64), kind="stable")
    with np.errstate(over="ignore"):
        w = np.exp((x[order].astype(np.float64) - float(x.max())) / float(np.float32(T)))
    keep = np.ones(n, bool)
    if k is not None and 0 < k < n:
        keep[k:] = False
    if p is not None and p < 1:
        c = np.cumsum(w * keep)
        first = np.searchsorted(c, float(np.float32(p)) * c[-1], side="left")
        keep[max(first, 0) + 1:] = False
    if m is not None and m > 0:
        keep &= w >= float(np.float32(m))
    keep[0] = True
    kept = np.zeros(n)
    kept[order] = w * keep
    c = np.cumsum(kept)
    ok = np.flatnonzero((c >= float(np.float32(r)) * c[-1]) & (kept > 0))
    return int(ok[0]) if len(ok) else int(np.flatnonzero(kept)[-1])
