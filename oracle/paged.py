"""Paged-cache and logit-adjustment oracle (TEST INFRASTRUCTURE ONLY; see oracle/__init__.py).

No reference counterpart (its caches are contiguous and it rejects penalties); the definitions of `aib_paged_append`,
`aib_paged_attn` and `aib_adjust_logits` in numpy float64. Inputs are float64 arrays of exactly representable values.
"""
import numpy as np


def rows_of(table_row, page, p):
    """(page id, row in page) of positions p."""
    p = np.asarray(p)
    return np.asarray(table_row)[p // page], p % page


def norm_rope(x, w, inv, p, eps):
    """RMSNorm (w None: none) and half-split rotation by p * inv (None: none) of head vectors x [..., HD]."""
    x = np.asarray(x, np.float64)
    if w is not None:
        x = np.asarray(w, np.float64) * x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if inv is None:
        return x
    a = float(p) * np.asarray(inv, np.float64)
    c, s, h = np.cos(a), np.sin(a), x.shape[-1] // 2
    return np.concatenate([x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s], -1)


def append(kc, vc, table, pos, cu, q, k, v, qn, kn, inv, eps):
    """kc, vc float64 [pages, KV, page, HD], updated in place (unrounded); returns q_out (NaN where not written) and
    the list of (page id, row) written."""
    page, pages, width = kc.shape[2], kc.shape[0], np.shape(table)[1]
    out = None if q is None else np.full(q.shape, np.nan)
    at = []
    for b in range(len(pos)):
        if pos[b] < 0:
            continue
        for t in range(cu[b], cu[b + 1]):
            p = int(pos[b]) + t - cu[b]
            if q is not None:
                out[t] = norm_rope(q[t], qn, inv, p, eps)
            if p // page >= width or not 0 <= table[b][p // page] < pages:
                continue
            i, r = int(table[b][p // page]), p % page
            kc[i, :, r] = norm_rope(k[t], kn, inv, p, eps)
            vc[i, :, r] = v[t]
            at.append((i, r))
    return out, at


def attention(q, kc, vc, table, pos, window, scale):
    """out [B, H, HD], lse [B, H] and, for error bounds, the weighted |v| sum of every output and the largest
    sum |q||k| of every head."""
    B, H, HD = q.shape
    pages, KV, page, _ = kc.shape
    G, width = H // KV, np.shape(table)[1]
    out, mag = np.zeros((B, H, HD)), np.zeros((B, H, HD))
    lse, dot = np.full((B, H), -np.inf), np.zeros((B, H))
    for b in range(B):
        hi = min(int(pos[b]) + 1, width * page)
        j = np.arange(max(0, int(pos[b]) + 1 - window) if window else 0, max(hi, 0))
        i, r = rows_of(table[b], page, j)
        ok = (i >= 0) & (i < pages)
        i, r = i[ok], r[ok]
        if not len(i):
            continue
        for h in range(H):
            K, V = kc[i, h // G, r], vc[i, h // G, r]
            s = (K @ q[b, h]) * scale
            m = s.max()
            e = np.exp(s - m)
            out[b, h], mag[b, h] = e @ V / e.sum(), e @ np.abs(V) / e.sum()
            lse[b, h] = m + np.log(e.sum())
            dot[b, h] = (np.abs(K) @ np.abs(q[b, h])).max() * abs(scale)
    return out, lse, mag, dot


def adjust(x, prior, rep, pres, freq, ids, bias, mask):
    """One row [V] of float64 logits. Returns the adjusted row and, for error bounds, the sum of the magnitudes of
    the terms that met in each value."""
    x = np.array(x, np.float64)
    mag = np.abs(x)
    V = len(x)
    if prior is not None:
        p = np.asarray(prior)
        u, n = np.unique(p[(p >= 0) & (p < V)], return_counts=True)
        y = np.where(x[u] < 0, x[u] * rep, x[u] / rep)
        x[u] = y - (n * freq + pres)
        mag[u] = np.abs(y) + np.abs(n * freq) + abs(pres)
    if ids is not None:
        for i, z in zip(ids, bias):
            if 0 <= i < V:
                x[i] += z
                mag[i] += abs(z)
    if mask is not None:
        j = np.arange(V)
        x[(np.asarray(mask).view(np.uint32)[j >> 5] >> (j & 31).astype(np.uint32)) & 1 == 0] = -np.inf
    return x, mag
