"""The paged-cache operators in 64 bits, entry by entry (numpy, no torch).

A batch as the library takes it: cu_rows [n_seqs + 1], lens [n_seqs], pages
[n_seqs, pages_per_seq]; caches [n_pages, n_kv, page_size, head_dim].
"""
import numpy as np


def place(pages, n_pages, page_size, s, e):
    """(page, place) of entry e of sequence s, or None."""
    if e < 0 or e // page_size >= pages.shape[1]:
        return None
    p = int(pages[s, e // page_size])
    return (p, e % page_size) if 0 <= p < n_pages else None


def rows_of(cu_rows, n_rows):
    """(sequence, place among its rows) of each row; None for a row of no sequence."""
    out = [None] * n_rows
    for s in range(len(cu_rows) - 1):
        for t in range(max(int(cu_rows[s]), 0), min(int(cu_rows[s + 1]), n_rows)):
            out[t] = (s, t - int(cu_rows[s]))
    return out


def head_norm(x, w, eps):
    if w is None:
        return x
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def rotate(x, cos, sin):
    """(rotated, sum of the magnitudes that each value is made of)."""
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    y = np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)
    size = np.concatenate([abs(a * cos) + abs(b * sin), abs(b * cos) + abs(a * sin)], -1)
    return y, size


def append(q, k, v, n_pages, page_size, pages, cu_rows, lens, cos, sin, positions=None, q_norm=None, k_norm=None,
           eps=1e-6):
    """{row: (q, q size)} and {(page, place): (k, k size, v)} of the rows that are written."""
    qs, entries = {}, {}
    for t, at in enumerate(rows_of(cu_rows, q.shape[0])):
        if at is None:
            continue
        e = int(lens[at[0]]) + at[1]
        where = place(pages, n_pages, page_size, at[0], e)
        pos = e if positions is None else int(positions[t])
        if where is None or not 0 <= pos < cos.shape[0]:
            continue
        qs[t] = rotate(head_norm(q[t], q_norm, eps), cos[pos], sin[pos])
        entries[where] = rotate(head_norm(k[t], k_norm, eps), cos[pos], sin[pos]) + (v[t],)
    return qs, entries


def attention(q, k_cache, v_cache, pages, cu_rows, lens, scale, tree_mask=None):
    """(out, size, score): of each output value its sum of p |v|, of each row
    and head the largest sum of |q k| scale; rows of no sequence are NaN."""
    n, H, D = q.shape
    n_pages, KV, ps, _ = k_cache.shape
    out = np.full((n, H, D), np.nan)
    size = np.zeros((n, H, D))
    score = np.zeros((n, H))
    for t, at in enumerate(rows_of(cu_rows, n)):
        if at is None:
            continue
        s, i = at
        count = int(cu_rows[s + 1]) - int(cu_rows[s])
        seen = []
        for e in range(int(lens[s]) + count):
            j = e - int(lens[s])
            if j >= 0:
                if tree_mask is None:
                    if j > i:
                        continue
                elif j // 32 >= tree_mask.shape[1] or not int(tree_mask[t, j // 32]) >> (j % 32) & 1:
                    continue
            w = place(pages, n_pages, ps, s, e)
            if w is not None:
                seen.append(w)
        if not seen:
            out[t] = 0.0
            continue
        pg, pl = np.array(seen).T
        for h in range(H):
            kk, vv = k_cache[pg, h // (H // KV), pl], v_cache[pg, h // (H // KV), pl]
            z = kk @ q[t, h] * scale
            p = np.exp(z - z.max())
            p /= p.sum()
            out[t, h] = p @ vv
            size[t, h] = p @ abs(vv)
            score[t, h] = (abs(kk) @ abs(q[t, h])).max() * abs(scale)
    return out, size, score


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log probability, distance of u to the nearer end of the token's interval) of one row."""
    x = np.asarray(x, np.float64)
    if not temperature > 0:
        bad = np.isnan(x)
        return (int(bad.argmax()) if bad.any() else int(x.argmax())), 0.0, 1.0
    if np.isnan(x).any() or not np.isfinite(x.max()):
        return len(x) - 1, float("nan"), 1.0
    w = np.exp((x - x.max()) / temperature)
    order = np.lexsort((np.arange(len(x)), -x))
    kept = order[:top_k] if top_k > 0 else order
    if top_p < 1:
        total = w[kept].sum()
        above, n = 0.0, 0
        while n < len(kept):  # a group of equal values at a time
            if n and not above < top_p * total:
                break
            m = n
            while m < len(kept) and x[kept[m]] == x[kept[n]]:
                m += 1
            above += w[kept[n:m]].sum()
            n = m
        kept = kept[:n]
    kept = np.sort(kept[w[kept] >= min(min_p, 1.0)])
    c = np.cumsum(w[kept])
    j = min(int(np.searchsorted(c, u * c[-1], side="right")), len(kept) - 1)
    while w[kept[j]] == 0:
        j -= 1
    lo = c[j - 1] if j else 0.0
    return int(kept[j]), float(np.log(w[kept[j]] / c[-1])), float(min(abs(u - lo / c[-1]), abs(c[j] / c[-1] - u)))
