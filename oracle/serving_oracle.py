"""Numpy / float64 restatement of the serving operators (test infrastructure only): slot maps,
the 8-bit paged cache, the attention over it, and sampling. Row by row and token by token,
from the definitions in ``include/dsalt_b200.h``."""
from __future__ import annotations

import math

import numpy as np

E_MIN = -110
BIG = 448.0


# --------------------------------------------------------------------------- slots
def reserve(tables, seq_lens, new_lens, free_pages, n_free, page, n_tokens):
    """``(tables, slots, positions, cu_new, granted, seq_lens, n_free)`` after the call."""
    tables = tables.copy()
    S, max_pages = tables.shape
    n_free = min(max(int(n_free), 0), len(free_pages))
    slots = np.full(n_tokens, -1, np.int64)
    positions = np.zeros(n_tokens, np.int32)
    cu = np.zeros(S + 1, np.int32)
    granted = np.zeros(S, bool)
    lens = np.zeros(S, np.int32)
    at, order = 0, 0
    left = n_free
    for s in range(S):
        old, new = max(int(seq_lens[s]), 0), max(int(new_lens[s]), 0)
        have, want = -(-old // page), -(-(old + new) // page)
        fits = want <= max_pages and at + new <= n_tokens
        need = want - have if fits else 0
        order += need
        granted[s] = fits and (need == 0 or order <= n_free)
        lens[s] = old + new if granted[s] else old
        if granted[s]:
            for j in range(need):
                tables[s, have + j] = free_pages[n_free - 1 - (order - need + j)]
            left -= need
            for r in range(new):
                pos = old + r
                if tables[s, pos // page] >= 0:
                    slots[at + r] = int(tables[s, pos // page]) * page + pos % page
                positions[at + r] = pos
        at += new
        cu[s + 1] = min(at, n_tokens)
    return tables, slots, positions, cu, granted, lens, left


def release(tables, seq_lens, flags, free_pages, n_free, page):
    """``(tables, seq_lens, free_pages, n_free)`` after the call."""
    tables, lens, free = tables.copy(), seq_lens.copy(), free_pages.copy()
    given = []
    for s in np.flatnonzero(flags):
        held = -(-max(int(lens[s]), 0) // page)
        given += [int(p) for p in tables[s, :held]]
        tables[s, :held] = -1
        lens[s] = 0
    for j, p in enumerate(given):
        free[n_free + len(given) - 1 - j] = p
    return tables, lens, free, n_free + len(given)


# --------------------------------------------------------------------------- cache
def e4m3_values():
    """The 256 values of e4m3 (NaN at 0x7f and 0xff)."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m / 8.0 * 2.0 ** -6, (1 + m / 8.0) * 2.0 ** (e - 7.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b < 128, v, -v)


VALUES = e4m3_values()


def to_e4m3(x):
    """Nearest e4m3 value, ties to even; beyond the largest, and for infinities: the largest."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), BIG)
    _, e = np.frexp(np.maximum(a, 2.0 ** -6))
    step = np.ldexp(1.0, e - 4)
    r = np.minimum(np.rint(np.where(np.isnan(a), 0, a) / step) * step, BIG)
    return np.where(np.isnan(x), np.nan, np.copysign(r, x))


def need_exponent(amax):
    if amax == 0:
        return E_MIN
    e = math.ceil(math.log2(amax / BIG)) + 1
    while e > E_MIN and amax <= BIG * 2.0 ** (e - 1):
        e -= 1
    return max(e, E_MIN)


def append(x, cache, scale, slots, page):
    """One of K / V: ``x [T, H, D]``, ``cache [n_pages, H, page, D]`` values (not bytes), ``scale
    [n_pages, H]``; returns the new ``(cache, scale)`` in float64."""
    x, cache, scale = np.asarray(x, np.float64), np.array(cache, np.float64), np.array(scale, np.float64)
    n_pages, H = scale.shape
    ok = (slots >= 0) & (slots < n_pages * page)
    for p in np.unique(slots[ok] // page):
        toks = np.flatnonzero(ok & (slots // page == p))
        offs = slots[toks] % page
        fresh = (offs == 0).any()
        for h in range(H):
            new = x[toks, h]
            fin = np.abs(new[np.isfinite(new)])
            e = need_exponent(float(fin.max()) if fin.size else 0.0)
            if not fresh:
                old = max(int(math.log2(scale[p, h])), E_MIN) if scale[p, h] > 0 else E_MIN
                e = max(e, old)
                if e > old:
                    cache[p, h] = to_e4m3(cache[p, h] * 2.0 ** (old - e))
            scale[p, h] = 2.0 ** e
            cache[p, h, offs] = to_e4m3(new * 2.0 ** -e)
    return cache, scale


# --------------------------------------------------------------------------- attention
def attention(q, k_cache, v_cache, k_scale, v_scale, tables, seq_lens, cu_q, w, lmk, bias):
    """``(out [T, H, D], lse [T, H], spread [T, H, D], size [T, H], n [T, H])``. ``spread`` is
    ``sum p|v| / sum p`` and ``size`` the largest ``sum_d |q_d k_d| / sqrt(D)`` of a row's keys: what
    rounding errors are relative to; ``n`` the number of keys. Caches are values."""
    T, H, D = q.shape
    Hkv, page = k_cache.shape[1], k_cache.shape[2]
    S = len(seq_lens)
    out, spread = np.zeros((T, H, D)), np.zeros((T, H, D))
    lse, size, count = np.full((T, H), -np.inf), np.zeros((T, H)), np.zeros((T, H), int)
    for s in range(S):
        t0, t1 = (s, s + 1) if cu_q is None else (int(cu_q[s]), int(cu_q[s + 1]))
        n = int(seq_lens[s])
        for t in range(t0, t1):
            i = n - (t1 - t0) + (t - t0)
            if i < 0:
                continue
            lo = max(0, i - max(int(w[t]), 1) + 1) if w is not None else 0
            for h in range(H):
                keys, add = list(range(lo, i + 1)), [0.0] * (i + 1 - lo)
                if lmk is not None:
                    for c, p in enumerate(lmk[h, s]):
                        if 0 <= p < lo:
                            keys.append(int(p))
                            add.append(0.0 if bias is None else float(bias[h, s, c]))
                keys = np.array(keys)
                pages = tables[s, keys // page]
                inside = (pages >= 0) & (pages < len(k_scale))
                keys, pages, add = keys[inside], pages[inside], np.array(add)[inside]
                if not len(keys):
                    continue
                hk = h // (H // Hkv)
                kk = k_cache[pages, hk, keys % page] * k_scale[pages, hk][:, None]
                vv = v_cache[pages, hk, keys % page] * v_scale[pages, hk][:, None]
                x = kk @ q[t, h] / math.sqrt(D) + add
                m = x.max()
                if m == -np.inf:
                    continue
                p = np.exp(x - m)
                out[t, h] = p @ vv / p.sum()
                spread[t, h] = p @ np.abs(vv) / p.sum()
                lse[t, h] = m + math.log(p.sum())
                size[t, h] = (np.abs(kk) @ np.abs(q[t, h])).max() / math.sqrt(D)
                count[t, h] = len(keys)
    return out, lse, spread, size, count


# --------------------------------------------------------------------------- sampling
def sample(logits, u, temperature, top_k, top_p, min_p):
    """One row: ``(token, logprob, margin)``; ``margin`` is how far, relative to the mass, the
    nearest decision (the top-p border, the draw) lies from the other side."""
    l = np.where(np.isnan(logits), -np.inf, np.asarray(logits, np.float64))
    V = len(l)
    top = l.max()
    if top == -np.inf:
        return 0, -np.inf, 1.0
    if not temperature > 0:
        return int(np.argmax(l)), 0.0, 1.0
    with np.errstate(invalid="ignore"):
        w = np.where(l == top, 1.0, np.where(l == -np.inf, 0.0, np.exp((l - top) / temperature)))
    order = np.lexsort((np.arange(V), -l))
    margin = 1.0
    if 0 < top_k < V:
        order = order[:top_k]
    if top_p < 1:
        mass = np.cumsum(w[order])
        gap = (mass - w[order] - top_p * mass[-1]) / mass[-1]
        n = max(1, int((gap < 0).sum()))
        margin = min(margin, float(np.abs(gap[1:]).min()) if V > 1 and len(gap) > 1 else 1.0)
        order = order[:n]
    if min_p > 0:
        order = order[:max(1, int((w[order] >= min_p).sum()))]
    kept = np.sort(order)
    mass = np.cumsum(w[kept])
    x = min(max(float(u), 0.0), 1.0) * mass[-1]
    at = min(int((mass <= x).sum()), int(np.flatnonzero(w[kept])[-1]))
    edges = np.abs(mass[:-1][w[kept][1:] > 0] - x) / mass[-1] if len(kept) > 1 else np.ones(1)
    if len(edges) and x > 0:
        margin = min(margin, float(edges.min()))
    return int(kept[at]), math.log(w[kept[at]] / mass[-1]), margin
