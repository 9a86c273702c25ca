"""Plain restatements of the ragged decode operators for the tests: lengths and
tables in whole numbers, the cache write in the 32-bit steps of its definition,
attention and sampling in 64 bits."""
from __future__ import annotations

import math

import numpy as np


def plan(held, keep, q, table, ring, state, P, T):
    """(table, ring, state, kv_len, cu_q, tok_req, tok_pos, slots, status)"""
    held, keep, q = (np.asarray(a, np.int64) for a in (held, keep, q))
    table, ring = table.copy(), ring.copy()
    B, cols = table.shape
    cap, (head, count) = len(ring), state
    bad = (held < 0) | (keep < 0) | (keep > held) | (q < 0) | (held > cols * P) | (keep + q > cols * P)
    good = ~bad
    have, need = -(-held // P), -(-(keep + q) // P)
    take, give = np.where(good, np.maximum(need - have, 0), 0), np.where(good, np.maximum(have - need, 0), 0)
    status = (1 if take.sum() > count else 0) | (2 if bad.any() else 0) | (4 if q[good].sum() > T else 0)
    req, pos, slots = np.full(T, -1), np.full(T, -1), np.full(T, -1)
    if status:
        return table, ring, (head, count), held, np.zeros(B + 1, np.int64), req, pos, slots, status
    old_ring, old_table, at, put, t, cu = ring.copy(), table.copy(), head, head + count, 0, [0]
    for b in range(B):
        for c in range(have[b], need[b]):
            table[b, c] = old_ring[at % cap]
            at += 1
        for c in range(need[b], have[b]):
            ring[put % cap] = old_table[b, c]
            put += 1
        for i in range(q[b]):
            p = keep[b] + i
            req[t], pos[t], slots[t] = b, p, table[b, p // P] * P + p % P
            t += 1
        cu.append(t)
    return table, ring, (at % cap, count - take.sum() + give.sum()), keep + q, np.array(cu), req, pos, slots, 0


def append(codes, scales, table, lens, cu, x, P, t):
    """New (codes, scales) after writing rows x [T][Hkv][D] to the requests' last positions."""
    codes, scales, x = codes.copy(), scales.copy(), x.astype(np.float32)
    f = np.float32
    with np.errstate(all="ignore"):
        for b in range(len(lens)):
            q = cu[b + 1] - cu[b]
            start = lens[b] - q
            if q == 0:
                continue
            for p0 in range(start // t * t, lens[b], t):
                lo, hi = max(p0, start), min(p0 + t, lens[b])
                page, off = table[b, p0 // P], p0 % P
                new = x[cu[b] + lo - start:cu[b] + hi - start]  # [n][H][D]
                a = np.where(np.isfinite(new), np.abs(new), 0).max((0, 2)).astype(f)
                old = scales[page, :, off // t] if lo > p0 else np.zeros_like(a)
                s = np.maximum(old, a * (f(1) / f(127)))
                s = np.where(s < f(2.0 ** -126), f(0), s)
                grown = s > old
                factor = np.where(grown, old / np.where(s > 0, s, f(1)), f(1)).astype(f)
                was = codes[page, :, off:off + lo - p0].astype(f)
                codes[page, :, off:off + lo - p0] = np.rint(was * factor[:, None, None]).astype(np.int8)
                inv = np.where(s > 0, f(1) / np.where(s > 0, s, f(1)), f(0))
                c = np.rint(new * inv[None, :, None])
                c = np.where(np.isnan(new) | (s == 0)[None, :, None], 0, np.clip(c, -127, 127))
                codes[page, :, off + lo - p0:off + hi - p0] = c.transpose(1, 0, 2).astype(np.int8)
                scales[page, :, off // t] = s
    return codes, scales


def attend(q, codes_k, codes_v, sk, sv, table, lens, cu, P, t, scale, window):
    """(out, lse, largest |v| seen) in 64 bits of q [T][H][D]."""
    T, H, D = q.shape
    Hkv, n_pages = codes_k.shape[1], codes_k.shape[0]
    G = H // Hkv
    out, lse, big = np.zeros((T, H, D)), np.full((T, H), -math.inf), np.zeros((T, H))
    for b in range(len(lens)):
        n, L = cu[b + 1] - cu[b], lens[b]
        pages = [table[b, p // P] for p in range(L)]
        ok = np.array([0 <= g < n_pages for g in pages], bool)
        idx = np.array([g if 0 <= g < n_pages else 0 for g in pages], np.int64)
        off = np.arange(L) % P
        for h in range(Hkv):
            with np.errstate(all="ignore"):
                k = codes_k[idx, h, off].astype(np.float64) * sk[idx, h, off // t].astype(np.float64)[:, None]
                v = codes_v[idx, h, off].astype(np.float64) * sv[idx, h, off // t].astype(np.float64)[:, None]
            for i in range(n):
                p = L - n + i
                seen = (np.arange(L) <= p) & ok
                if window:
                    seen &= np.arange(L) > p - window
                if not seen.any():
                    continue
                for hh in range(h * G, (h + 1) * G):
                    s = scale * (k[seen] @ q[cu[b] + i, hh].astype(np.float64))
                    m = s.max()
                    e = np.exp(s - m)
                    out[cu[b] + i, hh] = e @ v[seen] / e.sum()
                    lse[cu[b] + i, hh] = m + math.log(e.sum())
                    big[cu[b] + i, hh] = np.abs(v[seen]).max()
    return out, lse, big


def sample_row(l, T, k, top_p, min_p):
    """(z, kept weights in float64, z's order) of one row of float32 logits, before a draw."""
    l = np.where(np.isnan(l), -np.inf, l).astype(np.float32)
    with np.errstate(all="ignore"):
        z = (l / np.float32(T)).astype(np.float32)
        high = z.max()
        d = (z - high).astype(np.float32).astype(np.float64)
        e = np.where(z == high, 1.0, np.exp(d))
    w = np.floor(e * 2.0 ** 31)
    by = np.argsort(-z.astype(np.float64), kind="stable")
    if k > 0:
        by = by[:k]
    if top_p < 1:
        run = np.cumsum(w[by])
        most = max(1.0, math.floor(np.rint(np.float32(max(top_p, 0)) * 2 ** 24) * run[-1] / 2 ** 24))
        by = by[run - w[by] < most]
    by = by[e[by] >= min(min_p, 1.0)]
    kept = np.zeros_like(w)
    kept[by] = w[by]
    return z, kept, by
