"""CPU oracle (numpy, float64) of the grouped-query operators: attention over
packed prompts, and the e4m3 cache with a scale per block and head (append,
attention, attention weights, eviction).  Straight from the definitions in
include/dsv4b.h; positions that a query does not see never enter a sum.

Caches are uint8 arrays [num_blocks, P, h_kv, d].
"""
from __future__ import annotations

import numpy as np


def _decode_table():
    t = np.zeros(256)
    for b in range(256):
        s, e, m = b >> 7, (b >> 3) & 15, b & 7
        x = np.nan if (e == 15 and m == 7) else (m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
        t[b] = -x if s else x
    return t


E4M3 = _decode_table()
_POS = E4M3[:127]  # 0 .. 448, ascending


def e4m3_encode(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3, ties to even, +-448 beyond; NaN keeps no sign."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.where(np.isnan(x), 0, np.abs(x)), 448.0)
    hi = np.clip(np.searchsorted(_POS, a, side="left"), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    pick = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    code = pick.astype(np.uint8) | (np.signbit(x).astype(np.uint8) << 7)
    return np.where(np.isnan(x), np.uint8(0x7F), code)


def softmax_row(s: np.ndarray, v: np.ndarray):
    """(out, lse, sum_t p |v|) of one row over the keys it sees (s [n], v [n, d])."""
    d = v.shape[1]
    if s.size == 0:
        return np.zeros(d), -np.inf, np.zeros(d)
    m = s.max() if not np.isnan(s).any() else np.nan
    with np.errstate(invalid="ignore", over="ignore"):
        p = np.exp(s - m)
        l = p.sum()
        p = p / l
        out = (p[:, None] * v).sum(0)
        mag = (p[:, None] * np.abs(v)).sum(0)
        return out, m + np.log(l), mag


def prefill(q, k, v, cu_q, cu_k, scale, causal):
    """out [Tq, h_q, d_v], lse [Tq, h_q], sum p|v| like out, and per row the
    largest scale * sum |q||k| that it sees.  Rows of no sequence are NaN."""
    tq, h_q, _ = q.shape
    g = h_q // k.shape[1]
    out = np.full((tq, h_q, v.shape[2]), np.nan)
    mag, lse, size = out.copy(), np.full((tq, h_q), np.nan), np.zeros((tq, h_q))
    for i in range(len(cu_q) - 1):
        q0, q1, k0, k1 = cu_q[i], cu_q[i + 1], cu_k[i], cu_k[i + 1]
        n_q, n_k = q1 - q0, k1 - k0
        for h in range(h_q):
            kk, vv = k[k0:k1, h // g], v[k0:k1, h // g]
            with np.errstate(invalid="ignore"):
                s = (q[q0:q1, h] @ kk.T) * scale
                a = (np.abs(q[q0:q1, h]) @ np.abs(kk).T) * scale
            for x in range(n_q):
                n = max(0, min(n_k, x + n_k - n_q + 1)) if causal else n_k
                out[q0 + x, h], lse[q0 + x, h], mag[q0 + x, h] = softmax_row(s[x, :n], vv[:n])
                size[q0 + x, h] = a[x, :n].max() if n else 0
    return out, lse, mag, size


def held(cache, scale, table, length, h):
    """Values [n, d] and positions [n] that sequence's head h holds below `length`."""
    P, nb = cache.shape[1], cache.shape[0]
    pos = np.array([t for t in range(min(length, len(table) * P)) if 0 <= table[t // P] < nb], np.int64)
    if pos.size == 0:
        return np.zeros((0, cache.shape[3])), pos
    blk = np.asarray(table)[pos // P]
    return E4M3[cache[blk, pos % P, h]] * scale[blk, h].astype(np.float64)[:, None], pos


def decode(q, kc, vc, ks, vs, table, ctx, scale):
    """out [b, s_q, h_q, d], lse [b, h_q, s_q], sum p|v| like out, size like lse, and
    sum |v| over the seen positions like out."""
    b, s_q, h_q, d = q.shape
    g = h_q // kc.shape[2]
    out, mag, vsum = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape)
    lse, size = np.full((b, h_q, s_q), -np.inf), np.zeros((b, h_q, s_q))
    for i in range(b):
        for kvh in range(kc.shape[2]):
            k, pos = held(kc, ks, table[i], int(ctx[i]), kvh)
            v, _ = held(vc, vs, table[i], int(ctx[i]), kvh)
            for h in range(kvh * g, (kvh + 1) * g):
                for x in range(s_q):
                    see = pos <= ctx[i] - s_q + x
                    with np.errstate(invalid="ignore"):
                        s = (k[see] @ q[i, x, h]) * scale
                        a = (np.abs(k[see]) @ np.abs(q[i, x, h])) * scale
                    out[i, x, h], lse[i, h, x], mag[i, x, h] = softmax_row(s, v[see])
                    size[i, h, x] = a.max() if a.size else 0
                    vsum[i, x, h] = np.abs(v[see]).sum(0)
    return out, lse, mag, size, vsum


def weights(q, lse, kc, ks, table, ctx, scale, width):
    """[b, h_kv, width], and the same of p * (1 + |lse| + scale sum |q||k|), for tolerances."""
    b, s_q, h_q, d = q.shape
    g = h_q // kc.shape[2]
    w, e = np.zeros((b, kc.shape[2], width)), np.zeros((b, kc.shape[2], width))
    for i in range(b):
        for kvh in range(kc.shape[2]):
            k, pos = held(kc, ks, table[i], min(int(ctx[i]), width), kvh)
            for h in range(kvh * g, (kvh + 1) * g):
                for x in range(s_q):
                    see = pos <= ctx[i] - s_q + x
                    if lse[i, h, x] == -np.inf:
                        continue
                    p = np.exp((k[see] @ q[i, x, h]) * scale - lse[i, h, x])
                    a = (np.abs(k[see]) @ np.abs(q[i, x, h])) * scale
                    w[i, kvh, pos[see]] += p
                    e[i, kvh, pos[see]] += p * (1 + abs(lse[i, h, x]) + a)
    return w, e


def block_exponent(amax: float) -> int:
    if amax == 0:
        return -100
    e = int(np.ceil(np.log2(amax / 448.0)))
    while amax > 448.0 * 2.0 ** e:
        e += 1
    while amax <= 448.0 * 2.0 ** (e - 1):
        e -= 1
    return max(-100, e)


def append(x, cu, ctx, table, cache, scale):
    """One of K and V, in place (cache uint8, scale fp32)."""
    nb, P, h_kv, _ = cache.shape
    for i in range(len(ctx)):
        n = cu[i + 1] - cu[i]
        start, t = ctx[i] - n, 0
        while t < n:
            p = start + t
            if p < 0:
                t += 1
                continue
            m = min(P - p % P, n - t)
            blk = table[i][p // P] if p // P < len(table[i]) else -1
            if 0 <= blk < nb:
                for h in range(h_kv):
                    new = x[cu[i] + t:cu[i] + t + m, h].astype(np.float64)
                    fin = np.abs(new[np.isfinite(new)])
                    s = np.float32(2.0 ** block_exponent(fin.max() if fin.size else 0.0))
                    old = p % P
                    if old:
                        s0 = scale[blk, h]
                        s = max(s, s0)
                        if s != s0:
                            r = np.float32(s0) / np.float32(s)
                            vals = (E4M3[cache[blk, :old, h]].astype(np.float32) * r).astype(np.float64)
                            cache[blk, :old, h] = e4m3_encode(vals)
                    scale[blk, h] = s
                    with np.errstate(over="ignore"):
                        cache[blk, old:old + m, h] = e4m3_encode((new.astype(np.float32) / s).astype(np.float64))
            t += m


def evict(kc, vc, ks, vs, table, ctx, w, budget, recent, new_table):
    """kept, new_weights, new_lens; writes the new blocks in place."""
    nb, P, h_kv, _ = kc.shape
    b = len(ctx)
    kept = np.full((b, h_kv, budget), -1, np.int32)
    new_w = np.zeros((b, h_kv, budget), np.float32)
    lens = np.zeros(b, np.int32)
    for i in range(b):
        n = max(0, min(int(ctx[i]), w.shape[2], table.shape[1] * P))
        lens[i] = m = min(n, budget)
        for h in range(h_kv):
            if n > budget:
                old = w[i, h, :n - recent]
                key = np.where(np.isnan(old), np.inf, old)
                order = sorted(range(n - recent), key=lambda t: (0 if np.isnan(old[t]) else 1, -key[t], t))
                pos = sorted(order[:budget - recent]) + list(range(n - recent, n))
            else:
                pos = list(range(n))
            kept[i, h, :m] = pos
            new_w[i, h, :m] = w[i, h, pos]
            for j0 in range(0, m, P):
                rows = pos[j0:j0 + P]
                dest = new_table[i][j0 // P] if j0 // P < new_table.shape[1] else -1
                if not 0 <= dest < nb:
                    continue
                for cache, scale in ((kc, ks), (vc, vs)):
                    src = [(table[i][t // P], t % P) for t in rows]
                    ok = [0 <= p < nb for p, _ in src]
                    s = np.array([scale[p, h] if o else 0 for (p, _), o in zip(src, ok)], np.float32)
                    top = max(np.float32(0), s.max())
                    for r, ((p, off), o) in enumerate(zip(src, ok)):
                        if not o:
                            cache[dest, r, h] = 0
                        elif s[r] == top:
                            cache[dest, r, h] = cache[p, off, h]
                        else:
                            x = E4M3[cache[p, off, h]].astype(np.float32) * (s[r] / top)
                            cache[dest, r, h] = e4m3_encode(x.astype(np.float64))
                    scale[dest, h] = top
    return kept, new_w, lens
