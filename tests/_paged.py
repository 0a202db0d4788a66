"""Plain 64-bit restatements of the paged-cache operators and of sampling
(include/ptmi.h), and what their tests share."""
import ctypes

import numpy as np

import pitorch_amd as pa

SENTINEL = np.float32(-7.5e33)      # what outputs hold before a call


def bf16(x):
    """x rounded to the nearest bf16, ties to even, as its 16 bits."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + (u >> 16 & 1)) >> 16).astype(np.uint16)
    return np.where((u & 0x7FFFFFFF) > 0x7F800000, (u >> 16 | 0x40).astype(np.uint16), r)


def from_bf16(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def pages_for(n, page):
    return -(-n // page)


def pages_struct(k, v, kind, n_pages, page, kv_heads, hd, strides=None):
    st = strides or (page * kv_heads * hd, kv_heads * hd, hd)
    return pa.Pages(k, v, kind, n_pages, page, kv_heads, hd, *st)


def place(strides, slots, page, heads, hd):
    """Element offsets [slots, heads, hd] of slots in a cache of these strides."""
    slots = np.asarray(slots, np.int64)
    at = slots // page * strides[0] + slots % page * strides[1]
    return at[:, None, None] + (np.arange(heads) * strides[2])[None, :, None] + np.arange(hd)


def plan(past, fresh, pool, n_pages, page, table, max_rows):
    """(kv_len, pool, row_start, row_pos, row_slot, status); table is changed in place."""
    S, W = table.shape
    n = lambda t: pages_for(t, page) if t > 0 else 0  # noqa: E731
    status, give, take = 0, [], 0
    if not 0 <= len(pool) <= n_pages:
        status |= 8
    rows = 0
    for i in range(S):
        p, f = int(past[i]), int(fresh[i])
        if p < 0 or f < -1 or p + f > 2**31 - 1 or f > 2**24 or n(p) > 2**24:
            status |= 8
            continue
        if n(p + max(f, 0)) > W:
            status |= 2
        elif f < 0:
            give += table[i, :n(p)].tolist()
        if f >= 0:
            take += n(p + f) - n(p)
            rows += f
        elif n(p) > W:
            give += [0] * n(p)
    if len(pool) + len(give) > n_pages:
        status |= 8
    if take > len(pool) + len(give):
        status |= 1
    if rows > max_rows:
        status |= 4
    kv, start = np.array(past, np.int32), np.zeros(S + 1, np.int32)
    pos, slot = np.full(max_rows, -1, np.int32), np.full(max_rows, -1, np.int32)
    if status:
        return kv, list(pool), start, pos, slot, status
    pool = list(pool) + give
    r = 0
    for i in range(S):
        start[i] = r
        p, f = int(past[i]), int(fresh[i])
        kv[i] = 0 if f < 0 else p + f
        for j in range(n(p), n(p + f) if f >= 0 else 0):
            table[i, j] = pool.pop()
        for t in range(p, p + max(f, 0)):
            pg = table[i, t // page]
            pos[r], slot[r] = t, pg * page + t % page if 0 <= pg < n_pages else -1
            r += 1
    start[S] = r
    return kv, pool, start, pos, slot, 0


def rotate(x, pos, rope):
    """x [rows, heads, hd] in fp32 as the store rotates it (no fused roundings)."""
    c, s = rope[pos][:, None, :, 0], rope[pos][:, None, :, 1]
    u, v = x[..., 0::2], x[..., 1::2]
    return np.stack((u * c - v * s, u * s + v * c), -1).reshape(x.shape)


def attention(q, k, v, table, page, n_pages, row_start, kv_len, scale, out):
    """fp64 results written over `out` [rows, heads, hd], and a bound on |error| of a
    result summed in fp32 in any order:
    a score is off by (hd + 8) 2^-24 scale sum|q k|, d at most over the row, and e^s by a
    factor 1 + 2d; normalised sums of `keys` terms by 2 (keys + 16) 2^-24 sum p|v|.
    k, v: [n_pages*page, kv_heads, hd] as the cache holds them."""
    bound = np.zeros_like(out)
    H, hd = q.shape[1:]
    G = H // k.shape[1]
    W = table.shape[1]
    for s in range(len(kv_len)):
        L = min(max(int(kv_len[s]), 0), W * page)
        n = row_start[s + 1] - row_start[s]
        if n <= 0:
            continue
        t = np.arange(L)
        pg = table[s, t // page] if L else np.zeros(0, np.int64)
        ok = (pg >= 0) & (pg < n_pages)
        t, slot = t[ok], (pg.astype(np.int64) * page + t % page)[ok]
        kk, vv = k[slot].astype(np.float64), v[slot].astype(np.float64)
        for i in range(n):
            r = row_start[s] + i
            if not 0 <= r < len(out):
                continue
            see = t <= L - n + i
            for h in range(H):
                K, Vv, x = kk[see, h // G], vv[see, h // G], q[r, h].astype(np.float64)
                if not len(K):
                    out[r, h] = 0
                    continue
                sc = (K @ x) * scale
                d = (hd + 8) * 2.0**-24 * np.max(np.abs(K) @ np.abs(x)) * abs(scale)
                p = np.exp(sc - sc.max())
                p /= p.sum()
                out[r, h] = p @ Vv
                bound[r, h] = (2 * d + 2 * (len(K) + 16) * 2.0**-24) * (p @ np.abs(Vv)) + 1e-37
    return bound


def sample(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
    """One row; also the least distance of a decision from its border, relative to the sum there."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    top = x.max()
    if top == -np.inf:
        return -1, 1.0
    order = np.argsort(-x, kind="stable")
    if not temperature > 0:
        return int(order[0]), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / np.float64(temperature)))
    w[w < 2.0**-45] = 0
    margin = 1.0
    keep = np.ones(len(x), bool)
    if top_k > 0:
        keep[order[top_k:]] = False
    mp = min(max(min_p, 0.0), 1.0) if min_p == min_p else 0.0
    keep &= w >= mp
    keep[order[0]] = True
    ws = np.where(keep, w, 0)[order]
    before = np.concatenate(([0.0], np.cumsum(ws)[:-1]))
    if not top_p >= 1:
        lim = top_p * ws.sum() if top_p > 0 else 0.0
        margin = min(margin, np.min(np.abs(before[1:] - lim)) / ws.sum() if len(ws) > 1 else 1.0)
        drop = ~(before < lim)
        drop[0] = False
        keep[order[drop]] = False
    c = np.cumsum(np.where(keep, w, 0))
    u = min(max(u, 0.0), 1 - 2.0**-24) if u == u else 0.0
    target = u * c[-1]
    token = int(np.sum(c <= target))
    margin = min(margin, np.min(np.abs(np.concatenate(([0.0] if u else [], c)) - target)) / c[-1])
    return token, margin


def byref(s):
    return ctypes.byref(s)
