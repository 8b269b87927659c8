"""Plain 64-bit forms of the paged 8-bit KV cache and of the row sampler, on the
host, written from their definitions (include/brolm_hip.h)."""
from __future__ import annotations

import math

import numpy as np

NO_PAGES, TABLE_FULL, ROWS_FULL, BAD_LENGTH, BAD_RING = 1, 2, 4, 8, 16


def plan(past, delta, page, n_pages, table, ring, ends, max_rows):
    """(lens, starts, slots, pos, ends, status); table and ring change in place."""
    n = len(past)
    width = table.shape[1]
    head, tail = int(ends[0]), int(ends[1])
    blocks = lambda x: -(-x // page)
    status, rows, take, give = 0, 0, 0, 0
    for a, d in zip(past, delta):
        a, d = int(a), int(d)
        if a < 0 or a + d < 0 or a > width * page:
            status |= BAD_LENGTH
        elif a + d > width * page:
            status |= TABLE_FULL
        else:
            rows += max(0, d)
            take += max(0, blocks(a + d) - blocks(a))
            give += max(0, blocks(a) - blocks(a + d))
    if head < 0 or tail < head or tail - head > n_pages or tail - head + give > n_pages:
        status |= BAD_RING
    elif take > tail - head:
        status |= NO_PAGES
    if rows > max_rows:
        status |= ROWS_FULL
    slots, pos = np.full(max_rows, -1, np.int64), np.full(max_rows, -1, np.int32)
    if status:
        return np.array(past, np.int32), np.zeros(n + 1, np.int32), slots, pos, np.array(ends, np.int64), status
    starts, back = [0], []
    for r in range(n):
        a, d = int(past[r]), int(delta[r])
        for b in range(blocks(a), blocks(a + d)):
            table[r, b] = ring[head % n_pages]
            head += 1
        back += [table[r, b] for b in range(blocks(a + d), blocks(a))]
        for i in range(max(0, d)):
            p = a + i
            pg = int(table[r, p // page])
            pos[starts[-1] + i] = p
            slots[starts[-1] + i] = pg * page + p % page if 0 <= pg < n_pages else -1
        starts.append(starts[-1] + max(0, d))
    for g in back:
        ring[tail % n_pages] = g
        tail += 1
    return (np.array(past, np.int32) + np.array(delta, np.int32), np.array(starts, np.int32), slots, pos,
            np.array([head, tail], np.int64), 0)


def empty_cache(n_pages, n_kv, page, hd, rng=None):
    """Codes and scales as numpy arrays; random bytes when rng is given (memory need not be cleared)."""
    if rng is None:
        return dict(kc=np.zeros((n_pages, n_kv, page, hd), np.int8), vc=np.zeros((n_pages, n_kv, hd, page), np.int8),
                    ks=np.zeros((n_pages, n_kv), np.float32), vs=np.zeros((n_pages, n_kv), np.float32))
    return dict(kc=rng.integers(-128, 128, (n_pages, n_kv, page, hd)).astype(np.int8),
                vc=rng.integers(-128, 128, (n_pages, n_kv, hd, page)).astype(np.int8),
                ks=rng.uniform(1e-3, 1e-1, (n_pages, n_kv)).astype(np.float32),
                vs=rng.uniform(1e-3, 1e-1, (n_pages, n_kv)).astype(np.float32))


def append(cache, k, v, slots):
    """k, v (rows, n_kv, hd) float16 into the cache, in place."""
    n_pages, n_kv, page, hd = cache["kc"].shape
    i = 0
    while i < len(slots):
        s0 = int(slots[i])
        if not 0 <= s0 < n_pages * page:
            i += 1
            continue
        n = 1
        while i + n < len(slots) and slots[i + n] == s0 + n and (s0 + n) % page:
            n += 1
        pg, off = s0 // page, s0 % page
        for x, codes, scales in ((k, cache["kc"][pg], cache["ks"][pg]),
                                 (v, np.swapaxes(cache["vc"][pg], 1, 2), cache["vs"][pg])):
            for h in range(n_kv):
                rows = x[i:i + n, h].astype(np.float64)
                old = scales[h] if off else np.float32(0)
                with np.errstate(invalid="ignore"):
                    new = np.maximum(old, np.float32(np.abs(rows).max() / 127))   # a NaN stays
                scales[h] = new
                if not (new > 0 and np.isfinite(new)):
                    codes[h, off:off + n] = 0
                    if off and new != old:
                        codes[h, :off] = 0
                    continue
                if off and new != old:
                    codes[h, :off] = np.rint(codes[h, :off].astype(np.float64) * float(old) / float(new))
                codes[h, off:off + n] = np.rint(rows / float(new))
        i += n


def values(cache, pages):
    """K and V (tokens of the pages in order, n_kv, hd) in 64 bits."""
    with np.errstate(invalid="ignore"):
        k = cache["kc"][pages].astype(np.float64) * cache["ks"][pages][:, :, None, None].astype(np.float64)
        v = cache["vc"][pages].astype(np.float64) * cache["vs"][pages][:, :, None, None].astype(np.float64)
    n_kv, hd = k.shape[1], k.shape[3]
    return (k.transpose(0, 2, 1, 3).reshape(-1, n_kv, hd), v.transpose(0, 3, 1, 2).reshape(-1, n_kv, hd))


def attention(cache, q, starts, lens, table, n_kv, window=0):
    """(out, bound): out (rows, n_q, hd) in 64 bits for the rows of q (rows, n_q, hd)
    float16, and how far an FP16 result computed as documented may be from it.

    The bound adds: the output's rounding, 2^-11 |o|; the rounding of every P to
    FP16, 2^-11 A with A the mean of |v| under the weights; q as 256 hi + lo times a power
    of two, off by at most half a step, max|q| 2^k being 16319.75 at least: a score by d =
    max|q| / 32639 sum|k| / sqrt(hd) and the weights by a factor within e^(+-2d); FP32 sums of n
    products and FP32 exponentials, (n + 64) 2^-23 A, and the FP32 rounding of a score
    of magnitude x (2^-22 x in the exponent, twice); P below FP16's normal range, at most
    n 2^-24 of the largest scale times 127 / 2^7."""
    n_pages, _, page, hd = cache["kc"].shape
    rows, n_q = q.shape[:2]
    out, bound = np.zeros((rows, n_q, hd)), np.zeros((rows, n_q, hd))
    group = n_q // n_kv
    for r in range(len(lens)):
        n, m = int(lens[r]), int(starts[r + 1]) - int(starts[r])
        if n <= 0 or m <= 0:
            continue
        pages = table[r, :-(-n // page)]
        ok = np.repeat((pages >= 0) & (pages < n_pages), page)[:n]
        k, v = values(cache, np.where((pages >= 0) & (pages < n_pages), pages, 0))
        key = np.arange(n)
        for i in range(m):
            p = n - m + i
            see = ok & (key <= p)
            if window > 0:
                see &= key > p - window
            if not see.any():
                continue
            for h in range(n_q):
                g = h // group
                kk, vv = k[:n][see][:, g], v[:n][see][:, g]
                qq = q[int(starts[r]) + i, h].astype(np.float64)
                s = kk @ qq / math.sqrt(hd)
                w = np.exp(s - s.max())
                w /= w.sum()
                o, a = w @ vv, w @ np.abs(vv)
                d = np.abs(qq).max() / 32639 * np.abs(kk).sum(1).max() / math.sqrt(hd)
                d += 2.0 ** -21 * np.abs(s).max()
                c = int(see.sum())
                out[int(starts[r]) + i, h] = o
                bound[int(starts[r]) + i, h] = (2.0 ** -11 * np.abs(o) + a * (2.0 ** -11 + math.expm1(2 * d) + (c + 64) * 2.0 ** -23)
                                                + c * 2.0 ** -24 * np.abs(vv).max())
    return out, bound


def sample(x, t, k, p, m, u):
    """The id drawn from one row of FP16 logits, and how near (in units of the kept
    mass) the draw or a cut lies to another answer."""
    x = x.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    if not t > 0:
        return int(np.argmax(x)), 1.0
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        e = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / float(t)))
    e = np.where(e >= 0, e, 0.0)
    run = np.cumsum(e)
    n, near = len(x), 1.0
    if k > 0:
        n = min(n, int(k))
    if not m <= 0:
        n = min(n, max(1, int((e >= float(m)).sum())))
        near = min(near, np.abs(e - float(m)).min())
    if p < 1:
        goal = float(p) * run[-1]
        n = min(n, int(np.argmax(run >= goal)) + 1)
        near = min(near, np.abs(run - goal).min() / run[-1])
    kept = run[:n]
    goal = u * kept[-1]
    near = min(near, np.abs(kept - goal).min() / kept[-1])
    hit = np.nonzero(kept > goal)[0]
    return int(order[hit[0] if len(hit) else n - 1]), near
