"""Plain 64-bit forms of a paged serving step with shared prefixes, on the host, written
from their definitions (include/brolm_hip.h)."""
from __future__ import annotations

import math

import numpy as np

import paged_util as pu


def plan(parent, shared_lens, starts, lens, pos_in):
    """(pos, shared, order, groups, group_starts)."""
    n, rows = len(parent), len(pos_in)
    pos, shared = np.array(pos_in, np.int32), np.zeros(rows, np.int32)
    members = {}
    for r in range(n):
        p = int(parent[r])
        s = max(0, min(int(shared_lens[r]), int(lens[p]))) if 0 <= p < n and p != r else 0
        for i in range(int(starts[r]), int(starts[r + 1])):
            shared[i] = s
            if pos[i] >= 0:
                pos[i] += s
            if s:
                members.setdefault(p, []).append(i)
    order, groups, first = [], [], []
    for p in sorted(members):
        groups.append(p)
        first.append(len(order))
        order += members[p]
    fill = lambda x, m, v: np.array(x + [v] * (m - len(x)), np.int32)
    return pos, shared, fill(order, rows, -1), fill(groups, n, -1), fill(first, n + 1, len(order))


def norm_rope(x, gain, eps, pos, cos, sin):
    """(rows, heads, hd) in 64 bits: head RMSNorm (gain None: none), then the rotation of pairs."""
    x = x.astype(np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * gain.astype(np.float64)
    c, s = cos[pos].astype(np.float64)[:, None], sin[pos].astype(np.float64)[:, None]
    a, b = x[..., 0::2], x[..., 1::2]
    y = np.empty_like(x)
    y[..., 0::2], y[..., 1::2] = a * c - b * s, a * s + b * c
    return y


def tables(rows, hd, theta=1e4):
    a = np.arange(rows)[:, None] * theta ** (-2.0 * np.arange(hd // 2) / hd)
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def attention(cache, q, starts, lens, table, parent, shared_lens, n_kv, window=0):
    """(out, bound) as paged_util.attention gives them, over the shared keys and then the own
    ones.  The bound is the one derived there: parts are joined in FP32, whose products and sums
    are counted among its (n + 64) 2^-23."""
    n_pages, _, page, hd = cache["kc"].shape
    rows, n_q = q.shape[:2]
    out, bound = np.zeros((rows, n_q, hd)), np.zeros((rows, n_q, hd))
    group = n_q // n_kv

    def keys(r, n):
        pages = table[r, :-(-n // page)]
        ok = (pages >= 0) & (pages < n_pages)
        k, v = pu.values(cache, np.where(ok, pages, 0))
        return k[:n], v[:n], np.repeat(ok, page)[:n]

    for r in range(len(lens)):
        n, m = max(0, int(lens[r])), int(starts[r + 1]) - int(starts[r])
        if m <= 0:
            continue
        p = int(parent[r])
        s = max(0, min(int(shared_lens[r]), int(lens[p]))) if 0 <= p < len(lens) and p != r else 0
        parts = [keys(p, s)] * (s > 0) + [keys(r, n)] * (n > 0)
        if not parts:
            continue
        k, v, ok = (np.concatenate([x[i] for x in parts]) for i in range(3))
        key = np.arange(s + n)
        for i in range(m):
            at = s + int(lens[r]) - m + i
            see = ok & ((key < s) | (key <= at))
            if window > 0:
                see &= key > at - window
            if not see.any():
                continue
            for g in range(n_kv):
                kk, vv = k[see][:, g], v[see][:, g]
                qq = q[int(starts[r]) + i, g * group:(g + 1) * group].astype(np.float64)
                x = qq @ kk.T / math.sqrt(hd)
                w = np.exp(x - x.max(1, keepdims=True))
                w /= w.sum(1, keepdims=True)
                o, a = w @ vv, w @ np.abs(vv)
                d = np.abs(qq).max(1) / 32639 * np.abs(kk).sum(1).max() / math.sqrt(hd) + 2.0 ** -21 * np.abs(x).max(1)
                c = int(see.sum())
                to = slice(g * group, (g + 1) * group)
                out[int(starts[r]) + i, to] = o
                bound[int(starts[r]) + i, to] = (2.0 ** -11 * np.abs(o) + a * (2.0 ** -11 + np.expm1(2 * d)[:, None] + (c + 64) * 2.0 ** -23)
                                                 + c * 2.0 ** -24 * np.abs(vv).max())
    return out, bound
