"""A paged serving step with shared prefixes on the GPU against plain 64-bit forms
(prefix_util.py): plan, q / k / v in one pass, attention, and a run of them together.
Plans, codes and scales are whole numbers or exactly rounded and compared bit for bit;
norms, rotation and attention within bounds derived there."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import paged_util as pu
import prefix_util as px
from gpu_util import call, dev, f16_dev, hip, host, ptr, release, stream, torch
from test_gpu_paged import Cache, Plan, _f16, _tables

pytestmark = pytest.mark.gpu


def _i32(x):
    return dev(np.asarray(x, np.int32))


def _half(a):
    """float16 (rows, ...) as a (rows, -1) device tensor."""
    return dev(a.view(np.uint16)).view(torch().float16).reshape(a.shape[0], -1)


class Prefix:
    """Outputs of bx_prefix_plan."""

    def __init__(self, n_req, rows):
        t = torch()
        self.n_req, self.rows = n_req, rows
        self.pos, self.shared, self.order = (t.full((rows,), 77, dtype=t.int32, device="cuda") for _ in range(3))
        self.groups = t.full((n_req,), 77, dtype=t.int32, device="cuda")
        self.group_starts = t.full((n_req + 1,), 77, dtype=t.int32, device="cuda")

    def step(self, parent, shared_lens, starts, lens, pos_in):
        call("bx_prefix_plan", ptr(parent), ptr(shared_lens), ptr(starts), ptr(lens), self.n_req, ptr(pos_in), ptr(self.pos),
             ptr(self.shared), ptr(self.order), self.rows, ptr(self.groups), ptr(self.group_starts), stream())

    def outputs(self):
        return [host(x) for x in (self.pos, self.shared, self.order, self.groups, self.group_starts)]


def attend(c, q, starts, lens, table, p, n_q, max_new, max_len, max_groups, max_shared, window=0, out=None, ws=None):
    t = torch()
    rows, n_req = q.shape[0], lens.numel()
    if out is None:
        out = t.full((rows, n_q * c.hd), 9.0, dtype=t.float16, device="cuda")
    if ws is None:
        n = int(hip().bx_attention_prefix_q8_workspace_bytes(rows, n_req, n_q, c.n_kv, c.hd, max_new, max_len, max_groups, max_shared))
        ws = t.zeros(n, dtype=t.uint8, device="cuda")
        ws[512 * 1024:] = 0xff   # what lies behind the counters may hold anything
    call("bx_attention_prefix_q8_f16", ptr(q), q.stride(0), rows, ptr(starts), ptr(lens), n_req, max_new, max_len,
         ptr(p.pos), ptr(p.shared), ptr(p.order), ptr(p.groups), ptr(p.group_starts), max_groups, max_shared, ptr(table),
         table.shape[1], *c.args(), n_q, c.n_kv, c.hd, window, ptr(out), out.stride(0), ptr(ws), C.c_size_t(ws.numel()),
         stream())
    return out


# ---------------------------------------------------------------------- plan

@pytest.mark.parametrize("n,most,extra", [(1, 3, 2), (2, 1, 0), (5, 40, 3), (64, 2, 1), (65, 9, 0), (700, 3, 700), (4096, 2, 5)])
def test_prefix_plan(n, most, extra):
    """Parents of every kind, among them none, itself and numbers out of range; requests without rows."""
    rng = np.random.default_rng(n + most)
    for turn, spread in enumerate((1, max(1, n // 50), n)):
        news = rng.integers(0, most + 1, n)
        starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        lens = np.where(rng.random(n) < 0.1, 0, rng.integers(0, 3000, n)).astype(np.int32)
        parent = rng.integers(0, spread, n)
        parent = np.where(rng.random(n) < 0.15, rng.choice([-1, n, -2 ** 31, 2 ** 31 - 1], n), parent).astype(np.int32)
        shared_lens = rng.choice([0, -1, 1, 700, 2 ** 31 - 1, -2 ** 31], n).astype(np.int32)
        rows = int(starts[-1]) + extra or 1
        pos_in = np.full(rows, -1, np.int32)
        pos_in[:starts[-1]] = rng.integers(0, 5000, int(starts[-1]))
        want = px.plan(parent, shared_lens, starts, lens, pos_in)
        p = Prefix(n, rows)
        args = [_i32(x) for x in (parent, shared_lens, starts, lens, pos_in)]
        print(f"[prefix plan] n={n} turn={turn} rows={rows}", flush=True)
        p.step(*args)
        for got, w, name in zip(p.outputs(), want, ("pos", "shared", "order", "groups", "group_starts")):
            np.testing.assert_array_equal(got, w, err_msg=name)
        # the positions in place
        p.pos = args[4]
        p.step(*args)
        for got, w in zip(p.outputs(), want):
            np.testing.assert_array_equal(got, w)
    release()


def test_prefix_plan_without_rows():
    """After a step that bx_kv_plan could not lay out: no row, no group."""
    p = Prefix(3, 6)
    p.step(_i32([-1, 0, 0]), _i32([0, 5, 5]), _i32([0, 0, 0, 0]), _i32([9, 4, 4]), _i32([-1] * 6))
    for got, want in zip(p.outputs(), ([-1] * 6, [0] * 6, [-1] * 6, [-1] * 3, [0] * 4)):
        np.testing.assert_array_equal(got, want)
    release()


def test_prefix_plan_positions_at_the_end_of_the_type():
    p = Prefix(2, 2)
    p.step(_i32([-1, 0]), _i32([0, 2 ** 31 - 1]), _i32([0, 0, 2]), _i32([2 ** 31 - 1, 5]), _i32([0, 7]))
    assert list(host(p.pos)) == [2 ** 31 - 1] * 2 and list(host(p.shared)) == [2 ** 31 - 1] * 2
    release()


# ------------------------------------------------------------ q, k, v in one pass

def _qkv(c, q, k, v, gains, eps, pos, cos, sin, slots, n_q, q_out=None):
    t = torch()
    if q_out is None:
        q_out = t.full((q.shape[0], n_q * c.hd), 9.0, dtype=t.float16, device="cuda")
    call("bx_qkv_append_q8_f16", ptr(q), q.stride(0), ptr(k), k.stride(0), ptr(v), v.stride(0), q.shape[0], n_q, c.n_kv,
         c.hd, ptr(gains[0]), ptr(gains[1]), eps, ptr(pos), ptr(cos), ptr(sin), cos.shape[0], ptr(slots), *c.args(),
         ptr(q_out), q_out.stride(0), stream())
    return q_out


def _close(got, want, scale):
    """One rounding to FP16 (half a step, 2^-11 relative, 2^-25 among subnormals), and FP32
    arithmetic before it: a sum of up to 256 squares, a root, a quotient, two products and a sum of
    products of size `scale`, below 2^-18 of that."""
    err = np.abs(got.astype(np.float64) - want)
    return (err <= 2.0 ** -11 * np.abs(want) + 2.0 ** -18 * scale + 2.0 ** -24).all()


@pytest.mark.parametrize("n_q,n_kv,hd,page", [(2, 1, 64, 16), (16, 8, 128, 64), (5, 5, 128, 16), (9, 3, 256, 32),
                                            (24, 8, 64, 128), (4, 2, 256, 128), (33, 1, 64, 64)])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("shape", ["step", "mixed", "prompts"])
def test_qkv_append(n_q, n_kv, hd, page, norm, shape):
    """Single rows, runs of every length at every place of a page, prompts of more than 2,048 rows."""
    rng = np.random.default_rng(n_q + hd + page + norm)
    t = torch()
    n_pages = {"step": 9, "mixed": 20, "prompts": 2400 // page + 30}[shape]
    want = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    c = Cache(want)
    slots = []
    for pg in rng.permutation(n_pages):
        off = int(rng.integers(0, page))
        n = {"step": 1, "mixed": int(rng.integers(1, page - off + 1)), "prompts": page - off if rng.random() < 0.3 else page}[shape]
        off = 0 if n == page else off
        slots += list(pg * page + off + np.arange(n))
        if rng.random() < 0.2:
            slots += [-1]
        if rng.random() < 0.1:
            slots += [n_pages * page + 3]
    slots = np.array(slots, np.int64)
    rows = slots.size
    cos, sin = px.tables(5000, hd)
    pos = rng.integers(0, 5000, rows).astype(np.int32)
    off_table = rng.random(rows) < 0.05
    pos[off_table] = rng.choice([-1, 5000, 2 ** 31 - 1, -2 ** 31], int(off_table.sum()))
    size = rng.choice([0.0, 1e-3, 1.0, 30.0], (rows, 1, 1), p=[0.1, 0.2, 0.5, 0.2])
    # q, k and v side by side, as one projection leaves them, at an odd distance and address
    wide = np.zeros((rows, (n_q + 2 * n_kv) * hd + 5), np.float16)
    x = (rng.standard_normal((rows, n_q + 2 * n_kv, hd)) * size).astype(np.float16)
    wide[:, 3:-2] = x.reshape(rows, -1)
    d = _half(wide)
    a, b = 3 + n_q * hd, 3 + (n_q + n_kv) * hd
    gain = [(1 + 0.4 * rng.standard_normal(hd)).astype(np.float16) for _ in range(2)] if norm else [None, None]
    gd = [None if g is None else _half(g.reshape(1, -1)) for g in gain]
    eps = 1e-6
    print(f"[qkv] {n_q}/{n_kv} heads of {hd}, page {page}, rows {rows}", flush=True)
    out = _qkv(c, d[:, 3:a], d[:, a:b], d[:, b:b + n_kv * hd], gd, eps, dev(pos), dev(cos), dev(sin), dev(slots), n_q)
    got = host(out).reshape(rows, n_q, hd)
    at = np.where(off_table, 0, pos)
    exact = px.norm_rope(x[:, :n_q], gain[0], eps, at, cos, sin)
    scale = np.abs(exact).max(-1, keepdims=True) * 2
    assert _close(got[~off_table], exact[~off_table], scale[~off_table])
    assert (got[off_table] == 9.0).all()
    # rows of K as FP16, from the same kernel's q heads; then everything bit for bit
    spare = Cache(pu.empty_cache(1, n_kv, page, hd))
    k16 = host(_qkv(spare, d[:, a:b], d[:, a:b], d[:, a:b], [gd[1], gd[1]], eps, dev(pos), dev(cos), dev(sin),
                    dev(np.full(rows, -1, np.int64)), n_kv)).reshape(rows, n_kv, hd)
    k_exact = px.norm_rope(x[:, n_q:n_q + n_kv], gain[1], eps, at, cos, sin)
    assert _close(k16[~off_table], k_exact[~off_table], 2 * np.abs(k_exact).max(-1, keepdims=True)[~off_table])
    k16 = np.where(off_table[:, None, None], np.float16(0), k16)
    pu.append(want, k16, x[:, n_q + n_kv:], slots)
    have = c.host()
    live = slots[(slots >= 0) & (slots < n_pages * page)]
    np.testing.assert_array_equal(have["ks"], want["ks"])
    np.testing.assert_array_equal(have["vs"], want["vs"])
    first = {}
    for s in live:
        first[s // page] = max(first.get(s // page, 0), int(s % page) + 1)
    for pg, n in first.items():
        np.testing.assert_array_equal(have["kc"][pg][:, :n], want["kc"][pg][:, :n])
        np.testing.assert_array_equal(have["vc"][pg][:, :, :n], want["vc"][pg][:, :, :n])
    release()


@pytest.mark.parametrize("hd,n_q,n_kv", [(64, 6, 2), (128, 16, 8), (256, 3, 1)])
def test_qkv_append_beside_the_separate_operators(hd, n_q, n_kv):
    """Near what bx_rms_norm, bx_rope_rows_f16 and bx_kv_append_q8_f16 give in turn, which round
    the normed values to FP16 as well; q in place."""
    rng = np.random.default_rng(hd)
    t = torch()
    rows, page = 70, 32
    cos, sin = (dev(x) for x in px.tables(200, hd))
    pos, slots = _i32(rng.integers(0, 200, rows)), dev(np.arange(7, 7 + rows).astype(np.int64))
    x = [_f16(rng, rows, h, hd, scale=2.0) for h in (n_q, n_kv, n_kv)]
    q, k, v = (_half(y) for y in x)
    gains = [_half((1 + 0.3 * rng.standard_normal((1, hd))).astype(np.float16)) for _ in range(2)]
    sep, one = (Cache(pu.empty_cache(4, n_kv, page, hd)) for _ in range(2))
    qn, kn = t.empty_like(q), t.empty_like(k)
    for src, g, dst, h in ((q, gains[0], qn, n_q), (k, gains[1], kn, n_kv)):
        call("bx_rms_norm", ptr(src), 0, ptr(g), 1e-6, ptr(dst), rows * h, hd, stream())
        call("bx_rope_rows_f16", ptr(dst), ptr(dst), rows, hd, h, ptr(pos), ptr(cos), ptr(sin), 200, stream())
    sep.append(kn, v, slots)
    _qkv(one, q, k, v, gains, 1e-6, pos, cos, sin, slots, n_q, q_out=q)
    a, b = (host(y).astype(np.float64).reshape(rows, n_q, hd) for y in (q, qn))
    # the pair's other element was rounded too: a step of 2^-10 of the larger of the two
    pair = np.abs(b).reshape(rows, n_q, -1, 2).max(-1).repeat(2, -1)
    assert (np.abs(a - b) <= 2.0 ** -10 * 2 * pair + 2.0 ** -23).all()
    (ka, va), (kb, vb) = one.read(slots), sep.read(slots)
    np.testing.assert_array_equal(host(va), host(vb))
    ka, kb = (host(y).astype(np.float64).reshape(rows, n_kv, hd) for y in (ka, kb))
    step = host(sep.ks).max()
    assert (np.abs(ka - kb) <= 1.01 * step + 2.0 ** -9 * np.abs(kb)).all()
    release()


def test_qkv_append_nan_and_infinity():
    """A NaN or an infinity in a head makes that head's row NaN (after a norm) and with it its page and head."""
    rng = np.random.default_rng(3)
    n_q, n_kv, hd, page, rows = 2, 2, 64, 16, 4
    cos, sin = (dev(x) for x in px.tables(50, hd))
    x = [_f16(rng, rows, h, hd) for h in (n_q, n_kv, n_kv)]
    x[0][1, 0, 5], x[1][2, 1, 9], x[2][0, 0, 3] = np.nan, np.inf, -np.inf
    q, k, v = (_half(y) for y in x)
    gains = [_half(np.ones((1, hd), np.float16))] * 2
    c = Cache(pu.empty_cache(2, n_kv, page, hd))
    out = host(_qkv(c, q, k, v, gains, 1e-6, _i32([1, 2, 3, 4]), cos, sin, dev(np.array([0, 1, 2, 16], np.int64)), n_q))
    out = out.reshape(rows, n_q, hd)
    assert np.isnan(out[1, 0]).all() and np.isfinite(np.delete(out.reshape(-1, hd), 2, 0)).all()
    ks, vs = host(c.ks), host(c.vs)
    assert np.isnan(ks[0, 1]) and np.isfinite([ks[0, 0], ks[1, 0], ks[1, 1]]).all()
    assert np.isinf(vs[0, 0]) and np.isfinite([vs[0, 1], vs[1, 0], vs[1, 1]]).all()
    release()


# ----------------------------------------------------------------- attention

def _pool(rng, lens, page, n_kv, hd):
    table, n_pages = _tables(rng, [max(0, n) for n in lens], page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    cache["ks"] = (0.02 * rng.uniform(0.7, 1.4, cache["ks"].shape)).astype(np.float32)
    cache["vs"] = (0.02 * 2.0 ** -rng.choice([0, 0, 0, 1, 3, 9], cache["vs"].shape)).astype(np.float32)
    return table, cache


def _planned(parent, shared_lens, lens, news, rows):
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    pos = np.full(rows, -1, np.int32)
    for r, (n, m) in enumerate(zip(lens, news)):
        pos[starts[r]:starts[r + 1]] = np.arange(n - m, n)
    p = Prefix(len(lens), rows)
    p.step(*(_i32(x) for x in (parent, shared_lens, starts, lens, pos)))
    return starts, p


def _case(rng, lens, news, parent, shared_lens, n_q, n_kv, hd, page, window=0, pad=2, q_scale=1.0, **loose):
    table, cache = _pool(rng, lens, page, n_kv, hd)
    rows = int(sum(news)) + pad
    starts, p = _planned(parent, shared_lens, lens, news, rows)
    q = _f16(rng, rows, n_q, hd, scale=q_scale)
    c = Cache(cache)
    shape = dict(max_new=max(1, max(news)), max_len=max(1, max(lens)), max_groups=len(set(parent)),
                 max_shared=max(1, max(lens)))
    shape.update(loose)
    out = attend(c, _half(q), dev(starts), _i32(lens), dev(table), p, n_q, window=window, **shape)
    want, bound = px.attention(cache, q, starts, lens, table, parent, shared_lens, n_kv, window)
    got, n = host(out).astype(np.float64).reshape(rows, n_q, hd), int(starts[-1])
    assert np.isfinite(got).all()
    err = np.abs(got - want)[:n]
    print(f"[attention] worst error / bound {np.max(err / np.maximum(bound[:n], 1e-30)):.3f}", flush=True)
    assert (err <= bound[:n] + 2.0 ** -25).all()
    assert (got[n:] == 9.0).all()   # rows behind the last request
    release()


CASES = [  # lens, news, parent, shared_lens
    ([5, 1, 1], [0, 1, 1], [-1, 0, 0], [0, 5, 5]),                                        # a handful of keys
    ([700, 3, 90, 17, 64], [0, 1, 1, 1, 1], [-1, 0, 0, 0, 0], [0, 700, 700, 1, 333]),     # forks at several places
    ([130, 200, 1, 40, 9, 60], [0, 0, 1, 1, 1, 1], [-1, -1, 1, 0, 1, -1], [0, 0, 200, 128, 64, 50]),
    ([300, 40, 50, 80], [1, 2, 5, 30], [-1, 0, 0, 0], [0, 300, 257, 299]),                # a parent with rows of its own
    ([90, 120, 120, 7], [70, 120, 65, 1], [-1, 0, 0, 0], [0, 20, 63, 64]),                # chunks behind a prefix being written
    ([64, 2, 3, 4], [0, 1, 1, 1], [-1, 0, 1, 2], [0, 64, 2, 3]),                          # a parent's parent is not followed
    ([40, 3, 5], [0, 3, 5], [-1, 0, 0], [0, 40, 40]),                                     # no own key before the rows
]


@pytest.mark.parametrize("n_q,n_kv,hd,page", [(2, 2, 64, 16), (16, 8, 128, 64), (6, 2, 128, 16), (16, 1, 64, 128),
                                            (4, 1, 256, 32)])
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("window", [0, 1, 37, 150])
@pytest.mark.parametrize("path", ["walk", "tiles"])
def test_attention_prefix(n_q, n_kv, hd, page, case, window, path):
    """Tiles that walk the shared keys and then the own ones; tiles of shared keys that are joined with those of
    the own ones (a bound on the shared keys that allows for far more)."""
    lens, news, parent, shared_lens = CASES[case]
    rng = np.random.default_rng(case * 7 + window + hd)
    loose = {} if path == "walk" else dict(max_shared=1 << 22)
    _case(rng, lens, news, parent, shared_lens, n_q, n_kv, hd, page, window, **loose)


@pytest.mark.parametrize("n_q,n_kv,hd,page,prefixes,requests,longest", [
    (8, 2, 128, 64, 1, 70, 1500), (4, 4, 64, 16, 9, 40, 700), (32, 8, 64, 32, 3, 45, 300), (3, 1, 256, 128, 2, 100, 600),
    (16, 1, 128, 16, 1, 33, 2000), (5, 5, 128, 32, 40, 41, 130)])
@pytest.mark.parametrize("window", [0, 400])
@pytest.mark.parametrize("path", ["walk", "tiles"])
def test_attention_prefix_of_many_requests(n_q, n_kv, hd, page, prefixes, requests, longest, window, path):
    """Several tiles of 128 columns a group, groups of a few columns, keys over many workgroups."""
    rng = np.random.default_rng(requests + longest)
    lens = list(rng.integers(1, longest + 1, prefixes)) + list(rng.integers(1, 40, requests))
    news = [0] * prefixes + [1] * requests
    parent = [-1] * prefixes + list(rng.integers(-1, prefixes, requests))
    shared_lens = [0] * prefixes + [int(rng.integers(1, longest + 1)) for _ in range(requests)]
    loose = {} if path == "walk" else dict(max_shared=1 << 18)
    _case(rng, lens, news, parent, shared_lens, n_q, n_kv, hd, page, window, max_groups=prefixes + 1, **loose)


@pytest.mark.parametrize("n_q,n_kv,hd,page", [(8, 2, 128, 64), (6, 2, 64, 16), (4, 1, 256, 32)])
@pytest.mark.parametrize("window", [0, 250])
def test_attention_prefix_chunks_of_large_batches(n_q, n_kv, hd, page, window):
    """Own keys in tiles of 128 columns as well: bounds that allow for far more work."""
    rng = np.random.default_rng(hd + window)
    _case(rng, [300, 130, 64, 200, 40], [0, 50, 64, 1, 3], [-1, 0, 0, 0, -1], [0, 300, 129, 300, 0], n_q, n_kv, hd, page,
          window, max_new=400, max_len=1 << 21, max_groups=5, max_shared=1 << 21)


WIDE = [  # prefixes' lengths, requests, rows each, heads, kv heads, hd, page
    ([700], 65, 1, 8, 2, 128, 64), ([700], 64, 1, 8, 2, 64, 16), ([300, 1000], 88, 1, 6, 2, 128, 16), ([513, 64], 50, 3, 16, 4, 64, 128),
    ([90], 7, 40, 3, 3, 128, 32), ([2000], 33, 1, 16, 1, 128, 128), ([129], 260, 1, 1, 1, 64, 32)]


@pytest.mark.parametrize("case", range(len(WIDE)))
@pytest.mark.parametrize("window", [0, 77, 400])
def test_attention_prefix_wide_tiles(case, window):
    """Tiles of 256 columns, whole and with a half to 128 and less: a bound on the shared keys that
    allows for far more work; forks everywhere, a third from the first tile."""
    prefixes, requests, m, n_q, n_kv, hd, page = WIDE[case]
    rng = np.random.default_rng(case * 5 + window)
    k = len(prefixes)
    parent = [-1] * k + [int(i % k) for i in range(requests)]
    shared_lens = [0] * k + [int(rng.integers(1, 65)) if rng.random() < 0.3 else int(rng.integers(1, prefixes[p] + 1)) for p in parent[k:]]
    lens = prefixes + [int(rng.integers(m, m + 20)) for _ in range(requests)]
    # 2^25 pairs of a row's head and a shared key and more
    _case(rng, lens, [0] * k + [m] * requests, parent, shared_lens, n_q, n_kv, hd, page, window, max_groups=k,
          max_shared=(1 << 25) // (requests * m * n_q) + 1)


@pytest.mark.parametrize("hd,rows", [(64, 140), (128, 150)])
def test_attention_prefix_wide_tiles_long(hd, rows):
    """Many tiles of keys to a workgroup, more than its buffers hold."""
    rng = np.random.default_rng(rows)
    lens, parent = [14500] + [3] * rows, [-1] + [0] * rows
    shared_lens = [0] + [int(rng.choice([14500, 14399, 9000])) for _ in range(rows)]
    _case(rng, lens, [0] + [1] * rows, parent, shared_lens, 16, 1, hd, 64)


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_prefix_wide_tiles_of_odd_pages(hd):
    """Pages that are none and pages of NaN and infinite scales among those of a wide tile's keys."""
    rng = np.random.default_rng(hd)
    n_q, n_kv, page, requests = 4, 2, 16, 130
    lens, news = [320] + [2] * requests, [0] + [1] * requests
    parent = [-1] + [0] * requests
    shared_lens = [0] + [320 if i % 3 == 0 else 160 if i % 3 == 1 else 48 for i in range(requests)]
    table, cache = _pool(rng, lens, page, n_kv, hd)
    table[0, 2], table[0, 7] = -1, cache["ks"].shape[0] + 3
    cache["vs"][table[0, 12], 0], cache["vs"][table[0, 13], 1], cache["ks"][table[0, 14], 1] = np.inf, np.nan, np.nan
    starts, p = _planned(parent, shared_lens, lens, news, requests)
    q = _f16(rng, requests, n_q, hd)
    out = attend(Cache(cache), _half(q), dev(starts), _i32(lens), dev(table), p, n_q, 1, 2, 1, 1 << 20)
    got = host(out).astype(np.float64).reshape(requests, n_q, hd)
    clean = dict(cache, ks=np.nan_to_num(cache["ks"], nan=0.01), vs=np.nan_to_num(cache["vs"], nan=0.01, posinf=0.01))
    want, bound = px.attention(clean, q, starts, lens, table, parent, shared_lens, n_kv)
    for i in range(requests):
        if shared_lens[i + 1] == 320:   # sees the infinite V scale of head 0 and the NaNs of head 1
            assert not np.isfinite(got[i, :2]).all() and np.isnan(got[i, 2:]).all(), i
        else:
            assert (np.abs(got[i] - want[i]) <= bound[i] + 2.0 ** -25).all(), i
    release()


def test_attention_prefix_small_bounds():
    """max_len and max_shared below the true lengths only shape the launch."""
    rng = np.random.default_rng(5)
    _case(rng, [900, 300, 7], [0, 1, 1], [-1, 0, 0], [0, 900, 800], 8, 2, 128, 64, max_len=1, max_shared=1)


def test_attention_prefix_of_nobody():
    """No request shares any key: the bits of bx_attention_paged_q8_f16."""
    rng = np.random.default_rng(6)
    n_q, n_kv, hd, page, lens, news = 8, 2, 128, 32, [300, 20, 1], [1, 3, 1]
    table, cache = _pool(rng, lens, page, n_kv, hd)
    starts, p = _planned([-1] * 3, [0] * 3, lens, news, 7)
    q, c = _half(_f16(rng, 7, n_q, hd)), Cache(cache)
    b = c.attention(q, dev(starts), _i32(lens), dev(table), n_q, 3, 300)
    for max_shared in (1, 1 << 22):
        a = attend(c, q, dev(starts), _i32(lens), dev(table), p, n_q, 3, 300, 1, max_shared)
        np.testing.assert_array_equal(host(a).view(np.uint16), host(b).view(np.uint16))
    release()


@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("max_shared", [160, 1 << 22])
def test_attention_prefix_as_copies(window, max_shared):
    """A prefix of whole pages that every request's table names by itself gives the same to the bound."""
    rng = np.random.default_rng(7)
    n_q, n_kv, hd, page = 8, 2, 128, 16
    lens, news = [160, 33, 5, 48], [0, 1, 4, 1]
    parent, shared_lens = [-1, 0, 0, 0], [0, 160, 160, 160]
    table, cache = _pool(rng, lens, page, n_kv, hd)
    starts, p = _planned(parent, shared_lens, lens, news, 6)
    q, c = _f16(rng, 6, n_q, hd), Cache(cache)
    a = host(attend(c, _half(q), dev(starts), _i32(lens), dev(table), p, n_q, 4, 48, 1, max_shared, window)).astype(np.float64)
    wide = np.full((4, 15), -1, np.int32)
    wide[:, :10] = table[0, :10]
    wide[1:, 10:10 + table.shape[1] - 1] = table[1:, :5][:, :wide.shape[1] - 10]
    all_lens = [160] + [160 + n for n in lens[1:]]
    b = host(c.attention(_half(q), dev(starts), _i32(all_lens), dev(wide), n_q, 4, 208, window)).astype(np.float64)
    _, bound = px.attention(cache, q, starts, lens, table, parent, shared_lens, n_kv, window)
    assert (np.abs(a - b) <= 2 * bound.reshape(a.shape) + 2.0 ** -24).all()
    release()


@pytest.mark.parametrize("max_shared", [100, 1 << 22])
def test_attention_prefix_pages_that_are_none(max_shared):
    """Entries of the shared table that name no page hide their keys; all of them: the own keys alone."""
    rng = np.random.default_rng(8)
    n_q, n_kv, hd, page = 4, 2, 64, 16
    lens, news = [100, 20, 30, 64, 12], [0, 1, 1, 0, 1]
    parent, shared_lens = [-1, 0, 0, -1, 3], [0, 100, 50, 0, 64]
    table, cache = _pool(rng, lens, page, n_kv, hd)
    table[0, 1], table[0, 4], table[3, :] = -1, cache["ks"].shape[0], 2 ** 31 - 1
    starts, p = _planned(parent, shared_lens, lens, news, 3)
    q = _f16(rng, 3, n_q, hd)
    out = attend(Cache(cache), _half(q), dev(starts), _i32(lens), dev(table), p, n_q, 1, 30, 2, max_shared)
    want, bound = px.attention(cache, q, starts, lens, table, parent, shared_lens, n_kv)
    assert (np.abs(host(out).astype(np.float64).reshape(want.shape) - want) <= bound + 2.0 ** -25).all()
    release()


@pytest.mark.parametrize("max_shared", [64, 1 << 22])
def test_attention_prefix_nan_stays_where_it_is_seen(max_shared):
    """A page of NaN scale at the end of the prefix reaches only the rows that share it; one without
    own keys and without a seen shared one gives zeros."""
    rng = np.random.default_rng(9)
    n_q, n_kv, hd, page = 4, 2, 128, 16
    lens, news = [64, 3, 3, 3, 0], [0, 1, 1, 1, 1]
    parent, shared_lens = [-1, 0, 0, 0, 0], [0, 48, 64, 49, 16]
    table, cache = _pool(rng, lens, page, n_kv, hd)
    cache["ks"][table[0, 3]] = np.nan
    cache["vs"][table[0, 3]] = np.nan
    starts, p = _planned(parent, shared_lens, lens, news, 4)
    q = _f16(rng, 4, n_q, hd)
    # window 1: the last row's only position is its own, whose key does not exist
    for window in (0, 1):
        out = host(attend(Cache(cache), _half(q), dev(starts), _i32(lens), dev(table), p, n_q, 1, 3, 1, max_shared, window))
        out = out.astype(np.float64).reshape(4, n_q, hd)
        if window:
            assert np.isfinite(out).all()
            continue
        assert np.isnan(out[1]).all() and np.isnan(out[2]).all()
        clean = dict(cache, ks=np.nan_to_num(cache["ks"]), vs=np.nan_to_num(cache["vs"]))
        want, bound = px.attention(clean, q, starts, lens, table, parent, shared_lens, n_kv)
        for i in (0, 3):
            assert (np.abs(out[i] - want[i]) <= bound[i] + 2.0 ** -25).all()
    release()


@pytest.mark.parametrize("max_shared", [100, 1 << 22])
def test_attention_prefix_strided_rows_and_odd_addresses(max_shared):
    rng = np.random.default_rng(10)
    t = torch()
    n_q, n_kv, hd, page, lens, news = 8, 2, 128, 16, [100, 33, 60], [0, 1, 20]
    parent, shared_lens = [-1, 0, 0], [0, 100, 70]
    table, cache = _pool(rng, lens, page, n_kv, hd)
    starts, p = _planned(parent, shared_lens, lens, news, 21)
    w = n_q * hd
    wide = rng.standard_normal((21, w + 77)).astype(np.float16)
    out = t.full((21, w + 31), 9.0, dtype=t.float16, device="cuda")
    attend(Cache(cache), _half(wide)[:, 3:3 + w], dev(starts), _i32(lens), dev(table), p, n_q, 20, 60, 1, max_shared, out=out[:, 5:5 + w])
    want, bound = px.attention(cache, wide[:, 3:3 + w].reshape(21, n_q, hd), starts, lens, table, parent, shared_lens, n_kv)
    got = host(out).astype(np.float64)
    assert (np.abs(got[:, 5:5 + w].reshape(21, n_q, hd) - want) <= bound + 2.0 ** -25).all()
    assert (got[:, :5] == 9).all() and (got[:, 5 + w:] == 9).all()
    release()


def test_attention_prefix_one_workspace_for_many_shapes_and_repeats():
    """Shapes in turn on one workspace, twice each with the same bits, counters back at zero."""
    rng = np.random.default_rng(11)
    t = torch()
    n_q, n_kv, hd, page = 8, 2, 64, 16
    shapes = [([3000, 500, 9], [0, 1, 1], [-1, 0, 0], [0, 3000, 2900]), ([64] + [40] * 60, [0] + [1] * 60, [-1] + [0] * 60, [0] + [50] * 60),
              ([700, 300, 90], [0, 100, 1], [-1, 0, 0], [0, 700, 1])]
    calls, sizes = [], []
    for lens, news, parent, shared_lens in shapes:
        table, cache = _pool(rng, lens, page, n_kv, hd)
        rows = sum(news)
        starts, p = _planned(parent, shared_lens, lens, news, rows)
        q = _f16(rng, rows, n_q, hd)
        args = (Cache(cache), _half(q), dev(starts), _i32(lens), dev(table), p, n_q, max(news), max(lens), 1, lens[0])
        sizes.append(int(hip().bx_attention_prefix_q8_workspace_bytes(rows, len(lens), n_q, n_kv, hd, *args[7:])))
        calls.append((args, px.attention(cache, q, starts, lens, table, parent, shared_lens, n_kv)))
    ws, seen = t.zeros(max(sizes), dtype=t.uint8, device="cuda"), {}
    for turn in range(4):
        for i in rng.permutation(len(calls)):
            args, (want, bound) = calls[i]
            got = host(attend(*args, ws=ws))
            assert (np.abs(got.astype(np.float64).reshape(want.shape) - want) <= bound + 2.0 ** -25).all(), (turn, i)
            np.testing.assert_array_equal(got, seen.setdefault(i, got))
    assert not host(ws)[:512 * 1024].any()
    release()


@pytest.mark.parametrize("max_shared", [100, 1 << 22])
def test_attention_prefix_more_rows_than_keys(max_shared):
    """Rows before the first own key attend all shared keys, the others the last `window` of theirs."""
    rng = np.random.default_rng(17)
    n_q, n_kv, hd, page, window = 8, 2, 128, 16, 37
    lens, news, parent, shared_lens = [100, 2, 0], [0, 5, 2], [-1, 0, 0], [0, 100, 90]
    table, cache = _pool(rng, lens, page, n_kv, hd)
    starts, p = _planned(parent, shared_lens, lens, news, 7)
    q = _f16(rng, 7, n_q, hd)
    got = host(attend(Cache(cache), _half(q), dev(starts), _i32(lens), dev(table), p, n_q, 5, 100, 1, max_shared, window=window))
    before = np.array([True, True, True, False, False, True, True])
    whole, last = (px.attention(cache, q, starts, lens, table, parent, shared_lens, n_kv, w) for w in (0, window))
    want, bound = (np.where(before[:, None, None], x, y) for x, y in zip(whole, last))
    assert (np.abs(got.astype(np.float64).reshape(want.shape) - want) <= bound + 2.0 ** -25).all()
    release()


def test_attention_prefix_captured_calls_share_a_workspace():
    """Graphs of calls of several kinds on one workspace, replayed in turn with eager calls between."""
    t = torch()
    rng = np.random.default_rng(19)
    n_q, n_kv, hd, page = 8, 2, 128, 64
    shapes = [([700, 300, 9], [0, 1, 1], [-1, 0, 0], [0, 700, 650]),                       # few rows
              ([900] + [60] * 70, [0] + [4] * 70, [-1] + [0] * 70, [0] + [900] * 70),       # tiles of 128 columns
              ([9000, 400, 300], [0, 400, 300], [-1, 0, 0], [0, 9000, 8000])]               # tiles of 256
    calls, sizes = [], []
    for lens, news, parent, shared_lens in shapes:
        table, cache = _pool(rng, lens, page, n_kv, hd)
        rows = sum(news)
        starts, p = _planned(parent, shared_lens, lens, news, rows)
        out = t.zeros((rows, n_q * hd), dtype=t.float16, device="cuda")
        calls.append(((Cache(cache), _half(_f16(rng, rows, n_q, hd)), dev(starts), _i32(lens), dev(table), p, n_q, max(news),
                       max(lens), 1, lens[0]), out))
        sizes.append(int(hip().bx_attention_prefix_q8_workspace_bytes(rows, len(lens), n_q, n_kv, hd, max(news), max(lens), 1,
                                                                      lens[0])))
    ws = t.zeros(max(sizes), dtype=t.uint8, device="cuda")
    alone, graphs = [], []
    for args, out in calls:
        alone.append(host(attend(*args, out=out, ws=ws)))
        graphs.append(t.cuda.CUDAGraph())
        with t.cuda.graph(graphs[-1]):
            attend(*args, out=out, ws=ws)
    for turn in range(6):
        for i in rng.permutation(len(calls)):
            calls[i][1].zero_()
            graphs[i].replay()
            k = int(rng.integers(len(calls)))
            got = host(calls[i][1])
            np.testing.assert_array_equal(got, alone[i], err_msg=f"turn {turn}, call {i}")
            attend(*calls[k][0], out=calls[k][1], ws=ws)
            np.testing.assert_array_equal(host(calls[k][1]), alone[k])
    release()


def test_attention_prefix_pool_beyond_32_bits():
    """Shared pages whose codes lie more than 2^32 bytes into the pool."""
    t = torch()
    rng = np.random.default_rng(12)
    n_q, n_kv, hd, page, lens = 4, 2, 128, 64, [200, 70]
    n_pages = (5 << 30) // (n_kv * page * hd)
    small = pu.empty_cache(8, n_kv, page, hd, rng)
    c = Cache(small)
    ids = np.array([n_pages - 1 - 3 * i for i in range(8)])
    for name in ("kc", "vc", "ks", "vs"):
        big = t.empty((n_pages,) + small[name].shape[1:], dtype=getattr(c, name).dtype, device="cuda")
        big[dev(ids)] = getattr(c, name)
        setattr(c, name, big)
    c.n_pages = n_pages
    table = np.array([[2, 3, 4, 5], [0, 1, -1, -1]], np.int32)
    far = np.where(table >= 0, ids[table], -1).astype(np.int32)
    starts, p = _planned([-1, 0], [0, 190], lens, [0, 1], 1)
    q = _f16(rng, 1, n_q, hd)
    want, bound = px.attention(small, q, starts, lens, table, [-1, 0], [0, 190], n_kv)
    for max_shared in (190, 1 << 22):
        out = attend(c, _half(q), dev(starts), _i32(lens), dev(far), p, n_q, 1, 70, 1, max_shared)
        assert (np.abs(host(out).astype(np.float64).reshape(want.shape) - want) <= bound + 2.0 ** -25).all()
    del c
    release()
    t.cuda.empty_cache()


# ------------------------------------------------- a step as a serving loop runs it

@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("max_shared", [None, 1 << 20])
@pytest.mark.parametrize("n_q,n_kv,hd,page,news", [(4, 2, 64, 16, [0, 1, 1, 9]), (8, 2, 128, 64, [1]), (4, 1, 256, 32, [1, 30])])
def test_serving_loop_with_prefixes(n_q, n_kv, hd, page, news, graph, max_shared):
    """Plan, prefix plan, q / k / v and attention of a layer, step after step: two prefixes are written
    in chunks, requests join, fork elsewhere, end and start over; also captured once and replayed."""
    t = torch()
    rng = np.random.default_rng(hd + graph)
    n_req, width = 9, -(-260 // page)
    n_pages, rows = n_req * width, n_req * max(max(news), 40) + 3
    table = np.full((n_req, width), -1, np.int32)
    ring, ends = rng.permutation(n_pages).astype(np.int32), np.array([0, n_pages], np.int64)
    past = np.zeros(n_req, np.int32)
    wanted = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    d, c, p = Plan(n_req, page, n_pages, width, rows, ring, ends, table, past), Cache(wanted), Prefix(n_req, rows)
    cos, sin = px.tables(1000, hd)
    gain = [(1 + 0.3 * rng.standard_normal(hd)).astype(np.float16) for _ in range(2)]
    cosd, sind, gd = dev(cos), dev(sin), [_half(g.reshape(1, -1)) for g in gain]
    x = t.empty((rows, (n_q + 2 * n_kv) * hd), dtype=t.float16, device="cuda")
    q_rot = t.empty((rows, n_q * hd), dtype=t.float16, device="cuda")
    out = t.empty_like(q_rot)
    delta, parent_d, shared_d = (t.zeros(n_req, dtype=t.int32, device="cuda") for _ in range(3))
    max_new, max_len = max(max(news), 40), width * page
    max_shared = max_shared or max_len
    nb = int(hip().bx_attention_prefix_q8_workspace_bytes(rows, n_req, n_q, n_kv, hd, max_new, max_len, 3, max_shared))
    ws = t.zeros(nb, dtype=t.uint8, device="cuda")

    def step():
        d.step(delta)
        p.step(parent_d, shared_d, d.starts, d.past, d.pos)
        a, b = n_q * hd, (n_q + n_kv) * hd
        _qkv(c, x[:, :a], x[:, a:b], x[:, b:], gd, 1e-6, p.pos, cosd, sind, d.slots, n_q, q_out=q_rot)
        attend(c, q_rot, d.starts, d.past, d.table, p, n_q, max_new, max_len, 3, max_shared, out=out, ws=ws)

    captured = None
    for i in range(9):
        change = rng.choice(news, n_req).astype(np.int32)
        change[:2] = 40 if i < 3 else 0
        change = np.where(past + change > 250, -past, change).astype(np.int32)
        parent = np.array([-1, -1] + [int(rng.integers(-1, 3)) for _ in range(n_req - 2)], np.int32)
        shared_lens = np.where(parent >= 0, rng.integers(1, 140, n_req), 0).astype(np.int32)
        raw = _f16(rng, rows, n_q + 2 * n_kv, hd, scale=1.5)
        x.copy_(_half(raw))
        for dst, src in ((delta, change), (parent_d, parent), (shared_d, shared_lens)):
            dst.copy_(dev(src))
        out.fill_(9.0)
        t.cuda.synchronize()
        print(f"[serve] step {i}", flush=True)
        if graph and i == 1:
            captured = t.cuda.CUDAGraph()
            with t.cuda.graph(captured):
                step()
        captured.replay() if captured is not None else step()
        lens, starts, slots, pos, ends, status = pu.plan(past, change, page, n_pages, table, ring, ends, rows)
        assert status == 0 == int(host(d.status)[0])
        plan = px.plan(parent, shared_lens, starts, lens, pos)
        for got, want in zip(p.outputs(), plan):
            np.testing.assert_array_equal(got, want)
        n = int(starts[-1])
        exact = px.norm_rope(raw[:n, :n_q], gain[0], 1e-6, plan[0][:n], cos, sin)
        qr = host(q_rot).reshape(rows, n_q, hd)
        assert _close(qr[:n], exact, 2 * np.abs(exact).max(-1, keepdims=True))
        # K in FP16 may round the other way where the exact value is near a border, so the cache is taken
        # as the device holds it: each value within half a code and those roundings of the exact row
        have = c.host()
        at = slots[:n]
        kv, vv = pu.values(have, np.arange(n_pages))
        k_exact = px.norm_rope(raw[:n, n_q:n_q + n_kv], gain[1], 1e-6, plan[0][:n], cos, sin)
        for got, want, sc in ((kv[at], k_exact, have["ks"]), (vv[at], raw[:n, n_q + n_kv:].astype(np.float64), have["vs"])):
            assert (np.abs(got - want) <= 0.5001 * sc[at // page][..., None] + 2.0 ** -10 * np.abs(want).max(-1, keepdims=True)).all()
        want, bound = px.attention(have, qr, starts, lens, table, parent, shared_lens, n_kv)
        got = host(out).astype(np.float64).reshape(rows, n_q, hd)
        assert (np.abs(got - want)[:n] <= bound[:n] + 2.0 ** -25).all()
        assert (got[n:] == 9.0).all()
        past = lens
    release()


def test_two_streams_with_their_own_workspaces():
    """Two pools served at the same time on two streams give what they give alone."""
    t = torch()
    rng = np.random.default_rng(13)
    n_q, n_kv, hd, page = 8, 2, 128, 64
    lens, news, parent, shared_lens = [3000, 700, 100], [0, 1, 1], [-1, 0, 0], [0, 3000, 2000]
    sides = []
    for _ in range(2):
        table, cache = _pool(rng, lens, page, n_kv, hd)
        starts, p = _planned(parent, shared_lens, lens, news, 2)
        sides.append((Cache(cache), _half(_f16(rng, 2, n_q, hd)), dev(starts), _i32(lens), dev(table), p, n_q, 1, 700, 1, 3000))
    alone = [host(attend(*s)) for s in sides]
    n = int(hip().bx_attention_prefix_q8_workspace_bytes(2, 3, n_q, n_kv, hd, 1, 700, 1, 3000))
    spaces = [t.zeros(n, dtype=t.uint8, device="cuda") for _ in range(2)]
    outs = [t.zeros((2, n_q * hd), dtype=t.float16, device="cuda") for _ in range(2)]
    streams = [t.cuda.Stream() for _ in range(2)]
    t.cuda.synchronize()
    for _ in range(20):
        for s, ws, out, st in zip(sides, spaces, outs, streams):
            with t.cuda.stream(st):
                attend(*s, out=out, ws=ws)
    t.cuda.synchronize()
    for out, want in zip(outs, alone):
        np.testing.assert_array_equal(host(out), want)
    release()
