"""bx_sample_rows_f16 against a plain 64-bit sampler (paged_util.sample): the same
id for every row, ties and cuts included.  The kernel decides in FP64, so a row
may differ only where the draw or a cut lies within 1e-12 of the mass from another
answer (summation order); the inputs here stay clear of that, which is asserted."""
from __future__ import annotations

import numpy as np
import pytest

import paged_util as pu
from gpu_util import call, dev, host, ptr, release, stream, torch

pytestmark = pytest.mark.gpu


def _run(x, t, k, p, m, u, stride=None, offset=0):
    rows, V = x.shape
    stride = stride or V
    buf = np.zeros(rows * stride + offset + 8, np.float16)
    for i in range(rows):
        buf[offset + i * stride:offset + i * stride + V] = x[i]
    d = dev(buf.view(np.uint16))
    out = torch().full((rows + 1,), -9, dtype=torch().int32, device="cuda")
    opt = lambda a, ty: None if a is None else ptr(dev(np.asarray(a, ty)))
    import ctypes as C
    call("bx_sample_rows_f16", C.c_void_p(d.data_ptr() + 2 * offset), stride, rows, V, ptr(dev(np.asarray(t, np.float32))),
         opt(k, np.int32), opt(p, np.float32), opt(m, np.float32), ptr(dev(np.asarray(u, np.float64))), ptr(out), stream())
    got = host(out)
    assert got[rows] == -9
    release()
    return got[:rows]


def _check(x, t, k, p, m, u, **kw):
    rows = x.shape[0]
    got = _run(x, t, k, p, m, u, **kw)
    z = np.zeros(rows)
    for i in range(rows):
        want, near = pu.sample(x[i], np.float32(t[i]), (k if k is not None else z)[i],
                               np.float32((p if p is not None else z + 1)[i]), np.float32((m if m is not None else z)[i]), u[i])
        assert got[i] == want or near < 1e-12, (i, got[i], want, t[i], near)
        assert near > 0 or got[i] == want


def _settings(rng, rows):
    return (rng.choice([0.0, 0.3, 0.7, 1.0, 1.7], rows), rng.choice([0, 1, 2, 40, 3000], rows),
            rng.choice([1.0, 0.95, 0.5, 0.01, 0.0], rows), rng.choice([0.0, 0.05, 0.3, 1.0], rows), rng.random(rows))


@pytest.mark.parametrize("V", [1, 2, 7, 8, 63, 1000, 8191, 65535, 65536, 65537, 151936, 200003])
def test_rows_match_the_plain_sampler(V):
    rng = np.random.default_rng(V)
    rows = 24 if V < 100000 else 12
    x = (rng.standard_normal((rows, V)) * rng.choice([0.01, 1.0, 4.0], (rows, 1))).astype(np.float16)
    print(f"[sample_rows] V={V}", flush=True)
    _check(x, *_settings(rng, rows))


@pytest.mark.parametrize("V", [1000, 151936])
def test_each_cut_alone_and_none(V):
    rng = np.random.default_rng(V + 1)
    rows = 8
    x = (rng.standard_normal((rows, V)) * 2).astype(np.float16)
    t, u = np.full(rows, 0.9), rng.random(rows)
    _check(x, t, None, None, None, u)
    _check(x, t, np.full(rows, 17), None, None, u)
    _check(x, t, None, np.full(rows, 0.8), None, u)
    _check(x, t, None, None, np.full(rows, 0.02), u)


@pytest.mark.parametrize("V", [4096, 151936])
def test_ties(V):
    """Forty levels over the whole vocabulary: every cut and draw ends inside a group of
    equal logits; whole rows of one value (more than 65,535 of them in the larger)."""
    rng = np.random.default_rng(V + 2)
    rows = 24
    levels = rng.choice(np.linspace(-4, 6, 200).astype(np.float16), 40, replace=False)
    x = levels[rng.integers(0, 40, (rows, V))]
    x[3] = np.float16(1.5)
    x[4] = np.float16(-60000)
    x[5, 10:] = np.float16(0.0)
    x[5, 500:] = np.float16(-0.0)     # one level with +0
    t, k, p, m, u = _settings(rng, rows)
    t[3:6], k[3:6], p[3:6], m[3:6] = 1.0, 0, 1.0, 0.0
    _check(x, t, k, p, m, u)


@pytest.mark.parametrize("V", [1000, 151936])
def test_masked_vocabularies(V):
    """Most ids at -infinity or at the type's lowest value, one id left, none left, NaN, +infinity."""
    rng = np.random.default_rng(V + 3)
    rows = 14
    x = (rng.standard_normal((rows, V)) * 2).astype(np.float16)
    keep = rng.random((rows, V)) < 30 / V
    keep[:, V // 2] = True
    x[:4] = np.where(keep[:4], x[:4], np.float16(-np.inf))
    x[4:8] = np.where(keep[4:8], x[4:8], np.finfo(np.float16).min)
    x[8] = -np.inf
    x[8, V - 1] = -3
    x[9] = -np.inf                                  # nothing left: every id alike
    x[10, ::3] = np.nan
    x[11, 5] = x[11, V - 2] = np.inf
    x[12].view(np.uint16)[::5] = 0x7c01             # a signalling NaN, and a negative one
    x[12].view(np.uint16)[1::5] = 0xfe01
    x[13] = np.nan
    t, k, p, m, u = _settings(rng, rows)
    for row in (0, 4, 8, 9, 10, 11, 12, 13):
        t[row] = max(t[row], 0.5)
    _check(x, t, k, p, m, u)
    _check(x, np.where(np.arange(rows) % 2, 1.0, 0.0), None, None, None, u)


def test_settings_at_their_ends():
    rng = np.random.default_rng(5)
    V = 5000
    x = np.tile((rng.standard_normal(V) * 3).astype(np.float16), (10, 1))
    inf, nan = np.inf, np.nan
    t = [1e-30, 1e30, inf, 1.0, 1.0, 1.0, -1.0, nan, 1.0, 1.0]
    k = [0, 0, 0, -5, V, 10 ** 9, 0, 0, 1, 0]
    p = [1.0, 1.0, 1.0, 2.0, 1.0, 1.0, 0.5, 0.5, 1.0, -1.0]
    m = [0.0, 0.0, 0.0, -1.0, 2.0, 0.0, 0.5, 0.5, 0.0, 0.0]
    u = [0.5, 0.5, 0.25, 0.0, 0.99, np.nextafter(1.0, 0.0), 0.5, 0.5, 0.9, 0.9]
    _check(x, np.array(t), np.array(k), np.array(p), np.array(m), np.array(u))


def test_rows_apart_and_odd_addresses():
    rng = np.random.default_rng(6)
    x = (rng.standard_normal((9, 3001)) * 2).astype(np.float16)
    args = _settings(rng, 9)
    for stride, offset in ((3001, 1), (3007, 3), (4096, 0), (3002, 7)):
        _check(x, *args, stride=stride, offset=offset)


def test_many_rows_and_replays():
    """More rows than compute units, captured once and replayed with other numbers."""
    t = torch()
    rng = np.random.default_rng(7)
    rows, V = 600, 2000
    x = (rng.standard_normal((rows, V)) * 2).astype(np.float16)
    tt, k, p, m, u = _settings(rng, rows)
    _check(x, tt, k, p, m, u)
    xd = dev(x.view(np.uint16))
    par = [dev(np.asarray(a, ty)) for a, ty in ((tt, np.float32), (k, np.int32), (p, np.float32), (m, np.float32))]
    ud, out = t.zeros(rows, dtype=t.float64, device="cuda"), t.zeros(rows, dtype=t.int32, device="cuda")

    def run():
        call("bx_sample_rows_f16", ptr(xd), V, rows, V, *map(ptr, par), ptr(ud), ptr(out), stream())

    run()
    t.cuda.synchronize()
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g):
        run()
    for _ in range(4):
        u = rng.random(rows)
        ud.copy_(dev(u))
        g.replay()
        got = host(out).copy()
        want = [pu.sample(x[i], np.float32(tt[i]), k[i], np.float32(p[i]), np.float32(m[i]), u[i])[0] for i in range(0, rows, 7)]
        np.testing.assert_array_equal(got[::7], want)
        run()
        np.testing.assert_array_equal(host(out), got)
    release()


def test_a_draw_between_two_levels_far_apart():
    """Empty keys between the levels of a row: their running mass is that of the level before them
    to the last bit, so that a draw next to it takes one of the row's ids."""
    x = np.array([[7.76171875, 7.51171875, 7.26171875, 6.76171875]], np.float16)
    got = _run(x, [0.360554575920105], None, None, None, [0.9655433869199928])
    assert got[0] in (2, 3)


def test_draws_around_every_border():
    """u at each border between two ids of small rows, and up to 48 steps of FP64 to either
    side: one of the two ids beside the border."""
    rng = np.random.default_rng(8)
    x, t, u, ids = [], [], [], []
    for _ in range(120):
        row = (rng.integers(-400, 400, 5) / 32).astype(np.float16)
        temp = np.float32(rng.uniform(0.5, 6))
        order = np.argsort(-row.astype(np.float64), kind="stable")
        run = np.cumsum(np.exp((row[order].astype(np.float64) - float(row.max())) / float(temp)))
        for j in range(4):
            border = run[j] / run[-1]
            if border > 1 - 2.0 ** -40:
                continue
            for k in range(-48, 49):
                x.append(row)
                t.append(temp)
                u.append(border + k * np.spacing(border))
                ids.append((order[j], order[j + 1]))
    got = _run(np.array(x), t, None, None, None, u)
    ids = np.array(ids)
    bad = np.nonzero((got != ids[:, 0]) & (got != ids[:, 1]))[0]
    assert bad.size == 0, [(x[i].tolist(), float(t[i]), u[i], int(got[i])) for i in bad[:4]]


@pytest.mark.parametrize("V", [1000, 151936])
def test_rows_match_the_one_row_sampler_and_the_oracle(V):
    """The settings of bx_sample_f16 (no min-p) give its ids, and those of the oracle's sample_token,
    on the same logits and draws.  Both of these sum in FP32: an id may differ where the draw lies
    within 1e-5 of the kept mass from the end of the id's interval, and among equal logits."""
    import ctypes as C

    import oracle
    from gpu_util import empty, hip
    rng = np.random.default_rng(V + 9)
    cases = [(1.0, 0, 1.0), (0.7, 50, 1.0), (1.0, 0, 0.9), (1.3, 40, 0.8), (0.5, 5, 0.5), (1.0, 0, 0.01), (2.0, 300, 0.95)]
    t, k, p = (np.array(c) for c in zip(*(cases * 6)))
    rows = t.size
    # the ids that a cut falls among are all different: a permutation of FP16 values
    x = np.empty((rows, V), np.float16)
    for i in range(rows):
        top = rng.choice(V, 600, replace=False)
        x[i] = rng.uniform(-9, 0.9, V).astype(np.float16)
        x[i, top] = rng.choice(np.arange(0x3C00, 0x4A00, dtype=np.uint16), 600, replace=False).view(np.float16)   # [1, 12)
    u = rng.random(rows)
    got = _run(x, t, k, p, None, u)
    ws = empty(int(hip().bx_sample_workspace_bytes(V)))
    one = torch().full((rows,), -9, dtype=torch().int32, device="cuda")
    xd = dev(x.view(np.uint16))
    for i in range(rows):
        call("bx_sample_f16", C.c_void_p(xd.data_ptr() + 2 * V * i), V, C.c_float(t[i]), int(k[i]), C.c_float(p[i]),
             C.c_double(u[i]), C.c_void_p(one.data_ptr() + 4 * i), ptr(ws), stream())
    one = host(one)
    near = 0
    for i in range(rows):
        want, margin = oracle.sample_token(x[i].astype(np.float32), float(np.float32(t[i])), int(k[i]), float(np.float32(p[i])), u[i])
        for other in (want, int(one[i])):
            if x[i, got[i]] != x[i, other]:
                assert margin < 1e-5, (i, got[i], other, margin, t[i], k[i], p[i])
                near += 1
    assert near <= 4
    release()
