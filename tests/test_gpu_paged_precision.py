"""How exact the attention over the paged 8-bit cache is where its tiles mix things that
a row's result must not depend on: pages of very different V scales, rows that
see different pages, strong query channels, splits of a long context.  The reference is the
softmax in 64 bits over the cache's values."""
from __future__ import annotations

import math

import numpy as np
import pytest

import paged_util as pu
from gpu_util import dev, host, release, torch
from test_gpu_paged import Cache, _tables

pytestmark = pytest.mark.gpu


def _attend(cache, q, starts, lens, table, n_kv, window=0, pair=True):
    """(out, bound) in 64 bits.  pair: P in two FP16 parts (tiles of 16 columns), else one (tiles
    of 128 columns).

    The bound adds: the output's rounding, 2^-11 |o| + 2^-25; P's, 2^-21 A (its remainder's half
    step) or 2^-11 A with A the mean of |v| under the weights, and below FP16's normal range 2^-25 of
    a P whose largest is at least 2^7, for each of c keys, times a code of at most 127; a
    score's error twice in the exponent: FP32 sums of hd products (hd 2^-24 sum |q k|), q to 2^-23
    of its largest, and six FP32 roundings of an exponent of at most (|s| log2(e) + 64), whose
    logarithm of a V scale adds 2^-18; FP32 sums of c products, (c + 64) 2^-23 A."""
    n_pages, _, page, hd = cache["kc"].shape
    rows, n_q = q.shape[:2]
    group = n_q // n_kv
    out, bound = np.zeros((rows, n_q, hd)), np.zeros((rows, n_q, hd))
    for r in range(len(lens)):
        n, m = int(lens[r]), int(starts[r + 1] - starts[r])
        if n <= 0 or m <= 0:
            continue
        pages = table[r, :-(-n // page)]
        k, v = pu.values(cache, pages)
        sv = np.repeat(cache["vs"][pages].astype(np.float64), page, axis=0)[:n]   # (n, n_kv)
        k, v = k[:n], v[:n]
        for i in range(m):
            p = n - m + i
            lo = max(0, p - window + 1) if window else 0
            if p < 0:
                continue
            row = int(starts[r]) + i
            for g in range(n_kv):
                qq = q[row, g * group:(g + 1) * group].astype(np.float64)
                kk, vv, ss = k[lo:p + 1, g], v[lo:p + 1, g], sv[lo:p + 1, g]
                s = qq @ kk.T / math.sqrt(hd)
                w = np.exp(s - s.max(1, keepdims=True))
                w /= w.sum(1, keepdims=True)
                o, a = w @ vv, w @ np.abs(vv)
                d = (hd * 2.0 ** -24 * (np.abs(qq) @ np.abs(kk).T) + 2.0 ** -23 * np.abs(qq).max() * np.abs(kk).sum(1)) / math.sqrt(hd)
                d = d.max(1) + 6 * 2.0 ** -24 * (np.abs(s).max(1) + 64) + 2.0 ** -18
                c = p + 1 - lo
                rel = (2.0 ** -21 if pair else 2.0 ** -11) + np.expm1(2 * d) + (c + 64) * 2.0 ** -23
                at = slice(g * group, (g + 1) * group)
                out[row, at] = o
                bound[row, at] = (2.0 ** -11 * np.abs(o) + 2.0 ** -25 + a * rel[:, None] +
                                  c * 127 * 2.0 ** -32 * (w * ss).max(1)[:, None])
    return out, bound


def _run(cache, q, starts, lens, table, n_q, max_new, max_len, window=0):
    rows = q.shape[0]
    out = Cache(cache).attention(dev(q.view(np.uint16)).view(torch().float16).reshape(rows, -1),
                                 dev(np.asarray(starts, np.int32)), dev(np.asarray(lens, np.int32)), dev(table), n_q,
                                 max_new, max_len, window)
    got = host(out).astype(np.float64).reshape(q.shape)
    release()
    return got


def _within(got, want, bound, what):
    worst = np.max(np.abs(got - want) / bound)
    print(f"[precision] {what}: worst error / bound {worst:.3f}", flush=True)
    assert np.isfinite(got).all() and worst <= 1, what


def _grid(rng, *shape, scale=1.0):
    """Queries in steps of 1/8: 16 bits hold them exactly."""
    return (np.rint(np.clip(rng.standard_normal(shape) * scale, -15, 15) * 8) / 8).astype(np.float16)


# rows, max_new, max_len: one tile of 16 columns, several of them, tiles of 128 columns
KINDS = [("one", 4, 4, 50), ("narrow", 40, 40, 50), ("wide", 40, 105, 1 << 21)]


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kind,news,max_new,max_len", KINDS)
def test_rows_that_do_not_see_a_page_of_large_values(kind, news, max_new, max_len, hd):
    """The last page holds values 2^26 times the others'; the rows before it, in the same tile of
    columns, keep the bits of their own."""
    rng = np.random.default_rng(hd + news)
    n_q, n_kv, page, lens = 4, 2, 16, [50]
    table, n_pages = _tables(rng, lens, page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    cache["ks"][:] = 0.02
    cache["vs"][:] = 7e-6
    cache["vs"][table[0, 3]] = 470.0
    q = _grid(rng, news, n_q, hd)
    got = _run(cache, q, [0, news], lens, table, n_q, max_new, max_len)
    want, bound = _attend(cache, q, [0, news], lens, table, n_kv, pair=kind != "wide")
    _within(got, want, bound, kind)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("large", [0, 9, 40])
@pytest.mark.parametrize("kind,news,max_new,max_len", [("one", 1, 1, 700), ("narrow", 40, 40, 700), ("wide", 40, 105, 1 << 21)])
def test_weight_on_pages_of_small_values(kind, news, max_new, max_len, large, hd):
    """A page of values 2^26 times the others' that the rows see and give no weight to."""
    rng = np.random.default_rng(hd + news + large)
    n_q, n_kv, page, lens = 4, 2, 16, [700]
    table, n_pages = _tables(rng, lens, page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    cache["ks"][:] = 0.005
    cache["vs"][:] = 7e-6
    cache["vs"][table[0, large]] = 470.0
    cache["ks"][table[0, large]] = 0.04
    cache["kc"][table[0, large]] = -120        # q is positive: far below all other scores
    q = np.abs(_grid(rng, news, n_q, hd, scale=3.0))
    got = _run(cache, q, [0, news], lens, table, n_q, max_new, max_len)
    want, bound = _attend(cache, q, [0, news], lens, table, n_kv, pair=kind != "wide")
    _within(got, want, bound, kind)


@pytest.mark.parametrize("kind,news,max_new,max_len", [("one", 1, 1, 300), ("wide", 40, 105, 1 << 21)])
def test_pages_of_zeros_and_extreme_scales(kind, news, max_new, max_len):
    """V scales of zero (a page of zeros) and of 1e-36 beside ordinary ones: weights are shared
    as the scores say, whatever the scale of what they weigh."""
    rng = np.random.default_rng(news)
    n_q, n_kv, hd, page, lens = 4, 2, 64, 32, [300]
    table, n_pages = _tables(rng, lens, page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    cache["ks"][:] = 0.02
    cache["vs"][:] = 0.02
    cache["vs"][table[0, 1]] = 0.0
    cache["vs"][table[0, 4], 0] = 1e-36
    cache["vs"][table[0, 7], 1] = 1e-42
    q = _grid(rng, news, n_q, hd)
    got = _run(cache, q, [0, news], lens, table, n_q, max_new, max_len)
    want, bound = _attend(cache, q, [0, news], lens, table, n_kv, pair=kind != "wide")
    _within(got, want, bound, kind)
    cache["vs"][:] = 0.0   # only zeros in sight
    assert (_run(cache, q, [0, news], lens, table, n_q, max_new, max_len) == 0).all()


def _strong(rng, q, ratio):
    """One channel of every head `ratio` times the others."""
    q[..., 5] = np.where(rng.random(q.shape[:-1]) < 0.5, ratio, -ratio)
    return q


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("ratio", [300, 3000])
@pytest.mark.parametrize("kind,news,max_new,max_len", [("one", 2, 2, 9), ("narrow", 40, 40, 50), ("wide", 40, 105, 1 << 21)])
def test_strong_query_channels(kind, news, max_new, max_len, ratio, hd):
    """A channel that outweighs the others' size, where the keys have nothing: the scores are what
    the other channels say."""
    rng = np.random.default_rng(hd + ratio + news)
    n_q, n_kv, page, lens = 4, 2, 16, [max(9, news)]
    table, n_pages = _tables(rng, lens, page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    cache["ks"][:] = 0.01
    cache["vs"][:] = 0.02
    cache["kc"][..., 5] = 0
    q = _strong(rng, rng.standard_normal((news, n_q, hd)), ratio).astype(np.float16)
    got = _run(cache, q, [0, news], lens, table, n_q, max_new, max_len)
    want, bound = _attend(cache, q, [0, news], lens, table, n_kv, pair=kind != "wide")
    _within(got, want, bound, kind)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("ratio", [0, 300])
@pytest.mark.parametrize("kind,news,max_new,max_len", [("one", 1, 1, 2000), ("narrow", 32, 32, 2000), ("wide", 40, 105, 1 << 21)])
def test_relative_error(kind, news, max_new, max_len, ratio, hd):
    """The error's size over all outputs.  A rounding to FP16 is uniform over a step of at most
    2^-10 of the value: 2^-11 / sqrt(3) = 2.82e-4 of it in the mean square, for the output, and once
    more where P is one part (values of either sign: the errors add like the products).  All
    other steps are below 1e-5."""
    rng = np.random.default_rng(hd + ratio + news)
    n_q, n_kv, page, lens = 8, 2, 64, [2000]
    table, n_pages = _tables(rng, lens, page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    cache["ks"][:] = 0.01 * rng.uniform(0.7, 1.4, cache["ks"].shape)
    cache["vs"][:] = 0.5 * rng.uniform(0.7, 1.4, cache["vs"].shape)
    q = rng.standard_normal((news, n_q, hd))
    if ratio:
        cache["kc"][..., 5] = 0
        q = _strong(rng, q, ratio)
    q = q.astype(np.float16)
    got = _run(cache, q, [0, news], lens, table, n_q, max_new, max_len)
    want, _ = _attend(cache, q, [0, news], lens, table, n_kv)
    rel = math.sqrt(np.mean((got - want) ** 2) / np.mean(want ** 2))
    print(f"[precision] {kind} {hd} {ratio}: relative error {rel:.2e}", flush=True)
    assert rel <= 2.82e-4 * (1 if kind != "wide" else math.sqrt(2)) + 1e-5


@pytest.mark.parametrize("n_q,n_kv,hd,page,lens,news", [
    (8, 2, 256, 16, [900, 1, 330], [70, 1, 40]), (4, 1, 256, 128, [900, 1, 330], [70, 1, 40]),
    (8, 2, 64, 32, [1100, 700, 64], [150, 90, 2]), (8, 1, 128, 64, [1100, 40], [33, 40])])
@pytest.mark.parametrize("window", [0, 250])
def test_chunks_of_many_tiles(n_q, n_kv, hd, page, lens, news, window):
    """Tiles of 128 columns over contexts of many tiles of keys, in several parts that are joined."""
    rng = np.random.default_rng(sum(lens) + window)
    table, n_pages = _tables(rng, lens, page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    cache["ks"][:] = 0.01 * rng.uniform(0.7, 1.4, cache["ks"].shape)
    cache["vs"][:] = 0.02 * 2.0 ** -rng.choice([0, 0, 1, 5], cache["vs"].shape)
    starts = np.concatenate([[0], np.cumsum(news)])
    q = rng.standard_normal((int(starts[-1]), n_q, hd)).astype(np.float16)
    got = _run(cache, q, starts, lens, table, n_q, max(news) + 65, 1 << 21, window)
    again = _run(cache, q, starts, lens, table, n_q, max(news) + 65, 1 << 21, window)
    want, bound = _attend(cache, q, starts, lens, table, n_kv, window, pair=False)
    _within(got, want, bound, "chunks")
    np.testing.assert_array_equal(got, again)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 1111])
@pytest.mark.parametrize("kind,news,length,max_new,max_len", [
    ("one", 1, 9000, 1, 9000), ("one", 3, 2500, 4, 9000), ("narrow", 32, 3000, 32, 3000), ("wide", 70, 3000, 135, 1 << 21)])
def test_every_key_counts_once(kind, news, length, max_new, max_len, window, hd):
    """Values with one head dim each, so that an output is the sum of a few weights: one key lost
    or counted twice, at a tile's, a part's or the window's edge, is far outside the bound."""
    rng = np.random.default_rng(hd + length + window)
    n_q, n_kv, page, lens = 4, 1, 64, [length]
    table, n_pages = _tables(rng, lens, page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    cache["ks"][:] = 0.001
    cache["vs"][:] = 0.01
    cache["vc"][:] = 0
    key = np.arange(length)
    cache["vc"][table[0, key // page], 0, (7 * key + key // hd) % hd, key % page] = 100
    q = rng.standard_normal((news, n_q, hd)).astype(np.float16)
    got = _run(cache, q, [0, news], lens, table, n_q, max_new, max_len, window)
    want, bound = _attend(cache, q, [0, news], lens, table, n_kv, window, pair=kind != "wide")
    _within(got, want, bound, kind)
    # the oracle without one key is found out, whichever it is, by every row that sees it
    at = np.arange(length - news, length)
    for lost in (length - news, length - 64, length - 65, length - 700, *rng.integers(length - (window or length) + news, length - news, 3)):
        less = {k: v.copy() for k, v in cache.items()}
        less["vc"][table[0, lost // page], 0, :, lost % page] = 0
        off, _ = _attend(less, q, [0, news], lens, table, n_kv, window, pair=kind != "wide")
        found = (np.abs(off - want) > 2 * bound).any(axis=(1, 2))
        sees = (at >= lost) & ((at < lost + window) | (window == 0))
        assert sees.any() and found[sees].all(), lost


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("kind,news,max_new,max_len", KINDS)
def test_rows_beside_a_page_without_values(kind, news, max_new, max_len, bad, hd):
    """The last page's V scale is NaN or infinite for one KV head: the rows before it in the same
    tile, and the other head, have their values as exactly as ever."""
    rng = np.random.default_rng(hd + news)
    n_q, n_kv, page, lens = 4, 2, 16, [50]
    table, n_pages = _tables(rng, lens, page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    cache["ks"][:] = 0.02
    cache["vs"][:] = 0.02 * 2.0 ** rng.integers(-20, 8, cache["vs"].shape)
    plain = {k: v.copy() for k, v in cache.items()}
    cache["vs"][table[0, 3], 1] = bad
    q = _grid(rng, news, n_q, hd)
    got = _run(cache, q, [0, news], lens, table, n_q, max_new, max_len)
    want, bound = _attend(plain, q, [0, news], lens, table, n_kv, pair=kind != "wide")
    sees = np.zeros((news, n_q), bool)
    sees[np.arange(50 - news, 50) >= 48, 2:] = True
    assert sees.any() and not np.isfinite(got[sees]).any()
    _within(got[~sees], want[~sees], bound[~sees], kind)
