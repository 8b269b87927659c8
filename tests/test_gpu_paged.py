"""The paged 8-bit KV cache on the GPU against plain 64-bit forms (paged_util.py):
plan, append, read, attention, and a run of them together as a serving loop makes
it.  Codes, scales, slots and tables are whole numbers or exactly rounded, so
they are compared bit for bit; attention within a bound derived there."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import paged_util as pu
from gpu_util import call, dev, empty, f16_dev, hip, host, ptr, release, stream, torch

pytestmark = pytest.mark.gpu


def _f16(rng, *shape, scale=1.0):
    return (rng.standard_normal(shape) * scale).astype(np.float16)


# ------------------------------------------------------------------ plumbing

class Plan:
    """Device state of a pool of requests, planned by bx_kv_plan in place."""

    def __init__(self, n_req, page, n_pages, max_blocks, max_rows, ring, ends, table, past):
        t = torch()
        self.n_req, self.page, self.n_pages, self.max_rows = n_req, page, n_pages, max_rows
        self.table, self.ring, self.ends, self.past = dev(table), dev(ring), dev(ends), dev(past)
        self.starts = t.full((n_req + 1,), 77, dtype=t.int32, device="cuda")
        self.slots = t.full((max_rows,), 77, dtype=t.int64, device="cuda")
        self.pos = t.full((max_rows,), 77, dtype=t.int32, device="cuda")
        self.status = t.full((1,), 77, dtype=t.int32, device="cuda")
        self.max_blocks = max_blocks
        self.ws = t.zeros(int(hip().bx_kv_plan_workspace_bytes()), dtype=t.uint8, device="cuda")

    def step(self, delta):
        call("bx_kv_plan", ptr(self.past), ptr(delta), self.n_req, self.page, self.n_pages, ptr(self.table),
             self.max_blocks, ptr(self.ring), ptr(self.ends), ptr(self.ends), ptr(self.past), ptr(self.starts),
             ptr(self.slots), ptr(self.pos), self.max_rows, ptr(self.status), ptr(self.ws), C.c_size_t(self.ws.numel()),
             stream())


class Cache:
    def __init__(self, c):
        self.n_pages, self.n_kv, self.page, self.hd = c["kc"].shape
        self.kc, self.vc, self.ks, self.vs = (dev(c[x]) for x in ("kc", "vc", "ks", "vs"))

    def args(self):
        return (self.page, self.n_pages, ptr(self.kc), ptr(self.vc), ptr(self.ks), ptr(self.vs))

    def host(self):
        return dict(kc=host(self.kc), vc=host(self.vc), ks=host(self.ks), vs=host(self.vs))

    def append(self, k, v, slots, k_stride=None, v_stride=None, rows=None):
        w = self.n_kv * self.hd
        call("bx_kv_append_q8_f16", k if isinstance(k, C.c_void_p) else ptr(k), k_stride or w,
             v if isinstance(v, C.c_void_p) else ptr(v), v_stride or w, rows or slots.numel(), self.n_kv, self.hd,
             ptr(slots), *self.args(), stream())

    def read(self, slots, fill=0.0):
        t = torch()
        w = self.n_kv * self.hd
        k, v = (t.full((slots.numel(), w), fill, dtype=t.float16, device="cuda") for _ in range(2))
        call("bx_kv_read_q8_f16", ptr(slots), slots.numel(), self.n_kv, self.hd, *self.args(), ptr(k), w, ptr(v), w, stream())
        return k, v

    def attention(self, q, starts, lens, table, n_q, max_new, max_len, window=0, out=None, ws=None):
        t = torch()
        rows, n_req = q.shape[0], lens.numel()
        if out is None:
            out = t.full((rows, n_q * self.hd), 9.0, dtype=t.float16, device="cuda")
        n = int(hip().bx_attention_paged_q8_workspace_bytes(rows, n_req, n_q, self.n_kv, self.hd, max_new, max_len))
        if ws is None:
            ws = t.zeros(n, dtype=t.uint8, device="cuda")
        call("bx_attention_paged_q8_f16", ptr(q), q.stride(0), rows, ptr(starts), ptr(lens), n_req, max_new, max_len,
             ptr(table), table.shape[1], *self.args(), n_q, self.n_kv, self.hd, window, ptr(out), out.stride(0), ptr(ws),
             C.c_size_t(ws.numel()), stream())
        return out


def _same_cache(got, want, pages):
    for name in ("ks", "vs", "kc", "vc"):
        np.testing.assert_array_equal(got[name][pages].view(np.uint8), want[name][pages].view(np.uint8), err_msg=name)


def _tables(rng, lens, page, spare=2, width=None):
    blocks = [-(-n // page) for n in lens]
    n_pages = sum(blocks) + spare
    order = rng.permutation(n_pages).astype(np.int32)
    table = np.full((len(lens), width or max(blocks + [1]) + 1), -1, np.int32)
    at = 0
    for r, b in enumerate(blocks):
        table[r, :b] = order[at:at + b]
        at += b
    return table, n_pages


def _slots(table, r, a, b, page):
    p = np.arange(a, b)
    return table[r, p // page].astype(np.int64) * page + p % page


# ---------------------------------------------------------------------- plan

PLANS = [  # requests, page, longest, chunk, extra rows
    (1, 16, 40, 1, 0), (5, 16, 100, 40, 3), (16, 64, 1500, 1, 5), (300, 32, 400, 90, 11), (4096, 16, 60, 3, 1),
    (3, 128, 3000, 2500, 2)]


@pytest.mark.parametrize("n,page,longest,chunk,extra", PLANS)
def test_plan_steps(n, page, longest, chunk, extra):
    """Six steps in place: growth by 0 .. chunk, requests cut short or ended, the ring wrapping around."""
    rng = np.random.default_rng(n + page)
    width = -(-(longest + 6 * chunk) // page) + 1
    past = rng.integers(0, longest + 1, n).astype(np.int32)
    table, used = _tables(rng, past, page, spare=0, width=width)
    n_pages = used + -(-6 * chunk // page) * n + 6 * n
    ring = np.full(n_pages, -7, np.int32)
    free = rng.permutation(np.arange(used, n_pages)).astype(np.int32)
    ends = np.array([3 * n_pages - 2, 3 * n_pages - 2 + free.size], np.int64)
    ring[(ends[0] + np.arange(free.size)) % n_pages] = free
    max_rows = n * chunk + extra
    d = Plan(n, page, n_pages, width, max_rows, ring, ends, table, past)
    for step in range(6):
        delta = rng.integers(0, chunk + 1, n)
        cut = rng.random(n) < 0.2
        delta = np.where(cut, -rng.integers(0, past + 1), delta)
        delta = np.where(rng.random(n) < 0.05, -past, delta).astype(np.int32)
        print(f"[plan] n={n} page={page} step={step}", flush=True)
        d.step(dev(delta))
        lens, starts, slots, pos, ends, status = pu.plan(past, delta, page, n_pages, table, ring, ends, max_rows)
        assert status == 0 == int(host(d.status)[0])
        for got, want in ((d.past, lens), (d.starts, starts), (d.slots, slots), (d.pos, pos), (d.ends, ends),
                          (d.table, table), (d.ring, ring)):
            np.testing.assert_array_equal(host(got), want)
        past = lens
    # every page is in the ring or in a table, once
    held = np.concatenate([table[r, :-(-int(past[r]) // page)] for r in range(n)])
    free = ring[(ends[0] + np.arange(ends[1] - ends[0])) % n_pages]
    assert np.array_equal(np.sort(np.concatenate([held, free])), np.arange(n_pages))
    release()


@pytest.mark.parametrize("what,status", [
    ("pages", pu.NO_PAGES), ("table", pu.TABLE_FULL), ("rows", pu.ROWS_FULL), ("past", pu.BAD_LENGTH),
    ("cut", pu.BAD_LENGTH), ("ring", pu.BAD_RING), ("order", pu.BAD_RING)])
def test_plan_all_or_nothing(what, status):
    """A step that cannot be laid out changes nothing and says why."""
    n, page, width, n_pages, max_rows = 3, 16, 4, 12, 40
    past, delta = np.array([20, 0, 33], np.int32), np.array([3, 20, -5], np.int32)
    table = np.array([[4, 5, -1, -1], [-1, -1, -1, -1], [0, 2, 7, -1]], np.int32)
    ring = np.array([1, 3, 6, 8, 9, 10, 11] + [-1] * 5, np.int32)
    ends = np.array([0, 7], np.int64)
    if what == "pages":
        ends[0] = 6
    elif what == "table":
        delta[0] = 45
    elif what == "rows":
        delta[1] = 38
    elif what == "past":
        past[1] = -1
    elif what == "cut":
        delta[2] = -34
    elif what == "ring":
        ends[1] = 13
    else:
        ends[:] = 5, 4
    d = Plan(n, page, n_pages, width, max_rows, ring, ends, table, past)
    d.step(dev(delta))
    assert int(host(d.status)[0]) == status
    for got, want in ((d.past, past), (d.table, table), (d.ring, ring), (d.ends, ends), (d.starts, np.zeros(n + 1)),
                      (d.slots, np.full(max_rows, -1)), (d.pos, np.full(max_rows, -1))):
        np.testing.assert_array_equal(host(got), want)
    release()


def test_plan_pages_outside_the_pool():
    """A table entry that names no page gives its rows no slot; the append and the attention skip them."""
    page, n_pages = 16, 8
    table = np.array([[3, 99, -1], [-5, -1, -1]], np.int32)
    past = np.array([30, 10], np.int32)
    d = Plan(2, page, n_pages, 3, 8, np.arange(n_pages, dtype=np.int32), np.array([0, 4], np.int64), table, past)
    d.step(dev(np.array([3, 2], np.int32)))
    want = [-1, -1, 0 * page, -1, -1, -1, -1, -1]   # the third row opens a page of the ring
    np.testing.assert_array_equal(host(d.slots), want)
    np.testing.assert_array_equal(host(d.pos), [30, 31, 32, 10, 11, -1, -1, -1])
    release()


def test_plan_most_rows():
    """A step of 2^31 - 1 rows at most: those behind the last one are all marked."""
    t = torch()
    page, rows = 64, 2 ** 31 - 1
    d = Plan(2, page, 8, 4, 1, np.arange(8, dtype=np.int32), np.array([0, 8], np.int64), np.full((2, 4), -1, np.int32),
             np.zeros(2, np.int32))
    d.max_rows = rows
    d.slots = t.full((rows,), 77, dtype=t.int64, device="cuda")
    d.pos = t.full((rows,), 77, dtype=t.int32, device="cuda")
    d.step(dev(np.array([3, 70], np.int32)))
    assert host(d.status)[0] == 0
    np.testing.assert_array_equal(host(d.pos[:73]), list(range(3)) + list(range(70)))
    np.testing.assert_array_equal(host(d.slots[:73]), list(range(3)) + list(range(64, 64 + 70)))
    for x in (d.pos, d.slots):
        for a in range(73, rows, 1 << 28):
            assert bool((x[a:a + (1 << 28)] == -1).all()), a
    del d, x
    release()
    t.cuda.empty_cache()


# ----------------------------------------------------------- append and read

@pytest.mark.parametrize("n_kv,hd,page", [(1, 64, 16), (2, 128, 64), (3, 256, 32), (8, 128, 128), (2, 64, 128), (5, 128, 16)])
def test_append_runs(n_kv, hd, page):
    """Runs of every length at every place of a page, over memory that was never cleared; small,
    large and zero rows, so that scales grow, stay and start at zero."""
    rng = np.random.default_rng(hd + page)
    n_pages = 40
    want = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    c = Cache(want)
    filled = np.zeros(n_pages, int)
    touched = np.zeros(n_pages, bool)
    for step in range(7):
        slots = []
        for pg in rng.permutation(n_pages)[:25]:
            n = min(page - filled[pg], int(rng.choice([1, 1, 2, 15, 16, 17, page])))
            if n == 0:
                filled[pg] = 0   # the page starts over
                n = int(rng.integers(1, page + 1))
            slots += list(pg * page + filled[pg] + np.arange(n))
            filled[pg] += n
            touched[pg] = True
            if rng.random() < 0.3:
                slots += [-1]
            if rng.random() < 0.1:
                slots += [n_pages * page + 5]
        slots = np.array(slots, np.int64)
        rows = slots.size
        size = rng.choice([0.0, 1e-3, 1.0, 30.0], (rows, 1, 1), p=[0.1, 0.2, 0.5, 0.2])
        k, v = ((rng.standard_normal((rows, n_kv, hd)) * size).astype(np.float16) for _ in range(2))
        print(f"[append] n_kv={n_kv} hd={hd} page={page} step={step} rows={rows}", flush=True)
        c.append(f16_dev(k), f16_dev(v), dev(slots))
        pu.append(want, k, v, slots)
        got = c.host()
        for pg in np.nonzero(touched)[0]:
            n = filled[pg]
            np.testing.assert_array_equal(got["ks"][pg], want["ks"][pg])
            np.testing.assert_array_equal(got["vs"][pg], want["vs"][pg])
            np.testing.assert_array_equal(got["kc"][pg][:, :n], want["kc"][pg][:, :n])
            np.testing.assert_array_equal(got["vc"][pg][:, :, :n], want["vc"][pg][:, :, :n])
        others = np.nonzero(~touched)[0]
        _same_cache(got, want, others)   # pages of nobody stay as they were
    # the rows back, in any order, repeated, and outside the pool
    live = np.concatenate([pg * page + np.arange(filled[pg]) for pg in np.nonzero(touched)[0]])
    slots = np.concatenate([live, rng.permutation(live), [-1, n_pages * page], live[3:20], live[:1]]).astype(np.int64)
    kg, vg = (host(x).reshape(-1, n_kv, hd) for x in c.read(dev(slots), fill=5.0))
    kw, vw = pu.values(want, np.arange(n_pages))
    inside = (slots >= 0) & (slots < n_pages * page)
    at = np.where(inside, slots, 0)
    for g, w in ((kg, kw[at]), (vg, vw[at])):
        # the product rounded to FP32, then to FP16: half a step each
        tol = np.abs(w) * (2.0 ** -11 + 2.0 ** -24) + 2.0 ** -25
        err = np.abs(g.astype(np.float64) - w)
        assert (err <= tol)[inside].all()
        assert (g[~inside] == 5.0).all()
    release()


@pytest.mark.parametrize("n_kv,hd,page", [(3, 64, 16), (3, 128, 32), (3, 64, 64), (1, 128, 128), (2, 256, 64), (5, 64, 32)])
def test_append_runs_of_long_prompts(n_kv, hd, page):
    """More than 2,048 rows in a call, runs of every length at every place of a page: several
    runs, short and long, begin in one workgroup's share of the rows, and long ones leave it."""
    rng = np.random.default_rng(hd + page + n_kv)
    n_pages = 6000 // page + 120
    want = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    c = Cache(want)
    filled = np.zeros(n_pages, int)
    for step in range(3):
        slots = []
        for pg in rng.permutation(n_pages):
            n = min(page - filled[pg], int(rng.choice([1, 2, 7, 15, 16, 17, page - 1, page], p=[.15, .1, .1, .1, .1, .1, .1, .25])))
            if n == 0:
                filled[pg] = 0   # the page starts over
                n = int(rng.integers(1, page + 1))
            slots += list(pg * page + filled[pg] + np.arange(n))
            filled[pg] += n
            if rng.random() < 0.2:
                slots += [-1] * int(rng.integers(1, 4))
        slots = np.array(slots, np.int64)
        rows = slots.size
        assert rows > 2048
        size = rng.choice([0.0, 1e-3, 1.0, 30.0], (rows, 1, 1), p=[0.1, 0.2, 0.5, 0.2])
        k, v = ((rng.standard_normal((rows, n_kv, hd)) * size).astype(np.float16) for _ in range(2))
        print(f"[append] n_kv={n_kv} hd={hd} page={page} step={step} rows={rows}", flush=True)
        c.append(f16_dev(k), f16_dev(v), dev(slots))
        pu.append(want, k, v, slots)
        got = c.host()
        np.testing.assert_array_equal(got["ks"], want["ks"])
        np.testing.assert_array_equal(got["vs"], want["vs"])
        for pg in range(n_pages):
            n = filled[pg]
            np.testing.assert_array_equal(got["kc"][pg][:, :n], want["kc"][pg][:, :n])
            np.testing.assert_array_equal(got["vc"][pg][:, :, :n], want["vc"][pg][:, :, :n])
    release()


def test_append_rounds_ties_to_even():
    """Codes that fall exactly between two integers, new and requantized."""
    page, hd = 16, 64
    want = pu.empty_cache(2, 1, page, hd)
    c = Cache(want)
    x = np.zeros((3, 1, hd), np.float16)
    x[0, 0, :8] = [127, 0.5, 1.5, 2.5, -0.5, -1.5, 63.5, -126.5]   # scale 1: halves are ties
    x[1, 0, :4] = [254, 1, 3, -5]                                  # scale 2: odd codes are ties, old and new
    x[2, 0, :2] = [1, 65504]
    for i in range(3):
        s = np.array([i], np.int64)
        c.append(f16_dev(x[i:i + 1]), f16_dev(x[i:i + 1] * np.float16(-1)), dev(s))
        pu.append(want, x[i:i + 1], -x[i:i + 1], s)
        got = c.host()
        np.testing.assert_array_equal(got["ks"][0], want["ks"][0])
        np.testing.assert_array_equal(got["kc"][0, 0, :i + 1], want["kc"][0, 0, :i + 1])
        np.testing.assert_array_equal(got["vc"][0, 0, :, :i + 1], want["vc"][0, 0, :, :i + 1])
    release()


@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64), (256, 128)])
def test_append_values_next_to_halves(hd, page):
    """Values whose quotient with the scale is as near to n + 1/2 as FP16 allows, on either side
    of it, for scales that are powers of two (exact halves) and others."""
    rng = np.random.default_rng(hd)
    n_kv, pages = 2, 24
    rows = pages * page
    amax = np.where(rng.random((pages, 1, n_kv, 1)) < 0.5, 127.0 * 2.0 ** rng.integers(-15, 9, (pages, 1, n_kv, 1)),
                    rng.uniform(1e-4, 6e4, (pages, 1, n_kv, 1))).astype(np.float16)
    scale = (amax.astype(np.float32) / np.float32(127)).astype(np.float64)
    x = ((rng.integers(-127, 127, (pages, page, n_kv, hd)) + 0.5) * scale).astype(np.float16)
    step = rng.integers(-1, 2, x.shape)
    x = np.where(step == 0, x, np.nextafter(x, np.where(step > 0, np.float16(np.inf), np.float16(-np.inf)).astype(np.float16)))
    x = np.clip(x, -amax, amax).astype(np.float16)
    x[:, 0, :, 0] = amax[:, 0, :, 0]
    k = x.reshape(rows, n_kv, hd)
    v = np.roll(k, 1, axis=2)
    cache = pu.empty_cache(pages, n_kv, page, hd, rng)
    slots = np.arange(rows, dtype=np.int64)
    c = Cache(cache)
    t = torch()
    c.append(dev(k.view(np.uint16)).view(t.float16).reshape(rows, -1), dev(v.view(np.uint16)).view(t.float16).reshape(rows, -1),
             dev(slots))
    pu.append(cache, k, v, slots)
    _same_cache(c.host(), cache, np.arange(pages))
    release()


def test_append_nan_and_infinity_stay_in_their_page_and_head():
    page, hd, n_kv = 16, 64, 3
    rng = np.random.default_rng(5)
    want = pu.empty_cache(4, n_kv, page, hd)
    c = Cache(want)
    k, v = _f16(rng, 40, n_kv, hd), _f16(rng, 40, n_kv, hd)
    k[20, 1, 7] = np.nan
    v[20, 2, 9] = -np.inf
    slots = np.arange(40, dtype=np.int64)
    for a, b in ((0, 18), (18, 40)):
        c.append(f16_dev(k[a:b].astype(np.float32)), f16_dev(v[a:b].astype(np.float32)), dev(slots[a:b]))
        pu.append(want, k[a:b], v[a:b], slots[a:b])
    kg, vg = (host(x).reshape(-1, n_kv, hd) for x in c.read(dev(slots)))
    bad_k, bad_v = np.zeros((40, n_kv), bool), np.zeros((40, n_kv), bool)
    bad_k[16:32, 1] = True
    bad_v[16:32, 2] = True
    assert np.isnan(kg[bad_k]).all() and np.isfinite(kg[~bad_k]).all()
    assert not np.isfinite(vg[bad_v]).any() and np.isfinite(vg[~bad_v]).all()
    np.testing.assert_array_equal(np.isnan(host(c.ks)), np.isnan(want["ks"]))
    release()


def test_append_strided_and_odd_addresses():
    """K and V as parts of wider rows (a fused projection's output), at 2-byte offsets."""
    page, hd, n_kv, rows = 32, 128, 2, 70
    rng = np.random.default_rng(8)
    w = n_kv * hd
    both = rng.standard_normal((rows, 3 * w + 5)).astype(np.float16)
    base = f16_dev(both.astype(np.float32)).reshape(-1)
    slots = np.concatenate([np.arange(3, 60), 96 + np.arange(13)]).astype(np.int64)
    want = pu.empty_cache(4, n_kv, page, hd)
    c = Cache(want)
    st = 3 * w + 5
    for off_k, off_v in ((1, w + 3), (2 * w + 5, 0)):
        k = C.c_void_p(base.data_ptr() + 2 * off_k)
        v = C.c_void_p(base.data_ptr() + 2 * off_v)
        c.append(k, v, dev(slots), st, st, rows)
        pu.append(want, both[:, off_k:off_k + w].reshape(rows, n_kv, hd), both[:, off_v:off_v + w].reshape(rows, n_kv, hd),
                  slots)
        got, exp = c.read(dev(slots)), pu.values(want, np.arange(4))
        for g, e in zip(got, exp):
            e = e[slots]
            assert (np.abs(host(g).reshape(e.shape).astype(np.float64) - e) <= np.abs(e) * 2.0 ** -10 + 2.0 ** -24).all()
    release()


# ----------------------------------------------------------------- attention

def _attention_case(rng, lens, news, n_q, n_kv, hd, page, window=0, q_scale=1.0, pad=0, max_new=None, max_len=None):
    table, n_pages = _tables(rng, lens, page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    # scales of a cache of unit-variance keys and values, some pages far smaller
    cache["ks"] = (0.02 * rng.uniform(0.7, 1.4, cache["ks"].shape)).astype(np.float32)
    cache["vs"] = (0.02 * 2.0 ** -rng.choice([0, 0, 0, 1, 3, 9], cache["vs"].shape)).astype(np.float32)
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    rows = int(starts[-1]) + pad
    q = _f16(rng, rows, n_q, hd, scale=q_scale)
    c = Cache(cache)
    out = c.attention(f16_dev(q.astype(np.float32)).reshape(rows, -1).view(torch().float16), dev(starts),
                      dev(np.array(lens, np.int32)), dev(table), n_q, max_new or max(news), max_len or max(lens), window)
    want, bound = pu.attention(cache, q, starts, lens, table, n_kv, window)
    got = host(out).astype(np.float64).reshape(rows, n_q, hd)
    n = int(starts[-1])
    err = np.abs(got - want)[:n]
    assert np.isfinite(got).all()
    print(f"[attention] worst error / bound {np.max(err / np.maximum(bound[:n], 1e-30)):.3f}", flush=True)
    assert (err <= bound[:n] + 2.0 ** -25).all()
    assert (got[n:] == 9.0).all()   # rows behind the last request
    release()


@pytest.mark.parametrize("n_q,n_kv,hd,page", [
    (4, 2, 64, 16), (16, 8, 128, 64), (8, 1, 128, 32), (2, 2, 256, 16), (16, 1, 64, 128), (6, 2, 128, 16), (5, 1, 256, 64)])
@pytest.mark.parametrize("lens", [[1], [2, 63, 64, 65], [300, 1, 17, 129], [1000]])
def test_attention_decode(n_q, n_kv, hd, page, lens):
    rng = np.random.default_rng(sum(lens) + n_q + hd)
    _attention_case(rng, lens, [1] * len(lens), n_q, n_kv, hd, page, pad=2)


@pytest.mark.parametrize("n_q,n_kv,hd,page,lens,news", [
    (4, 2, 128, 64, [40, 300, 5], [3, 2, 4]),                 # several tokens a request, 16 columns at most
    (8, 2, 128, 16, [200, 64, 1, 700], [50, 64, 1, 1]),       # chunks and single tokens together
    (8, 1, 64, 32, [130, 129], [130, 65]),
    (6, 2, 256, 16, [100, 7], [33, 7]),
    (3, 3, 128, 128, [400], [170]),
    (16, 1, 128, 64, [90], [21]),
    (4, 4, 64, 16, [257, 1, 80], [257, 1, 16])])
@pytest.mark.parametrize("window", [0, 1, 37, 64, 250])
def test_attention_chunks(n_q, n_kv, hd, page, lens, news, window):
    rng = np.random.default_rng(sum(lens) + window)
    _attention_case(rng, lens, news, n_q, n_kv, hd, page, window, pad=3)


@pytest.mark.parametrize("n_q,n_kv,hd,page,lens,news", [
    (8, 2, 128, 16, [200, 64, 1, 700], [50, 64, 1, 1]),
    (8, 1, 64, 32, [130, 129], [130, 65]),
    (6, 2, 256, 16, [100, 7], [33, 7]),
    (3, 3, 128, 128, [400], [170]),
    (16, 1, 128, 64, [90], [21]),
    (4, 4, 64, 16, [257, 1, 80], [257, 1, 16]),
    (4, 1, 128, 64, [2600, 1, 90], [300, 0, 4])])
@pytest.mark.parametrize("window", [0, 37, 250])
def test_attention_chunks_of_large_batches(n_q, n_kv, hd, page, lens, news, window):
    """Tiles of 128 columns: bounds on rows and lengths that allow for far more work."""
    rng = np.random.default_rng(sum(lens) + window + 1)
    _attention_case(rng, lens, news, n_q, n_kv, hd, page, window, pad=3, max_new=max(news) + 65, max_len=1 << 21)


@pytest.mark.parametrize("n_req,most", [(5, 40), (63, 9), (64, 9), (65, 9), (200, 5), (256, 5), (257, 5)])
def test_attention_short_runs_of_many_requests(n_req, most):
    """Zero to some rows a request, so that tiles begin and end anywhere; 257 requests are laid
    out otherwise."""
    rng = np.random.default_rng(n_req)
    news = rng.integers(0, most + 1, n_req)
    news[[0, -1]] = most
    lens = news + rng.integers(0, 150, n_req)
    _attention_case(rng, lens.tolist(), news.tolist(), 8, 1, 64, 16, window=int(n_req == 65) * 70, pad=1)


def test_attention_single_tokens_under_a_loose_bound():
    """max_new and max_len far above what comes."""
    for max_new, max_len in ((7, 1 << 20), (64, 200), (64, 1 << 20)):
        _attention_case(np.random.default_rng(max_new), [33, 150, 64], [1, 1, 1], 8, 2, 128, 32, pad=4, max_new=max_new,
                        max_len=max_len)


@pytest.mark.parametrize("news", [[1, 1], [30, 1]])
def test_attention_long(news):
    """Thousands of keys: many splits, merged by the last workgroup."""
    rng = np.random.default_rng(3)
    _attention_case(rng, [9000, 2500], news, 4, 1, 128, 64)


def test_attention_peaked_scores():
    """Large queries: one key takes nearly all the weight, the running maximum moves often."""
    rng = np.random.default_rng(4)
    _attention_case(rng, [700, 90], [1, 20], 8, 2, 128, 32, q_scale=12.0)


def test_attention_rows_without_keys():
    """Idle requests, a request with more rows than keys, tables that name no page."""
    rng = np.random.default_rng(6)
    n_q, n_kv, hd, page = 4, 2, 128, 16
    table, n_pages = _tables(rng, [40, 40, 40, 40], page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    table[2, 1] = n_pages + 3
    table[3] = -1
    news, lens = [0, 5, 2, 3], [0, 3, 40, 40]
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    q = _f16(rng, 12, n_q, hd)
    c = Cache(cache)
    for max_new in (5, 4):   # tiles over all columns, and a tile a request
        use = starts if max_new == 5 else np.array([0, 0, 4, 6, 9], np.int32)
        out = c.attention(f16_dev(q.astype(np.float32)).view(torch().float16).reshape(12, -1), dev(use),
                          dev(np.array(lens, np.int32)), dev(table), n_q, max_new, 40)
        want, bound = pu.attention(cache, q, use, lens, table, n_kv)
        got = host(out).astype(np.float64).reshape(12, n_q, hd)
        n = int(use[-1])
        assert (np.abs(got - want)[:n] <= bound[:n] + 2.0 ** -25).all()
        first = int(use[1])
        assert (got[first:first + (int(use[2]) - first - 3)] == 0).all()      # rows before the first key
        assert (got[int(use[3]):n] == 0).all()                                # no page at all
        assert (got[n:] == 9.0).all()
    release()


@pytest.mark.parametrize("max_new,max_len", [(4, 40), (40, 40), (100, 1 << 21)])
def test_attention_windows_and_lengths_at_their_ends(max_new, max_len):
    """The widest window with rows before the first key, and a length far below zero (no keys):
    single-token tiles, several of them, tiles of 128 columns."""
    rng = np.random.default_rng(max_new)
    n_q, n_kv, hd, page, window = 4, 1, 64, 16, 2 ** 31 - 1
    news, lens = [4, 2, 3, 1], [2, 40, -2 ** 31, 0]
    if max_new > 4:
        news[0] = max_new
    table, n_pages = _tables(rng, [16, 40, 16, 16], page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    n = int(starts[-1])
    q = _f16(rng, n, n_q, hd)
    out = Cache(cache).attention(dev(q.view(np.uint16)).view(torch().float16).reshape(n, -1), dev(starts),
                                 dev(np.array(lens, np.int32)), dev(table), n_q, max_new, max_len, window)
    got = host(out).astype(np.float64).reshape(n, n_q, hd)
    want, bound = pu.attention(cache, q, starts, np.maximum(lens, 0).tolist(), table, n_kv)
    assert (np.abs(got - want) <= bound + 2.0 ** -25).all()
    assert (got[:int(starts[1]) - 2] == 0).all() and (got[int(starts[2]):] == 0).all()
    release()


def test_attention_nan_stays_where_it_is_seen():
    """A NaN in a page's scale, in codes behind the last token, or in one query row
    reaches the rows that see it and no others."""
    rng = np.random.default_rng(7)
    n_q, n_kv, hd, page = 4, 2, 64, 16
    lens, news = [50, 50], [50, 1]
    table, n_pages = _tables(rng, lens, page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    cache["ks"][table[0, 1], 0] = np.nan     # keys 16 .. 31 of request 0, KV head 0
    cache["vs"][table[0, 2], 1] = np.inf     # values 32 .. 47, KV head 1
    q = _f16(rng, 51, n_q, hd)
    q[5, 3, 2] = np.nan
    starts = np.array([0, 50, 51], np.int32)
    c = Cache(cache)
    qd = dev(q.view(np.uint16)).view(torch().float16).reshape(51, -1)
    got = host(c.attention(qd, dev(starts), dev(np.array(lens, np.int32)), dev(table), n_q, 50, 50)).reshape(51, n_q, hd)
    bad = np.zeros((51, n_q), bool)
    bad[16:50, :2] = True
    bad[32:50, 2:] = True
    bad[5, 3] = True
    assert not np.isfinite(got[bad]).all(-1).any()
    assert np.isfinite(got[~bad]).all()
    release()


@pytest.mark.parametrize("news", [[1, 1], [30, 1], [200, 3]])
def test_attention_pages_behind_the_window_may_hold_anything(news):
    """Pages that no row's window reaches have been given back: their codes and scales (NaN,
    infinite, huge) change nothing, nor do those of tokens behind the last one."""
    rng = np.random.default_rng(sum(news))
    n_q, n_kv, hd, page, window, lens = 8, 2, 128, 16, 90, [700, 333]
    table, n_pages = _tables(rng, lens, page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    q = _f16(rng, int(starts[-1]), n_q, hd)
    want, bound = pu.attention(cache, q, starts, lens, table, n_kv, window)
    for r, (n, m) in enumerate(zip(lens, news)):
        gone = table[r, :max(0, n - m - window + 1) // page]   # pages before the first row's window
        for name, bad in (("ks", [np.nan, np.inf, 3e38]), ("vs", [3e38, np.nan, np.inf])):
            cache[name][gone] = np.resize(np.array(bad, np.float32), (gone.size, n_kv))
        last = table[r, (n - 1) // page]
        cache["kc"][last][:, (n - 1) % page + 1:] = -128
        cache["vc"][last][:, :, (n - 1) % page + 1:] = 127
    c = Cache(cache)
    out = c.attention(dev(q.view(np.uint16)).view(torch().float16).reshape(q.shape[0], -1), dev(starts),
                      dev(np.array(lens, np.int32)), dev(table), n_q, max(news), max(lens), window)
    got = host(out).astype(np.float64).reshape(q.shape)
    assert (np.abs(got - want) <= bound + 2.0 ** -25).all()
    release()


def test_attention_one_workspace_for_many_shapes():
    """Calls of different shapes in turn on one workspace, sized for the largest of them."""
    t = torch()
    rng = np.random.default_rng(21)
    n_q, n_kv, hd, page = 8, 2, 64, 16
    shapes = [([3000], [1], 0), ([40, 2000, 7], [40, 1, 3], 300), ([900] * 40, [1] * 40, 20), ([5000, 3], [20, 1], 0)]
    sizes = [int(hip().bx_attention_paged_q8_workspace_bytes(sum(m), len(n), n_q, n_kv, hd, max(m), max(n))) for n, m, _ in shapes]
    ws = t.zeros(max(sizes), dtype=t.uint8, device="cuda")
    calls = []
    for lens, news, window in shapes:
        table, n_pages = _tables(rng, lens, page)
        cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
        starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
        q = _f16(rng, int(starts[-1]), n_q, hd)
        args = (dev(q.view(np.uint16)).view(t.float16).reshape(q.shape[0], -1), dev(starts), dev(np.array(lens, np.int32)),
                dev(table), n_q, max(news), max(lens), window)
        calls.append((Cache(cache), args, pu.attention(cache, q, starts, lens, table, n_kv, window)))
    for turn in range(6):
        for i in rng.permutation(len(calls)):
            c, args, (want, bound) = calls[i]
            got = host(c.attention(*args, ws=ws)).astype(np.float64).reshape(want.shape)
            assert (np.abs(got - want) <= bound + 2.0 ** -25).all(), (turn, i)
    assert not host(ws)[:512 * 1024].any()   # every counter back at zero
    release()


def test_attention_strided_rows_and_odd_addresses():
    rng = np.random.default_rng(9)
    n_q, n_kv, hd, page, lens, news = 8, 2, 128, 16, [100, 33], [20, 1]
    table, n_pages = _tables(rng, lens, page)
    cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    starts = np.array([0, 20, 21], np.int32)
    w = n_q * hd
    wide = rng.standard_normal((21, w + 77)).astype(np.float16)
    qd = dev(wide.view(np.uint16)).view(torch().float16)
    c = Cache(cache)
    t = torch()
    out = t.full((21, w + 31), 9.0, dtype=t.float16, device="cuda")
    c.attention(qd[:, 3:3 + w], dev(starts), dev(np.array(lens, np.int32)), dev(table), n_q, 20, 100, out=out[:, 5:5 + w])
    want, bound = pu.attention(cache, wide[:, 3:3 + w].reshape(21, n_q, hd), starts, lens, table, n_kv)
    got = host(out).astype(np.float64)
    assert (np.abs(got[:, 5:5 + w].reshape(21, n_q, hd) - want) <= bound + 2.0 ** -25).all()
    assert (got[:, :5] == 9).all() and (got[:, 5 + w:] == 9).all()
    release()


def test_attention_pool_beyond_32_bits():
    """Pages whose codes lie more than 2^32 bytes into the pool (the last pages of 5 GiB)."""
    t = torch()
    rng = np.random.default_rng(10)
    n_q, n_kv, hd, page, lens = 4, 2, 128, 64, [70, 200]
    n_pages = (5 << 30) // (n_kv * page * hd)
    small = pu.empty_cache(8, n_kv, page, hd, rng)
    kc = t.empty((n_pages, n_kv, page, hd), dtype=t.int8, device="cuda")
    vc = t.empty((n_pages, n_kv, hd, page), dtype=t.int8, device="cuda")
    ks = t.empty((n_pages, n_kv), device="cuda")
    vs = t.empty((n_pages, n_kv), device="cuda")
    ids = np.array([n_pages - 1 - 3 * i for i in range(8)])
    c = Cache(small)
    for big, name in ((kc, "kc"), (vc, "vc"), (ks, "ks"), (vs, "vs")):
        big[dev(ids)] = dev(small[name])
    c.n_pages, c.kc, c.vc, c.ks, c.vs = n_pages, kc, vc, ks, vs
    table = np.array([[0, 1, -1, -1], [2, 3, 4, 5]], np.int32)
    far = np.where(table >= 0, ids[table], -1).astype(np.int32)
    # a new token each, appended through slots beyond 2^32, then attended
    slots = np.array([far[0, 1] * page + 5, int(far[1, 3]) * page + 7], np.int64)
    k, v = _f16(rng, 2, n_kv, hd, scale=2.5), _f16(rng, 2, n_kv, hd, scale=2.5)
    c.append(f16_dev(k), f16_dev(v), dev(slots))
    pu.append(small, k, v, np.array([1 * page + 5, 5 * page + 7], np.int64))
    q = _f16(rng, 2, n_q, hd)
    starts, lens = np.array([0, 1, 2], np.int32), np.array([70, 200], np.int32)
    out = c.attention(f16_dev(q).view(t.float16).reshape(2, -1), dev(starts), dev(lens), dev(far), n_q, 1, 200)
    want, bound = pu.attention(small, q, starts, lens, table, n_kv)
    assert (np.abs(host(out).astype(np.float64).reshape(2, n_q, hd) - want) <= bound + 2.0 ** -25).all()
    kr, vr = c.read(dev(slots))
    kw, vw = pu.values(small, np.arange(8))
    at = [1 * page + 5, 5 * page + 7]
    assert np.allclose(host(kr).reshape(2, n_kv, hd), kw[at], rtol=2.0 ** -10, atol=2.0 ** -24)
    assert np.allclose(host(vr).reshape(2, n_kv, hd), vw[at], rtol=2.0 ** -10, atol=2.0 ** -24)
    release()


# ------------------------------------------------- a step as a serving loop runs it

def _serve(c, d, wanted, rng, table, ring, ends, past, steps, n_q, graph=False, news=None):
    """Steps of plan -> append -> attention against the host forms; returns nothing, asserts."""
    t = torch()
    n_kv, hd, page, n_pages = c.n_kv, c.hd, c.page, c.n_pages
    rows = d.max_rows
    k = t.empty((rows, n_kv * hd), dtype=t.float16, device="cuda")
    v = t.empty_like(k)
    q = t.empty((rows, n_q * hd), dtype=t.float16, device="cuda")
    out = t.empty_like(q)
    delta = t.empty(d.n_req, dtype=t.int32, device="cuda")
    max_new, max_len = max(news), d.max_blocks * page
    nb = int(hip().bx_attention_paged_q8_workspace_bytes(rows, d.n_req, n_q, n_kv, hd, max_new, max_len))
    ws = t.zeros(nb, dtype=t.uint8, device="cuda")

    def step():
        d.step(delta)
        c.append(k, v, d.slots)
        c.attention(q, d.starts, d.past, d.table, n_q, max_new, max_len, out=out, ws=ws)

    captured = None
    for i in range(steps):
        change = rng.choice(news, d.n_req).astype(np.int32)
        over = past + change > d.max_blocks * page
        change = np.where(over, -past, change).astype(np.int32)
        kk, vv, qq = (_f16(rng, rows, h, hd, scale=s) for h, s in ((n_kv, 1 + i), (n_kv, 1.0), (n_q, 1.0)))
        for dst, src in ((k, kk), (v, vv), (q, qq)):
            dst.copy_(dev(src.view(np.uint16)).view(t.float16).reshape(dst.shape))
        delta.copy_(dev(change))
        out.fill_(9.0)
        t.cuda.synchronize()
        print(f"[serve] step {i}", flush=True)
        if graph and captured is None and i == 1:
            captured = t.cuda.CUDAGraph()
            with t.cuda.graph(captured):
                step()
        if captured is not None:
            captured.replay()
        else:
            step()
        lens, starts, slots, pos, ends, status = pu.plan(past, change, page, n_pages, table, ring, ends, rows)
        assert status == 0 == int(host(d.status)[0])
        np.testing.assert_array_equal(host(d.slots), slots)
        np.testing.assert_array_equal(host(d.past), lens)
        pu.append(wanted, kk, vv, slots)
        want, bound = pu.attention(wanted, qq, starts, lens, table, n_kv)
        got = host(out).astype(np.float64).reshape(rows, n_q, hd)
        n = int(starts[-1])
        assert (np.abs(got - want)[:n] <= bound[:n] + 2.0 ** -25).all()
        assert (got[n:] == 9.0).all()
        past = lens


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("n_req,page,hd,news", [(6, 16, 64, [0, 1, 1, 9]), (9, 32, 128, [1]), (3, 64, 128, [1, 70])])
def test_serving_loop(n_req, page, hd, news, graph):
    """Requests grow, end and start over on the pages of others; captured into a graph
    and replayed as well (the state stays in place, so replays continue it)."""
    rng = np.random.default_rng(n_req * page + graph)
    n_q, n_kv = 4, 2
    width = -(-150 // page)
    n_pages = n_req * width
    table = np.full((n_req, width), -1, np.int32)
    ring, ends = rng.permutation(n_pages).astype(np.int32), np.array([0, n_pages], np.int64)
    past = np.zeros(n_req, np.int32)
    wanted = pu.empty_cache(n_pages, n_kv, page, hd, rng)
    d = Plan(n_req, page, n_pages, width, n_req * max(news) + 2, ring, ends, table, past)
    c = Cache(wanted)
    _serve(c, d, wanted, rng, table, ring, ends, past, 12, n_q, graph, news)
    release()


def test_two_streams_with_their_own_workspaces():
    """Two pools served at the same time on two streams give what they give alone."""
    t = torch()
    rng = np.random.default_rng(12)
    n_q, n_kv, hd, page, lens = 8, 2, 128, 64, [3000, 700, 1500]
    sides = []
    for _ in range(2):
        table, n_pages = _tables(rng, lens, page)
        cache = pu.empty_cache(n_pages, n_kv, page, hd, rng)
        q = _f16(rng, 3, n_q, hd)
        sides.append((Cache(cache), dev(q.view(np.uint16)).view(t.float16).reshape(3, -1), dev(table)))
    starts, ln = dev(np.array([0, 1, 2, 3], np.int32)), dev(np.array(lens, np.int32))
    alone = [host(c.attention(q, starts, ln, tb, n_q, 1, 3000)) for c, q, tb in sides]
    n = int(hip().bx_attention_paged_q8_workspace_bytes(3, 3, n_q, n_kv, hd, 1, 3000))
    spaces = [t.zeros(n, dtype=t.uint8, device="cuda") for _ in range(2)]
    outs = [t.zeros((3, n_q * hd), dtype=t.float16, device="cuda") for _ in range(2)]
    streams = [t.cuda.Stream() for _ in range(2)]
    t.cuda.synchronize()
    for _ in range(20):
        for (c, q, tb), ws, out, st in zip(sides, spaces, outs, streams):
            with t.cuda.stream(st):
                c.attention(q, starts, ln, tb, n_q, 1, 3000, out=out, ws=ws)
    t.cuda.synchronize()
    for out, want in zip(outs, alone):
        np.testing.assert_array_equal(host(out), want)
    release()
