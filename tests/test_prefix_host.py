"""What the entry points of a step with shared prefixes refuse, on the CPU: every check
stands before the first GPU call; and the host forms against each other."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import paged_util as pu
import prefix_util as px
from test_paged_host import CACHE, EINVAL, EUNSUPPORTED, P, _refused, _with


def _p(i):
    return C.c_void_p(0x10000 * i)   # never read: the call is refused first


PLAN = [("parent", _p(1)), ("shared_lens", _p(2)), ("starts", _p(3)), ("lens", _p(4)), ("n_req", 4), ("pos_in", _p(5)),
        ("pos", _p(6)), ("shared", _p(7)), ("order", _p(8)), ("max_rows", 10), ("groups", _p(9)), ("group_starts", _p(10)),
        ("stream", None)]


@pytest.mark.parametrize("kw,code,word", [
    (dict(parent=None), EINVAL, "null"), (dict(shared_lens=None), EINVAL, "null"), (dict(pos_in=None), EINVAL, "null"),
    (dict(order=None), EINVAL, "null"), (dict(group_starts=None), EINVAL, "null"), (dict(n_req=0), EINVAL, "shape"),
    (dict(n_req=-3), EINVAL, "shape"), (dict(max_rows=0), EINVAL, "shape"), (dict(n_req=4097), EUNSUPPORTED, "4096"),
    (dict(shared=_p(5)), EINVAL, "lie over"), (dict(order=_p(4)), EINVAL, "lie over"), (dict(pos=_p(1)), EINVAL, "lie over"),
    (dict(pos=_p(7)), EINVAL, "lie over"), (dict(groups=_p(10)), EINVAL, "lie over")])
def test_prefix_plan_refuses(native, kw, code, word):
    _refused(native, "bx_prefix_plan", _with(PLAN, **kw), code, word)


QKV = [("q", P), ("q_stride", 2048), ("k", P), ("k_stride", 1024), ("v", P), ("v_stride", 1024), ("rows", 5), ("n_q", 16),
       ("n_kv", 8), ("hd", 128), ("q_gain", P), ("k_gain", P), ("eps", 1e-6), ("pos", P), ("cos", P), ("sin", P),
       ("tab_rows", 100), ("slots", P)] + CACHE + [("q_out", P), ("q_out_stride", 2048), ("stream", None)]


@pytest.mark.parametrize("kw,code,word", [
    (dict(q=None), EINVAL, "null"), (dict(k=None), EINVAL, "null"), (dict(v=None), EINVAL, "null"),
    (dict(pos=None), EINVAL, "null"), (dict(cos=None), EINVAL, "null"), (dict(sin=None), EINVAL, "null"),
    (dict(slots=None), EINVAL, "null"), (dict(q_out=None), EINVAL, "null"), (dict(kc=None), EINVAL, "null cache"),
    (dict(q_gain=None), EINVAL, "gains"), (dict(k_gain=None), EINVAL, "gains"), (dict(rows=0), EINVAL, "shape"),
    (dict(n_q=0), EINVAL, "shape"), (dict(tab_rows=0), EINVAL, "shape"), (dict(q_stride=2047), EINVAL, "shape"),
    (dict(k_stride=1023), EINVAL, "shape"), (dict(v_stride=1), EINVAL, "shape"), (dict(q_out_stride=2047), EINVAL, "shape"),
    (dict(eps=-1.0), EINVAL, "eps"), (dict(eps=float("nan")), EINVAL, "eps"), (dict(n_kv=0), EINVAL, "cache shape"),
    (dict(n_pages=0), EINVAL, "cache shape"), (dict(page=48), EUNSUPPORTED, "pages hold"), (dict(hd=96), EUNSUPPORTED, "head_dim"),
    (dict(vc=C.c_void_p(0x1008)), EINVAL, "aligned"), (dict(q_out_stride=2056), EINVAL, "another stride"),
    (dict(rows=2 ** 31 - 1, n_kv=64, k_stride=8192, v_stride=8192), EUNSUPPORTED, "too many"),
    (dict(n_q=(1 << 24) + 1, q_stride=1 << 32, q_out_stride=1 << 32), EUNSUPPORTED, "too many")])
def test_qkv_append_refuses(native, kw, code, word):
    _refused(native, "bx_qkv_append_q8_f16", _with(QKV, **kw), code, word)


ATTN = [("q", P), ("q_stride", 2048), ("rows", 5), ("starts", P), ("lens", P), ("n_req", 3), ("max_new", 2), ("max_len", 500),
        ("pos", P), ("shared", P), ("order", P), ("groups", P), ("group_starts", P), ("max_groups", 1), ("max_shared", 900),
        ("table", P), ("max_blocks", 10)] + CACHE + [
            ("n_q", 16), ("n_kv", 8), ("hd", 128), ("window", 0), ("out", P), ("out_stride", 2048), ("ws", P),
            ("ws_bytes", 1 << 40), ("stream", None)]


@pytest.mark.parametrize("kw,code,word", [
    (dict(q=None), EINVAL, "null"), (dict(starts=None), EINVAL, "null"), (dict(pos=None), EINVAL, "null"),
    (dict(shared=None), EINVAL, "null"), (dict(order=None), EINVAL, "null"), (dict(groups=None), EINVAL, "null"),
    (dict(group_starts=None), EINVAL, "null"), (dict(ws=None), EINVAL, "null"), (dict(kc=None), EINVAL, "null cache"),
    (dict(rows=0), EINVAL, "shape"), (dict(n_req=0), EINVAL, "shape"), (dict(max_new=0), EINVAL, "shape"),
    (dict(max_len=0), EINVAL, "shape"), (dict(max_groups=0), EINVAL, "shape"), (dict(max_shared=0), EINVAL, "shape"),
    (dict(max_blocks=0), EINVAL, "shape"), (dict(n_q=15), EINVAL, "shape"), (dict(window=-1), EINVAL, "shape"),
    (dict(n_q=136), EUNSUPPORTED, "larger than 16"), (dict(q_stride=2047), EINVAL, "stride"),
    (dict(out_stride=2047), EINVAL, "stride"), (dict(max_blocks=1 << 25), EUNSUPPORTED, "tokens a request"),
    (dict(ws_bytes=16), EINVAL, "workspace"), (dict(ws=C.c_void_p(0x1008)), EINVAL, "workspace"),
    (dict(hd=80), EUNSUPPORTED, "head_dim"), (dict(page=0), EUNSUPPORTED, "pages hold"),
    (dict(kc=C.c_void_p(0x1001)), EINVAL, "aligned"),
    (dict(n_q=1 << 18, n_kv=1 << 18, page=128, q_stride=1 << 26, out_stride=1 << 26), EUNSUPPORTED, "2^31 bytes")])
def test_attention_prefix_refuses(native, kw, code, word):
    _refused(native, "bx_attention_prefix_q8_f16", _with(ATTN, **kw), code, word)


def test_attention_prefix_workspace_query(native):
    f = native.hip().bx_attention_prefix_q8_workspace_bytes
    own = native.hip().bx_attention_paged_q8_workspace_bytes
    assert f(0, 1, 16, 8, 128, 1, 100, 1, 100) == 0 and f(1, 1, 15, 8, 128, 1, 100, 1, 100) == 0
    assert f(1, 1, 16, 8, 128, 1, 100, 0, 100) == 0 and f(1, 1, 16, 8, 128, 1, 100, 1, 0) == 0
    assert f(4, 5, 16, 8, 128, 1, 100, 1, 100) >= own(4, 5, 16, 8, 128, 1, 100)
    assert f(300, 5, 16, 8, 128, 60, 100, 1, 100) > own(300, 5, 16, 8, 128, 60, 100)
    assert f(4, 5, 16, 8, 128, 1, 100, 1, 100000) > f(4, 5, 16, 8, 128, 1, 100, 1, 100)


def test_host_plan_and_attention_agree_with_copies():
    """The plain form over shared keys equals the plain form of independent requests that hold copies."""
    rng = np.random.default_rng(1)
    n_kv, n_q, hd, page = 2, 4, 64, 16
    cache = pu.empty_cache(20, n_kv, page, hd, rng)
    table = np.array([[3, 7, 9, -1, -1], [1, 2, -1, -1, -1], [4, -1, -1, -1, -1]], np.int32)
    lens, starts = [48, 20, 5], np.array([0, 0, 3, 4])
    q = rng.standard_normal((4, n_q, hd)).astype(np.float16)
    copies = np.array([[3, 7, 9, -1, -1], [3, 7, 9, 1, 2], [3, 7, 4, -1, -1]], np.int32)
    for window in (0, 30):
        a = px.attention(cache, q, starts, lens, table, [-1, 0, 0], [0, 48, 32], n_kv, window)
        b = pu.attention(cache, q, starts, [48, 68, 37], copies, n_kv, window)
        np.testing.assert_allclose(a[0], b[0], rtol=1e-12, atol=1e-14)
        np.testing.assert_allclose(a[1], b[1], rtol=1e-9, atol=1e-12)
    pos, shared, order, groups, first = px.plan([-1, 0, 0], [0, 48, 32], starts, lens, [17, 18, 19, 4, -1])
    assert list(pos) == [65, 66, 67, 36, -1] and list(shared) == [48, 48, 48, 32, 0]
    assert list(order) == [0, 1, 2, 3, -1] and list(groups) == [0, -1, -1] and list(first) == [0, 4, 4, 4]
