"""What the paged-cache and row-sampling entry points refuse, on the CPU: every
check stands before the first GPU call."""
from __future__ import annotations

import ctypes as C

import pytest

P = C.c_void_p(0x1000)   # never read: the call is refused first
EINVAL, EUNSUPPORTED = -1, -3


def _refused(native, name, args, code, word):
    h = native.hip()
    assert getattr(h, name)(*args) == code, (name, args)
    msg = h.bx_last_error().decode()
    assert word in msg, msg


def _with(base, **kw):
    keys, vals = zip(*base)
    return [kw.get(k, v) for k, v in zip(keys, vals)]


PLAN = [("past", P), ("delta", C.c_void_p(0x2000)), ("n_req", 4), ("page", 64), ("n_pages", 100), ("table", P),
        ("max_blocks", 10), ("ring", P), ("ends_in", P), ("ends_out", P), ("lens", P), ("starts", C.c_void_p(0x3000)),
        ("slots", P), ("pos", P), ("max_rows", 10), ("status", P), ("ws", P), ("ws_bytes", 256), ("stream", None)]


@pytest.mark.parametrize("kw,code,word", [
    (dict(past=None), EINVAL, "null"), (dict(status=None), EINVAL, "null"), (dict(ws=None), EINVAL, "null"),
    (dict(n_req=0), EINVAL, "shape"), (dict(max_rows=0), EINVAL, "shape"), (dict(n_pages=-1), EINVAL, "shape"),
    (dict(n_req=4097), EUNSUPPORTED, "4096"), (dict(page=48), EUNSUPPORTED, "pages hold"),
    (dict(page=256), EUNSUPPORTED, "pages hold"), (dict(max_blocks=1 << 26), EUNSUPPORTED, "tokens a request"),
    (dict(ws_bytes=255), EINVAL, "workspace"), (dict(ws=C.c_void_p(0x1004)), EINVAL, "workspace"),
    (dict(lens=C.c_void_p(0x2000)), EINVAL, "over past"), (dict(starts=P), EINVAL, "over past")])
def test_plan_refuses(native, kw, code, word):
    assert native.hip().bx_kv_plan_workspace_bytes() == 256
    _refused(native, "bx_kv_plan", _with(PLAN, **kw), code, word)


CACHE = [("page", 64), ("n_pages", 100), ("kc", P), ("vc", P), ("ks", P), ("vs", P)]
APPEND = [("k", P), ("k_stride", 1024), ("v", P), ("v_stride", 1024), ("rows", 5), ("n_kv", 8), ("hd", 128),
          ("slots", P)] + CACHE + [("stream", None)]
READ = [("slots", P), ("rows", 5), ("n_kv", 8), ("hd", 128)] + CACHE + [("k", P), ("k_stride", 1024), ("v", P),
                                                                      ("v_stride", 1024), ("stream", None)]
CACHE_REFUSALS = [
    (dict(k=None), EINVAL, "null"), (dict(slots=None), EINVAL, "null"), (dict(kc=None), EINVAL, "null cache"),
    (dict(vs=None), EINVAL, "null cache"), (dict(rows=0), EINVAL, "shape"), (dict(k_stride=1023), EINVAL, "shape"),
    (dict(v_stride=0), EINVAL, "shape"), (dict(n_kv=0), EINVAL, "cache shape"), (dict(n_pages=0), EINVAL, "cache shape"),
    (dict(page=8), EUNSUPPORTED, "pages hold"), (dict(hd=96), EUNSUPPORTED, "head_dim"),
    (dict(vc=C.c_void_p(0x1008)), EINVAL, "aligned")]


@pytest.mark.parametrize("kw,code,word", CACHE_REFUSALS)
@pytest.mark.parametrize("name,base", [("bx_kv_append_q8_f16", APPEND), ("bx_kv_read_q8_f16", READ)])
def test_append_and_read_refuse(native, name, base, kw, code, word):
    _refused(native, name, _with(base, **kw), code, word)


ATTN = [("q", P), ("q_stride", 2048), ("rows", 5), ("starts", P), ("lens", P), ("n_req", 3), ("max_new", 2),
        ("max_len", 500), ("table", P), ("max_blocks", 10)] + CACHE + [
            ("n_q", 16), ("n_kv", 8), ("hd", 128), ("window", 0), ("out", P), ("out_stride", 2048), ("ws", P),
            ("ws_bytes", 1 << 40), ("stream", None)]


@pytest.mark.parametrize("kw,code,word", [
    (dict(q=None), EINVAL, "null"), (dict(table=None), EINVAL, "null"), (dict(ws=None), EINVAL, "null"),
    (dict(kc=None), EINVAL, "null cache"), (dict(rows=0), EINVAL, "shape"), (dict(n_req=0), EINVAL, "shape"),
    (dict(max_new=0), EINVAL, "shape"), (dict(max_len=0), EINVAL, "shape"), (dict(n_q=15), EINVAL, "shape"),
    (dict(window=-1), EINVAL, "shape"), (dict(n_q=136), EUNSUPPORTED, "larger than 16"),
    (dict(q_stride=2047), EINVAL, "stride"), (dict(out_stride=2047), EINVAL, "stride"),
    (dict(max_blocks=1 << 25), EUNSUPPORTED, "tokens a request"), (dict(ws_bytes=16), EINVAL, "workspace"),
    (dict(ws=C.c_void_p(0x1008)), EINVAL, "workspace"), (dict(hd=80), EUNSUPPORTED, "head_dim"),
    (dict(page=0), EUNSUPPORTED, "pages hold"), (dict(kc=C.c_void_p(0x1001)), EINVAL, "aligned")])
def test_attention_refuses(native, kw, code, word):
    _refused(native, "bx_attention_paged_q8_f16", _with(ATTN, **kw), code, word)


def test_attention_workspace_query(native):
    f = native.hip().bx_attention_paged_q8_workspace_bytes
    assert f(0, 1, 16, 8, 128, 1, 100) == 0 and f(1, 1, 15, 8, 128, 1, 100) == 0
    assert f(1, 1, 16, 8, 128, 1, 100) > 0
    assert f(1, 1, 16, 8, 128, 1, 100000) > f(1, 1, 16, 8, 128, 1, 100)


SAMPLE = [("logits", P), ("stride", 1000), ("rows", 4), ("vocab", 1000), ("t", P), ("k", None), ("p", None),
          ("m", None), ("u", P), ("out", P), ("stream", None)]


@pytest.mark.parametrize("kw,code,word", [
    (dict(logits=None), EINVAL, "null"), (dict(t=None), EINVAL, "null"), (dict(u=None), EINVAL, "null"),
    (dict(out=None), EINVAL, "null"), (dict(rows=0), EINVAL, "shape"), (dict(vocab=0), EINVAL, "shape"),
    (dict(stride=999), EINVAL, "shape"), (dict(vocab=4194305, stride=1 << 23), EUNSUPPORTED, "4194304")])
def test_sample_rows_refuses(native, kw, code, word):
    _refused(native, "bx_sample_rows_f16", _with(SAMPLE, **kw), code, word)
