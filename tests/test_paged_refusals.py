"""Argument checks of the paged KV cache and logits entry points, on the host
(no GPU): each refusal returns its code and launches nothing."""

from __future__ import annotations

import ctypes

import pytest

from tvarant_b200 import capi

P = ctypes.c_void_p(256)  # never dereferenced: every call below is refused, or empty


def cache(**kw):
    d = dict(k=256, v=256, page_type=0, num_pages=4, page_size=16, kv_heads=2, head_dim=64)
    d.update(kw)
    strides = (ctypes.c_int64 * 3)(2048, 1024, 64)
    return capi.PagedKV(d["k"], d["v"], d["page_type"], 0, d["num_pages"], d["page_size"],
                        d["kv_heads"], d["head_dim"], strides, strides)


def pool(**kw):
    d = dict(table=256, stride=8, max_pages=8, requests=4, free=256, num_pages=16, page_size=16)
    d.update(kw)
    return capi.PagePool(d["table"], d["stride"], d["max_pages"], d["requests"], d["free"],
                         d["num_pages"], d["page_size"])


def plan(pl, seq=P, new=P, seq_out=P, count=P, count_out=P, slots=P, tokens=4, per=0):
    return capi.try_call("tvr_page_plan", pl, seq, new, seq_out, count, count_out, slots, None,
                         None, tokens, per, None)


@pytest.mark.parametrize("kw, text", [
    (dict(page_size=0), "page size"), (dict(page_size=(1 << 20) + 1), "page size"),
    (dict(requests=-1), "negative"), (dict(max_pages=-1), "negative"),
    (dict(num_pages=-1), "negative"), (dict(stride=7), "stride"),
    (dict(table=None), "block table"), (dict(free=None), "free pages"),
    (dict(max_pages=1 << 28, stride=1 << 28), "too many"),
    (dict(num_pages=0x7fffffff), "too many"),
])
def test_page_plan_refuses_a_bad_pool(kw, text):
    assert plan(pool(**kw)) == capi.ERR_INVALID
    assert text in capi.last_error()


@pytest.mark.parametrize("kw, text", [
    (dict(seq=None), "null lengths"), (dict(new=None), "null lengths"),
    (dict(seq_out=None), "null lengths"), (dict(count=None), "free count"),
    (dict(count_out=None), "free count"), (dict(slots=None), "null slots"),
    (dict(tokens=-1), "negative"), (dict(per=-1), "negative"),
    (dict(tokens=1 << 32), "too many"),
])
def test_page_plan_refuses_bad_arguments(kw, text):
    assert plan(pool(), **kw) == capi.ERR_INVALID
    assert text in capi.last_error()


def test_page_plan_takes_8192_requests_at_most():
    assert plan(pool(requests=8193)) == capi.ERR_UNSUPPORTED
    assert "8192" in capi.last_error()
    assert capi.try_call("tvr_page_plan", None, P, P, P, P, P, P, None, None, 0, 0,
                         None) == capi.ERR_INVALID


def append(c, k=P, v=P, strides=True, slots=P, tokens=3):
    st = (ctypes.c_int64 * 4)(128, 64, 128, 64) if strides else None
    return capi.try_call("tvr_paged_append", c, k, v, st, slots, tokens, None)


@pytest.mark.parametrize("c, kw, text", [
    (dict(page_type=3), {}, "page type"), (dict(page_type=-1), {}, "page type"),
    (dict(page_size=0), {}, "page size"), (dict(num_pages=-1), {}, "negative"),
    (dict(kv_heads=70000), {}, "too many"), (dict(k=None), {}, "null pages"),
    ({}, dict(k=None), "null pointer"), ({}, dict(v=None), "null pointer"),
    ({}, dict(strides=False), "null pointer"), ({}, dict(slots=None), "null pointer"),
    ({}, dict(tokens=-1), "negative"),
])
def test_paged_append_refuses(c, kw, text):
    assert append(cache(**c), **kw) == capi.ERR_INVALID
    assert text in capi.last_error()


def test_empty_calls_launch_nothing():
    assert append(cache(), k=None, v=None, slots=None, tokens=0) == capi.OK
    assert append(cache(kv_heads=0)) == capi.OK
    assert attend(cache(), requests=0, q=None, lens=None) == capi.OK
    assert capi.try_call("tvr_adjust_logits", None, 0, None, 0, 0, 100, capi.LogitRules(),
                         None) == capi.OK
    assert capi.try_call("tvr_history_append", None, 32, 0, None, None, None, 0, 0,
                         None) == capi.OK


def attend(c, q=P, k_new=None, v_new=None, slots=None, table=P, stride=8, max_pages=8, lens=P,
           out=P, requests=2, heads=4, strides=True, scale=0.125, ws=P, ws_bytes=1 << 30):
    st = (ctypes.c_int64 * 8)(256, 64, 128, 64, 128, 64, 256, 64) if strides else None
    return capi.try_call("tvr_paged_attention", c, q, k_new, v_new, slots, table, stride, max_pages,
                         lens, out, None, requests, heads, st, scale, ws, ws_bytes, None)


@pytest.mark.parametrize("c, kw, text", [
    (dict(page_type=7), {}, "page type"), (dict(page_size=0), {}, "page size"),
    ({}, dict(requests=-1), "negative"), ({}, dict(max_pages=-1), "negative"),
    ({}, dict(heads=5), "share"), (dict(kv_heads=0), {}, "share"),
    ({}, dict(q=None), "null pointer"), ({}, dict(out=None), "null pointer"),
    ({}, dict(lens=None), "null pointer"), ({}, dict(strides=False), "null pointer"),
    ({}, dict(table=None), "block table"), (dict(v=None), {}, "null pages"),
    ({}, dict(slots=P), "together"), ({}, dict(k_new=P, v_new=P), "together"),
    ({}, dict(k_new=P, slots=P), "together"), ({}, dict(stride=7), "stride"),
    ({}, dict(max_pages=1 << 28, stride=1 << 28), "too many"),
    ({}, dict(requests=1 << 30), "too many"),
    ({}, dict(scale=float("nan")), "finite"), ({}, dict(scale=float("inf")), "finite"),
])
def test_paged_attention_refuses(c, kw, text):
    assert attend(cache(**c), **kw) == capi.ERR_INVALID
    assert text in capi.last_error()


def test_paged_attention_needs_its_workspace():
    size = ctypes.c_int64()
    capi.call("tvr_paged_attention_workspace", 4, 2, 64, ctypes.byref(size))
    assert size.value > 0
    for kw in (dict(ws=None), dict(ws_bytes=size.value - 1)):
        assert attend(cache(), **kw) == capi.ERR_INVALID
        assert "workspace" in capi.last_error()
    assert attend(cache(), ws=ctypes.c_void_p(264)) == capi.ERR_INVALID
    assert "aligned" in capi.last_error()


def test_paged_attention_takes_256_dimensions_at_most():
    assert attend(cache(head_dim=264)) == capi.ERR_UNSUPPORTED
    assert "256" in capi.last_error()
    assert capi.try_call("tvr_paged_attention_workspace", 5, 2, 64,
                         ctypes.byref(ctypes.c_int64())) == capi.ERR_INVALID
    assert capi.try_call("tvr_paged_attention_workspace", 4, 2, 64, None) == capi.ERR_INVALID


def rules(**kw):
    r = capi.LogitRules()
    for k, v in kw.items():
        setattr(r, k, v)
    return r


@pytest.mark.parametrize("r, kw, text", [
    (rules(), dict(rows=-1), "negative"), (rules(), dict(x=None), "null pointer"),
    (rules(), dict(stride=99), "stride"), (rules(), dict(rows=70000), "too many"),
    (rules(), dict(out=P, x=P, out_stride=200), "in place"),
    (rules(tokens=256, token_bits=16, total_lens=256), {}, "token_bits"),
    (rules(tokens=256, token_bits=32), {}, "lengths"),
    (rules(tokens=256, token_bits=32, total_lens=256, tokens_stride=-1), {}, "stride"),
    (rules(bias_ids=256), {}, "values"),
    (rules(bias_ids=256, bias_values=256, bias_stride=-1), {}, "stride"),
    (rules(masks=256, mask_stride=3, n_masks=2), {}, "mask row"),
    (rules(masks=256, mask_stride=4, n_masks=2), dict(rows=3), "fewer masks"),
])
def test_adjust_logits_refuses(r, kw, text):
    a = dict(x=P, stride=100, out=ctypes.c_void_p(4096), out_stride=100, rows=2, vocab=100)
    a.update(kw)
    assert capi.try_call("tvr_adjust_logits", a["x"], a["stride"], a["out"], a["out_stride"],
                         a["rows"], a["vocab"], r, None) == capi.ERR_INVALID
    assert text in capi.last_error()
    assert capi.try_call("tvr_adjust_logits", P, 100, P, 100, 2, 100, None,
                         None) == capi.ERR_INVALID


@pytest.mark.parametrize("kw, text", [
    (dict(bits=8), "token_bits"), (dict(rows=-1), "negative"), (dict(lens=None), "null pointer"),
    (dict(ids=None), "null pointer"), (dict(tokens=None), "null pointer"),
    (dict(stride=9), "stride"), (dict(capacity=1 << 33, stride=1 << 33), "32 bits"),
])
def test_history_append_refuses(kw, text):
    a = dict(tokens=P, bits=32, stride=10, lens=P, ids=P, rows=2, capacity=10)
    a.update(kw)
    assert capi.try_call("tvr_history_append", a["tokens"], a["bits"], a["stride"], a["lens"],
                         a["ids"], None, a["rows"], a["capacity"], None) == capi.ERR_INVALID
    assert text in capi.last_error()
