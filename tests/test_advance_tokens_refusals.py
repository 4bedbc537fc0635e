"""Argument checks of tvr_advance_tokens, on the host (no GPU)."""

from __future__ import annotations

import ctypes

import pytest

from tvarant_b200 import capi

P = ctypes.c_void_p(256)  # never dereferenced: every call below is refused, or empty


@pytest.mark.parametrize("kw, text", [
    (dict(current=None), "null pointer"), (dict(nxt=None), "null pointer"),
    (dict(slots=None), "null pointer"), (dict(tokens=None), "null pointer"),
    (dict(bits=8), "token_bits"), (dict(rows=-1), "negative"), (dict(capacity=-1), "negative"),
    (dict(stride=9), "stride"), (dict(capacity=1 << 33, stride=1 << 33), "32 bits"),
])
def test_advance_tokens_refuses(kw, text):
    a = dict(current=P, nxt=P, slots=P, tokens=P, bits=32, stride=10, lens=P, rows=2, capacity=10)
    a.update(kw)
    assert capi.try_call("tvr_advance_tokens", a["current"], a["nxt"], a["slots"], a["tokens"],
                         a["bits"], a["stride"], a["lens"], a["rows"], a["capacity"],
                         None) == capi.ERR_INVALID
    assert text in capi.last_error()


def test_no_rows():
    assert capi.try_call("tvr_advance_tokens", None, None, None, None, 32, 0, None, 0, 0,
                         None) == capi.OK
