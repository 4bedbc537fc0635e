"""A request none of whose positions counts, since every page id is out of
range, gives what a request of length 0 gives: a zero row and lse = -inf (the
scores of positions that count may all be -inf: that is 0 / 0, as the formula
says)."""

from __future__ import annotations

import math

import numpy as np
import pytest

from conftest import rel_frobenius
from test_paged_gpu import BAD_INDEX, TOL, Case, _status, clean_status, lib  # noqa: F401

pytestmark = pytest.mark.gpu

FORMS = [(2, 2, 64, "float32"), (2, 2, 128, "float16"), (8, 2, 64, "float32"), (8, 1, 128, "float16"),
         (4, 1, 128, "bfloat16"), (24, 2, 128, "bfloat16"), (16, 1, 64, "float16"),
         (6, 2, 256, "float32"), (2, 2, 5, "float32"), (6, 2, 33, "float16")]


@pytest.mark.parametrize("heads, kv_heads, dim, dtype", FORMS)
def test_every_page_id_is_bad(lib, heads, kv_heads, dim, dtype):  # noqa: F811
    # whole requests, and one cut into parts
    c = Case(lib, [40, 100, 7, 3000 if dim > 33 else 300], heads, kv_heads, dim, 16, dtype)
    c.table[0] = 1 << 30
    c.table[3] = -1
    out, lse = c.run()
    assert _status(lib) == BAD_INDEX
    want, want_lse = c.want()
    for r in (0, 3):
        assert (out[r] == 0).all() and (lse[r] == -np.inf).all()
    assert rel_frobenius(out[1:3], want[1:3]) <= TOL
    assert np.max(np.abs(lse[1:3] - want_lse[1:3])) <= 1e-5 * max(1, np.abs(want_lse[1:3]).max())


@pytest.mark.parametrize("heads, kv_heads, dim, dtype", FORMS)
def test_one_page_counts(lib, heads, kv_heads, dim, dtype):  # noqa: F811
    """The parts without a position add nothing to the one that has some."""
    n = 3000 if dim > 33 else 300
    c = Case(lib, [n], heads, kv_heads, dim, 16, dtype)
    keep = (2 * n // 3) // 16
    good = int(c.table[0, keep])
    c.table[0] = -1
    c.table[0, keep] = good
    k, v = c.rows[0]
    c.rows[0] = k[:, keep * 16:keep * 16 + 16], v[:, keep * 16:keep * 16 + 16]
    out, lse = c.run()
    want, want_lse = c.want()
    assert rel_frobenius(out, want) <= TOL and np.max(np.abs(lse - want_lse)) <= 1e-5 * 10
    # that page's scores -inf: NaN and -inf, whatever the others are
    if dtype == "float32":
        c.q[:] = 0.0
        c.q[..., 0] = 1.0
        c.k[good] = 0.0
        c.k[good, :, :, 0] = -math.inf
        out, lse = c.run()
        assert np.isnan(out).all()
        if heads == kv_heads:  # an infinite key may make a group's scores NaN
            assert (lse == -np.inf).all()
