"""Scores and queries so large that their rounding or their range shows: the
outputs stay finite, and equal to the formula where the scores' bits decide it."""

from __future__ import annotations

import math

import numpy as np
import pytest

from conftest import rel_frobenius
from test_paged_gpu import Case, _status, clean_status, lib  # noqa: F401

pytestmark = pytest.mark.gpu

F16 = [(8, 1, 64, "float16"), (8, 1, 128, "float16"), (16, 1, 128, "float16"), (4, 2, 256, "float16")]
OTHERS = [(8, 1, 64, "float32"), (8, 1, 64, "bfloat16"), (4, 1, 128, "bfloat16"),
          (2, 2, 64, "float16"), (2, 2, 7, "float32")]


def _two_levels(lib, heads, kv_heads, dim, dtype, power, step):  # noqa: F811
    """Scores (in the exp2 domain) of 1.5 * 2^power at the first 128 positions
    and `step` more at the other 128."""
    requests = 64 if heads == 16 else 1  # enough for units of 16 heads
    c = Case(lib, [256] * requests, heads, kv_heads, dim, 16, dtype, spare=0)
    up = 1.0 / (np.float64(np.float32(c.scale)) * math.log2(math.e))
    c.q[:] = 0.0
    c.q[..., 0] = 1.5 * 2.0**power * up
    c.q[..., 1] = step * up
    c.k[:] = 0.0
    c.k[..., 0] = 1.0
    for r in range(requests):
        for i in range(8, 16):
            c.k[int(c.table[r, i]), :, :, 1] = 1.0
        k, _ = c.rows[r]
        k[:] = 0.0
        k[:, :, 0] = 1.0
        k[:, 128:, 1] = 1.0
    return c


@pytest.mark.parametrize("heads, kv_heads, dim, dtype", F16)
@pytest.mark.parametrize("power, step", [(20, 4.0), (24, 4.0), (25, 8.0)])
def test_f16_weights_of_large_scores(lib, heads, kv_heads, dim, dtype, power, step):  # noqa: F811
    """A step that scores of 22 bits still hold (2^(power - 22) divides it).
    All keys share the large part of their scores, whose rounding falls
    out; weights of 1 and 2^step are exact, so the outputs are good to the
    errors of sums of 256 of them."""
    c = _two_levels(lib, heads, kv_heads, dim, dtype, power, step)
    out, _ = c.run()
    assert np.isfinite(out).all()
    for r in range(len(c.lens)):
        v = np.repeat(c.rows[r][1], heads // kv_heads, 0)
        w = np.where(np.arange(256) < 128, 2.0**-step, 1.0)
        want = np.einsum("j,hjd->hd", w / w.sum(), v)
        # the step itself is a query of 24 bits times the scale: 2^-22 of `step`
        assert rel_frobenius(out[r], want) <= 1e-5
    assert _status(lib) == 0


@pytest.mark.parametrize("heads, kv_heads, dim, dtype", F16 + OTHERS)
def test_outputs_stay_finite(lib, heads, kv_heads, dim, dtype):  # noqa: F811
    for power in (24, 25, 26, 27, 28, 100):
        for step in (2.0, 8.0, 16.0, 64.0):
            out, lse = _two_levels(lib, heads, kv_heads, dim, dtype, power, step).run()
            assert np.isfinite(out).all() and np.isfinite(lse).all(), (power, step)


@pytest.mark.parametrize("heads, kv_heads, dim, dtype", F16 + OTHERS)
def test_queries_near_the_largest(lib, heads, kv_heads, dim, dtype):  # noqa: F811
    """Queries of 2^118: the position of the largest score takes all of the
    weight, and its value is the output, to the 22 bits of an fp32 value's two
    terms at least."""
    c = Case(lib, [50, 200], heads, kv_heads, dim, 16, dtype)
    c.q *= 2.0**118
    out, _ = c.run()
    q = c.q.cpu().double().numpy()
    for r in range(2):
        k, v = c.rows[r]
        for h in range(heads):
            g = h // (heads // kv_heads)
            z = np.sort(k[g] @ q[r, h])
            if z[-1] - z[-2] > 1e-4 * abs(z[-1]):  # not a tie within the scores' errors
                one = v[g, np.argmax(k[g] @ q[r, h])]
                assert np.max(np.abs(out[r, h] - one)) <= 2.0**-20 * np.max(np.abs(one))
