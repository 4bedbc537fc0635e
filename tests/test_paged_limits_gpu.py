"""The paged operators at their limits: a plan of 8192 requests, rows of more
than 1024 tokens, and one workspace for attention calls of every shape."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

from test_paged_gpu import (CACHE_FULL, Case, _plan_oracle, _pool_state, _run_plan, _status,  # noqa: F401
                            clean_status, lib)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("requests, news, spare, per", [
    (8192, [-1, 0, 1, 1, 1], 9000, 0),       # more tokens than one CTA takes
    (8192, [-1, 0, 0, 0, 0, 0, 0, 0, 0, 1], 20, 0),  # fewer; some of them refused
    (8192, [-1, 0, 1], 300, 1),
    (700, [-1, 0, 1, 2, 5], 3000, 4),        # requests with more than their row
])
def test_plans_of_many_requests(lib, requests, news, spare, per, in_place):  # noqa: F811
    rng = np.random.default_rng(requests + spare)
    lens = rng.integers(0, 30, requests).astype(np.int32)
    new = rng.choice(news, requests).astype(np.int32)
    table, free = _pool_state(rng, lens, 8, 5, spare)
    tokens = requests * per if per else int(new[new > 0].sum()) + 3
    want = _plan_oracle(table, lens, new, free, spare, 8, tokens, per)
    got = _run_plan(lib, table, lens, new, free, spare, 8, tokens, per, in_place)
    for name, g, w in zip(("table", "lens", "free", "count", "slots", "positions", "rows"), got,
                          [*want[:3], np.array([want[3]]), *want[4:7]]):
        assert np.array_equal(g, w), name
    assert _status(lib) == (CACHE_FULL if want[7] else 0)


def test_one_workspace_for_every_shape(lib):  # noqa: F811
    """Each call leaves all counters at zero and does not read what the call
    before it left behind them."""
    cases = []
    for heads, kv_heads, dim, dtype, lens in (
            (12, 12, 64, "float32", [5000, 3]), (16, 1, 128, "float16", [12345]),
            (40, 1, 128, "bfloat16", [20000]), (24, 2, 256, "float32", [3000, 0, 40]),
            (4, 1, 128, "bfloat16", [9, 30000]), (16, 1, 64, "float16", [100] * 70 + [9000]),
            (2, 2, 128, "float32", [40] * 200)):
        cases.append(Case(lib, lens, heads, kv_heads, dim, 16, dtype))
    alone = [c.check() for c in cases]
    size = max(c.workspace.numel() for c in cases)
    workspace = cases[0].torch.zeros(size, dtype=cases[0].torch.uint8, device="cuda")
    counters = 3 * 640 * ctypes.sizeof(ctypes.c_int)
    for c in cases:
        c.workspace = workspace
    for order in (range(len(cases)), reversed(range(len(cases)))):
        for i in order:
            out, lse = cases[i].run()
            assert np.array_equal(out, alone[i][0]) and np.array_equal(lse, alone[i][1])
            assert not workspace[:counters].any()
