"""Requests end at ``max_len`` positions, whole pages or not: the page plan
refuses what goes past it, and GPT-2 never computes a position that it has no
embedding for."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpt2_paged_refused_gpu import CACHE_FULL, Server, model  # noqa: F401
from test_paged_gpu import _plan_oracle, _pool_state, _status, clean_status, lib  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_len, page", [(128, 24), (128, 16), (61, 8)])
def test_a_request_ends_at_max_len(model, max_len, page):  # noqa: F811
    rng = np.random.default_rng(max_len + page)
    prompt = rng.integers(0, 1009, max_len - 2).tolist()
    s = Server(model, [prompt, [3]], 20, page, False, max_len)
    s.step([1, 1], advances=[0, 1])
    s.step([1, 1], advances=[0, 1])
    assert s.status() == 0
    s.step([1, 1], advances=[1])
    assert s.status() == CACHE_FULL and s.cache.seq_lens.cpu().tolist() == [max_len, 4]


def _run(lib, pool, s, n, c, tokens, per):  # noqa: F811
    import torch

    slots = torch.full((tokens,), -99, dtype=torch.int64, device="cuda")
    pos, rows = (torch.full((tokens,), -99, dtype=torch.int32, device="cuda") for _ in range(2))
    lib.call("tvr_page_plan", pool, s.data_ptr(), n.data_ptr(), s.data_ptr(), c.data_ptr(),
             c.data_ptr(), slots.data_ptr(), pos.data_ptr(), rows.data_ptr(), tokens, per,
             torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return [x.cpu().numpy() for x in (slots, pos, rows)]


@pytest.mark.parametrize("per", [0, 9])
@pytest.mark.parametrize("requests", [5, 300])
def test_plan_refuses_past_max_positions(lib, requests, per):  # noqa: F811
    """As if the requests that would go past it asked for more than their table
    has: those are refused, the others get what they get without them."""
    import torch

    rng = np.random.default_rng(requests + per)
    page, limit, max_pages, spare = 16, 41, 8, 4 * requests
    lens = rng.integers(0, limit + 1, requests).astype(np.int32)
    new = rng.choice([-1, 0, 1, 1, 2, 9], requests).astype(np.int32)
    lens[:3], new[:3] = [limit, limit - 1, limit], [1, 1, 0]
    table, free = _pool_state(rng, lens, page, max_pages, spare)
    tokens = requests * per if per else int(new[new > 0].sum()) + 3
    t, s, n, f = (torch.from_numpy(x).cuda() for x in (table, lens, new, free))
    c = torch.tensor([spare], dtype=torch.int32, device="cuda")
    pool = lib.PagePool(t.data_ptr(), max_pages, max_pages, requests, f.data_ptr(), f.numel(), page,
                        limit)
    slots, pos, rows = _run(lib, pool, s, n, c, tokens, per)
    over = (new > 0) & (lens + new > limit)
    assert over.any()
    served = np.where(over, 0, new).astype(np.int32)
    total = requests * per if per else int(served[served > 0].sum())
    want = _plan_oracle(table, lens, served, free, spare, page, total, per)
    assert not want[7]
    assert np.array_equal(t.cpu().numpy(), want[0]) and np.array_equal(s.cpu().numpy(), want[1])
    assert np.array_equal(f.cpu().numpy(), want[2]) and int(c) == want[3]
    # the tokens of refused requests have their places, and no slots
    gone = np.isin(rows, np.nonzero(over)[0])
    assert (slots[gone] == -1).all() and gone.sum() == new[over].sum()
    assert np.array_equal(slots[slots >= 0], want[4][want[4] >= 0])
    assert np.array_equal(pos[slots >= 0], want[5][want[4] >= 0])
    assert _status(lib) == CACHE_FULL
