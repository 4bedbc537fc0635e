"""Lengths that GPT-2 has no positions for are refused on the host (no GPU)."""

from __future__ import annotations

import pytest
import torch

from tvarant_b200 import gpt2
from tvarant_b200.paged import PagedCache


@pytest.fixture(scope="module")
def model():
    return gpt2.init_gpt2(gpt2.GPT2Config(n_layer=1, d_model=64, n_head=2, d_ff=64, vocab=50,
                                          n_ctx=20))


def cache(pages, max_len):
    z = torch.zeros(1, dtype=torch.int32)
    k = [torch.zeros(4, 2, 8, 32)]
    return PagedCache(k, k, torch.zeros(1, pages, dtype=torch.int32), z, torch.zeros(4), z,
                      torch.zeros(1, dtype=torch.uint8), max_len)


def test_a_cache_past_the_context_is_refused(model):
    with pytest.raises(ValueError, match="21 positions"):
        gpt2.new_paged_cache(model, 1, 4, 8, 21, "tvarant")


@pytest.mark.parametrize("tokens, c", [(21, cache(3, 20)), (11, cache(2, 10)), (17, cache(2, 0))])
def test_a_prompt_past_the_cache_is_refused(model, tokens, c):
    with pytest.raises(ValueError, match=f"{tokens} positions"):
        gpt2.paged_prefill(model, torch.zeros(1, tokens, dtype=torch.int64), c, 0)


def test_steps_over_a_cache_past_the_context_are_refused(model):
    for c in (cache(3, 0), cache(4, 21)):  # 24 positions, and 21
        with pytest.raises(ValueError, match="context of 20"):
            gpt2.paged_decode_step(model, torch.zeros(1, 1, dtype=torch.int64), c,
                                   torch.ones(1, dtype=torch.int32))
        with pytest.raises(ValueError, match="context of 20"):
            gpt2.paged_prefill(model, torch.zeros(1, 3, dtype=torch.int64), c, 0)


def test_a_negative_limit_is_refused():
    from tvarant_b200 import capi

    pool = capi.PagePool(256, 8, 8, 4, 256, 16, 16, -1)
    assert capi.try_call("tvr_page_plan", pool, 256, 256, 256, 256, 256, 256, None, None, 4, 0,
                         None) == capi.ERR_INVALID
    assert "negative" in capi.last_error()
