"""The first token after a prompt under the rules of its request
(``LogitRules.row``): masked, penalised and biased like the later ones, and in
the history that they are penalised by."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpt2_paged_gpu import model  # noqa: F401  (a fixture: its tokens repeat)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mask_rows", [True, False])
def test_the_first_token_is_chosen_by_the_rules(model, mask_rows):  # noqa: F811
    import torch

    from tvarant_b200 import gpt2
    from tvarant_b200.paged import LogitRules

    torch.tvarant.clear_status()
    R, V, cap = 3, 1009, 30
    cache = gpt2.new_paged_cache(model, R, 20, 16, 100, "tvarant")
    prompts = [[5, 6, 7], [400, 3, 9, 11, 2], [1]]
    allowed = [range(100, 140), range(V), range(200, 260)]
    words = np.zeros((R, -(-V // 32)), np.uint32)
    for r, tokens in enumerate(allowed):
        for v in tokens:
            words[r, v // 32] |= np.uint32(1 << (v % 32))
    order = [2, 0, 1] if mask_rows else [0, 1, 2]  # mask_rows[r] = order[r]
    held = np.empty_like(words)
    held[order] = words
    tokens = torch.full((R, cap), -1, dtype=torch.int32)
    for r, p in enumerate(prompts):
        tokens[r, : len(p)] = torch.tensor(p)
    lens = torch.tensor([len(p) for p in prompts], dtype=torch.int32)
    rules = LogitRules(
        tokens=tokens.to("tvarant"), prompt_lens=lens.to("tvarant"),
        total_lens=lens.clone().to("tvarant"),
        presence=torch.full((R,), 1e4).to("tvarant"),
        masks=torch.from_numpy(held.view(np.int32)).to("tvarant"),
        mask_rows=torch.tensor(order, dtype=torch.int32).to("tvarant") if mask_rows else None,
        bias_ids=torch.tensor([[120], [77], [250]], dtype=torch.int32).to("tvarant"),
        bias_values=torch.full((R, 1), 100.0).to("tvarant"))
    ids = torch.zeros(R, 1, dtype=torch.int64)
    chosen = []
    for r, p in enumerate(prompts):
        logits = gpt2.paged_prefill(model, torch.tensor([p]).to("tvarant"), cache, r)
        one = rules.row(r)
        first = one.apply(logits[:, -1]).argmax(-1)
        torch.ops.tvarant.history_append_(one.tokens, one.total_lens, first)
        ids[r] = first.cpu()
        chosen.append([int(ids[r])])
    assert [c[0] for c in chosen] == [120, 77, 250]  # the bias, where the mask allows it
    assert rules.total_lens.cpu().tolist() == [4, 6, 2]
    ids, live = ids.to("tvarant"), torch.ones(R, dtype=torch.int32).to("tvarant")
    for _ in range(12):
        gpt2.paged_decode_step(model, ids, cache, live, rules)
        for c, x in zip(chosen, ids.cpu().view(-1).tolist()):
            c.append(x)
    for r, c in enumerate(chosen):
        assert len(set(c)) == len(c) and set(c) <= set(allowed[r])  # none twice, the first among them
        n = int(lens[r])
        assert rules.tokens.cpu()[r, n:n + 13].tolist() == c
    assert torch.tvarant.get_status() == 0


def test_a_row_of_absent_parts():
    from tvarant_b200.paged import LogitRules

    assert all(v is None for v in vars(LogitRules().row(0)).values())
