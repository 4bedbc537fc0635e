"""GPT-2 over the paged cache (tvarant_b200.gpt2.paged_prefill and
paged_decode_step): requests of different lengths that start and end at
different steps choose the tokens that each of them chooses alone, decoded with
``forward`` over its whole sequence; also captured as a CUDA graph, with 16-bit
pages and with logit rules.

Tokens are compared where the two best logits of ``forward`` are further apart
than the two paths' difference can be (both compute GEMMs in 3xTF32: 1e-5
relative; the margin is 1e-3 of the logits' spread).
"""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    import torch

    import torch_tvarant  # noqa: F401
    from tvarant_b200 import gpt2

    old = torch.get_float32_matmul_precision()
    torch.set_float32_matmul_precision("highest")
    cfg = gpt2.GPT2Config(n_layer=3, d_model=256, n_head=4, d_ff=512, vocab=1009, n_ctx=128)
    m = gpt2.init_gpt2(cfg, seed=3)
    yield m.to("tvarant")
    torch.set_float32_matmul_precision(old)


def _forward_next(model, tokens):
    """The logits after `tokens`, over the whole sequence."""
    import torch

    from tvarant_b200 import gpt2

    ids = torch.tensor([tokens], dtype=torch.int64).to("tvarant")
    return gpt2.forward(model, ids, attention="bmm")[0, -1].cpu()


def _clear_best(logits, tol):
    top = logits.topk(2).values
    return float(top[0] - top[1]) > tol * float(logits.std())


@pytest.mark.parametrize("dtype, tol", [("float32", 1e-3), ("bfloat16", 5e-2)])
@pytest.mark.parametrize("graph", [False, True])
def test_requests_that_start_and_end(model, dtype, tol, graph):
    import torch

    from tvarant_b200 import gpt2
    from tvarant_b200.graphs import Graph

    torch.tvarant.clear_status()
    R = 3
    cache = gpt2.new_paged_cache(model, R, 40, 8, 100, "tvarant", getattr(torch, dtype))
    ids = torch.zeros(R, 1, dtype=torch.int64).to("tvarant")
    live = torch.zeros(R, dtype=torch.int32).to("tvarant")
    rng = np.random.default_rng(7)
    held = {}  # request -> its tokens, the last one not in the cache yet
    host_ids, host_live = [0] * R, [0] * R

    def start(r, n):
        prompt = rng.integers(0, 1009, n).tolist()
        logits = gpt2.paged_prefill(model, torch.tensor([prompt]).to("tvarant"), cache, r)[0, -1].cpu()
        want = _forward_next(model, prompt)
        assert float((logits - want).abs().max()) <= 1e-3 * float(want.std())
        held[r] = [*prompt, int(logits.argmax())]
        host_ids[r], host_live[r] = held[r][-1], 1

    def push():
        ids.copy_(torch.tensor(host_ids, dtype=torch.int64).view(R, 1))
        live.copy_(torch.tensor(host_live, dtype=torch.int32))

    captured = None
    if graph:  # capturing runs the step; with nobody live it changes nothing
        captured = Graph(lambda: gpt2.paged_decode_step(model, ids, cache, live))
        assert cache.seq_lens.cpu().tolist() == [0] * R
    checked = 0
    for step in range(24):
        if step == 0:
            start(0, 5)
        if step == 3:
            start(2, 17)
        if step == 6:
            start(1, 1)
        if step == 12:
            host_live[2] = -1  # ends in this step
        if step == 15:
            start(2, 9)
        push()
        if graph:
            captured.replay()
        else:
            gpt2.paged_decode_step(model, ids, cache, live)
        torch.tvarant.synchronize()
        got = ids.cpu().view(-1).tolist()
        for r in list(held):
            if host_live[r] < 0:
                host_live[r] = 0
                del held[r]
                continue
            want = _forward_next(model, held[r])
            if _clear_best(want, tol):
                assert got[r] == int(want.argmax()), (step, r)
                checked += 1
            held[r].append(got[r])
            host_ids[r] = got[r]
    assert checked > 30
    lens = [len(held[r]) - 1 if r in held else 0 for r in range(R)]
    assert cache.seq_lens.cpu().tolist() == lens
    assert int(cache.free_count.cpu()) == 40 - sum(-(-n // 8) for n in lens)
    assert torch.tvarant.get_status() == 0
    if captured is not None:
        captured.close()


def test_rules_steer_the_choice(model):
    """A grammar mask, a bias and a repetition penalty, with the histories
    growing on the device."""
    import torch

    from tvarant_b200 import gpt2
    from tvarant_b200.paged import LogitRules

    torch.tvarant.clear_status()
    R, V, cap = 2, 1009, 40
    cache = gpt2.new_paged_cache(model, R, 20, 16, 100, "tvarant")
    prompts = [[5, 6, 7], [400, 3, 9, 11, 2]]
    words = np.zeros((1, -(-V // 32)), np.uint32)
    for v in range(100, 140):
        words[0, v // 32] |= np.uint32(1 << (v % 32))
    tokens = torch.full((R, cap), -1, dtype=torch.int32)
    for r, p in enumerate(prompts):
        tokens[r, : len(p)] = torch.tensor(p)
    lens = torch.tensor([len(p) for p in prompts], dtype=torch.int32)
    rules = LogitRules(
        tokens=tokens.to("tvarant"), prompt_lens=lens.to("tvarant"),
        total_lens=lens.clone().to("tvarant"),
        presence=torch.tensor([0.0, 1e4]).to("tvarant"),
        masks=torch.from_numpy(words.view(np.int32)).to("tvarant"),
        mask_rows=torch.tensor([0, -1], dtype=torch.int32).to("tvarant"),
        bias_ids=torch.tensor([[120], [77]], dtype=torch.int32).to("tvarant"),
        bias_values=torch.tensor([[100.0], [100.0]]).to("tvarant"))
    ids = torch.zeros(R, 1, dtype=torch.int64)
    for r, p in enumerate(prompts):
        logits = gpt2.paged_prefill(model, torch.tensor([p]).to("tvarant"), cache, r)
        ids[r, 0] = int(logits[0, -1].cpu().argmax())
    ids, live = ids.to("tvarant"), torch.ones(R, dtype=torch.int32).to("tvarant")
    chosen = []
    for _ in range(12):
        gpt2.paged_decode_step(model, ids, cache, live, rules)
        chosen.append(ids.cpu().view(-1).tolist())
    a, b = zip(*chosen)
    assert all(x == 120 for x in a)                # allowed by its mask, and favoured
    assert b[0] == 77 and len(set(b)) == len(b)    # no token twice under that penalty
    assert rules.total_lens.cpu().tolist() == [3 + 12, 5 + 12]
    assert rules.tokens.cpu()[0, 3:15].tolist() == list(a)
    assert rules.tokens.cpu()[1, 5:17].tolist() == list(b)
    assert torch.tvarant.get_status() == 0


def test_a_pool_without_pages_says_so(model):
    import torch

    from tvarant_b200 import gpt2

    torch.tvarant.clear_status()
    cache = gpt2.new_paged_cache(model, 2, 1, 4, 100, "tvarant")
    gpt2.paged_prefill(model, torch.tensor([[1, 2, 3, 4]]).to("tvarant"), cache, 0)
    torch.tvarant.synchronize()
    assert torch.tvarant.get_status() == 0
    ids = torch.zeros(2, 1, dtype=torch.int64).to("tvarant")
    live = torch.tensor([1, 0], dtype=torch.int32).to("tvarant")
    gpt2.paged_decode_step(model, ids, cache, live)
    torch.tvarant.synchronize()
    assert torch.tvarant.get_status() == 7  # TVR_DEV_CACHE_FULL
    assert cache.seq_lens.cpu().tolist() == [4, 0]
    torch.tvarant.clear_status()
