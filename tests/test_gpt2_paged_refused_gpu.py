"""Rows that do not advance in ``gpt2.paged_decode_step`` (refused by the page
plan for want of pages, paused, or ended): their current token, their history
and their length stay, so that a refused or paused request goes on later with
the tokens that it would have chosen without the interruption.

Tokens are compared as in test_gpt2_paged_gpu: where the two best logits of
``forward`` are clearly apart.
"""

from __future__ import annotations

import pytest

from test_gpt2_paged_gpu import _clear_best, _forward_next

pytestmark = pytest.mark.gpu

CACHE_FULL = 7


@pytest.fixture(scope="module")
def model():
    """Weights large enough that the next token is hardly ever the current one."""
    import torch

    import torch_tvarant  # noqa: F401
    from tvarant_b200 import gpt2

    old = torch.get_float32_matmul_precision()
    torch.set_float32_matmul_precision("highest")
    cfg = gpt2.GPT2Config(n_layer=3, d_model=256, n_head=4, d_ff=512, vocab=1009, n_ctx=128)
    m = gpt2.init_gpt2(cfg, seed=3)
    for layer in m.layers:
        for name in ("w_qkv", "w_proj", "w_fc", "w_out"):
            getattr(layer, name).mul_(6)
    yield m.to("tvarant")
    torch.set_float32_matmul_precision(old)


class Server:
    """Requests with their tokens on the host, decoded eagerly or by a graph."""

    def __init__(self, model, prompts, num_pages, page_size, graph, max_len=100):
        import torch

        from tvarant_b200 import gpt2
        from tvarant_b200.graphs import Graph
        from tvarant_b200.paged import LogitRules

        torch.tvarant.clear_status()
        self.torch, self.model = torch, model
        R, cap = len(prompts), 40 + max(map(len, prompts))
        self.cache = gpt2.new_paged_cache(model, R, num_pages, page_size, max_len, "tvarant")
        tokens = torch.full((R, cap), -1, dtype=torch.int32)
        for r, p in enumerate(prompts):
            tokens[r, : len(p)] = torch.tensor(p)
        self.lens = [len(p) for p in prompts]
        lens = torch.tensor(self.lens, dtype=torch.int32)
        self.rules = LogitRules(tokens=tokens.to("tvarant"), prompt_lens=lens.to("tvarant"),
                                total_lens=lens.clone().to("tvarant"))
        self.ids = torch.zeros(R, 1, dtype=torch.int64).to("tvarant")
        self.live = torch.zeros(R, dtype=torch.int32).to("tvarant")
        step = lambda: gpt2.paged_decode_step(model, self.ids, self.cache, self.live, self.rules)  # noqa: E731
        self.captured = Graph(step) if graph else None
        self.step_once = self.captured.replay if graph else step
        self.held = []
        for r, p in enumerate(prompts):
            logits = gpt2.paged_prefill(model, torch.tensor([p]).to("tvarant"), self.cache, r)
            self.held.append([*p, int(logits[0, -1].cpu().argmax())])
        self.ids.copy_(torch.tensor([h[-1] for h in self.held]).view(R, 1))
        self.chosen = [[] for _ in prompts]

    def step(self, live, advances):
        """A step; the requests of `advances` choose what ``forward`` chooses,
        the others keep what they had."""
        torch = self.torch
        before = self.ids.cpu().view(-1).tolist()
        histories = self.rules.tokens.cpu().clone()
        self.live.copy_(torch.tensor(live, dtype=torch.int32))
        self.step_once()
        torch.tvarant.synchronize()
        got = self.ids.cpu().view(-1).tolist()
        for r, h in enumerate(self.held):
            if r not in advances:
                assert got[r] == before[r], r
                assert torch.equal(self.rules.tokens.cpu()[r], histories[r]), r
                continue
            want = _forward_next(self.model, h)
            if _clear_best(want, 1e-3):
                assert got[r] == int(want.argmax()), r
            h.append(got[r])
            self.chosen[r].append(got[r])
        totals = [n + len(c) for n, c in zip(self.lens, self.chosen)]
        assert self.rules.total_lens.cpu().tolist() == totals
        for r, c in enumerate(self.chosen):
            assert self.rules.tokens.cpu()[r, self.lens[r]:totals[r]].tolist() == c

    def status(self):
        got = self.torch.tvarant.get_status()
        self.torch.tvarant.clear_status()
        return got

    def close(self):
        if self.captured is not None:
            self.captured.close()


@pytest.mark.parametrize("graph", [False, True])
def test_a_refused_request_goes_on_when_pages_are_free(model, graph):
    s = Server(model, [[5, 6, 7, 8], [400, 3, 9, 11, 2, 1, 900, 33], [17]], 4, 4, graph)
    # the pool is empty: requests 0 and 1 need a page, request 2 has room in its own
    s.step([1, 1, 1], advances=[2])
    assert s.status() == CACHE_FULL and s.cache.seq_lens.cpu().tolist() == [4, 8, 2]
    s.step([1, 1, 1], advances=[2])
    assert s.status() == CACHE_FULL and s.cache.seq_lens.cpu().tolist() == [4, 8, 3]
    # request 1 ends: its pages serve request 0
    s.step([1, -1, 0], advances=[0])
    assert s.status() == 0 and s.cache.seq_lens.cpu().tolist() == [5, 0, 3]
    for _ in range(3):
        s.step([1, 0, 0], advances=[0])
    s.step([1, 0, 1], advances=[0, 2])
    assert s.status() == 0 and s.cache.seq_lens.cpu().tolist() == [9, 0, 4]
    s.close()


@pytest.mark.parametrize("graph", [False, True])
def test_a_paused_request_goes_on(model, graph):
    s = Server(model, [[5, 6, 7], [400, 3, 9, 11, 2]], 20, 8, graph)
    for live in ([1, 1], [1, 0], [0, 0], [1, 0], [0, 1], [1, 1], [1, 1]):
        s.step(live, advances=[r for r in range(2) if live[r]])
    assert s.status() == 0 and s.cache.seq_lens.cpu().tolist() == [8, 9]
    s.close()


@pytest.mark.parametrize("kind", ["strided", "int32"])
def test_ids_of_other_layouts(model, kind):
    import torch

    from tvarant_b200 import gpt2

    s = Server(model, [[5, 6, 7], [400, 3]], 20, 8, False)
    s.live.copy_(torch.tensor([1, 0], dtype=torch.int32))
    wide = torch.stack([s.ids.cpu(), torch.full((2, 1), -5)], 1).view(2, 2).to("tvarant")
    ids = wide[:, :1] if kind == "strided" else s.ids.int()
    gpt2.paged_decode_step(model, ids, s.cache, s.live)
    want = _forward_next(model, s.held[0])
    assert ids.cpu().view(-1).tolist() == [int(want.argmax()), s.held[1][-1]]
    assert wide.cpu()[:, 1].tolist() == [-5, -5]


@pytest.mark.parametrize("bits", [32, 64])
def test_advance_tokens(bits):
    import torch

    import torch_tvarant  # noqa: F401

    def dev(values, dtype):
        return torch.tensor(values, dtype=dtype).to("tvarant")

    ops = torch.ops.tvarant
    dt = torch.int32 if bits == 32 else torch.int64
    tokens = dev([[-1] * 3 for _ in range(5)], dt)
    lens = dev([0, 2, 3, 1, -1], torch.int32)
    current, nxt = dev([1, 2, 3, 4, 5], torch.int64), dev([11, 12, 13, 14, 15], torch.int64)
    slots = dev([0, 1 << 40, 7, -1, 8], torch.int64)
    ops.advance_tokens_(current, nxt, slots, tokens, lens)
    # a full history, and one of a negative length, stay as they are
    assert current.cpu().tolist() == [11, 12, 13, 4, 15] and lens.cpu().tolist() == [1, 3, 3, 1, -1]
    assert tokens.cpu().tolist() == [[11, -1, -1], [-1, -1, 12], *[[-1] * 3] * 3]
    ops.advance_tokens_(current, dev([6] * 5, torch.int64), dev([-1, -1, -1, 0, -1], torch.int64))
    assert current.cpu().tolist() == [11, 12, 13, 6, 15] and lens.cpu().tolist() == [1, 3, 3, 1, -1]
    for bad in (lambda: ops.advance_tokens_(current, nxt, slots[:2]),
                lambda: ops.advance_tokens_(current, nxt, slots, tokens),
                lambda: ops.advance_tokens_(current, nxt, slots, tokens[:2], lens),
                lambda: ops.advance_tokens_(current, nxt, slots, tokens, lens[:2]),
                lambda: ops.advance_tokens_(lens, lens, slots)):
        with pytest.raises(RuntimeError):
            bad()
