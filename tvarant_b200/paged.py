"""A paged KV cache for many requests of different lengths on the tvarant device.

The keys and values of every layer live in pages of ``page_size`` positions
that are shared out among the requests: request ``r``'s position ``j`` is row
``j % page_size`` of page ``block_table[r, j // page_size]``.  All of the
bookkeeping is on the device (``torch.ops.tvarant.page_plan``), so one step
serves requests that grow, finish and start, and can be captured once as a CUDA
graph.  ``tvarant_b200.gpt2.paged_prefill`` and ``paged_decode_step`` run GPT-2
over it.  The reference has no KV cache.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch


@dataclass
class PagedCache:
    """The pages of every layer and the state of the requests that share them.

    ``k`` / ``v``: per layer ``[pages, kv heads, page size, head dim]`` in
    float32, float16 or bfloat16 (new rows are rounded to it; attention
    computes in fp32).  ``block_table`` ``[requests, max pages]``, ``seq_lens``
    ``[requests]``, ``free_pages`` and ``free_count`` are int32.
    A request has at most ``max_len`` positions (0: what its row of the table
    holds).  ``workspace`` belongs to the attention calls: two steps that may run at
    the same time need a cache object with a workspace of its own each.
    """

    k: list
    v: list
    block_table: torch.Tensor
    seq_lens: torch.Tensor
    free_pages: torch.Tensor
    free_count: torch.Tensor
    workspace: torch.Tensor
    max_len: int = 0

    @property
    def requests(self) -> int:
        return self.block_table.shape[0]

    @property
    def page_size(self) -> int:
        return self.k[0].shape[2]

    @property
    def max_positions(self) -> int:
        """The positions that a request can have."""
        held = self.block_table.shape[1] * self.page_size
        return min(held, self.max_len) if self.max_len > 0 else held

    def plan(self, new_lens: torch.Tensor, tokens: int = 0, tokens_per_request: int = 0):
        """Block tables and slot maps for ``new_lens[r]`` new tokens of each
        request (int32, on the device; negative: the request ends and gives up
        its pages).  Returns ``(slots, positions, rows)`` of the tokens, packed
        ``[tokens]`` in the order of the requests, or ``[requests,
        tokens_per_request]``.  A request that the pool cannot serve, or that
        would have more than ``max_positions``, keeps its length, its slots are -1, and the device status word becomes 7
        (``TVR_DEV_CACHE_FULL``)."""
        return torch.ops.tvarant.page_plan(self.block_table, self.seq_lens, new_lens,
                                           self.free_pages, self.free_count, self.page_size,
                                           tokens, tokens_per_request, self.max_len)

    def append(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor,
               slots: torch.Tensor) -> None:
        """Writes ``[tokens, kv heads, head dim]`` rows into their slots."""
        torch.ops.tvarant.paged_append_(self.k[layer], self.v[layer], k_new, v_new, slots)

    def attend(self, layer: int, q: torch.Tensor, scale: float) -> torch.Tensor:
        """One query per request, ``[requests, heads, head dim]``, over its
        cached positions."""
        return torch.ops.tvarant.paged_attention(q, self.k[layer], self.v[layer],
                                                 self.block_table, self.seq_lens, scale,
                                                 self.workspace)[0]

    def append_attend(self, layer: int, q: torch.Tensor, k_new: torch.Tensor,
                      v_new: torch.Tensor, slots: torch.Tensor, scale: float) -> torch.Tensor:
        """``append`` of each request's last position (slots ``[requests]``,
        -1 for none), then ``attend``, in one launch."""
        return torch.ops.tvarant.paged_attention_append(
            q, k_new, v_new, self.k[layer], self.v[layer], slots, self.block_table,
            self.seq_lens, scale, self.workspace)[0]


def new_paged_cache(layers: int, requests: int, num_pages: int, page_size: int, max_len: int,
                    heads: int, kv_heads: int, head_dim: int, device,
                    dtype: torch.dtype = torch.float32) -> PagedCache:
    """An empty cache: ``num_pages`` free pages for ``requests`` requests of up
    to ``max_len`` positions each."""
    if dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"pages are float32, float16 or bfloat16, got {dtype}")
    if heads % kv_heads != 0:
        raise ValueError(f"{heads} heads do not share {kv_heads} key heads evenly")
    max_pages = -(-max_len // page_size)
    shape = (num_pages, kv_heads, page_size, head_dim)
    pages = [[torch.zeros(shape, dtype=dtype, device=device) for _ in range(layers)]
             for _ in range(2)]

    def ints(t):
        return t.to(torch.int32).to(device)

    size = torch.ops.tvarant.paged_attention_workspace(heads, kv_heads, head_dim)
    return PagedCache(pages[0], pages[1], ints(torch.zeros(requests, max_pages)),
                      ints(torch.zeros(requests)),
                      ints(torch.arange(num_pages - 1, -1, -1)),  # page 0 on top
                      ints(torch.tensor([num_pages])),
                      torch.zeros(max(1, size), dtype=torch.uint8, device=device), max_len)


@dataclass
class LogitRules:
    """What ``torch.ops.tvarant.adjust_logits`` applies to the logits of a step
    (include/tvarant.h, ``tvr_adjust_logits``); an absent part is None.  With
    ``tokens`` the histories grow by the tokens that
    ``gpt2.paged_decode_step`` chooses.  A prompt's tokens, and the first token
    after it (``row``), are for the caller to put there."""

    tokens: torch.Tensor | None = None        # [requests, capacity] int32 or int64
    prompt_lens: torch.Tensor | None = None   # [requests] int32
    total_lens: torch.Tensor | None = None    # [requests] int32
    repetition: torch.Tensor | None = None    # [requests] float32, as are the next two
    presence: torch.Tensor | None = None
    frequency: torch.Tensor | None = None
    bias_ids: torch.Tensor | None = None      # [requests, biases] int32
    bias_values: torch.Tensor | None = None   # [requests, biases] float32
    bias_counts: torch.Tensor | None = None   # [requests] int32
    masks: torch.Tensor | None = None         # [masks, words] int32, a bit a token
    mask_rows: torch.Tensor | None = None     # [requests] int32, -1: no mask

    def row(self, r: int) -> LogitRules:
        """The rules of request ``r`` alone, for logits ``[1, vocab]``: views, so
        that its history grows in place.  The first token after a prompt, with
        ``logits`` from ``gpt2.paged_prefill``::

            one = rules.row(r)
            first = one.apply(logits[:, -1]).argmax(-1)
            torch.ops.tvarant.history_append_(one.tokens, one.total_lens, first)
        """
        def cut(t):
            return None if t is None else t[r:r + 1]

        return LogitRules(
            cut(self.tokens), cut(self.prompt_lens), cut(self.total_lens), cut(self.repetition),
            cut(self.presence), cut(self.frequency), cut(self.bias_ids), cut(self.bias_values),
            cut(self.bias_counts), self.masks if self.mask_rows is not None else cut(self.masks),
            cut(self.mask_rows))

    def apply(self, logits: torch.Tensor) -> torch.Tensor:
        return torch.ops.tvarant.adjust_logits(
            logits, self.tokens, self.prompt_lens, self.total_lens, self.repetition,
            self.presence, self.frequency, self.bias_ids, self.bias_values, self.bias_counts,
            self.masks, self.mask_rows)
