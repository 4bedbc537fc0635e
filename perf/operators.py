"""The operators of a paged decode step, as measured cases: the page plan, the append of new keys
and values to their pages, one new token's attention over the pages, and the adjustment of logits.

``run`` computes a case in its plain form (elementary torch operations in fp32), or, where ``own``
is set, makes the call that a user makes of the framework (the C ABI through
``tvarant_b200.capi``, on raw device pointers and the current stream).
"""

import ctypes
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # A decode step of a small batch: a page is needed now and then.  Launch latency.
        {"name": "plan_decode", "op": "plan", "requests": 8, "page": 16, "lo": 20, "hi": 900,
         "decode": 8, "prompt": 0, "finished": 0, "extra": 100},
        # A full server: most requests decode, some bring prompts, some finish.
        {"name": "plan_mixed", "op": "plan", "requests": 1000, "page": 16, "lo": 1, "hi": 8000,
         "decode": 900, "prompt": 2047, "finished": 60, "extra": 9000},
        # One prompt of the GPT-2 configuration (12 heads of 64) written into fp32 pages.
        {"name": "append_prompt", "op": "append", "tokens": 611, "kv_heads": 12, "dim": 64,
         "page": 16, "type": "f32", "layout": "head", "fused": True},
        # Prompts of many requests into bf16 pages, 8 heads of 128.
        {"name": "append_prompts", "op": "append", "tokens": 16385, "kv_heads": 8, "dim": 128,
         "page": 64, "type": "bf16", "layout": "token", "fused": False},
        # One request of the GPT-2 configuration, the smallest call of a decode step.
        {"name": "attend_one", "op": "attend", "requests": 1, "heads": 12, "kv_heads": 12,
         "dim": 64, "lo": 777, "hi": 777, "idle": 0, "page": 16, "type": "f32", "layout": "head",
         "append": True},
        # A ragged batch of that configuration, two of its rows idle.
        {"name": "attend_batch", "op": "attend", "requests": 16, "heads": 12, "kv_heads": 12,
         "dim": 64, "lo": 30, "hi": 1024, "idle": 2, "page": 16, "type": "f32", "layout": "head",
         "append": True},
        # A few long documents, heads shared by groups of four, 16-bit pages.
        {"name": "attend_long", "op": "attend", "requests": 2, "heads": 32, "kv_heads": 8,
         "dim": 128, "lo": 40000, "hi": 100001, "idle": 0, "page": 32, "type": "bf16",
         "layout": "token", "append": False},
        # Many requests of very different lengths, heads shared by groups of eight.
        {"name": "attend_grouped", "op": "attend", "requests": 61, "heads": 64, "kv_heads": 8,
         "dim": 128, "lo": 100, "hi": 16000, "idle": 1, "page": 16, "type": "f16",
         "layout": "head", "append": True},
        # The largest: a full server of fp32 pages.
        {"name": "attend_many", "op": "attend", "requests": 128, "heads": 12, "kv_heads": 12,
         "dim": 64, "lo": 200, "hi": 8000, "idle": 0, "page": 16, "type": "f32", "layout": "head",
         "append": True},
        # One row over the GPT-2 vocabulary.
        {"name": "logits_one", "op": "logits", "rows": 1, "vocab": 50257, "history": 300,
         "biases": 5, "masks": 1},
        # A decode batch over that vocabulary.
        {"name": "logits_batch", "op": "logits", "rows": 48, "vocab": 50257, "history": 1024,
         "biases": 40, "masks": 7},
        # A full server, a larger vocabulary, long histories, a grammar for most rows.
        {"name": "logits_many", "op": "logits", "rows": 400, "vocab": 129280, "history": 20000,
         "biases": 300, "masks": 300},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "logits"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    if op == "plan":
        n = _log(rng, 1, 1500)
        hi = _log(rng, 10, 10000)
        return {"op": op, "requests": n, "page": page, "lo": rng.randint(1, 10), "hi": hi,
                "decode": rng.randint(0, n), "prompt": _log(rng, 1, 3000),
                "finished": rng.randint(0, n // 4), "extra": _log(rng, 50, 20000)}
    if op == "append":
        return {"op": op, "tokens": _log(rng, 1, 16000), "kv_heads": rng.choice([1, 4, 8, 12]),
                "dim": rng.choice([32, 64, 96, 128, 256]) // 2, "page": page,
                "type": rng.choice(list(TYPES)), "layout": rng.choice(["head", "token"]),
                "fused": rng.choice([True, False])}
    if op == "attend":
        heads, kv_heads, dim = rng.choice([
            (12, 12, 64), (12, 12, 64), (32, 32, 128), (32, 8, 128), (64, 8, 128), (40, 8, 128),
            (16, 1, 128), (6, 2, 96), (8, 4, 256), (9, 3, 80), (14, 2, 64), (4, 4, 32)])
        kind = rng.choice(list(TYPES))
        per_key = kv_heads * dim * (4 if kind == "f32" else 2)
        keys = 180_000_000 // per_key  # half of the bytes of the largest listed case's keys
        n = min(_log(rng, 1, 150), max(1, keys // 64))
        hi = min(_log(rng, 16, 60000), keys // n)
        return {"op": op, "requests": n, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "lo": max(1, int(hi * rng.uniform(0.01, 1.0))), "hi": hi,
                "idle": rng.randint(0, n // 8), "page": page, "type": kind,
                "layout": rng.choice(["head", "token"]), "append": rng.choice([True, True, False])}
    vocab = rng.choice([50257, 32000, 65537, 128256, 151936, 1003])
    rows = _log(rng, 1, min(400, 50_000_000 // vocab))
    return {"op": op, "rows": rows, "vocab": vocab, "history": _log(rng, 1, 20000),
            "biases": _log(rng, 1, 300), "masks": rng.randint(1, rows)}


# ---- inputs ---------------------------------------------------------------


def _lengths(case):
    """Lengths lo..hi, spread over their logarithm, the idle requests' zero: the same set for every
    seed (``prepare`` deals it out), so that the work of a case is known."""
    n, idle = case["requests"], case["idle"]
    lo, hi, live = case["lo"], case["hi"], case["requests"] - case["idle"]
    lens = [max(1, round(lo * (hi / lo) ** ((i + 1) / live))) for i in range(live)]
    return [0] * (n - live) + lens


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pages(g, shape, kind, layout):
    """[pages, heads, page, dim], the heads outside the positions of a page or inside them."""
    p, h, s, d = shape
    if layout == "head":
        return torch.randn(p, h, s, d, generator=g, device=DEV).to(TYPES[kind])
    return torch.randn(p, s, h, d, generator=g, device=DEV).to(TYPES[kind]).transpose(1, 2)


def _descriptor(case, k, v):
    """The paged cache as the C ABI takes it."""
    from tvarant_b200 import capi

    capi.load()
    capi.call("tvr_init")
    code = {"f32": capi.PAGE_F32, "f16": capi.PAGE_F16, "bf16": capi.PAGE_BF16}[case["type"]]
    return capi.PagedKV(k.data_ptr(), v.data_ptr(), code, 0, k.shape[0], k.shape[2], k.shape[1],
                        k.shape[3], (ctypes.c_int64 * 3)(*k.stride()[:3]),
                        (ctypes.c_int64 * 3)(*v.stride()[:3]))


def _prepare_plan(case, g):
    n, page = case["requests"], case["page"]
    lo, hi = case["lo"], case["hi"]
    lens = [round(lo * (hi / lo) ** ((i + 1) / n)) for i in range(n)]
    news = [1] * case["decode"] + [-1] * min(case["finished"], n - case["decode"])
    rest = n - len(news)  # prompts of 1..prompt tokens; without prompts, idle requests
    news += [1 + (i * case["prompt"]) // max(1, rest) if case["prompt"] else 0 for i in range(rest)]
    order = torch.randperm(n, generator=g, device=DEV)
    seq = _ints(lens)[order]
    new = _ints(news)[torch.randperm(n, generator=g, device=DEV)]
    tokens = sum(max(0, x) for x in news)
    max_pages = -(-(hi + max(1, case["prompt"])) // page)
    held = [-(-x // page) for x in lens]
    num_pages = sum(held) + case["extra"]
    ids = torch.randperm(num_pages, generator=g, device=DEV).to(torch.int32)
    first = (-(-seq // page)).cumsum(0) - (-(-seq // page))
    column = torch.arange(max_pages, device=DEV)
    table = ids[(first[:, None] + column).clamp(max=num_pages - 1)].contiguous()
    free = torch.zeros(num_pages, dtype=torch.int32, device=DEV)
    free[: case["extra"]] = ids[sum(held):]
    s = {"table": table, "seq": seq, "new": new, "free": free,
         "count": _ints([case["extra"]]), "tokens": max(1, tokens), "page": page}
    if own:
        from tvarant_b200 import capi

        capi.load()
        capi.call("tvr_init")
        s["pool"] = capi.PagePool(table.data_ptr(), table.stride(0), max_pages, n,
                                  free.data_ptr(), num_pages, page)
    return s


def _prepare_append(case, g):
    n, h, d, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
    num_pages = -(-n // page) + 3
    shape = (num_pages, h, page, d)
    k, v = (_pages(g, shape, case["type"], case["layout"]) for _ in range(2))
    if case["fused"]:  # the keys and values of a fused projection [tokens, 3, heads, dim]
        qkv = torch.randn(n, 3, h, d, generator=g, device=DEV)
        k_new, v_new = qkv[:, 1], qkv[:, 2]
    else:
        k_new, v_new = (torch.randn(n, h, d, generator=g, device=DEV) for _ in range(2))
    ids = torch.randperm(num_pages, generator=g, device=DEV)
    token = torch.arange(n, device=DEV)
    slots = ids[token // page] * page + token % page
    slots = torch.where(token % 97 == 96, -1, slots)  # tokens of a request that was refused
    s = {"k": k, "v": v, "k_new": k_new, "v_new": v_new, "slots": slots,
         "live": (slots >= 0).nonzero()[:, 0], "type": TYPES[case["type"]]}
    if own:
        s["cache"] = _descriptor(case, k, v)
        s["strides"] = (ctypes.c_int64 * 4)(*k_new.stride()[:2], *v_new.stride()[:2])
    return s


def _prepare_attend(case, g):
    n, h, d, page = case["requests"], case["kv_heads"], case["dim"], case["page"]
    order = torch.randperm(n, generator=g, device=DEV)
    lens = _ints(_lengths(case))[order]
    held = [-(-x // page) for x in _lengths(case)]
    max_pages, num_pages = max(held), sum(held) + 7
    pages = -(-lens // page)
    first = pages.cumsum(0) - pages
    ids = torch.randperm(num_pages, generator=g, device=DEV).to(torch.int32)
    column = torch.arange(max_pages, device=DEV)
    table = ids[(first[:, None] + column).clamp(max=num_pages - 1)].contiguous()
    shape = (num_pages, h, page, d)
    k, v = (_pages(g, shape, case["type"], case["layout"]) for _ in range(2))
    heads = case["heads"]
    qkv = torch.randn(n, heads + 2 * h, d, generator=g, device=DEV)  # a fused projection's rows
    last = (lens.long() - 1).clamp(min=0)
    slot = table.gather(1, (last // page)[:, None])[:, 0].long() * page + last % page
    slot = torch.where(lens > 0, slot, -1)
    s = {"q": qkv[:, :heads], "k_new": qkv[:, heads:heads + h], "v_new": qkv[:, heads + h:],
         "k": k, "v": v, "table": table, "lens": lens, "slots": slot, "append": case["append"],
         "live": (slot >= 0).nonzero()[:, 0], "type": TYPES[case["type"]],
         "scale": 1.0 / math.sqrt(d)}
    if own:
        s["cache"] = _descriptor(case, k, v)
        s["strides"] = (ctypes.c_int64 * 8)(*s["q"].stride()[:2], *s["k_new"].stride()[:2],
                                            *s["v_new"].stride()[:2], heads * d, d)
        from tvarant_b200 import capi

        size = ctypes.c_int64()
        capi.call("tvr_paged_attention_workspace", heads, h, d, ctypes.byref(size))
        s["workspace"] = torch.zeros(max(1, size.value), dtype=torch.uint8, device=DEV)
    return s


def _prepare_logits(case, g):
    n, vocab, hist, nb = case["rows"], case["vocab"], case["history"], case["biases"]

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    # histories of half to all of `history` tokens, the frequent ids often, padded with -1
    total = [hist // 2 + (hist - hist // 2) * (i + 1) // n for i in range(n)]
    total = _ints(total)[torch.randperm(n, generator=g, device=DEV)]
    prompt = (total * uniform(n)).to(torch.int32)
    tokens = (vocab * uniform(n, hist) ** 3).to(torch.int32).clamp(max=vocab - 1)
    tokens = torch.where(torch.arange(hist, device=DEV) < total[:, None], tokens, -1)
    counts = (nb * uniform(n)).to(torch.int32)
    words = -(-vocab // 32)
    bits = torch.randint(-2**31, 2**31, (case["masks"], words), generator=g, device=DEV)
    tight = torch.arange(case["masks"], device=DEV) % 3 == 2  # few tokens allowed
    sparse = bits * (uniform(case["masks"], words) < 0.01)
    s = {"logits": 4.0 * torch.randn(n, vocab, generator=g, device=DEV),
         "tokens": tokens, "prompt": prompt, "total": total,
         "repetition": 1.0 + 0.5 * uniform(n), "presence": 0.8 * uniform(n),
         "frequency": 0.4 * uniform(n),
         "bias_ids": torch.randint(0, vocab, (n, nb), generator=g, device=DEV).to(torch.int32),
         "bias_values": 5.0 * torch.randn(n, nb, generator=g, device=DEV), "bias_counts": counts,
         "masks": torch.where(tight[:, None], sparse, bits).to(torch.int32),
         # every mask has a row; the rows over the number of masks have none
         "mask_rows": torch.where(torch.arange(n, device=DEV) < case["masks"],
                                  torch.arange(n, device=DEV), -1).to(torch.int32)
         [torch.randperm(n, generator=g, device=DEV)]}
    if own:
        from tvarant_b200 import capi

        capi.load()
        capi.call("tvr_init")
        s["rules"] = capi.LogitRules(
            tokens.data_ptr(), 32, 0, tokens.stride(0), prompt.data_ptr(), total.data_ptr(),
            s["repetition"].data_ptr(), s["presence"].data_ptr(), s["frequency"].data_ptr(),
            s["bias_ids"].data_ptr(), s["bias_values"].data_ptr(), counts.data_ptr(), nb,
            s["masks"].data_ptr(), words, case["masks"], s["mask_rows"].data_ptr())
    return s


def prepare(case, seed):
    g = _generator(seed)
    s = {"plan": _prepare_plan, "append": _prepare_append, "attend": _prepare_attend,
         "logits": _prepare_logits}[case["op"]](case, g)
    s["op"] = case["op"]
    return s


# ---- the plain forms ------------------------------------------------------


def _plain_plan(s):
    page, seq, new, table = s["page"], s["seq"].long(), s["new"].long(), s["table"]
    n, max_pages = table.shape
    count, done, grow = s["count"].long(), new < 0, new.clamp(min=0)
    held = (seq + page - 1) // page
    # released pages go on top of the stack, in the order of the requests and their tables
    out = torch.where(done, held, 0)
    out_end = out.cumsum(0)
    column = torch.arange(max_pages, device=seq.device)
    last = s["free"].numel()
    stack = torch.cat([s["free"], s["free"].new_zeros(n * max_pages + 1)])
    at = torch.where(done[:, None] & (column < held[:, None]),
                     count + (out_end - out)[:, None] + column, stack.numel() - 1)
    stack[at] = table
    top = count + out_end[-1]
    # pages taken from the top
    need = (seq + grow + page - 1) // page - held
    fits = (held + need <= max_pages) & ~done
    need = torch.where(fits, need, 0)
    end = need.cumsum(0)
    take = fits & ((need == 0) | (end <= top))
    need = torch.where(take, need, 0)
    fresh = take[:, None] & (column >= held[:, None]) & (column < (held + need)[:, None])
    place = top - 1 - (end - need)[:, None] - (column - held[:, None])
    table = torch.where(fresh, stack[place.clamp(0, stack.numel() - 1)], table)
    top = top - need.sum()
    seq_out = torch.where(done, 0, torch.where(take, seq + grow, seq))
    keep = torch.arange(last, device=seq.device)
    free = torch.where((keep >= count) & (keep < top), stack[:last], s["free"])
    # the tokens, packed in the order of the requests
    stop = grow.cumsum(0)
    t = torch.arange(s["tokens"], device=seq.device)
    r = torch.searchsorted(stop, t, right=True)
    pad, r = r >= n, r.clamp(max=n - 1)
    at = seq[r] + t - (stop - grow)[r]
    slot = table[r, (at // page).clamp(max=max_pages - 1)].long() * page + at % page
    slot = torch.where(pad | ~take[r], -1, slot)
    return {"table": table, "seq": seq_out.int(), "count": top.int(), "free": free, "slots": slot,
            "positions": torch.where(pad, 0, at).int(), "rows": torch.where(pad, -1, r).int()}


def _write(s):
    """New rows of keys and values, rounded to the pages' type, into their slots."""
    page, live = s["k"].shape[2], s["live"]
    slot = s["slots"][live]
    s["k"][slot // page, :, slot % page] = s["k_new"][live].to(s["type"])
    s["v"][slot // page, :, slot % page] = s["v_new"][live].to(s["type"])


def _plain_append(s):
    _write(s)
    return {"k": s["k"], "v": s["v"]}


def _plain_attend(s):
    if s["append"]:
        _write(s)
    q, lens, table = s["q"], s["lens"], s["table"]
    n, heads, d = q.shape
    hk, page = s["k"].shape[1], s["k"].shape[2]
    keys = table.shape[1] * page
    k, v = (x[table].float().transpose(1, 2).reshape(n, hk, keys, d) for x in (s["k"], s["v"]))
    scores = (q.reshape(n, hk, heads // hk, d) @ k.transpose(2, 3)) * s["scale"]
    seen = torch.arange(keys, device=q.device) < lens[:, None]
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (scores - top).exp()
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).reshape(n, heads)
    got = {"out": out.reshape(n, heads, d), "lse": lse}
    return {**got, "k": s["k"], "v": s["v"]} if s["append"] else got


def _plain_logits(s):
    x, tokens = s["logits"], s["tokens"].long()
    n, vocab = x.shape
    at = torch.arange(tokens.shape[1], device=x.device)
    seen = at < s["total"][:, None]
    made = seen & (at >= s["prompt"][:, None])
    # whole numbers below 2^24: the fp32 counts are exact
    used = torch.zeros(n, vocab, device=x.device).scatter_add_(1, tokens.clamp(min=0), seen.float())
    count = torch.zeros(n, vocab, device=x.device).scatter_add_(1, tokens.clamp(min=0), made.float())
    r = s["repetition"][:, None]
    x = torch.where(used > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    listed_ = torch.arange(s["bias_ids"].shape[1], device=x.device) < s["bias_counts"][:, None]
    x = x.scatter_add_(1, s["bias_ids"].long(), torch.where(listed_, s["bias_values"], 0.0))
    v = torch.arange(vocab, device=x.device)
    word = s["masks"][s["mask_rows"].clamp(min=0).long()][:, v // 32]
    allowed = ((word >> (v % 32).int()) & 1) > 0
    return torch.where(allowed | (s["mask_rows"] < 0)[:, None], x, -math.inf)


# ---- the framework's calls ------------------------------------------------


def _own_plan(s, capi, stream):
    n, tokens = s["seq"].numel(), s["tokens"]
    seq_out, count_out = torch.empty_like(s["seq"]), torch.empty_like(s["count"])
    slots = torch.empty(tokens, dtype=torch.int64, device=DEV)
    positions = torch.empty(tokens, dtype=torch.int32, device=DEV)
    rows = torch.empty(tokens, dtype=torch.int32, device=DEV)
    capi.call("tvr_page_plan", s["pool"], s["seq"].data_ptr(), s["new"].data_ptr(),
              seq_out.data_ptr(), s["count"].data_ptr(), count_out.data_ptr(), slots.data_ptr(),
              positions.data_ptr(), rows.data_ptr(), tokens, 0, stream)
    return {"table": s["table"], "seq": seq_out, "count": count_out, "free": s["free"],
            "slots": slots, "positions": positions, "rows": rows}


def _own_append(s, capi, stream):
    capi.call("tvr_paged_append", s["cache"], s["k_new"].data_ptr(), s["v_new"].data_ptr(),
              s["strides"], s["slots"].data_ptr(), s["slots"].numel(), stream)
    return {"k": s["k"], "v": s["v"]}


def _own_attend(s, capi, stream):
    q, table = s["q"], s["table"]
    n, heads, d = q.shape
    out = torch.empty(n, heads, d, device=DEV)
    lse = torch.empty(n, heads, device=DEV)
    new = (s["k_new"].data_ptr(), s["v_new"].data_ptr(), s["slots"].data_ptr())
    k_new, v_new, slots = new if s["append"] else (None, None, None)
    capi.call("tvr_paged_attention", s["cache"], q.data_ptr(), k_new, v_new, slots,
              table.data_ptr(), table.stride(0), table.shape[1], s["lens"].data_ptr(),
              out.data_ptr(), lse.data_ptr(), n, heads, s["strides"], s["scale"],
              s["workspace"].data_ptr(), s["workspace"].numel(), stream)
    got = {"out": out, "lse": lse}
    return {**got, "k": s["k"], "v": s["v"]} if s["append"] else got


def _own_logits(s, capi, stream):
    x = s["logits"]
    out = torch.empty_like(x)
    capi.call("tvr_adjust_logits", x.data_ptr(), x.stride(0), out.data_ptr(), out.stride(0),
              x.shape[0], x.shape[1], s["rules"], stream)
    return out


def run(state):
    op = state["op"]
    if own:
        from tvarant_b200 import capi

        stream = torch.cuda.current_stream().cuda_stream
        return {"plan": _own_plan, "append": _own_append, "attend": _own_attend,
                "logits": _own_logits}[op](state, capi, stream)
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend,
            "logits": _plain_logits}[op](state)


# ---- what a pass cannot do without ----------------------------------------


def work(case):
    if case["op"] == "plan":
        n, page = case["requests"], case["page"]
        rest = n - case["decode"] - min(case["finished"], n - case["decode"])
        prompts = [1 + (i * case["prompt"]) // max(1, rest) if case["prompt"] else 0
                   for i in range(rest)]
        tokens = case["decode"] + sum(prompts)
        # lengths in and out; a page id read and written for each page of new tokens; the outputs
        return {"bytes": 12 * n + 8 * (tokens // page + 1) + 16 * tokens, "flops": 0}
    if case["op"] == "append":
        size = 4 if case["type"] == "f32" else 2
        values = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        return {"bytes": values * (4 + size) + 8 * case["tokens"], "flops": 0}
    if case["op"] == "attend":
        size = 4 if case["type"] == "f32" else 2
        lens, d = _lengths(case), case["dim"]
        n, keys = case["requests"], sum(_lengths(case))
        b = 2 * size * d * case["kv_heads"] * keys + 4 * sum(-(-x // case["page"]) for x in lens)
        b += n * case["heads"] * (8 * d + 4) + 4 * n
        if case["append"]:
            b += 2 * n * case["kv_heads"] * d * 4 + 8 * n
        return {"bytes": b, "flops": 4 * d * case["heads"] * keys}
    n, vocab, hist = case["rows"], case["vocab"], case["history"]
    b = 8 * n * vocab + 3 * n * hist + 4 * n * case["biases"]
    return {"bytes": b + min(n, case["masks"]) * (vocab // 8), "flops": 4 * n * vocab}


# ---- the definitions in 64 bits -------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(s)
    if case["op"] == "logits":
        return _exact_logits(s)
    return _exact_pages(s) if case["op"] == "append" else _exact_attend(s)


def _exact_plan(s):
    """Request by request, with a list as the stack of free pages."""
    page, table = s["page"], s["table"].tolist()
    seq, new, count = s["seq"].tolist(), s["new"].tolist(), int(s["count"])
    free = s["free"].tolist()
    stack = free[:count]
    for r, x in enumerate(new):
        if x < 0:
            stack += table[r][: -(-seq[r] // page)]
    slots, positions, rows, full = [], [], [], False
    for r, x in enumerate(new):
        if x < 0:
            seq[r] = 0
            continue
        held, want = -(-seq[r] // page), -(-(seq[r] + x) // page)
        fits = want <= len(table[r])
        if fits and want - held > len(stack):
            full = True  # nobody behind it gets a page either
        refused = not fits or (full and want > held)
        if not refused:
            for c in range(held, want):
                table[r][c] = stack.pop()
        for i in range(seq[r], seq[r] + x):
            slots.append(-1 if refused else table[r][i // page] * page + i % page)
            positions.append(i)
            rows.append(r)
        if not refused:
            seq[r] += x
    free[count:len(stack)] = stack[count:]
    pad = s["tokens"] - len(slots)
    i32, i64 = torch.int32, torch.int64
    return {"table": torch.tensor(table, dtype=i32), "seq": torch.tensor(seq, dtype=i32),
            "count": torch.tensor([len(stack)], dtype=i32), "free": torch.tensor(free, dtype=i32),
            "slots": torch.tensor(slots + [-1] * pad, dtype=i64),
            "positions": torch.tensor(positions + [0] * pad, dtype=i32),
            "rows": torch.tensor(rows + [-1] * pad, dtype=i32)}


def _exact_pages(s):
    """The pages' values, the new rows before their rounding."""
    got = {}
    for name in ("k", "v"):
        pages, page = s[name].double(), s[name].shape[2]
        for t, slot in enumerate(s["slots"].tolist()):
            if slot >= 0:
                pages[slot // page, :, slot % page] = s[name + "_new"][t].double()
        got[name] = pages
    return got


def _exact_attend(s):
    q, page = s["q"].double(), s["k"].shape[2]
    n, heads, d = q.shape
    group = heads // s["k"].shape[1]
    out = torch.zeros(n, heads, d, dtype=torch.float64, device=DEV)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64, device=DEV)
    for r, length in enumerate(s["lens"].tolist()):
        if not length:
            continue
        pages = s["table"][r, : -(-length // page)].long()
        k, v = (s[x][pages].transpose(0, 1).flatten(1, 2)[:, :length].double() for x in "kv")
        if s["append"]:
            k[:, -1] = s["k_new"][r].to(s["type"]).double()
            v[:, -1] = s["v_new"][r].to(s["type"]).double()
        z = torch.einsum("hgd,hkd->hgk", q[r].view(-1, group, d), k) * s["scale"]
        lse[r] = torch.logsumexp(z, -1).flatten()
        out[r] = torch.einsum("hgk,hkd->hgd", torch.softmax(z, -1), v).reshape(heads, d)
    got = {"out": out, "lse": lse}
    return {**got, "k": None, "v": None} if s["append"] else got


def _exact_logits(s):
    x = s["logits"].double()
    n, vocab = x.shape
    prompt, total, nb = s["prompt"].tolist(), s["total"].tolist(), s["bias_counts"].tolist()
    for r in range(n):
        row = x[r]
        used, times = s["tokens"][r, : total[r]].long().unique(return_counts=True)
        rep = s["repetition"][r].double()
        row[used] = torch.where(row[used] > 0, row[used] / rep, row[used] * rep)
        used, times = s["tokens"][r, prompt[r]: total[r]].long().unique(return_counts=True)
        row[used] -= s["frequency"][r].double() * times + s["presence"][r].double()
        row.index_add_(0, s["bias_ids"][r, : nb[r]].long(), s["bias_values"][r, : nb[r]].double())
        m = int(s["mask_rows"][r])
        if m >= 0:
            bits = (s["masks"][m][:, None] >> torch.arange(32, device=DEV)) & 1
            row[bits.flatten()[:vocab] == 0] = -math.inf
    return x
