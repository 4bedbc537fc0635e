"""The page plan, the append to pages and the attention of one new token over
them (include/tvarant.h: tvr_page_plan, tvr_paged_append, tvr_paged_attention)
against plain implementations in Python and in 64 bits, at the sizes, layouts
and contents where they can go wrong.

The plan and fp32 appends are exact; 16-bit appends equal the rounding to
nearest even.  Attention computes in fp32: with N(0, 1) operands a score of D
products has an error of about sqrt(D) 2^-24 |q k| <= 1e-6, the terms that the
tensor-core form cuts its operands into leave at most 2^-21 more, and a weight's
relative error is its score's absolute one, so the outputs, sums of such
weights, are within 1e-5 (relative Frobenius) with room for the summation; the
log-sum-exp within 1e-5 of max(1, |lse|).
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from conftest import rel_frobenius

pytestmark = pytest.mark.gpu

TOL = 1e-5
CACHE_FULL, BAD_INDEX = 7, 8
TYPES = ["float32", "float16", "bfloat16"]


@pytest.fixture(scope="module")
def lib():
    import torch  # noqa: F401

    from tvarant_b200 import capi

    capi.load()
    capi.call("tvr_init")
    return capi


@pytest.fixture(autouse=True)
def clean_status(lib):
    lib.call("tvr_clear_status", 0)
    yield
    lib.call("tvr_clear_status", 0)


def _status(lib):
    import torch

    torch.cuda.synchronize()
    return lib.get_status(0)


# ---- the plan ---------------------------------------------------------------


def _plan_oracle(table, seq, new, free, count, page, tokens, per):
    """Request by request, with a list as the stack of free pages."""
    table, seq, free = table.copy(), seq.copy(), free.copy()
    stack = list(free[:count])
    for r, x in enumerate(new):
        if x < 0:
            stack += list(table[r, : -(-seq[r] // page)])
    slots = np.full(tokens, -1, np.int64)
    positions = np.zeros(tokens, np.int32)
    rows = np.full(tokens, -1, np.int32)
    full = refused_any = False
    start = 0
    for r, x in enumerate(new):
        if x < 0:
            seq[r] = 0
            continue
        held, want = -(-seq[r] // page), -(-(seq[r] + x) // page)
        room = x <= per if per else start + x <= tokens or x == 0
        fits = want <= table.shape[1] and room
        if fits and want - held > len(stack):
            full = True
        refused = not fits or (full and want > held)
        refused_any |= refused
        if not refused:
            for c in range(held, want):
                table[r, c] = stack.pop()
        for i in range(x):
            t = r * per + i if per else start + i
            if t >= tokens or (per and i >= per):
                break
            positions[t], rows[t] = seq[r] + i, r
            if not refused:
                slots[t] = table[r, (seq[r] + i) // page] * page + (seq[r] + i) % page
        start += x
        if not refused:
            seq[r] += x
    free[count:len(stack)] = stack[count:]
    return table, seq, free, len(stack), slots, positions, rows, refused_any


def _run_plan(lib, table, seq, new, free, count, page, tokens, per=0, in_place=False,
              optional=True):
    import torch

    t, s, n, f = (torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (table, seq, new, free))
    c = torch.tensor([count], dtype=torch.int32, device="cuda")
    s2, c2 = (s, c) if in_place else (torch.full_like(s, -7), torch.full_like(c, -7))
    slots = torch.full((max(tokens, 1),), -99, dtype=torch.int64, device="cuda")
    pos, rows = (torch.full((max(tokens, 1),), -99, dtype=torch.int32, device="cuda")
                 for _ in range(2))
    pl = lib.PagePool(t.data_ptr(), t.stride(0), t.shape[1], t.shape[0], f.data_ptr(), f.numel(),
                      page)
    lib.call("tvr_page_plan", pl, s.data_ptr(), n.data_ptr(), s2.data_ptr(), c.data_ptr(),
             c2.data_ptr(), slots.data_ptr(), pos.data_ptr() if optional else None,
             rows.data_ptr() if optional else None, tokens, per,
             torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return [x.cpu().numpy() for x in (t, s2, f, c2, slots, pos, rows)]


def _pool_state(rng, lens, page, max_pages, spare):
    held = [-(-x // page) for x in lens]
    ids = rng.permutation(sum(held) + spare).astype(np.int32)
    table = rng.integers(-5, 5, (len(lens), max_pages)).astype(np.int32)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = ids[at:at + h]
        at += h
    free = np.full(len(ids), -3, np.int32)
    free[:spare] = ids[at:]
    return table, free


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("page", [1, 16, 24])
@pytest.mark.parametrize("requests, hi, news, spare, per", [
    (1, 40, [5], 10, 0),
    (7, 60, [1, 1, 0, -1, 200, -1, 3], 30, 0),     # the 200 may exceed the pool
    (8, 60, [1, 1, 0, -1, 4, -1, 3, 1], 0, 0),     # only what the ended ones give up
    (33, 90, None, 12, 0),
    (1025, 300, None, 400, 0),
    (6, 50, [1, 0, 1, 1, -1, 1], 9, 1),            # a decode step's row form
    (5, 50, [3, 9, 0, 8, 1], 40, 8),               # one request has more than its row
    (64, 33, None, 64, 4),
])
def test_plan_against_a_list(lib, requests, hi, news, spare, per, page, in_place):
    rng = np.random.default_rng(requests * 31 + page + spare)
    lens = rng.integers(0, hi, requests).astype(np.int32)
    new = (np.asarray(news, np.int32) if news is not None
           else rng.choice([-1, 0, 1, 1, 1, 2, 17], requests).astype(np.int32))
    max_pages = -(-(hi + 210) // page)
    table, free = _pool_state(rng, lens, page, max_pages, spare)
    total = int(new[new > 0].sum())
    tokens = requests * per if per else total + 3
    want = _plan_oracle(table, lens, new, free, spare, page, tokens, per)
    got = _run_plan(lib, table, lens, new, free, spare, page, tokens, per, in_place)
    for name, g, w in zip(("table", "lens", "free", "count", "slots", "positions", "rows"), got,
                          [*want[:3], np.array([want[3]]), *want[4:7]]):
        assert np.array_equal(g[:len(w)] if name in ("slots", "positions", "rows") else g, w), name
    assert _status(lib) == (CACHE_FULL if want[7] else 0)


def test_plan_refuses_tokens_past_the_arrays_and_pages_past_the_table(lib):
    rng = np.random.default_rng(3)
    lens = np.array([10, 20, 30, 40], np.int32)
    table, free = _pool_state(rng, lens, 16, 4, 20)
    # request 1 needs a fifth column; request 2's tokens end past the arrays
    new = np.array([1, 50, 4, 1], np.int32)
    want = _plan_oracle(table, lens, new, free, 20, 16, 54, 0)
    got = _run_plan(lib, table, lens, new, free, 20, 16, 54, optional=False)
    assert want[7] and np.array_equal(got[1], [11, 20, 30, 40])
    for g, w in zip(got[:5], [*want[:3], np.array([want[3]]), want[4]]):
        assert np.array_equal(g, w)
    assert _status(lib) == CACHE_FULL


def test_plan_without_requests_or_tokens(lib):
    got = _run_plan(lib, np.zeros((1, 4), np.int32), np.array([3], np.int32),
                    np.array([0], np.int32), np.arange(9, dtype=np.int32), 9, 16, 0)
    assert got[1][0] == 3 and got[3][0] == 9 and got[4][0] == -99
    assert _status(lib) == 0


def test_steps_of_a_server_neither_lose_nor_share_a_page(lib):
    """200 steps in place: requests start, grow, end; at every step the pages
    in use and the free ones are all pages, each once."""
    import torch

    rng = np.random.default_rng(9)
    R, page, max_pages, num = 12, 4, 10, 70
    table = torch.zeros(R, max_pages, dtype=torch.int32, device="cuda")
    seq = torch.zeros(R, dtype=torch.int32, device="cuda")
    free = torch.arange(num, dtype=torch.int32, device="cuda")
    count = torch.tensor([num], dtype=torch.int32, device="cuda")
    slots = torch.empty(R * 9, dtype=torch.int64, device="cuda")
    pl = lib.PagePool(table.data_ptr(), max_pages, max_pages, R, free.data_ptr(), num, page)
    for _ in range(200):
        new = torch.from_numpy(rng.choice([-1, 0, 1, 1, 1, 1, 1, 9], R).astype(np.int32)).cuda()
        lib.call("tvr_page_plan", pl, seq.data_ptr(), new.data_ptr(), seq.data_ptr(),
                 count.data_ptr(), count.data_ptr(), slots.data_ptr(), None, None, R * 9, 0,
                 torch.cuda.current_stream().cuda_stream)
        lens, tab = seq.cpu().numpy(), table.cpu().numpy()
        used = np.concatenate([tab[r, : -(-lens[r] // page)] for r in range(R)])
        rest = free.cpu().numpy()[: int(count)]
        assert sorted([*used, *rest]) == list(range(num))
        s = slots.cpu().numpy()
        s = s[s >= 0]
        assert len(set(s)) == len(s)
    assert _status(lib) in (0, CACHE_FULL)


# ---- pages --------------------------------------------------------------------


def _pages(lib, torch, shape, dtype, layout, fill, offset=0):
    """[pages, heads, page, dim] with the heads outside the positions ("head")
    or inside them ("token"); `offset` elements past an aligned address."""
    p, h, s, d = shape
    n = p * h * s * d
    flat = torch.full((n + offset,), fill, dtype=torch.float32).to(getattr(torch, dtype)).cuda()
    flat = flat[offset:]
    if layout == "head":
        return flat.view(p, h, s, d)
    return flat.view(p, s, h, d).transpose(1, 2)


def _cache(lib, k, v):
    code = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2}[str(k.dtype)]
    return lib.PagedKV(k.data_ptr(), v.data_ptr(), code, 0, k.shape[0], k.shape[2], k.shape[1],
                       k.shape[3], (ctypes.c_int64 * 3)(*k.stride()[:3]),
                       (ctypes.c_int64 * 3)(*v.stride()[:3]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("tokens, heads, dim, page, offset", [
    (1, 1, 64, 16, 0), (37, 3, 64, 16, 0), (501, 2, 128, 24, 0), (29, 5, 7, 4, 0),
    (33, 2, 64, 16, 1), (20, 1, 256, 1, 0),
])
def test_append_places_and_rounds(lib, dtype, layout, tokens, heads, dim, page, offset):
    import torch

    rng = np.random.default_rng(tokens + dim)
    num = -(-tokens // page) + 4
    k = _pages(lib, torch, (num, heads, page, dim), dtype, layout, 9.0, offset)
    v = _pages(lib, torch, (num, heads, page, dim), dtype, layout, -9.0, offset)
    # rows of a fused projection; values that f16 cannot hold, NaN and infinities among them
    src = (rng.standard_normal((tokens, 3, heads, dim)) * 10.0 ** rng.integers(-9, 6, (tokens, 3, heads, dim))
           ).astype(np.float32)
    src[0, 1, 0, 0], src[0, 2, 0, -1] = np.nan, np.inf
    dsrc = torch.from_numpy(src).cuda()
    kn, vn = dsrc[:, 1], dsrc[:, 2]
    slots = rng.permutation(num * page)[:tokens].astype(np.int64)
    slots[tokens // 3::5] = -1
    ds = torch.from_numpy(slots).cuda()
    want_k, want_v = k.cpu().clone(), v.cpu().clone()
    for t, s in enumerate(slots):
        if s >= 0:
            want_k[s // page, :, s % page] = torch.from_numpy(src[t, 1]).to(k.dtype)
            want_v[s // page, :, s % page] = torch.from_numpy(src[t, 2]).to(k.dtype)
    st = (ctypes.c_int64 * 4)(*kn.stride()[:2], *vn.stride()[:2])
    lib.call("tvr_paged_append", _cache(lib, k, v), kn.data_ptr(), vn.data_ptr(), st, ds.data_ptr(),
             tokens, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(k.cpu().nan_to_num(7), want_k.nan_to_num(7))
    assert torch.equal(v.cpu().nan_to_num(7), want_v.nan_to_num(7))
    assert _status(lib) == 0


def test_append_drops_slots_past_the_pages(lib):
    import torch

    k = torch.zeros(3, 2, 4, 8, device="cuda")
    v = torch.zeros(3, 2, 4, 8, device="cuda")
    src = torch.ones(3, 2, 8, device="cuda")
    slots = torch.tensor([12, 5, 1 << 40], dtype=torch.int64, device="cuda")
    st = (ctypes.c_int64 * 4)(16, 8, 16, 8)
    lib.call("tvr_paged_append", _cache(lib, k, v), src.data_ptr(), src.data_ptr(), st,
             slots.data_ptr(), 3, torch.cuda.current_stream().cuda_stream)
    assert _status(lib) == BAD_INDEX
    assert float(k.sum()) == 16.0 and float(k[1, :, 1].sum()) == 16.0


# ---- attention ------------------------------------------------------------------


class Case:
    """A cache of requests of the given lengths, its pages in random order and
    everything that no request holds NaN."""

    def __init__(self, lib, lens, heads, kv_heads, dim, page, dtype="float32", layout="head",
                 seed=0, offset=0, spare=2, spread=1.0):
        import torch

        self.lib, self.torch, self.lens = lib, torch, list(lens)
        rng = np.random.default_rng(seed + sum(lens) + dim)
        R = len(lens)
        held = [-(-max(x, 0) // page) for x in lens]
        self.max_pages = max(max(held), 1)
        num = sum(held) + spare
        ids = rng.permutation(num).astype(np.int32)
        table = rng.integers(-9, num + 9, (R, self.max_pages)).astype(np.int32)  # stale entries
        self.k = _pages(lib, torch, (num, kv_heads, page, dim), dtype, layout, math.nan, offset)
        self.v = _pages(lib, torch, (num, kv_heads, page, dim), dtype, layout, math.nan, offset)
        self.rows = []  # per request: keys, values as the pages hold them, in 64 bits
        at = 0
        for r, n in enumerate(lens):
            pages = ids[at:at + held[r]]
            table[r, :held[r]] = pages
            at += held[r]
            kr = torch.from_numpy(spread * rng.standard_normal((kv_heads, max(n, 0), dim))).to(self.k.dtype)
            vr = torch.from_numpy(rng.standard_normal((kv_heads, max(n, 0), dim))).to(self.k.dtype)
            for i, pg in enumerate(pages):
                lo, hi = i * page, min(n, (i + 1) * page)
                self.k[int(pg), :, : hi - lo] = kr[:, lo:hi].cuda()
                self.v[int(pg), :, : hi - lo] = vr[:, lo:hi].cuda()
            self.rows.append((kr.double().numpy(), vr.double().numpy()))
        qkv = rng.standard_normal((R, heads + 2 * kv_heads, dim)).astype(np.float32)
        self.qkv = torch.from_numpy(qkv).cuda()
        self.q = self.qkv[:, :heads]
        self.k_new, self.v_new = self.qkv[:, heads:heads + kv_heads], self.qkv[:, heads + kv_heads:]
        self.table = torch.from_numpy(table).cuda()
        self.seq = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.slots = torch.tensor(
            [int(table[r, (n - 1) // page]) * page + (n - 1) % page if n > 0 else -1
             for r, n in enumerate(lens)], dtype=torch.int64, device="cuda")
        self.heads, self.dim, self.page, self.scale = heads, dim, page, 1.0 / math.sqrt(dim)
        size = ctypes.c_int64()
        lib.call("tvr_paged_attention_workspace", heads, kv_heads, dim, ctypes.byref(size))
        self.workspace = torch.zeros(size.value, dtype=torch.uint8, device="cuda")

    def run(self, append=False, slots=None, out=None, stream=None, lse=True):
        torch, lib = self.torch, self.lib
        R = len(self.lens)
        if out is None:
            out = torch.full((R, self.heads, self.dim), math.nan, device="cuda")
        got_lse = torch.full((R, self.heads), math.nan, device="cuda")
        slots = self.slots if slots is None else slots
        st = (ctypes.c_int64 * 8)(*self.q.stride()[:2], *self.k_new.stride()[:2],
                                  *self.v_new.stride()[:2], *out.stride()[:2])
        new = (self.k_new.data_ptr(), self.v_new.data_ptr(), slots.data_ptr()) if append else (None,) * 3
        lib.call("tvr_paged_attention", _cache(lib, self.k, self.v), self.q.data_ptr(), *new,
                 self.table.data_ptr(), self.table.stride(0), self.max_pages, self.seq.data_ptr(),
                 out.data_ptr(), got_lse.data_ptr() if lse else None, R, self.heads, st, self.scale,
                 self.workspace.data_ptr(), self.workspace.numel(),
                 stream or torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return out.cpu().numpy(), got_lse.cpu().numpy()

    def want(self, append=False):
        R, kv = len(self.lens), self.k.shape[1]
        out = np.zeros((R, self.heads, self.dim))
        lse = np.full((R, self.heads), -np.inf)
        q = self.q.cpu().double().numpy()
        for r, n in enumerate(self.lens):
            if n <= 0:
                continue
            k, v = (x.copy() for x in self.rows[r])
            if append:
                k[:, -1] = self.k_new[r].to(self.k.dtype).double().cpu().numpy()
                v[:, -1] = self.v_new[r].to(self.k.dtype).double().cpu().numpy()
            for h in range(self.heads):
                g = h // (self.heads // kv)
                z = k[g] @ q[r, h] * self.scale
                m = z.max()
                w = np.exp(z - m)
                out[r, h] = w @ v[g] / w.sum()
                lse[r, h] = m + np.log(w.sum())
        return out, lse

    def check(self, append=False, **kw):
        out, lse = self.run(append, **kw)
        want, want_lse = self.want(append)
        assert np.isfinite(out).all()
        assert rel_frobenius(out, want) <= TOL, rel_frobenius(out, want)
        fin = np.isfinite(want_lse)
        assert np.array_equal(lse[~fin], want_lse[~fin])
        if fin.any():
            assert np.max(np.abs(lse[fin] - want_lse[fin]) / np.maximum(1, np.abs(want_lse[fin]))) <= 1e-5
        assert not self.workspace[:4096].any()  # left ready for the next call
        return out, lse


LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 129, 200, 513, 0, 31, 1000]


@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv_heads, dim", [
    (12, 12, 64), (4, 2, 64), (14, 2, 64), (18, 2, 64), (4, 4, 128), (8, 2, 128), (10, 2, 128),
    (16, 2, 128), (12, 1, 128), (40, 1, 128), (2, 2, 256), (6, 2, 256), (24, 2, 256), (3, 3, 32),
    (6, 3, 80), (5, 5, 96), (8, 1, 96), (2, 2, 200),
])
def test_attention_head_layouts(lib, heads, kv_heads, dim, dtype, append):
    c = Case(lib, LENS, heads, kv_heads, dim, 16, dtype)
    c.check(append)
    assert _status(lib) == 0


@pytest.mark.parametrize("layout", ["head", "token"])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 128])
@pytest.mark.parametrize("heads, kv_heads, dim, dtype", [
    (3, 3, 64, "float32"), (3, 3, 128, "bfloat16"), (8, 1, 128, "float16"), (4, 1, 128, "bfloat16"),
    (8, 2, 64, "float32"),
])
def test_attention_page_sizes(lib, page, layout, heads, kv_heads, dim, dtype):
    c = Case(lib, [0, 1, 7, 100, 333, 24, 48], heads, kv_heads, dim, page, dtype, layout, seed=page)
    c.check(append=page % 2 == 0)
    assert _status(lib) == 0


@pytest.mark.parametrize("heads, kv_heads, dim, dtype, offset", [
    (4, 2, 64, "float32", 1), (4, 2, 64, "bfloat16", 1), (6, 3, 7, "float32", 0),
    (6, 2, 33, "float16", 0), (2, 1, 4, "bfloat16", 0),
])
def test_attention_without_whole_chunks(lib, heads, kv_heads, dim, dtype, offset):
    """Rows that are not 16-byte chunks: the general form."""
    for append in (False, True):
        c = Case(lib, [0, 1, 5, 40, 129], heads, kv_heads, dim, 16, dtype, offset=offset)
        c.check(append)
    assert _status(lib) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv_heads, lens", [
    (12, 12, [5000]), (8, 1, [30011]), (32, 8, [9000, 3]), (4, 1, [20000]), (16, 1, [12345]),
    (12, 12, [40] * 130 + [3000]), (8, 8, [100] * 300), (32, 4, [70, 1, 300] * 60),
])
def test_attention_split_over_many_ctas(lib, heads, kv_heads, lens, dtype):
    """Requests cut into many parts, and many requests in a part; the same bits
    every time."""
    c = Case(lib, lens, heads, kv_heads, 64 if heads == 12 else 128, 16, dtype)
    out, lse = c.check(append=True)
    for _ in range(3):
        again, lse2 = c.run(append=True)
        assert np.array_equal(out, again) and np.array_equal(lse, lse2)
    assert _status(lib) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("heads, kv_heads, lens", [
    (16, 1, LENS * 4 + [33, 400, 70]), (16, 1, LENS * 4 + [33, 400, 70, 9]),
    (9, 1, [130] * 63 + [9000]), (40, 2, LENS * 3), (24, 1, [5] * 65),
])
def test_attention_of_more_heads_than_a_block_of_rows(lib, heads, kv_heads, lens, dim, dtype):
    """Units of 8 and of 16 heads, whole and with heads to spare, on both sides of
    64 (request, key head) pairs."""
    c = Case(lib, lens, heads, kv_heads, dim, 16, dtype, seed=dim)
    out, lse = c.check(append=True)
    again, lse2 = c.run(append=True)
    assert np.array_equal(out, again) and np.array_equal(lse, lse2)
    assert _status(lib) == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads, kv_heads", [(3, 3), (8, 2)])
def test_append_form_is_append_then_attend(lib, heads, kv_heads, dtype):
    import torch

    a = Case(lib, LENS, heads, kv_heads, 64, 16, dtype)
    b = Case(lib, LENS, heads, kv_heads, 64, 16, dtype)
    out, lse = a.run(append=True)
    st = (ctypes.c_int64 * 4)(*b.k_new.stride()[:2], *b.v_new.stride()[:2])
    lib.call("tvr_paged_append", _cache(lib, b.k, b.v), b.k_new.data_ptr(), b.v_new.data_ptr(), st,
             b.slots.data_ptr(), len(LENS), torch.cuda.current_stream().cuda_stream)
    out2, lse2 = b.run()
    assert np.array_equal(out, out2) and np.array_equal(lse, lse2)
    for x, y in ((a.k, b.k), (a.v, b.v)):
        assert torch.equal(x.nan_to_num(3), y.nan_to_num(3))
    # a request without a slot appends nothing and attends to what is there
    none = torch.full_like(a.slots, -1)
    c = Case(lib, LENS, heads, kv_heads, 64, 16, dtype)
    out3, _ = c.run(append=True, slots=none)
    assert rel_frobenius(out3, c.want()[0]) <= TOL


def test_strided_outputs_and_inputs(lib):
    import torch

    c = Case(lib, [3, 77, 0, 200], 6, 3, 64, 16)
    buf = torch.full((4, 2, 6, 65), math.nan, device="cuda")
    out = buf[:, 1, :, :64]  # rows 65 floats apart: not on 16-byte boundaries
    c.q = torch.randn(4, 6, 3, 64, device="cuda")[:, :, 1]
    c.check(out=out)
    assert torch.isnan(buf[:, 0]).all() and torch.isnan(buf[:, :, :, 64]).all()
    c.run(lse=False)


def test_scores_far_apart(lib):
    """Weights that underflow, running maxima that jump: keys up to 300 apart."""
    for heads, kv_heads, dtype in ((2, 2, "float32"), (8, 1, "float32"), (8, 1, "float16"),
                                   (4, 1, "bfloat16"), (7, 1, "bfloat16")):
        c = Case(lib, [700, 64, 1500], heads, kv_heads, 128, 16, dtype, spread=30.0)
        out, lse = c.run()
        want, want_lse = c.want()
        # scores of up to 340 carry errors of up to sqrt(128) 2^-24 340 = 2.3e-4
        # and, in the tensor-core form, 2^-21 340 = 1.6e-4
        assert rel_frobenius(out, want) <= 1e-3
        assert np.max(np.abs(lse - want_lse)) <= 1e-3
    assert _status(lib) == 0


def test_rows_of_minus_infinity_and_of_nan(lib):
    """A request whose scores are all -inf gives what the formula gives (NaN,
    lse -inf); one of its keys NaN, a NaN row; the others are untouched."""
    import torch

    for heads, kv_heads, dim in ((2, 2, 64), (2, 2, 7)):
        c = Case(lib, [20, 33, 50], heads, kv_heads, dim, 16)
        c.q[0] = 0.0
        c.q[0, :, 0] = 1.0
        page_ids = c.table[0, :2].cpu().tolist()
        for j in range(20):
            c.k[page_ids[j // 16], :, j % 16] = 0.0
            c.k[page_ids[j // 16], :, j % 16, 0] = -math.inf
        c.k[int(c.table[1, 1]), 0, 3, 1] = math.nan  # position 19 of request 1, head 0
        out, lse = c.run()
        assert np.isnan(out[0]).all() and (lse[0] == -np.inf).all()
        assert np.isnan(out[1, 0]).all() and np.isfinite(out[1, 1]).all()
        want, _ = c.want()
        assert rel_frobenius(out[2], want[2]) <= TOL
        torch.cuda.synchronize()


def test_bad_page_ids_are_dropped(lib):
    for heads, kv_heads, dim in ((2, 2, 64), (8, 1, 128), (2, 2, 5)):
        lib.call("tvr_clear_status", 0)
        c = Case(lib, [40, 100], heads, kv_heads, dim, 16)
        c.table[0, 1] = 1 << 30
        c.table[1, 2] = -1
        out, _ = c.run()
        assert _status(lib) == BAD_INDEX
        for r, (lo, hi) in enumerate(((16, 32), (32, 48))):
            k, v = c.rows[r]
            keep = np.r_[0:lo, hi:c.lens[r]]
            c.rows[r] = k[:, keep], v[:, keep]
        want, _ = c.want()
        assert rel_frobenius(out, want) <= TOL
    lib.call("tvr_clear_status", 0)
    c = Case(lib, [40], 2, 2, 64, 16)
    bad = c.torch.full_like(c.slots, 1 << 40)
    out, _ = c.run(append=True, slots=bad)  # appends nothing
    assert _status(lib) == BAD_INDEX
    assert rel_frobenius(out, c.want()[0]) <= TOL


def test_lengths_outside_the_table(lib):
    c = Case(lib, [64, 32], 2, 2, 64, 16)
    c.seq.copy_(c.torch.tensor([1 << 30, -5], dtype=c.torch.int32))
    c.lens = [64, -5]
    out, lse = c.run()
    want, want_lse = c.want()
    assert rel_frobenius(out, want) <= TOL and (out[1] == 0).all() and (lse[1] == -np.inf).all()


def test_on_a_stream_of_its_own(lib):
    import torch

    c = Case(lib, [300, 20], 12, 12, 64, 16)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    out, _ = c.run(append=True, stream=s.cuda_stream)
    assert rel_frobenius(out, c.want(append=True)[0]) <= TOL


def test_offsets_past_32_bits(lib):
    """Pages 2.4 GB apart: element offsets past 2^31 in every form."""
    import torch

    for dim, heads, kv_heads, dtype in ((64, 2, 2, "bfloat16"), (64, 8, 2, "float16"),
                                        (63, 2, 2, "bfloat16")):
        c = Case(lib, [40], heads, kv_heads, dim, 16, dtype, spare=0)
        want, _ = c.want(append=True)
        step = 1200000000
        big = torch.empty(2 * step + 16 * 2 * dim, dtype=c.k.dtype, device="cuda")
        far = big.as_strided((3, kv_heads, 16, dim), (step, 16 * dim, dim, 1))
        far.copy_(c.k)
        c.k = far
        big2 = torch.empty_like(big)
        far2 = big2.as_strided((3, kv_heads, 16, dim), (step, 16 * dim, dim, 1))
        far2.copy_(c.v)
        c.v = far2
        out, _ = c.run(append=True)
        assert rel_frobenius(out, want) <= TOL
        del c, far, far2, big, big2
        torch.cuda.empty_cache()
    assert _status(lib) == 0


def test_torch_operators(lib):
    """The tvarant device's operators give what the C entry points give, and
    refuse what they do not take."""
    import torch

    import torch_tvarant  # noqa: F401
    from tvarant_b200.paged import new_paged_cache

    ops = torch.ops.tvarant
    g = torch.Generator().manual_seed(4)
    for dtype in (torch.float32, torch.bfloat16):
        cache = new_paged_cache(1, 3, 20, 8, 64, 4, 2, 64, "tvarant", dtype)
        assert cache.requests == 3 and cache.page_size == 8
        new = torch.tensor([5, 0, 20], dtype=torch.int32).to("tvarant")
        slots, positions, rows = cache.plan(new, tokens=25)
        assert rows.cpu().tolist() == [0] * 5 + [2] * 20
        assert positions.cpu().tolist() == [*range(5), *range(20)]
        kv = torch.randn(25, 2, 2, 64, generator=g)
        d = kv.to("tvarant")
        cache.append(0, d[:, 0], d[:, 1], slots)
        q = torch.randn(3, 4, 64, generator=g)
        o = cache.attend(0, q.to("tvarant"), 0.125).cpu()
        x = kv.to(dtype).double()
        for r, (a, b) in ((0, (0, 5)), (2, (5, 25))):
            k, v = x[a:b, 0].repeat_interleave(2, 1), x[a:b, 1].repeat_interleave(2, 1)
            w = torch.softmax(torch.einsum("hd,khd->hk", q[r].double(), k) * 0.125, -1)
            want = torch.einsum("hk,khd->hd", w, v)
            assert rel_frobenius(o[r].numpy(), want.numpy()) <= TOL
        assert (o[1] == 0).all()
        # a decode step: the append form equals append, then attend
        one = torch.tensor([1, 0, 1], dtype=torch.int32).to("tvarant")
        slots, _, _ = cache.plan(one, tokens_per_request=1)
        assert slots.shape == (3, 1) and slots.cpu()[1, 0] == -1
        n = torch.randn(3, 2, 2, 64, generator=g).to("tvarant")
        o1 = cache.append_attend(0, q.to("tvarant"), n[:, 0], n[:, 1], slots.view(3), 0.125).cpu()
        assert torch.equal(o1, cache.attend(0, q.to("tvarant"), 0.125).cpu())
        end = torch.tensor([-1, -1, -1], dtype=torch.int32).to("tvarant")
        cache.plan(end, tokens=1)
        assert cache.seq_lens.cpu().tolist() == [0, 0, 0] and int(cache.free_count.cpu()) == 20
        qd = q.to("tvarant")
        for bad in (lambda: cache.attend(0, qd[:, :3], 0.125), lambda: cache.attend(0, qd[:2], 0.125),
                    lambda: cache.attend(0, qd[:, :, :32], 0.125),
                    lambda: ops.paged_append_(cache.k[0], cache.v[0], n[:, 0], n[:, 1],
                                              slots.view(3)[:2]),
                    lambda: cache.plan(one[:2], tokens=1), lambda: cache.plan(one, tokens=-1),
                    lambda: ops.paged_attention(qd, cache.k[0], cache.v[0], cache.block_table,
                                                cache.seq_lens, 0.125, cache.workspace[:64])):
            with pytest.raises(RuntimeError):
                bad()
    with pytest.raises(ValueError):
        new_paged_cache(1, 1, 1, 1, 1, 4, 3, 64, "tvarant")
    with pytest.raises(ValueError):
        new_paged_cache(1, 1, 1, 1, 1, 4, 4, 64, "tvarant", torch.float64)
    assert _status(lib) == 0
