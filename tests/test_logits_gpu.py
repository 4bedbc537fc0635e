"""tvr_adjust_logits and tvr_history_append against the formula in 64 bits.

Each logit goes through at most one product, one subtraction of a product, one
subtraction and the additions of its biases, each rounded to fp32: the error is
within (4 + biases of the token) 2^-24 of the largest magnitude on the way.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

BAD_INDEX = 8


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


def _make(rng, rows, vocab, history, biases, masks, bits=32):
    total = rng.integers(0, history + 1, rows).astype(np.int32)
    prompt = (total * rng.random(rows)).astype(np.int32)
    ids = (vocab * rng.random((rows, max(history, 1))) ** 3).astype(np.int32 if bits == 32 else np.int64)
    ids[rng.random(ids.shape) < 0.1] = -1              # ids that are no tokens
    ids[rng.random(ids.shape) < 0.05] = vocab
    ids[rng.random(ids.shape) < 0.02] = 2**31 - 1 if bits == 32 else 2**40
    words = -(-vocab // 32)
    bits_ = rng.integers(0, 2**32, (max(masks, 1), words), dtype=np.uint64).astype(np.uint32)
    bits_[::3] = 0                                     # nothing is allowed
    bits_[1::3] = 0xffffffff
    bias_ids = rng.integers(-2, vocab + 3, (rows, max(biases, 1))).astype(np.int32)
    bias_ids[:, ::4] = bias_ids[:, :1]                 # tokens of several biases
    d = dict(x=(4 * rng.standard_normal((rows, vocab))).astype(np.float32), tokens=ids,
             prompt=prompt, total=total,
             rep=rng.uniform(1, 2, rows).astype(np.float32),
             pres=rng.uniform(-1, 1, rows).astype(np.float32),
             freq=rng.uniform(-1, 1, rows).astype(np.float32), bias_ids=bias_ids,
             bias_values=(3 * rng.standard_normal(bias_ids.shape)).astype(np.float32),
             bias_counts=rng.integers(0, max(biases, 1) + 1, rows).astype(np.int32), masks=bits_,
             mask_rows=rng.integers(-1, max(masks, 1), rows).astype(np.int32), bits=bits)
    return d


def _want(d, parts):
    """The values, and the bound on their errors."""
    x = d["x"].astype(np.float64)
    rows, vocab = x.shape
    big = np.abs(x)
    ops = np.full(x.shape, 4.0)
    for r in range(rows):
        if "tokens" in parts:
            t = d["tokens"][r, : d["total"][r]]
            ok = (t >= 0) & (t < vocab)
            used = np.unique(t[ok])
            rep = float(d["rep"][r]) if "rep" in parts else 1.0
            x[r, used] = np.where(x[r, used] > 0, x[r, used] / rep, x[r, used] * rep)
            made = t[d["prompt"][r]:] if "prompt" in parts else t
            made = made[(made >= 0) & (made < vocab)]
            c = np.bincount(made, minlength=vocab)
            f = float(d["freq"][r]) if "freq" in parts else 0.0
            p = float(d["pres"][r]) if "pres" in parts else 0.0
            big[r] = np.maximum(big[r], np.abs(x[r])) + np.abs(f * c) + np.abs(p) * (c > 0)
            x[r] -= f * c + p * (c > 0)
        if "bias" in parts:
            n = d["bias_counts"][r] if "bias_counts" in parts else d["bias_ids"].shape[1]
            for i, v in zip(d["bias_ids"][r, :n], d["bias_values"][r, :n]):
                if 0 <= i < vocab:
                    x[r, i] += float(v)
                    big[r, i] += abs(float(v))
                    ops[r, i] += 1
        if "masks" in parts:
            m = d["mask_rows"][r] if "mask_rows" in parts else r
            if m >= 0:
                v = np.arange(vocab)
                x[r, ((d["masks"][m][v // 32] >> (v % 32)) & 1) == 0] = -np.inf
    return x, ops * 2.0**-24 * big


ALL = ("tokens", "prompt", "rep", "pres", "freq", "bias", "bias_counts", "masks", "mask_rows")


def _run(lib, d, parts, x=None, out=None):
    import torch

    g = {k: torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).cuda()
         for k, v in d.items() if isinstance(v, np.ndarray)}
    ptr = lambda name, key=None: g[key or name].data_ptr() if name in parts else None  # noqa: E731
    bias = "bias" in parts
    r = lib.LogitRules(
        ptr("tokens"), d["bits"], 0, g["tokens"].stride(0), ptr("prompt"), ptr("tokens", "total"),
        ptr("rep"), ptr("pres"), ptr("freq"), g["bias_ids"].data_ptr() if bias else None,
        g["bias_values"].data_ptr() if bias else None, ptr("bias_counts"), g["bias_ids"].shape[1],
        ptr("masks"), g["masks"].stride(0), g["masks"].shape[0], ptr("mask_rows"))
    x = g["x"] if x is None else x
    out = torch.full_like(x, math.nan) if out is None else out
    lib.call("tvr_adjust_logits", x.data_ptr(), x.stride(0), out.data_ptr(), out.stride(0),
             x.shape[0], x.shape[1], r, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def _check(got, want, bound):
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    fin = np.isfinite(want)
    assert (np.abs(got[fin] - want[fin]) <= bound[fin]).all()


@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("rows, vocab, history, biases, masks", [
    (1, 1, 1, 1, 1), (1, 50257, 300, 5, 1), (3, 1003, 50, 40, 2), (2, 31, 0, 1, 2),
    (5, 2048, 700, 9, 3), (17, 50257, 1000, 600, 17), (2, 129280, 20000, 300, 2),
    (4, 8193, 3, 0, 4), (300, 4099, 100, 3, 7),
])
def test_every_part(lib, rows, vocab, history, biases, masks, bits):
    rng = np.random.default_rng(rows * vocab)
    d = _make(rng, rows, vocab, history, biases, masks, bits)
    got = _run(lib, d, ALL)
    want, bound = _want(d, ALL)
    _check(got, want, bound)
    assert np.array_equal(got, _run(lib, d, ALL), equal_nan=True)  # the same bits again
    assert lib.get_status(0) == 0


@pytest.mark.parametrize("parts", [
    (), ("tokens",), ("tokens", "rep"), ("tokens", "prompt", "rep"), ("tokens", "freq"),
    ("tokens", "prompt", "pres"), ("bias",), ("bias", "bias_counts"), ("masks",),
    ("masks", "mask_rows"), ("bias", "masks"),
])
def test_parts_alone(lib, parts):
    rng = np.random.default_rng(len(parts))
    d = _make(rng, 6, 5003, 200, 30, 6)
    got = _run(lib, d, parts)
    want, bound = _want(d, parts)
    _check(got, want, bound)
    if not parts:
        assert np.array_equal(got, d["x"])


@pytest.mark.parametrize("history", [32767, 32768, 40000])
@pytest.mark.parametrize("vocab", [5003, 70001])
def test_counters_of_both_widths(lib, vocab, history):
    """A token that makes up the whole history, with or without a prompt before
    it, and others beside it: the counts of neighbours stay apart."""
    d = _make(np.random.default_rng(history), 3, vocab, history, 5, 3)
    d["total"][:] = history
    d["tokens"][0] = 4000
    d["tokens"][1] = 4001
    d["tokens"][1, ::2] = 4000
    d["tokens"][2, :9000] = 4097
    d["prompt"][:] = [0, 5, 0]
    d["freq"][:] = [0.001, -0.002, 0.5]
    got = _run(lib, d, ALL)
    want, bound = _want(d, ALL)
    _check(got, want, bound)


@pytest.mark.parametrize("bits", [32, 64])
@pytest.mark.parametrize("rows, vocab, history, biases, masks", [
    (700, 2053, 90, 10, 600), (900, 33, 5, 40, 3), (320, 4099, 700, 300, 320), (160, 40001, 300, 20, 7),
    (601, 9000, 0, 3, 0),
])
def test_many_rows(lib, rows, vocab, history, biases, masks, bits):
    """Rows enough for many CTAs an SM, also in place and with rows that start
    anywhere; the same bits every time."""
    import torch

    d = _make(np.random.default_rng(rows), rows, vocab, max(1, history), biases, max(1, masks), bits)
    parts = [x for x in ALL if (history or x not in ("tokens", "prompt")) and
             (masks or x not in ("masks", "mask_rows"))]
    want, bound = _want(d, parts)
    got = _run(lib, d, parts)
    _check(got, want, bound)
    assert np.array_equal(got, _run(lib, d, parts), equal_nan=True)
    buf = torch.full((rows, vocab + 10), math.nan, device="cuda")
    x = buf[:, 3:3 + vocab]
    x.copy_(torch.from_numpy(d["x"]))
    _check(_run(lib, d, parts, x=x, out=x), want, bound)
    assert torch.isnan(buf[:, :3]).all() and torch.isnan(buf[:, 3 + vocab:]).all()


def test_in_place_and_with_strides(lib):
    import torch

    rng = np.random.default_rng(1)
    d = _make(rng, 5, 1537, 100, 20, 5)
    want, bound = _want(d, ALL)
    for pad, shift, out_shift in ((0, 0, 0), (7, 3, 3), (5, 1, 2), (4, 0, 1)):
        buf = torch.full((5, 1537 + pad + 8), math.nan, device="cuda")
        x = buf[:, shift:shift + 1537]
        x.copy_(torch.from_numpy(d["x"]))
        obuf = torch.full((5, 1537 + pad + 8), math.nan, device="cuda")
        out = obuf[:, out_shift:out_shift + 1537]
        _check(_run(lib, d, ALL, x=x, out=out), want, bound)
        assert torch.isnan(obuf[:, :out_shift]).all()
        assert torch.isnan(obuf[:, out_shift + 1537:]).all()
        _check(_run(lib, d, ALL, x=x, out=x), want, bound)  # in place
        assert torch.isnan(buf[:, shift + 1537:]).all()


def test_nan_and_infinities(lib):
    """What a mask forbids is -inf whatever it was; elsewhere NaN and infinities
    stay what they are, and other logits do not see them."""
    rng = np.random.default_rng(2)
    d = _make(rng, 4, 3001, 60, 10, 4)
    d["x"][0, 10:20] = np.nan
    d["x"][1, 100] = np.inf
    d["x"][2, ::7] = -np.inf
    d["bias_values"][3, 0] = np.inf
    d["masks"][:] = 0xffffffff
    d["masks"][0, 0] = ~np.uint32((1 << 12) | 1)  # token 0 and token 12
    d["mask_rows"][:] = [0, -1, 0, 0]
    with np.errstate(invalid="ignore"):
        got = _run(lib, d, ALL)
        want, bound = _want(d, ALL)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert got[0, 12] == -np.inf and np.isnan(got[0, 13])
    fin = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fin)
    assert (np.abs(got[fin] - want[fin]) <= bound[fin]).all()


def test_biases_add_in_list_order(lib):
    """Large biases cancel in fp32 only in the order of the list."""
    d = _make(np.random.default_rng(3), 1, 100, 1, 70, 1)
    d["x"][:] = 1.0
    ids = np.full((1, 70), 5, np.int32)
    vals = np.zeros((1, 70), np.float32)
    vals[0, :4] = [1e8, 0.25, -1e8, 0.5]
    vals[0, 69] = 2.0
    d["bias_ids"], d["bias_values"] = ids, vals
    acc = np.float32(1.0)
    for v in vals[0]:
        acc = np.float32(acc + v)
    got = _run(lib, d, ("bias",))
    assert got[0, 5] == acc and (np.delete(got[0], 5) == 1.0).all()


def test_mask_rows_out_of_range(lib):
    d = _make(np.random.default_rng(4), 3, 100, 1, 1, 2)
    d["mask_rows"][:] = [0, 2, -1]
    got = _run(lib, d, ("masks", "mask_rows"))
    assert lib.get_status(0) == BAD_INDEX
    assert np.array_equal(got[1:], d["x"][1:])


def test_lengths_are_bounded_by_the_arrays(lib):
    d = _make(np.random.default_rng(5), 2, 500, 40, 6, 2)
    d["total"][:] = [2**30, -3]
    d["bias_counts"][:] = [2**30, -1]
    got = _run(lib, d, ALL)
    d["total"][:] = [40, 0]
    d["bias_counts"][:] = [6, 0]
    want, bound = _want(d, ALL)
    _check(got, want, bound)


@pytest.mark.parametrize("bits", [32, 64])
def test_history_append(lib, bits):
    import torch

    dt = torch.int32 if bits == 32 else torch.int64
    tokens = torch.full((4, 6), -1, dtype=dt, device="cuda")
    lens = torch.tensor([0, 5, 6, 2], dtype=torch.int32, device="cuda")
    ids = torch.tensor([7, 8, 9, 10], dtype=torch.int64, device="cuda")
    live = torch.tensor([1, 1, 1, 0], dtype=torch.int32, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    lib.call("tvr_history_append", tokens.data_ptr(), bits, 6, lens.data_ptr(), ids.data_ptr(),
             live.data_ptr(), 4, 6, st)
    assert lens.cpu().tolist() == [1, 6, 6, 2]
    assert tokens[0, 0] == 7 and tokens[1, 5] == 8 and (tokens[2:] == -1).all()
    lib.call("tvr_history_append", tokens.data_ptr(), bits, 6, lens.data_ptr(), ids.data_ptr(),
             None, 4, 6, st)
    assert lens.cpu().tolist() == [2, 6, 6, 3] and tokens[3, 2] == 10


def test_torch_operator(lib):
    import torch

    import torch_tvarant  # noqa: F401
    from tvarant_b200.paged import LogitRules

    d = _make(np.random.default_rng(6), 3, 1003, 30, 10, 3)
    dev = {k: torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).to("tvarant")
           for k, v in d.items() if isinstance(v, np.ndarray)}
    rules = LogitRules(dev["tokens"], dev["prompt"], dev["total"], dev["rep"], dev["pres"],
                       dev["freq"], dev["bias_ids"], dev["bias_values"], dev["bias_counts"],
                       dev["masks"], dev["mask_rows"])
    want, bound = _want(d, ALL)
    _check(rules.apply(dev["x"]).cpu().numpy(), want, bound)
    assert torch.equal(LogitRules().apply(dev["x"]).cpu(), dev["x"].cpu())
    ops = torch.ops.tvarant
    for bad in (lambda: ops.adjust_logits(dev["x"][0]),
                lambda: ops.adjust_logits(dev["x"], tokens=dev["tokens"]),
                lambda: ops.adjust_logits(dev["x"], repetition=dev["rep"][:2]),
                lambda: ops.adjust_logits(dev["x"], bias_ids=dev["bias_ids"]),
                lambda: ops.adjust_logits(dev["x"], masks=dev["masks"][:, :3]),
                lambda: ops.history_append_(dev["tokens"], dev["total"], dev["total"])):
        with pytest.raises(RuntimeError):
            bad()
