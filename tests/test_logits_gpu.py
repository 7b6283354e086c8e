"""nd_logits_penalty against the definition in 64 bits.

The kernel rounds every step to fp32: with M the largest magnitude of a value
on its way (and of what is added to it), each of the at most five steps is off
by at most 2^-24 M, a sum of n biases by n of them; a bf16 output adds 2^-8 of
the result.  The greedy token has to be the first index of the largest value
that was written.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _ops():
    from neurodsl_b200 import ops
    return ops


def reference(x, history, lens, rep, pres, freq, ids, bias, mask):
    """Rows of float64 values and the magnitude that bounds each one's roundings."""
    x = x.astype(np.float64)
    rows, V = x.shape
    mag = np.abs(x)
    steps = np.full((rows, V), 5.0)
    for r in range(rows):
        if history is not None:
            n = history.shape[1] if lens is None else min(max(lens[r], 0), history.shape[1])
            h = history[r, :n]
            tok, c = np.unique(h[(h >= 0) & (h < V)], return_counts=True)
            y = x[r, tok]
            if rep is not None:
                y = np.where(y > 0, y / np.float64(rep[r]), y * np.float64(rep[r]))
            mag[r, tok] = np.maximum(mag[r, tok], np.abs(y))
            if pres is not None:
                y = y - np.float64(pres[r])
                mag[r, tok] += abs(pres[r])
            if freq is not None:
                y = y - np.float64(freq[r]) * c
                mag[r, tok] += abs(freq[r]) * c
            x[r, tok] = y
        if ids is not None:
            for t, b in zip(ids[r], bias[r]):
                if 0 <= t < V:
                    x[r, t] += np.float64(b)
                    mag[r, t] += abs(b)
                    steps[r, t] += 1
    if mask is not None:
        m = np.broadcast_to(mask, (rows, mask.shape[-1]))
        bits = (m[:, :, None].astype(np.uint32) >> np.arange(32, dtype=np.uint32)) & 1
        x[bits.reshape(rows, -1)[:, :V] == 0] = -np.inf
    return x, steps * 2.0**-24 * mag


def check(out, idx, want, tol):
    got = out.float().cpu().numpy().astype(np.float64)
    fin = np.isfinite(want)
    np.testing.assert_array_equal(got[~fin], want[~fin])
    if out.dtype == torch.bfloat16:
        tol = tol + 2.0**-8 * np.abs(np.where(fin, want, 0)) * (1 + 2.0**-6) + 2.0**-133
    assert (np.abs(got[fin] - want[fin]) <= tol[fin]).all()
    if idx is not None:
        key = np.where(np.isnan(got), -np.inf, got)
        np.testing.assert_array_equal(idx.cpu().numpy(), key.argmax(1))


def run(rows, V, n_hist, n_bias=0, masked=False, dtype=torch.float32, out_dtype=None, seed=0,
        pad=0, in_place=False, lens=False, parts=("rep", "pres", "freq"), one_mask=False, dup=False):
    rng = np.random.default_rng(seed)
    base = torch.from_numpy(rng.standard_normal((rows, V + pad)).astype(np.float32) * 4).to(DEV).to(dtype)
    x = base[:, :V]
    hist = hl = rep = pres = freq = ids = bias = mask = None
    if n_hist:
        hist = rng.integers(0, max(1, V // 3), (rows, n_hist)).astype(np.int32)
        hist[rng.random(hist.shape) < 0.2] = -1
        hist[:, 0] = V - 1
        if lens:
            hl = rng.integers(0, n_hist + 1, rows).astype(np.int32)
        rep = rng.uniform(0.7, 1.6, rows).astype(np.float32) if "rep" in parts else None
        pres = rng.uniform(-1, 1, rows).astype(np.float32) if "pres" in parts else None
        freq = rng.uniform(-0.3, 0.6, rows).astype(np.float32) if "freq" in parts else None
    if n_bias:
        ids = rng.integers(0, max(1, V // 2) if not dup else max(1, min(V, 5)), (rows, n_bias)).astype(np.int32)
        ids[rng.random(ids.shape) < 0.2] = -1
        bias = rng.standard_normal((rows, n_bias)).astype(np.float32) * 3
    if masked:
        words = (V + 31) // 32
        mask = rng.integers(0, 2**32, (1 if one_mask else rows, words), dtype=np.uint64).astype(np.uint32)
        mask[0] = 0                       # a row that allows nothing
        if rows > 1 and not one_mask:
            mask[1] = 0
            mask[1, words // 2] = 1       # one token
    d = lambda a: None if a is None else torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).to(DEV)
    m_dev = d(mask)
    if one_mask:
        m_dev = m_dev[0]
    want, tol = reference(x.float().cpu().numpy(), hist, hl, rep, pres, freq, ids, bias, mask)
    out = x if in_place else None
    guard = base[:, V:].clone()
    y, idx = _ops().logits_penalty(x, history=d(hist), history_lens=d(hl), repetition=d(rep),
                                   presence=d(pres), frequency=d(freq), bias_ids=d(ids), bias=d(bias),
                                   mask=m_dev, out=out, out_dtype=out_dtype)
    torch.cuda.synchronize()
    check(y, idx, want, tol)
    assert torch.equal(base[:, V:], guard)
    assert _ops().device_error() == 0
    return y, idx


@pytest.mark.parametrize("rows, V", [(1, 1), (3, 31), (2, 32), (5, 33), (2, 4095), (3, 4097), (1, 50257), (7, 8192), (2, 131073)])
@pytest.mark.parametrize("dtype, out_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                              (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)])
def test_sizes_and_types(rows, V, dtype, out_dtype):
    run(rows, V, 40, 7, True, dtype, out_dtype, seed=V)


@pytest.mark.parametrize("n_hist", [0, 1, 255, 3000])
@pytest.mark.parametrize("n_bias", [0, 1, 33, 500])
def test_lists(n_hist, n_bias):
    run(3, 1000, n_hist, n_bias, seed=n_hist + n_bias, lens=True)


@pytest.mark.parametrize("parts", [(), ("rep",), ("pres",), ("freq",), ("rep", "freq")])
def test_each_penalty_alone(parts):
    run(2, 500, 60, parts=parts, seed=len(parts))


def test_strides_and_in_place():
    for dtype in (torch.float32, torch.bfloat16):
        run(4, 1001, 30, 5, True, dtype, pad=7, seed=1)
        run(4, 1001, 30, 5, True, dtype, pad=7, in_place=True, seed=2)
        run(4, 1024, 30, 5, True, dtype, in_place=True, seed=3)


def test_one_mask_for_all_rows():
    run(6, 777, 10, 0, True, one_mask=True)


def test_tokens_listed_many_times():
    """Biases of the same token add up in list order, the same bits each time."""
    a = run(2, 300, 100, 400, dup=True, seed=8)
    b = run(2, 300, 100, 400, dup=True, seed=8)
    assert torch.equal(a[0], b[0])


def test_many_rows():
    run(700, 257, 20, 3, True, seed=4)


def test_ties_infinities_and_nan():
    ops = _ops()
    x = torch.full((4, 9000), 1.0, device=DEV)
    x[1, 5000:] = math.inf
    x[2] = math.nan
    x[2, 8000] = -math.inf
    x[3] = -math.inf
    out, idx = ops.logits_penalty(x)
    assert idx.tolist() == [0, 5000, 8000, 0]
    assert torch.equal(out.nan_to_num(5.0), x.nan_to_num(5.0))
    # a token under the mask is gone even where its logit is NaN or +inf
    mask = torch.full((282,), -1, dtype=torch.int32, device=DEV)
    mask[5000 // 32:] = 0
    out, idx = ops.logits_penalty(x, mask=mask)
    assert (out[:, 5024:] == -math.inf).all() and idx.tolist()[:2] == [0, 0]
    # -inf stays -inf under every penalty
    hist = torch.arange(100, dtype=torch.int32, device=DEV).repeat(4, 1)
    one = torch.ones(4, device=DEV)
    out, _ = ops.logits_penalty(x, history=hist, repetition=2 * one, presence=one, frequency=one)
    assert (out[3] == -math.inf).all() and (out[1, 5000:] == math.inf).all()


def test_bad_tokens_are_skipped():
    ops = _ops()
    x = torch.zeros((2, 50), device=DEV)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    one = torch.ones(2, device=DEV)
    out, _ = ops.logits_penalty(x, history=i32([[50, 3], [-2, 2**31 - 1]]), presence=one)
    assert ops.device_error() == 16
    want = torch.zeros((2, 50), device=DEV)
    want[0, 3] = -1
    assert torch.equal(out, want)
    out, _ = ops.logits_penalty(x, bias_ids=i32([[50], [4]]), bias=torch.ones((2, 1), device=DEV))
    assert ops.device_error() == 16
    assert out[0].abs().max() == 0 and out[1, 4] == 1
    out, _ = ops.logits_penalty(x, history=i32([[1, 2], [1, 2]]), history_lens=i32([3, -1]), presence=one)
    assert ops.device_error() == 16
    assert out[0, 1] == -1 and out[0, 2] == -1 and out[1].abs().max() == 0


def test_greedy_only_and_buffers():
    ops = _ops()
    x = torch.randn(5, 3000, device=DEV)
    out, idx = ops.logits_penalty(x, greedy=False)
    assert idx is None and torch.equal(out, x)
    buf, ib = torch.empty(5, 3000, device=DEV), torch.empty(5, dtype=torch.int32, device=DEV)
    a, b = ops.logits_penalty(x, out=buf, idx=ib)
    assert a is buf and b is ib and torch.equal(ib.long(), x.argmax(1))


def test_captured():
    ops = _ops()
    x = torch.randn(3, 20000, device=DEV)
    hist = torch.randint(0, 20000, (3, 50), dtype=torch.int32, device=DEV)
    f = torch.full((3,), 0.5, device=DEV)
    out, idx = torch.empty_like(x), torch.empty(3, dtype=torch.int32, device=DEV)
    ops.logits_penalty(x, history=hist, frequency=f, out=out, idx=idx)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.logits_penalty(x, history=hist, frequency=f, out=out, idx=idx)
    for _ in range(3):
        x.copy_(torch.randn(3, 20000, device=DEV))
        g.replay()
        want = ops.logits_penalty(x, history=hist, frequency=f)
        assert torch.equal(out, want[0]) and torch.equal(idx, want[1])


def test_refusals():
    ops = _ops()
    x = torch.zeros((2, 50), device=DEV)
    h = torch.zeros((2, 3), dtype=torch.int32, device=DEV)
    for kw in (dict(history=h[:1]), dict(history=h, repetition=torch.ones(1, device=DEV)),
               dict(bias_ids=h), dict(mask=torch.zeros((2, 1), dtype=torch.int32, device=DEV)),
               dict(out=torch.zeros((2, 49), device=DEV)), dict(history=h, history_lens=h[0])):
        with pytest.raises(ValueError):
            ops.logits_penalty(x, **kw)
    for kw in (dict(history=h.long()), dict(mask=torch.zeros((2, 2), device=DEV)),
               dict(history=h, presence=torch.ones(2, dtype=torch.float64, device=DEV)),
               dict(history=h.cpu())):
        with pytest.raises(TypeError):
            ops.logits_penalty(x, **kw)
    with pytest.raises(RuntimeError):
        ops.logits_penalty(x, presence=torch.ones(2, device=DEV))      # a penalty without a history
    with pytest.raises(RuntimeError):
        big = torch.zeros(200, device=DEV)
        ops.logits_penalty(big[:100].view(2, 50), out=big[50:150].view(2, 50))


def test_out_beside_logits_in_one_buffer():
    ops = _ops()
    buf = torch.randn(4, 2000, device=DEV)
    x = buf[:, :1000].clone()
    out, idx = ops.logits_penalty(buf[:, :1000], out=buf[:, 1000:])
    assert torch.equal(out, x) and torch.equal(buf[:, :1000], x) and torch.equal(idx.long(), x.argmax(1))
    with pytest.raises(RuntimeError):
        ops.logits_penalty(buf[:, :1000], out=buf[:, 999:1999])


@pytest.mark.parametrize("n_hist, n_bias, V", [(9000, 0, 30000), (20000, 300, 9001), (7000, 7000, 70000), (1, 0, 300000)])
def test_long_lists(n_hist, n_bias, V):
    """Lists longer than the largest table, vocabularies longer than a bit map."""
    run(2, V, n_hist, n_bias, True, seed=n_hist, lens=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, V, n_hist, n_bias, pad", [
    (5, 4097, 700, 40, 0), (3, 4099, 64, 3, 7), (6, 33, 300, 20, 1), (2, 20011, 9000, 300, 2)])
def test_in_place_with_lists(dtype, rows, V, n_hist, n_bias, pad):
    """Listed tokens are computed from the logits that the stream overwrites."""
    run(rows, V, n_hist, n_bias, True, dtype, dtype, seed=V + pad, pad=pad, in_place=True, lens=True)


@pytest.mark.parametrize("V, n_hist", [(50257, 1024), (6000, 6000), (130001, 6144)])
def test_histories_of_different_tokens(V, n_hist):
    """Every entry another token: the fullest table."""
    rng = np.random.default_rng(V)
    rows = 3
    hist = np.stack([rng.permutation(V)[:n_hist] for _ in range(rows)]).astype(np.int32)
    x = torch.from_numpy(rng.standard_normal((rows, V)).astype(np.float32) * 4).to(DEV).to(torch.bfloat16)
    rep, freq = np.full(rows, 1.3, np.float32), np.full(rows, 0.2, np.float32)
    want, tol = reference(x.float().cpu().numpy(), hist, None, rep, None, freq, None, None, None)
    d = lambda a: torch.from_numpy(a).to(DEV)
    y, idx = _ops().logits_penalty(x, history=d(hist), repetition=d(rep), frequency=d(freq), out_dtype=torch.float32)
    check(y, idx, want, tol)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, V, pad", [(3, 8191, 1), (5, 9001, 47), (2, 5, 2), (300, 2050, 3)])
def test_padded_logits_and_a_tight_output(dtype, out_dtype, rows, V, pad):
    """Rows whose place within 16 bytes differs between input and output."""
    run(rows, V, 50, 5, True, dtype, out_dtype, seed=V, pad=pad, lens=True)


@pytest.mark.parametrize("dtype, out_dtype, in_place", [
    (torch.bfloat16, torch.bfloat16, False), (torch.bfloat16, torch.bfloat16, True),
    (torch.bfloat16, torch.float32, False), (torch.float32, torch.bfloat16, False)])
@pytest.mark.parametrize("V", [1, 2, 3, 8, 33, 4097])
def test_listed_tokens_at_the_ends_of_a_row(dtype, out_dtype, in_place, V):
    """Wherever in a word the row begins and ends; what lies beside it is none of
    the call's."""
    rng = np.random.default_rng(V)
    ids = np.array([[0, V - 1]], np.int32)
    hist = np.array([[V - 1, 0, V - 1]], np.int32)
    bias, freq = np.array([[1.5, -2.5]], np.float32), np.full(1, 0.25, np.float32)
    d = lambda a: torch.from_numpy(a).to(DEV)
    for first in range(4):
        buf = torch.full((first + V + 4,), math.nan, device=DEV).to(dtype)
        x = buf[first:first + V].view(1, V)
        x.copy_(torch.from_numpy(rng.standard_normal((1, V)).astype(np.float32)))
        want, tol = reference(x.float().cpu().numpy(), hist, None, None, None, freq, ids, bias, None)
        out, idx = _ops().logits_penalty(x, history=d(hist), frequency=d(freq), bias_ids=d(ids), bias=d(bias),
                                         out=x if in_place else None, out_dtype=out_dtype)
        check(out, idx, want, tol)
        assert buf[:first].isnan().all() and buf[first + V:].isnan().all()
    assert _ops().device_error() == 0


@pytest.mark.parametrize("direct", [True, False])
def test_an_empty_history(monkeypatch, direct):
    """[rows][0], as before the first token: nothing is penalised; a length that is
    not 0 is reported like any other outside [0, n]."""
    from neurodsl_b200 import _lib
    ops = _ops()
    if not direct:
        monkeypatch.setattr(_lib, "calls", False)
    x = torch.randn((3, 500), device=DEV)
    empty = torch.empty((3, 0), dtype=torch.int32, device=DEV)
    half = torch.full((3,), 0.5, device=DEV)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    for lens, code in ((None, 0), (i32([0, 0, 0]), 0), (i32([0, 1, 0]), 16), (i32([-1, 0, 0]), 16)):
        out, idx = torch.empty_like(x), i32([9, 9, 9])
        ops.logits_penalty(x, history=empty, history_lens=lens, repetition=1 + half, presence=half, frequency=half,
                           out=out, idx=idx)
        assert torch.equal(out, x) and torch.equal(idx.long(), x.argmax(1))
        assert ops.device_error() == code
    out, _ = ops.logits_penalty(x, history=empty, presence=half, bias_ids=i32([[7], [8], [9]]), bias=2 * half[:, None])
    want = x.clone()
    for r in range(3):
        want[r, 7 + r] += 1
    assert torch.equal(out, want)
    with pytest.raises(RuntimeError):
        ops.logits_penalty(x, presence=half)
