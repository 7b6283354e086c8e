"""nd_window_attn_fwd against the definition in 64 bits.

Tolerances.  With A = sum_j p_j |v_j| and O = sum_j p_j v_j (p the exact
weights): the kernel rounds each weight to bf16 before the second product,
once, and once more where a later half of the same K/V tile raises the row's
offset (relative 2^-8 each), and rounds a bf16 output once (2^-8 |O|).  The
fp32 part: a score is a sum of 64 products, its error at most
66 * 2^-24 * scale * sum |q k| =: E, which is a relative error of p; the sums
over n keys add at most n * 2^-23; the hardware exponential 2^-22.
"""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

D = 64


def _ops():
    from neurodsl_b200 import ops
    return ops


def reference(Q, K, V, window, sinks, scale):
    B, H, Sq, _ = Q.shape
    Hkv, Sk = K.shape[1], K.shape[2]
    q = Q.double()
    k = K.double().repeat_interleave(H // Hkv, 1)
    v = V.double().repeat_interleave(H // Hkv, 1)
    s = q @ k.transpose(-1, -2) * scale
    mag = (q.abs() @ k.abs().transpose(-1, -2)).max().item() * abs(scale)
    p = torch.arange(Sk - Sq, Sk, device="cuda")[:, None]
    j = torch.arange(Sk, device="cuda")[None, :]
    seen = (j <= p) & ((j > p - window) | (j < sinks))
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    w = torch.exp(s - lse[..., None])
    return w @ v, w @ v.abs(), lse, s.amax(-1), mag


def compare(got, want, out_dtype, n):
    O, lse, m = got
    ref, A, lse_ref, m_ref, mag = want
    E = 66 * 2.0**-24 * mag + n * 2.0**-23 + 2.0**-22
    tol = (2 * 2.0**-8 + 2 * E) * A
    if out_dtype == torch.bfloat16:
        tol = tol + 2.0**-8 * ref.abs() * (1 + 2.0**-6)
    assert ((O.double() - ref).abs() <= tol).all()
    assert ((lse.double() - lse_ref).abs() <= 2 * E + 2.0**-21 * (1 + lse_ref.abs())).all()
    assert ((m.double() - m_ref).abs() <= E + 2.0**-22 * (1 + m_ref.abs())).all()


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16)


def make(layout, B, H, Hkv, Sq, Sk, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    heads = lambda x, n: x.unflatten(-1, (n, D)).transpose(1, 2)
    if layout == "head":
        return (_randn(g, B, H, Sq, D), _randn(g, B, Hkv, Sk, D), _randn(g, B, Hkv, Sk, D),
                torch.empty(B, H, Sq, D, device="cuda", dtype=torch.bfloat16))
    out = heads(torch.empty(B, Sq, H * D, device="cuda", dtype=torch.bfloat16), H)
    if layout == "token":
        qkv = _randn(g, B, Sk, (H + 2 * Hkv) * D)
        return (heads(qkv[:, Sk - Sq:, :H * D], H), heads(qkv[..., H * D:(H + Hkv) * D], Hkv),
                heads(qkv[..., (H + Hkv) * D:], Hkv), out)
    # a cache whose rows past Sk hold anything
    k, v = _randn(g, B, Hkv, Sk + 37, D), _randn(g, B, Hkv, Sk + 37, D)
    k[:, :, Sk:] = math.nan
    v[:, :, Sk:] = math.inf
    return heads(_randn(g, B, Sq, H * D), H), k[:, :, :Sk], v[:, :, :Sk], out


CASES = [
    # B, H, Hkv, Sq, Sk, window, sinks
    (1, 1, 1, 1, 1, 1, 0),
    (2, 2, 2, 5, 5, 3, 0),
    (1, 2, 1, 1, 700, 64, 4),          # one query against many keys
    (1, 4, 2, 127, 128, 16, 1),
    (1, 12, 12, 213, 213, 64, 4),
    (2, 6, 2, 129, 1000, 128, 0),      # positions that do not start at a tile
    (1, 3, 3, 300, 300, 1, 0),         # a row sees itself alone
    (1, 2, 2, 300, 300, 1, 2),
    (1, 2, 2, 513, 513, 513, 7),
    (1, 2, 1, 640, 640, 2**31 - 1, 0),  # no window at all
    (1, 4, 1, 257, 777, 100, 300),     # sinks over several tiles
    (1, 1, 1, 1024, 1024, 256, 128),
    (1, 2, 2, 1000, 1000, 129, 129),
    (1, 2, 2, 900, 1111, 127, 130),    # sinks that end inside the window's first tile
    (1, 2, 2, 600, 600, 2, 2**31 - 1),  # every key a sink
    (2, 100, 50, 130, 130, 17, 2),     # more items than SMs
    (1, 1, 1, 5000, 5000, 700, 4),
]


@pytest.mark.parametrize("layout", ["head", "token", "cache"])
@pytest.mark.parametrize("B, H, Hkv, Sq, Sk, window, sinks", CASES)
def test_against_definition(B, H, Hkv, Sq, Sk, window, sinks, layout):
    Q, K, V, out = make(layout, B, H, Hkv, Sq, Sk)
    got = _ops().window_attn_fwd(Q, K, V, window, sinks=sinks, out=out)
    assert got[0] is out
    compare(got, reference(Q, K, V, window, sinks, 0.125), torch.bfloat16, Sk)


@pytest.mark.parametrize("layout", ["head", "token"])
def test_fp32_output_and_scale(layout):
    Q, K, V, _ = make(layout, 2, 4, 2, 300, 450, seed=3)
    got = _ops().window_attn_fwd(Q, K, V, 77, sinks=5, scale=0.3, out_dtype=torch.float32)
    compare(got, reference(Q, K, V, 77, 5, 0.3), torch.float32, 450)


def test_large_scores_move_the_offset():
    """Scores that grow by hundreds along the keys: the running offset is
    raised again and again, and the first keys of a window stop mattering."""
    Q, K, V, out = make("head", 1, 2, 1, 400, 400, seed=5)
    K *= torch.linspace(0.1, 30, 400, device="cuda")[None, None, :, None].to(torch.bfloat16)
    got = _ops().window_attn_fwd(Q, K, V, 150, sinks=3, out=out)
    compare(got, reference(Q, K, V, 150, 3, 0.125), torch.bfloat16, 400)


def test_writes_only_its_rows():
    """A chunk's output goes into a longer buffer; the rows around stay."""
    Q, K, V, _ = make("head", 2, 2, 2, 70, 200, seed=1)
    big = torch.full((2, 2, 75, D), 7.0, device="cuda", dtype=torch.bfloat16)
    lse = torch.full((2, 2, 70), math.nan, device="cuda")
    got = _ops().window_attn_fwd(Q, K, V, 50, sinks=1, out=big[:, :, :70], lse=lse)
    compare(got, reference(Q, K, V, 50, 1, 0.125), torch.bfloat16, 200)
    assert (big[:, :, 70:] == 7.0).all()


def test_full_window_is_causal_attention():
    """Small problems sum a row's keys in two groups, nd_flash_attn_fwd in one, so
    the two agree to rounding: each lies within the bounds above of the same
    exact result, hence within twice those of the other (bits: 2 * (2 * 2^-8 A +
    2^-8 |O|), and the fp32 terms of lse and the maxima, which no grouping
    changes for the maxima)."""
    ops = _ops()
    Q, K, V, out = make("token", 2, 4, 4, 333, 333, seed=2)
    a = ops.window_attn_fwd(Q, K, V, 333)
    b = ops.flash_attn_fwd(Q, K, V, causal=True)
    want = reference(Q, K, V, 333, 0, 0.125)
    compare(a, want, torch.bfloat16, 333)
    compare(b, want, torch.bfloat16, 333)
    assert torch.equal(a[2], b[2])


def test_same_bits_every_time_and_in_a_graph():
    ops = _ops()
    Q, K, V, out = make("cache", 2, 4, 2, 300, 500, seed=4)
    lse = torch.empty(2, 4, 300, device="cuda")
    m = torch.empty_like(lse)
    first = [t.clone() for t in ops.window_attn_fwd(Q, K, V, 90, sinks=4, out=out, lse=lse, row_max=m)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.window_attn_fwd(Q, K, V, 90, sinks=4, out=out, lse=lse, row_max=m)
    for _ in range(3):
        out.zero_()
        lse.zero_()
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip((out, lse, m), first):
            assert torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = ops.window_attn_fwd(Q, K, V, 90, sinks=4, stream=side)
    side.synchronize()
    assert torch.equal(got[0], first[0])


def test_refusals():
    ops = _ops()
    Q, K, V, out = make("head", 1, 4, 2, 10, 20)
    with pytest.raises(ValueError):
        ops.window_attn_fwd(Q, K, V[:, :1], 4)
    with pytest.raises(ValueError):
        ops.window_attn_fwd(Q, K, V, 4, out=out[:, :2])
    with pytest.raises(TypeError):
        ops.window_attn_fwd(Q.float(), K, V, 4)
    with pytest.raises(TypeError):
        ops.window_attn_fwd(Q, K.cpu(), V, 4)
    for kw in (dict(window=0), dict(window=4, sinks=-1), dict(window=4, scale=-1.0)):
        with pytest.raises(RuntimeError):
            ops.window_attn_fwd(Q, K, V, **kw)
    with pytest.raises(RuntimeError):
        ops.window_attn_fwd(K, Q[:, :2], Q[:, :2], 4)       # more queries than keys


@pytest.mark.parametrize("B, H, Hkv, Sq, Sk, window, sinks", [
    (2, 70, 35, 256, 300, 33, 2),      # two one-tile items for some SMs, streams of 1 to 3 tiles
    (1, 146, 73, 250, 640, 250, 1),
    (1, 3, 1, 384, 384, 384, 0),
    (4, 8, 8, 128, 128, 128, 0),       # a stream of one tile, shared by two groups
    (1, 2, 2, 1, 128, 128, 0),         # its last position alone: nothing to mask but the copy
    (1, 2, 2, 1, 129, 1, 0),
])
def test_one_tile_items(B, H, Hkv, Sq, Sk, window, sinks):
    Q, K, V, out = make("cache", B, H, Hkv, Sq, Sk, seed=Sk)
    got = _ops().window_attn_fwd(Q, K, V, window, sinks=sinks, out=out)
    compare(got, reference(Q, K, V, window, sinks, 0.125), torch.bfloat16, Sk)


def test_results_do_not_depend_on_the_sm_limit():
    ops = _ops()
    for shape in ((1, 8, 4, 300, 500), (2, 100, 50, 300, 300)):
        Q, K, V, _ = make("head", *shape, seed=7)
        want = ops.window_attn_fwd(Q, K, V, 70, sinks=4)
        with ops.sm_limit(5):
            got = ops.window_attn_fwd(Q, K, V, 70, sinks=4)
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_single_rows_of_any_stride():
    """The stride of a dimension of one row is never applied."""
    ops = _ops()
    Q, K, V, _ = make("head", 2, 4, 2, 1, 90, seed=8)
    want = ops.window_attn_fwd(Q, K, V, 40, sinks=1)
    odd = Q.as_strided(Q.shape, (4 * D, D, 3, 1))
    got = ops.window_attn_fwd(odd, K, V, 40, sinks=1)
    assert torch.equal(got[0], want[0])
    q, k, v, _ = make("head", 1, 2, 2, 1, 1, seed=9)
    got = ops.window_attn_fwd(q, k.as_strided(k.shape, (2 * D, D, 1, 1)), v, 2**40, sinks=2**40)
    compare(got, reference(q, k, v, 1, 0, 0.125), torch.bfloat16, 1)
