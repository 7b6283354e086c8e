"""The paged key-value cache (nd_paged_decode_attn, nd_paged_kv_store,
nd_paged_kv_evict) against the definitions in 64 bits.

Decode tolerances, with p the exact weights, A = sum_j p_j |v_j| and n keys:
a score is a sum of 64 products kept in fp32, then scaled by log2(e): absolute
error at most E1 = 66 * 2^-24 * scale * sum |q k| + 2^-22 * |s|, a relative
error of p; sums over keys and their joining add at most n * 2^-23, the
exponential and the divisions a few 2^-23.  So p, l and o are each within
E = E1 + (n + 32) * 2^-23, relative to A where they are summed.  A bf16 output
rounds each weight (2^-8 A) and the result (2^-8 |O|); an fp32 output splits
each weight into three bf16 terms (2^-24).
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

D = 64
DEV = "cuda"


def _ops():
    from neurodsl_b200 import ops
    return ops


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)


class Cache:
    """A pool in random page order whose unused rows hold NaN and infinities,
    and a table whose unused entries are no pages at all."""

    def __init__(self, lens, Hkv, page, seed=0, max_len=None, extra_pages=2, spare=0):
        g = self.g = _gen(seed)
        self.Hkv, self.page = Hkv, page
        B = len(lens)
        most = max(max(lens, default=0), max_len or 0)
        self.max_pages = -(-most // page) + extra_pages
        used = [-(-L // page) for L in lens]
        n = sum(used) + 3 + spare
        self.k = torch.full((n, Hkv, page, D), math.nan, device=DEV, dtype=torch.bfloat16)
        self.v = torch.full((n, Hkv, page, D), math.inf, device=DEV, dtype=torch.bfloat16)
        order = torch.randperm(n, generator=g, device=DEV).tolist()
        table = torch.full((B, self.max_pages), -(2**31), dtype=torch.int32)
        self.free = order[sum(used):]
        at = 0
        for b, L in enumerate(lens):
            ids = order[at:at + used[b]]
            at += used[b]
            table[b, :used[b]] = torch.tensor(ids, dtype=torch.int32)
            for i, p in enumerate(ids):
                r = min(page, L - i * page)
                self.k[p, :, :r] = _randn(g, Hkv, r, D)
                self.v[p, :, :r] = _randn(g, Hkv, r, D)
        self.table = table.to(DEV)
        self.lens_list = list(lens)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def rows(self, pool, b, h, L, table=None):
        t = (self.table if table is None else table)[b, :-(-L // self.page)].long()
        return pool[t, h].reshape(-1, D)[:L]


def visible(L, window, sinks):
    j = torch.arange(L, device=DEV)
    return j if window <= 0 else j[(j >= L - window) | (j < sinks)]


def check_decode(c, q, out, lse, window, sinks, scale, weights=None, weights0=None, k=None, v=None):
    k = c.k if k is None else k
    v = c.v if v is None else v
    B, H, _ = q.shape
    G = H // c.Hkv
    for b, L in enumerate(c.lens_list):
        j = visible(L, window, sinks)
        n = j.numel()
        if n == 0:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
            continue
        for h in range(c.Hkv):
            hs = slice(h * G, (h + 1) * G)
            kk, vv = c.rows(k, b, h, L)[j].double(), c.rows(v, b, h, L)[j].double()
            qq = q[b, hs].double()
            s = qq @ kk.T * scale
            l = torch.logsumexp(s, -1)
            p = torch.exp(s - l[:, None])
            ref, A = p @ vv, p @ vv.abs()
            E1 = (66 * 2.0**-24 * abs(scale) * (qq.abs() @ kk.abs().T).max() + 2.0**-22 * s.abs().max()).item()
            E = E1 + (n + 32) * 2.0**-23
            tol = 3 * E * A
            if out.dtype == torch.bfloat16:
                tol = tol + 2.0**-8 * (A + ref.abs()) * (1 + 2.0**-6)
            assert ((out[b, hs].double() - ref).abs() <= tol).all(), (b, h)
            assert ((lse[b, hs].double() - l).abs() <= 2 * E + 2.0**-22 * (1 + l.abs())).all(), (b, h)
            if weights is not None:
                want = weights0[b, h, j].double() + p.sum(0)
                wtol = 3 * E * p.sum(0) + 2.0**-23 * want.abs()
                assert ((weights[b, h, j].double() - want).abs() <= wtol).all(), (b, h)
        if weights is not None:    # nothing else moved
            rest = torch.ones(weights.shape[2], dtype=torch.bool, device=DEV)
            rest[j] = False
            assert torch.equal(weights[b][:, rest], weights0[b][:, rest])


def run_decode(c, H, window=0, sinks=0, append=False, out_dtype=torch.bfloat16, with_weights=False,
               scale=0.125, workspace=None, seed=1):
    ops = _ops()
    g = _gen(seed)
    B = len(c.lens_list)
    q = _randn(g, B, H, D)
    kn = vn = None
    k_want, v_want = c.k.clone(), c.v.clone()
    if append:
        kn, vn = _randn(g, B, c.Hkv, D), _randn(g, B, c.Hkv, D)
        for b, L in enumerate(c.lens_list):
            if L:
                p = int(c.table[b, (L - 1) // c.page])
                k_want[p, :, (L - 1) % c.page] = kn[b]
                v_want[p, :, (L - 1) % c.page] = vn[b]
    w = w0 = None
    if with_weights:
        w = torch.rand((B, c.Hkv, c.max_pages * c.page + 3), generator=g, device=DEV)
        w0 = w.clone()
    out, lse = ops.paged_decode_attn(q, c.k, c.v, c.table, c.lens, k_new=kn, v_new=vn, window=window,
                                     sinks=sinks, scale=scale, out_dtype=out_dtype, weights=w,
                                     workspace=workspace)
    torch.cuda.synchronize()
    # the pools hold the appended rows and nothing else changed (NaN included)
    assert torch.equal(c.k.view(torch.int16), k_want.view(torch.int16))
    assert torch.equal(c.v.view(torch.int16), v_want.view(torch.int16))
    check_decode(c, q, out, lse, window, sinks, scale, w, w0)
    assert ops.device_error() == 0
    return out, lse


RAGGED = [1, 0, 15, 16, 17, 63, 64, 65, 130, 300, 1]


@pytest.mark.parametrize("page", [1, 7, 16, 24, 64, 100, 512])
@pytest.mark.parametrize("append", [False, True])
def test_pages_and_lengths(page, append):
    run_decode(Cache(RAGGED, 2, page), 4, append=append)


@pytest.mark.parametrize("H, Hkv", [(1, 1), (12, 12), (3, 1), (8, 1), (9, 1), (16, 2), (32, 2), (40, 1)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_head_groups(H, Hkv, out_dtype):
    run_decode(Cache([200, 1, 77], Hkv, 16), H, append=True, out_dtype=out_dtype)


@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (16, 4), (64, 0), (64, 64), (100, 70),
                                           (128, 500), (1000, 4), (299, 1), (2**31 - 1, 2**31 - 1)])
@pytest.mark.parametrize("page", [16, 20])
def test_window_and_sinks(window, sinks, page):
    c = Cache([0, 1, 64, 65, 300, 1000], 2, page)
    run_decode(c, 6, window=window, sinks=sinks, append=True, with_weights=True)


def test_pages_outside_the_window_are_not_read():
    """Pages between the sinks and the window may have been given back: their
    table entries name no page."""
    c = Cache([1000], 1, 16)
    c.table[0, 1:(1000 - 100) // 16] = -1
    q = _randn(_gen(3), 1, 2, D)
    out, lse = _ops().paged_decode_attn(q, c.k, c.v, c.table, c.lens, window=100, sinks=4)
    check_decode(c, q, out, lse, 100, 4, 0.125)
    assert _ops().device_error() == 0


@pytest.mark.parametrize("lens", [[5000], [40000], [4097, 3, 9000], [1] * 300, [700] * 64])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_splits(lens, out_dtype):
    """One long sequence over all CTAs, many short ones, more than one per CTA."""
    run_decode(Cache(lens, 2, 32), 4, out_dtype=out_dtype, with_weights=True)


def test_one_workspace_for_many_shapes_and_same_bits():
    ops = _ops()
    ws = ops.paged_decode_workspace(64, 32, 2, 8192, weights=True)
    c = Cache([3000, 17, 0, 900], 2, 16)
    first = run_decode(c, 8, workspace=ws, with_weights=True)
    for lens, H in (([70] * 33, 2), ([5000], 32), ([1], 2)):
        run_decode(Cache(lens, 2, 16), H, workspace=ws)
        again = run_decode(c, 8, workspace=ws, with_weights=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_large_scores():
    c = Cache([500, 1200], 2, 16)
    c.k *= 20     # scores of hundreds: the running max moves, most weights vanish
    run_decode(c, 4, with_weights=True)


def test_contiguous_cache_is_a_pool_of_long_pages():
    """[B][H][L_max][64] caches are B pages of L_max rows: same numbers as the
    contiguous decode, up to the two roundings of a bf16 output."""
    ops = _ops()
    g = _gen(9)
    B, H, L_max, L = 3, 4, 300, 257
    k, v, q = _randn(g, B, H, L_max, D), _randn(g, B, H, L_max, D), _randn(g, B, H, D)
    table = torch.arange(B, dtype=torch.int32, device=DEV)[:, None].contiguous()
    lens = torch.full((B,), L, dtype=torch.int32, device=DEV)
    a, la = ops.paged_decode_attn(q, k, v, table, lens, out_dtype=torch.float32)
    b, lb = ops.kv_decode_attn(q, k, v, L, out_dtype=torch.float32)
    assert (a - b).abs().max() < 1e-4 and (la - lb).abs().max() < 1e-4


def test_bad_tables_and_lengths():
    """A page outside the pool reads as zeros and takes no write, a length past
    the table is cut and nothing appended; both set the device error word."""
    ops = _ops()
    for bad in (-1, 10**6, 2**31 - 1):
        c = Cache([100, 50], 2, 16)
        c.table[0, 2] = bad
        q = _randn(_gen(1), 2, 4, D)
        out, lse = ops.paged_decode_attn(q, c.k, c.v, c.table, c.lens)
        assert ops.device_error() == 16 and ops.device_error() == 0
        zero = c.free[0]
        c.k[zero] = 0
        c.v[zero] = 0
        c.table[0, 2] = zero
        check_decode(c, q, out, lse, 0, 0, 0.125)
    for L in (-5, 10**9):
        c = Cache([100, 50], 2, 16, extra_pages=0)
        k0, v0 = c.k.clone(), c.v.clone()
        lens = torch.tensor([L, 50], dtype=torch.int32, device=DEV)
        c.table[0] = torch.tensor(c.table[0].tolist())
        kn = _randn(_gen(2), 2, 2, D)
        q = _randn(_gen(1), 2, 4, D)
        ops.paged_decode_attn(q, c.k, c.v, c.table, lens, k_new=kn, v_new=kn)
        assert ops.device_error() == 16
        same = c.k.view(torch.int16) == k0.view(torch.int16)
        p = int(c.table[1, 49 // 16])
        same[p, :, 49 % 16] = True      # sequence 1's append
        assert same.all()


def test_bad_page_takes_no_append():
    ops = _ops()
    c = Cache([33], 1, 16)
    c.table[0, 2] = 77777
    k0 = c.k.clone()
    kn = _randn(_gen(2), 1, 1, D)
    ops.paged_decode_attn(_randn(_gen(1), 1, 1, D), c.k, c.v, c.table, c.lens, k_new=kn, v_new=kn)
    assert ops.device_error() == 16
    assert torch.equal(c.k.view(torch.int16), k0.view(torch.int16))


def test_shared_prefix_pages():
    c = Cache([96, 96, 96], 2, 16)
    c.table[1, :4] = c.table[0, :4]
    c.table[2, :4] = c.table[0, :4]
    run_decode(c, 4, append=True)


def test_offsets_past_32_bits():
    """Rows beyond 2^31 elements (and 2^32 bytes) of the pool."""
    page, Hkv = 128, 8
    n = 2**31 // (page * Hkv * D) + 3
    k = torch.empty((n, Hkv, page, D), dtype=torch.bfloat16, device=DEV)
    v = torch.empty((n, Hkv, page, D), dtype=torch.bfloat16, device=DEV)
    c = Cache([200], Hkv, page)
    t = c.table.clone()
    t[0, :2] = torch.tensor([n - 1, n - 2], dtype=torch.int32)
    for i in range(2):
        k[n - 1 - i] = c.k[int(c.table[0, i])]
        v[n - 1 - i] = c.v[int(c.table[0, i])]
    c.k, c.v, c.table = k, v, t
    ops = _ops()
    q = _randn(_gen(1), 1, 8, D)
    out, lse = ops.paged_decode_attn(q, k, v, t, c.lens)
    check_decode(c, q, out, lse, 0, 0, 0.125)
    src = _randn(_gen(2), 5, 2 * Hkv * D)
    ops.paged_kv_store(src, 0, Hkv * D, k, v, t, 1, 5, pos0=130)
    assert torch.equal(c.rows(k, 0, 3, 135)[130:], src[:, 3 * D:4 * D])
    assert torch.equal(c.rows(v, 0, 7, 135)[130:], src[:, (Hkv + 7) * D:])
    ot = torch.tensor([[n - 3]], dtype=torch.int32, device=DEV)
    w = torch.rand((1, Hkv, c.max_pages * page), device=DEV)
    kept, _, _ = ops.paged_kv_evict(k, v, t, c.lens, w, ot, 100, sinks=1, recent=1)
    for h in (0, 7):
        assert torch.equal(k[n - 3, h, :100], c.rows(k, 0, h, 200)[kept[0, h].long()])
    assert ops.device_error() == 0


def test_graphs_streams_and_device_lengths():
    """Two captured graphs with a workspace each, replayed at the same time;
    the lengths and tables are read when the graph runs."""
    ops = _ops()
    runs = []
    for seed in (1, 2):
        c = Cache([400, 1000, 3], 2, 16, seed=seed)
        q = _randn(_gen(seed), 3, 8, D)
        out = torch.empty_like(q)
        lse = torch.empty(3, 8, device=DEV)
        ws = ops.paged_decode_workspace(3, 8, 2, c.max_pages * 16)
        ops.paged_decode_attn(q, c.k, c.v, c.table, c.lens, out=out, lse=lse, workspace=ws)
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            ops.paged_decode_attn(q, c.k, c.v, c.table, c.lens, out=out, lse=lse, workspace=ws)
        runs.append((c, q, out, lse, g, s))
    for lens in ([400, 1000, 3], [399, 7, 0], [1, 64, 2]):
        for c, q, out, lse, g, s in runs:
            c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
            c.lens_list = lens
        torch.cuda.synchronize()
        for _ in range(5):
            for c, q, out, lse, g, s in runs:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for c, q, out, lse, g, s in runs:
            check_decode(c, q, out, lse, 0, 0, 0.125)


def test_side_stream_makes_its_own_workspace():
    ops = _ops()
    c = Cache([5000, 300], 2, 16)
    q = _randn(_gen(4), 2, 4, D)
    want = ops.paged_decode_attn(q, c.k, c.v, c.table, c.lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(8):
        got.append(ops.paged_decode_attn(q, c.k, c.v, c.table, c.lens, stream=s))
        torch.full((1 << 20,), 255, dtype=torch.uint8, device=DEV)   # would land in freed memory
    s.synchronize()
    for o, l in got:
        assert torch.equal(o, want[0]) and torch.equal(l, want[1])


def test_programmatic_launch_same_bits():
    ops = _ops()
    c = Cache([600, 31], 2, 16)
    ws = ops.paged_decode_workspace(2, 4, 2, c.max_pages * 16, weights=True)
    a = run_decode(c, 4, append=True, with_weights=True, workspace=ws)
    with ops.pdl(True):
        b = run_decode(c, 4, append=True, with_weights=True, workspace=ws)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_decode_refusals():
    ops = _ops()
    c = Cache([20, 30], 2, 16)
    q = _randn(_gen(1), 2, 4, D)
    call = lambda **kw: ops.paged_decode_attn(**{**dict(q=q, k_pages=c.k, v_pages=c.v,
                                                       block_table=c.table, lens=c.lens), **kw})
    call()
    for kw in (dict(q=q[:, :3].contiguous()), dict(window=-1), dict(sinks=-2),
               dict(workspace=torch.zeros(16, dtype=torch.uint8, device=DEV))):
        with pytest.raises(RuntimeError):
            call(**kw)
    for kw in (dict(lens=c.lens[:1]), dict(v_pages=c.v[:1]), dict(block_table=c.table[:1]),
               dict(k_new=q), dict(weights=torch.zeros(2, 1, 64, device=DEV)),
               dict(out=torch.zeros(2, 4, 64, device=DEV, dtype=torch.float16))):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(lens=c.lens.long()), dict(block_table=c.table.long()), dict(q=q.float()),
               dict(lens=c.lens.cpu()), dict(weights=torch.zeros(2, 2, 64, dtype=torch.float64, device=DEV))):
        with pytest.raises(TypeError):
            call(**kw)


# -------------------------------------------------------------------- store
@pytest.mark.parametrize("page", [1, 7, 16, 64, 300])
@pytest.mark.parametrize("ragged", [False, True])
def test_store(page, ragged):
    ops = _ops()
    B, S, Hkv = 4, 45, 3
    c = Cache([120] * B, Hkv, page)
    src = _randn(c.g, B * S, 2 * Hkv * D + 8)[:, :2 * Hkv * D]      # padded rows
    lens = [45, 0, 1, 17] if ragged else [S] * B
    pos0 = [0, 3, 70, 16] if ragged else [9] * B
    k_want, v_want = c.k.clone(), c.v.clone()
    for b in range(B):
        for s in range(lens[b]):
            p, r = int(c.table[b, (pos0[b] + s) // page]), (pos0[b] + s) % page
            k_want[p, :, r] = src[b * S + s, Hkv * D:].view(Hkv, D)
            v_want[p, :, r] = src[b * S + s, :Hkv * D].view(Hkv, D)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    if ragged:
        ops.paged_kv_store(src, Hkv * D, 0, c.k, c.v, c.table, B, S, pos0=i32(pos0), lens=i32(lens))
    else:
        ops.paged_kv_store(src, Hkv * D, 0, c.k, c.v, c.table, B, S, pos0=9)
    assert torch.equal(c.k.view(torch.int16), k_want.view(torch.int16))
    assert torch.equal(c.v.view(torch.int16), v_want.view(torch.int16))
    assert ops.device_error() == 0


def test_store_bad_positions():
    """Rows whose page or position does not exist go nowhere, the others do."""
    ops = _ops()
    c = Cache([64, 64], 1, 16, extra_pages=0)
    src = _randn(c.g, 2 * 20, 2 * D)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
    for pos0, lens, bad in (([50, 0], [20, 20], None), ([-3, 0], [20, 20], None),
                            ([0, 0], [99, 20], None), ([0, 0], [-1, 20], None),
                            ([0, 0], [20, 20], 12345)):
        c.table[0, 1] = c.free[0] if bad is None else bad
        k_want, v_want = c.k.clone(), c.v.clone()
        for b in range(2):
            for s in range(min(max(lens[b], 0), 20)):
                t = pos0[b] + s
                if 0 <= t < 64 and 0 <= int(c.table[b, t // 16]) < c.k.shape[0]:
                    k_want[int(c.table[b, t // 16]), 0, t % 16] = src[b * 20 + s, :D]
                    v_want[int(c.table[b, t // 16]), 0, t % 16] = src[b * 20 + s, D:]
        ops.paged_kv_store(src, 0, D, c.k, c.v, c.table, 2, 20, pos0=i32(pos0), lens=i32(lens))
        assert ops.device_error() == 16
        assert torch.equal(c.k.view(torch.int16), k_want.view(torch.int16))
        assert torch.equal(c.v.view(torch.int16), v_want.view(torch.int16))


def test_store_refusals():
    ops = _ops()
    c = Cache([64, 64], 1, 16, extra_pages=0)
    src = _randn(c.g, 40, 2 * D)
    with pytest.raises(RuntimeError):
        ops.paged_kv_store(src, 0, D, c.k, c.v, c.table, 2, 20, pos0=45)
    with pytest.raises(ValueError):
        ops.paged_kv_store(src, 0, D, c.k, c.v, c.table, 2, 21)
    with pytest.raises(ValueError):
        ops.paged_kv_store(src, 0, D + 8, c.k, c.v, c.table, 2, 20)
    with pytest.raises(RuntimeError):
        ops.paged_kv_store(src, 4, D, c.k, c.v, c.table, 2, 20)


# ----------------------------------------------------------------- eviction
def choose(w, L, budget, sinks, recent):
    """The positions that stay, by the definition."""
    if L <= budget:
        return np.arange(L)
    mid = w[sinks:L - recent].astype(np.float64)
    key = np.where(np.isnan(mid), -np.inf, mid)
    nan = np.isnan(mid)
    # largest first, NaN behind everything, lowest position among equals
    order = np.lexsort((np.arange(mid.size), -key, nan))
    best = np.sort(order[:budget - sinks - recent]) + sinks
    return np.concatenate([np.arange(sinks), best, np.arange(L - recent, L)])


def run_evict(lens, Hkv, page, budget, sinks, recent, change=None, seed=0, full=False):
    ops = _ops()
    B = len(lens)
    out_pages = -(-budget // page)
    c = Cache(lens, Hkv, page, seed=seed, spare=B * (out_pages + 1), extra_pages=0 if full else 2)
    w = torch.rand((B, Hkv, c.max_pages * page + 5), generator=c.g, device=DEV) ** 4
    w = torch.where(w < 0.05, torch.floor(w * 256) / 256, w)      # ties
    if change is not None:
        change(w)
    ot = torch.full((B, out_pages + 1), -7, dtype=torch.int32)
    for b in range(B):
        ot[b, :out_pages] = torch.tensor(c.free[b * out_pages:(b + 1) * out_pages], dtype=torch.int32)
    ot = ot.to(DEV)
    k_want, v_want = c.k.clone(), c.v.clone()
    w_out = torch.full((B, Hkv, budget + 11), 5.0, device=DEV)
    kept, new_lens, got_w = ops.paged_kv_evict(c.k, c.v, c.table, c.lens, w, ot, budget, sinks=sinks,
                                               recent=recent, weights_out=w_out)
    torch.cuda.synchronize()
    wn, kn = w.cpu().numpy(), kept.cpu().numpy()
    w_want = np.zeros(w_out.shape, np.float32)
    for b, L in enumerate(lens):
        n = min(L, budget)
        assert int(new_lens[b]) == n
        for h in range(Hkv):
            want = choose(wn[b, h], L, budget, sinks, recent)
            np.testing.assert_array_equal(kn[b, h, :n], want)
            assert (kn[b, h, n:] == -1).all()
            w_want[b, h, :n] = wn[b, h, want]
            if n:
                src = torch.from_numpy(want).to(DEV)
                slot = torch.arange(n, device=DEV)
                dst = ot[b].long()[slot // page]
                for pool, to in ((c.k, k_want), (c.v, v_want)):
                    to[dst, h, slot % page] = c.rows(pool, b, h, L)[src]
    np.testing.assert_array_equal(got_w.cpu().numpy(), w_want)
    assert torch.equal(c.k.view(torch.int16), k_want.view(torch.int16))
    assert torch.equal(c.v.view(torch.int16), v_want.view(torch.int16))
    assert ops.device_error() == 0


@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("budget, sinks, recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (32, 4, 8),
                                                   (33, 33, 0), (33, 0, 33), (100, 10, 90), (64, 0, 0)])
def test_evict(page, budget, sinks, recent):
    run_evict([200, 0, 33, 1, 101, 64], 2, page, budget, sinks, recent)


@pytest.mark.parametrize("L, budget", [(1024, 1023), (1025, 512), (5000, 3333), (20000, 700), (40000, 16384)])
def test_evict_long(L, budget):
    run_evict([L, L // 2], 2, 32, budget, 4, budget // 8, seed=L)


@pytest.mark.parametrize("lens, Hkv, budget", [
    ([8192], 2, 512), ([8000], 2, 2000), ([1000], 2, 600), ([1500, 1100], 64, 1200),
    ([1200, 0, 700], 64, 600), ([300, 257, 100, 99, 1], 70, 100),
    ([1100, 40, 1030, 500, 41, 39, 64, 1], 64, 40), ([600, 900, 1, 0], 45, 513)])
def test_evict_few_and_many_heads(lens, Hkv, budget):
    """Heads that leave SMs idle, fill them once or several times over, with one
    block a head and with two launches."""
    run_evict(lens, Hkv, 16, budget, 4, budget // 8, seed=budget)


@pytest.mark.parametrize("cap, budget", [(8192, 700), (16384, 3000), (24576, 500), (30000, 9000),
                                         (55296, 4000), (55328, 4000)])
def test_evict_where_the_weights_are_kept(cap, budget):
    """Capacities up to the last position of each place for the weights, the
    longest sequence filling it."""
    run_evict([cap, cap - 33, budget + 1, 5], 2, 32, budget, 4, budget // 8, seed=cap, full=True)


def test_evict_ties_and_unusual_weights():
    def all_equal(w):
        w.fill_(0.25)
    run_evict([500, 300], 2, 16, 100, 3, 10, all_equal)

    def zeros_of_both_signs(w):
        w.fill_(0.0)
        w[..., ::2] = -0.0
    run_evict([500, 300], 2, 16, 100, 3, 10, zeros_of_both_signs)

    def unusual(w):
        w[..., 10:40] = math.nan
        w[..., 50:60] = math.inf
        w[..., 70:90] = -math.inf
        w[..., 100:150] = -w[..., 100:150]
        w[..., 200:220] = 1e-42            # subnormal
    run_evict([500, 300], 2, 16, 100, 3, 10, unusual)
    run_evict([500, 300], 2, 16, 290, 0, 0, unusual)

    def nearly_all_nan(w):
        w.fill_(math.nan)
        w[..., 77] = -math.inf
    run_evict([500, 300], 2, 16, 20, 0, 0, nearly_all_nan)


def test_evict_bad_pages():
    """A source page outside the pool moves zeros, an output page outside it
    takes nothing."""
    ops = _ops()
    c = Cache([64], 1, 16, spare=4)
    w = torch.rand((1, 1, c.max_pages * 16), device=DEV)
    ot = torch.tensor([[c.free[0], 10**7]], dtype=torch.int32, device=DEV)
    c.table[0, 0] = -3
    before = c.k.clone()
    kept, new_lens, _ = ops.paged_kv_evict(c.k, c.v, c.table, c.lens, w, ot, 20, sinks=8)
    assert ops.device_error() == 16
    assert int(new_lens[0]) == 20
    assert (c.k[c.free[0], 0, :8] == 0).all()
    rest = [p for p in range(c.k.shape[0]) if p != c.free[0]]
    assert torch.equal(c.k[rest].view(torch.int16), before[rest].view(torch.int16))


def test_evict_refusals():
    ops = _ops()
    c = Cache([64], 1, 16, spare=4)
    w = torch.rand((1, 1, c.max_pages * 16), device=DEV)
    ot = torch.tensor([c.free[:2]], dtype=torch.int32, device=DEV)
    call = lambda budget=20, w=w, ot=ot, **kw: ops.paged_kv_evict(c.k, c.v, c.table, c.lens, w, ot, budget, **kw)
    call()
    for kw in (dict(budget=33), dict(budget=0), dict(sinks=12, recent=9), dict(sinks=-1),
               dict(w=w[..., :40].contiguous()), dict(weights_out=w),
               dict(weights_out=torch.zeros(1, 1, 19, device=DEV))):
        with pytest.raises(RuntimeError):
            call(**kw)
    for kw in (dict(kept=torch.zeros(3, dtype=torch.int32, device=DEV)),
               dict(new_lens=torch.zeros(3, dtype=torch.int32, device=DEV)), dict(w=w.view(1, 2, -1))):
        with pytest.raises(ValueError):
            call(**kw)


def test_empty_tables_and_batches():
    """No pages at all: every sequence is empty; no sequences: nothing to do."""
    ops = _ops()
    kp = torch.zeros((1, 2, 16, D), dtype=torch.bfloat16, device=DEV)
    q = _randn(_gen(1), 3, 4, D)
    table = torch.empty((3, 0), dtype=torch.int32, device=DEV)
    lens = torch.zeros(3, dtype=torch.int32, device=DEV)
    w = torch.ones((3, 2, 5), device=DEV)
    out, lse = ops.paged_decode_attn(q, kp, kp, table, lens, weights=w)
    assert (out == 0).all() and (lse == -math.inf).all() and (w == 1).all()
    out, lse = ops.paged_decode_attn(q[:0], kp, kp, table[:0], lens[:0])
    assert out.shape == (0, 4, D)
    ops.paged_kv_store(_randn(_gen(1), 0, 4 * D), 0, 2 * D, kp, kp, table[:0], 0, 7)
    assert ops.device_error() == 0


def test_window_past_31_bits_is_no_window():
    c = Cache([300, 20], 2, 16)
    run_decode(c, 4, window=2**40, sinks=2**40)


@pytest.mark.parametrize("page", [4, 8, 12, 20, 32, 48, 256])
def test_more_page_sizes(page):
    run_decode(Cache([1, 700, 64, 333], 2, page), 24, append=True, window=200, sinks=9, with_weights=True)


def test_tables_wider_than_used():
    """Tables and weights in longer rows, as views."""
    c = Cache([100, 40, 77], 2, 16)
    wide = torch.full((3, 20), 10**6, dtype=torch.int32, device=DEV)
    wide[:, 2:2 + c.max_pages] = c.table
    c.table = wide[:, 2:2 + c.max_pages]
    run_decode(c, 4, append=True, with_weights=True)


def test_store_then_contiguous_decode_with_programmatic_launch():
    """The contiguous decode attention reads cached rows before it waits for the
    kernel before it; a store right in front of it has to have ended by then."""
    ops = _ops()
    g = _gen(5)
    B, H, L_max, S = 8, 12, 2048, 2000
    kc = torch.zeros((B, H, L_max, D), dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    table = torch.arange(B, dtype=torch.int32, device=DEV)[:, None].contiguous()
    src = _randn(g, B * S, 2 * H * D)
    q = _randn(g, B, H, D)
    want = None
    for _ in range(5):
        kc.zero_()
        vc.zero_()
        with ops.pdl(True):
            ops.paged_kv_store(src, 0, H * D, kc, vc, table, B, S)
            out, lse = ops.kv_decode_attn(q, kc, vc, S)
        if want is None:
            torch.cuda.synchronize()
            want = ops.kv_decode_attn(q, kc, vc, S)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def spoil(what, c, q):
    """Numbers that are not finite in places that are seen."""
    b = len(c.lens_list) - 1
    L = c.lens_list[b]

    def keys(first, n, value):
        for j in range(first, first + n):
            c.k[int(c.table[b, j // c.page]), 0, j % c.page, 0] = value
    if what == "one query":
        q[b, 0, 5] = math.nan
    elif what == "one key":
        keys(L - 2, 1, math.nan)
    elif what == "first key":
        keys(0, 1, math.nan)
    elif what == "sixteen keys":       # all that one warp sees of a tile
        keys(16, 16, math.nan)
    elif what == "every key":
        keys(0, L, math.nan)
    elif what == "a tile and more":
        keys(64, 80, math.nan)
    elif what == "infinite key":       # +inf for the heads above zero there, -inf (weight 0) for the others
        keys(20, 1, math.inf)
    elif what == "infinite query":
        q[b, 1, 0] = math.inf
    else:                              # every score of every head -inf
        q[b, :, 0] = 1.0
        keys(0, L, -math.inf)


@pytest.mark.parametrize("what", ["one query", "one key", "first key", "sixteen keys", "every key", "a tile and more",
                                  "infinite key", "infinite query", "nothing left"])
@pytest.mark.parametrize("lens, H, page", [([0, 200], 2, 16), ([300, 5000], 4, 16), ([40, 9000], 18, 20)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_scores_that_are_not_finite_are_not_lost(what, lens, H, page, out_dtype):
    """By the definition a NaN among the scores, or +inf, or nothing above -inf,
    leaves no number in the row (lse: NaN, and -inf for the last); a key of -inf
    among others weighs nothing.  Only a sequence without keys is zeros."""
    ops = _ops()
    Hkv = 2
    G = H // Hkv
    c = Cache(lens, Hkv, page, seed=5)
    q = _randn(_gen(7), len(lens), H, D)
    spoil(what, c, q)
    w = torch.rand((len(lens), Hkv, c.max_pages * page), generator=c.g, device=DEV)
    w0 = w.clone()
    out, lse = ops.paged_decode_attn(q, c.k, c.v, c.table, c.lens, out_dtype=out_dtype, weights=w)
    assert ops.device_error() == 0
    bad_heads = 0
    for b, L in enumerate(lens):
        if L == 0:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all() and torch.equal(w[b], w0[b])
            continue
        for h in range(Hkv):
            k, v = c.rows(c.k, b, h, L).double(), c.rows(c.v, b, h, L).double()
            group_bad = False
            want_w, tol_w = w0[b, h, :L].double(), torch.zeros(L, dtype=torch.float64, device=DEV)
            for i in range(h * G, (h + 1) * G):
                s = (q[b, i].double() * k).sum(-1) * 0.125
                if s.isnan().any() or (s == math.inf).any():
                    assert out[b, i].isnan().all() and lse[b, i].isnan(), (b, i)
                    group_bad = True
                    continue
                seen = s > -math.inf
                if not seen.any():
                    assert out[b, i].isnan().all() and lse[b, i] == -math.inf, (b, i)
                    group_bad = True
                    continue
                l = torch.logsumexp(s, -1)
                p = torch.exp(s - l)
                ref, A = p @ v, p @ v.abs()
                E1 = (66 * 2.0**-24 * 0.125 * (q[b, i].double().abs() * k[seen].abs()).sum(-1).max()
                      + 2.0**-22 * s[seen].abs().max()).item()
                E = E1 + (L + 32) * 2.0**-23
                tol = 3 * E * A
                if out_dtype == torch.bfloat16:
                    tol = tol + 2.0**-8 * (A + ref.abs()) * (1 + 2.0**-6)
                assert ((out[b, i].double() - ref).abs() <= tol).all(), (b, i)
                assert (lse[b, i].double() - l).abs() <= 2 * E + 2.0**-22 * (1 + l.abs()), (b, i)
                want_w, tol_w = want_w + p, tol_w + 3 * E * p
            bad_heads += group_bad
            if group_bad:
                assert w[b, h, :L].isnan().all(), (b, h)
            else:
                assert ((w[b, h, :L].double() - want_w).abs() <= tol_w + 2.0**-23 * want_w.abs()).all(), (b, h)
            assert torch.equal(w[b, h, L:], w0[b, h, L:])
    assert bad_heads >= 1 or what == "infinite key"      # there it is for the signs of q


@pytest.mark.parametrize("lens, Hkv, budget", [([500, 300, 40], 2, 100), ([700] * 5, 70, 300), ([900, 20, 1100], 300, 200),
                                               ([5000, 9000], 3, 2500), ([-4, 10**8, 77], 90, 30)])
def test_evict_writes_the_lengths_in_place(lens, Hkv, budget):
    """new_lens = lens: every head of a sequence goes by the old length."""
    ops = _ops()
    page, B = 16, len(lens)
    fit = [1200 if L > 10**6 else max(L, 0) for L in lens]
    out_pages = -(-budget // page)
    c = Cache(fit, Hkv, page, seed=budget, spare=B * out_pages, extra_pages=0)
    c.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
    w = torch.rand((B, Hkv, c.max_pages * page), generator=c.g, device=DEV)
    ot = torch.tensor(c.free[:B * out_pages], dtype=torch.int32, device=DEV).view(B, out_pages)
    k0, v0 = c.k.clone(), c.v.clone()
    want = ops.paged_kv_evict(c.k, c.v, c.table, c.lens, w, ot, budget, sinks=2, recent=9)
    ops.device_error()
    k1, v1 = c.k.clone(), c.v.clone()
    c.k.copy_(k0)
    c.v.copy_(v0)
    got = ops.paged_kv_evict(c.k, c.v, c.table, c.lens, w, ot, budget, sinks=2, recent=9, new_lens=c.lens)
    assert got[1] is c.lens and torch.equal(c.lens, want[1])
    assert c.lens.tolist() == [min(L, budget) for L in fit]
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    assert torch.equal(c.k.view(torch.int16), k1.view(torch.int16))
    assert torch.equal(c.v.view(torch.int16), v1.view(torch.int16))
    assert ops.device_error() == (16 if lens != fit else 0)


@pytest.mark.parametrize("with_weights", [False, True])
def test_append_then_contiguous_decode_with_programmatic_launch(with_weights):
    """The row that a paged decode appends is one of those that a contiguous decode
    right behind it reads before it waits."""
    ops = _ops()
    g = _gen(6)
    B, H, L_max, L = 8, 12, 2048, 2000
    kc, vc = _randn(g, B, H, L_max, D), _randn(g, B, H, L_max, D)
    table = torch.arange(B, dtype=torch.int32, device=DEV)[:, None].contiguous()
    lens = torch.full((B,), L, dtype=torch.int32, device=DEV)
    q, kn, vn = _randn(g, B, H, D), 4 * _randn(g, B, H, D), 4 * _randn(g, B, H, D)
    q2 = kn.clone()          # attends mostly to the appended row
    ws = ops.paged_decode_workspace(B, H, H, L_max, weights=with_weights)
    w = torch.zeros((B, H, L_max), device=DEV) if with_weights else None
    want = None
    for _ in range(5):
        kc[:, :, L - 1] = 0
        vc[:, :, L - 1] = 0
        with ops.pdl(True):
            ops.paged_decode_attn(q, kc, vc, table, lens, k_new=kn, v_new=vn, weights=w, workspace=ws)
            out, lse = ops.kv_decode_attn(q2, kc, vc, L + 1)
        if want is None:
            torch.cuda.synchronize()
            assert torch.equal(kc[:, :, L - 1], kn) and torch.equal(vc[:, :, L - 1], vn)
            want = ops.kv_decode_attn(q2, kc, vc, L + 1)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    assert ops.device_error() == 0


@pytest.mark.parametrize("lens, H, Hkv, page", [([300, 64, 17], 12, 12, 16), ([900, 5000], 8, 2, 64), ([700], 18, 2, 20)])
def test_bf16_output_is_rounded_once(lens, H, Hkv, page):
    """A bf16 output keeps its weights to 2^-16 (two bf16 terms, the second of what
    the first leaves: 2^-8 of 2^-8), as the contiguous decode keeps them in fp32: off by
    its own rounding and the module's fp32 bounds, however small it is beside sum p |v|."""
    c = Cache(lens, Hkv, page, seed=3)
    q = _randn(_gen(2), len(lens), H, D)
    out, _ = _ops().paged_decode_attn(q, c.k, c.v, c.table, c.lens)
    G = H // Hkv
    for b, L in enumerate(lens):
        for h in range(Hkv):
            k, v = c.rows(c.k, b, h, L).double(), c.rows(c.v, b, h, L).double()
            qq = q[b, h * G:(h + 1) * G].double()
            s = qq @ k.T * 0.125
            p = torch.softmax(s, -1)
            ref, A = p @ v, p @ v.abs()
            E1 = (66 * 2.0**-24 * 0.125 * (qq.abs() @ k.abs().T).max() + 2.0**-22 * s.abs().max()).item()
            E = E1 + (L + 32) * 2.0**-23
            tol = (3 * E + 2.0**-16) * A + 2.0**-8 * ref.abs() * (1 + 2.0**-6)
            assert ((out[b, h * G:(h + 1) * G].double() - ref).abs() <= tol).all(), (b, h)
