"""The serving operators as a serving loop uses them, one after the other, and
through the operator graph, against a 64-bit mirror of the same loop.

Attention tolerance: with A = sum_j p_j |v_j|, a bf16 weight and a bf16 output
are off by at most 2^-8 each (the prefill may round a weight twice), and
scores of a few units in fp32 change p by less than 1e-4.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

D, DEV = 64, "cuda"


def _ops():
    from neurodsl_b200 import ops
    return ops


def attend(q, k, v, seen=None):
    """Rows q over k, v in 64 bits: O, A = sum p |v|, p."""
    s = q.double() @ k.double().transpose(-1, -2) * 0.125
    if seen is not None:
        s = s.masked_fill(~seen, -math.inf)
    p = torch.softmax(s, -1)
    return p @ v.double(), p @ v.double().abs(), p


def close(got, ref, A):
    tol = 2.0**-8 * (2 * A + ref.abs()) * (1 + 2.0**-6) + 1e-4 * A
    assert ((got.double() - ref).abs() <= tol).all()


def test_prompt_decode_evict_decode_choose():
    ops = _ops()
    g = torch.Generator(device=DEV)
    g.manual_seed(11)
    rn = lambda *s: torch.randn(s, generator=g, device=DEV).to(torch.bfloat16)
    B, H, Hkv, S, page, V = 3, 4, 2, 100, 16, 1003
    G, window, sinks, budget, keep_sinks, recent = H // Hkv, 48, 4, 40, 2, 16
    prompt = [37, 100, 64]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)

    # ---- the padded prompts: windowed attention in place on the projection,
    # keys and values into the pages
    qkv = rn(B, S, (H + 2 * Hkv) * D)
    heads = lambda x, n: x.unflatten(-1, (n, D)).transpose(1, 2)
    Q, K, Vv = (heads(qkv[..., :H * D], H), heads(qkv[..., H * D:(H + Hkv) * D], Hkv),
                heads(qkv[..., (H + Hkv) * D:], Hkv))
    O, _, _ = ops.window_attn_fwd(Q, K, Vv, window, sinks=sinks)
    max_pages = 10
    n_pages = B * max_pages + B * 6 + 1
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = order[:B * max_pages].view(B, max_pages).contiguous()
    kp = torch.full((n_pages, Hkv, page, D), math.nan, device=DEV, dtype=torch.bfloat16)
    vp = torch.full_like(kp, math.inf)
    lens = i32(prompt)
    ops.paged_kv_store(qkv.view(B * S, -1), H * D, (H + Hkv) * D, kp, vp, table, B, S, lens=lens)
    mirror = [[(K[b, h, :L].clone(), Vv[b, h, :L].clone()) for h in range(Hkv)] for b, L in enumerate(prompt)]
    for b, L in enumerate(prompt):
        i, j = torch.arange(L, device=DEV)[:, None], torch.arange(L, device=DEV)[None, :]
        seen = (j <= i) & ((j > i - window) | (j < sinks))
        for h in range(H):
            ref, A, _ = attend(Q[b, h, :L], *mirror[b][h // G], seen)
            close(O[b, h, :L], ref, A)

    # ---- decode steps, greedy tokens under penalties
    ws = ops.paged_decode_workspace(B, H, Hkv, max_pages * page, weights=True)
    weights = torch.zeros((B, Hkv, max_pages * page), device=DEV)
    w_mirror = [[torch.zeros(L, dtype=torch.float64, device=DEV) for _ in range(Hkv)] for L in prompt]
    head = rn(V, H * D)
    history = torch.full((B, 64), -1, dtype=torch.int32, device=DEV)
    one = torch.ones(B, device=DEV)
    n_tok = 0

    def step(table, weights, w_mirror):
        nonlocal n_tok
        q, kn, vn = rn(B, H, D), rn(B, Hkv, D), rn(B, Hkv, D)
        lens.add_(1)
        out, _ = ops.paged_decode_attn(q, kp, vp, table, lens, k_new=kn, v_new=vn, weights=weights,
                                       workspace=ws)
        for b in range(B):
            for h in range(Hkv):
                k, v = mirror[b][h]
                k, v = torch.cat([k, kn[b, h][None]]), torch.cat([v, vn[b, h][None]])
                mirror[b][h] = (k, v)
                ref, A, p = attend(q[b, h * G:(h + 1) * G], k, v)
                close(out[b, h * G:(h + 1) * G], ref, A)
                w_mirror[b][h] = torch.cat([w_mirror[b][h], torch.zeros(1, dtype=torch.float64, device=DEV)])
                w_mirror[b][h] += p.sum(0)
                got = weights[b, h, :k.shape[0]].double()
                assert ((got - w_mirror[b][h]).abs() <= 1e-4 * (1 + w_mirror[b][h])).all()
        logits = ops.linear(out.reshape(B, H * D), head, out_dtype=torch.float32)
        x, idx = ops.logits_penalty(logits, history=history, repetition=1.3 * one, presence=0.5 * one)
        want = logits.double()
        for b in range(B):
            tok = history[b][history[b] >= 0].long().unique()
            y = want[b, tok]
            want[b, tok] = torch.where(y > 0, y / 1.3, y * 1.3) - 0.5
        # two steps of fp32 rounding, and 1.3 itself in fp32
        assert ((x.double() - want).abs() <= 2.0**-22 * (logits.abs() + 1)).all()
        assert torch.equal(idx.long(), x.argmax(1))
        history[:, n_tok] = idx
        n_tok += 1

    for _ in range(20):
        step(table, weights, w_mirror)

    # ---- the caches are cut, onto fresh pages, and decoding goes on there
    out_table = torch.full((B, 6), -1, dtype=torch.int32, device=DEV)
    out_table[:, :3] = order[B * max_pages:B * max_pages + 3 * B].view(B, 3)
    kept, new_lens, w2 = ops.paged_kv_evict(kp, vp, table, lens, weights, out_table, budget,
                                            sinks=keep_sinks, recent=recent)
    for b in range(B):
        L = int(lens[b])
        n = min(L, budget)
        assert int(new_lens[b]) == n
        for h in range(Hkv):
            w = weights[b, h, :L].cpu().numpy()
            mid = np.argsort(-w[keep_sinks:L - recent], kind="stable")[:budget - keep_sinks - recent]
            rows = np.concatenate([np.arange(keep_sinks), np.sort(mid) + keep_sinks, np.arange(L - recent, L)])
            rows = rows if L > budget else np.arange(L)
            np.testing.assert_array_equal(kept[b, h, :n].cpu().numpy(), rows)
            r = torch.from_numpy(rows).to(DEV)
            mirror[b][h] = (mirror[b][h][0][r], mirror[b][h][1][r])
            w_mirror[b][h] = w2[b, h, :n].double()
    lens.copy_(new_lens)
    out_table[:, 3:] = order[B * max_pages + 3 * B:B * max_pages + 6 * B].view(B, 3)
    w2 = w2[:, :, :6 * page].contiguous()
    for _ in range(12):
        step(out_table, w2, w_mirror)
    assert ops.device_error() == 0


def test_serving_step_as_a_graph():
    """Decode, logits and the choice of the token captured once and replayed
    while the lengths grow on the device."""
    ops = _ops()
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    rn = lambda *s: torch.randn(s, generator=g, device=DEV).to(torch.bfloat16)
    B, H, page, V, max_pages = 2, 4, 16, 777, 4
    def state():
        gg = torch.Generator(device=DEV)
        gg.manual_seed(8)
        kp = torch.randn((B * max_pages, H, page, D), generator=gg, device=DEV).to(torch.bfloat16)
        return dict(kp=kp, vp=kp.flip(0).clone(), lens=torch.tensor([5, 20], dtype=torch.int32, device=DEV),
                    hist=torch.full((B, 40), -1, dtype=torch.int32, device=DEV),
                    at=torch.zeros(1, dtype=torch.int64, device=DEV))
    table = torch.arange(B * max_pages, dtype=torch.int32, device=DEV).view(B, max_pages)
    embed, head = rn(V, 3 * H * D), rn(V, H * D)
    tok0 = torch.tensor([1, 2], dtype=torch.int32, device=DEV)
    rep = torch.full((B,), 1.2, device=DEV)
    ws = ops.paged_decode_workspace(B, H, H, max_pages * page)

    def step(s, tok, out):
        qkv = embed[tok.long()].view(B, 3, H, D)
        s["lens"].add_(1)
        q, k, v = (qkv[:, i].contiguous() for i in range(3))
        o, _ = ops.paged_decode_attn(q, s["kp"], s["vp"], table, s["lens"], k_new=k, v_new=v, window=16,
                                     sinks=2, workspace=ws)
        logits = ops.linear(o.view(B, H * D), head, out_dtype=torch.float32)
        x, idx = ops.logits_penalty(logits, history=s["hist"], repetition=rep)
        s["hist"].index_copy_(1, s["at"], idx[:, None])
        s["at"].add_(1)
        tok.copy_(idx)
        out.copy_(x)

    a, tok, out = state(), tok0.clone(), torch.empty(B, V, device=DEV)
    eager = []
    for _ in range(25):
        step(a, tok, out)
        eager.append((tok.clone(), out.clone()))
    b, tok, out = state(), tok0.clone(), torch.empty(B, V, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):      # one uncaptured step on a copy
        step(state(), tok0.clone(), out.clone())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b, tok, out)
    for t, x in eager:
        graph.replay()
        assert torch.equal(tok, t) and torch.equal(out, x)
    assert torch.equal(a["kp"], b["kp"]) and ops.device_error() == 0


def test_operator_graph():
    """:window_attention, :paged_decode_attn and :logits_penalty as rules."""
    from neurodsl_b200 import graph as g_
    ops = _ops()
    rng = np.random.default_rng(0)
    bf = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda().to(torch.bfloat16)
    S, Sk, H, Hkv = 30, 75, 4, 2
    q, k, v = bf(S, H * D), bf(Sk, Hkv * D), bf(Sk, Hkv * D)
    kp, vp = bf(6, Hkv, 16, D), bf(6, Hkv, 16, D)
    table = torch.tensor([[4, 1, 0], [2, 5, 3]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([37, 16], dtype=torch.int32, device=DEV)
    qd, kn, vn = bf(2, H * D), bf(2, Hkv * D), bf(2, Hkv * D)
    kp0, vp0 = kp.clone(), vp.clone()
    logits = torch.from_numpy(rng.standard_normal((2, 500)).astype(np.float32)).cuda()
    hist = torch.from_numpy(rng.integers(0, 500, (2, 9)).astype(np.int32)).cuda()
    g = g_.NeuroGraph()
    for n, x in (("q", q), ("k", k), ("v", v), ("kp", kp), ("vp", vp), ("table", table), ("lens", lens),
                 ("qd", qd), ("kn", kn), ("vn", vn), ("logits", logits), ("hist", hist)):
        g_.set_(g, n, x)
    g_.addrule(g, g_.GraphRule("a", ["q", "k", "v"], "window_attention",
                               {"n_heads": H, "n_kv_heads": Hkv, "window": 20, "sinks": 3}))
    g_.addrule(g, g_.GraphRule("d", ["qd", "kp", "vp", "table", "lens", "kn", "vn"], "paged_decode_attn",
                               {"n_heads": H, "window": 12, "sinks": 1}))
    g_.addrule(g, g_.GraphRule("t", ["logits", "hist"], "logits_penalty",
                               {"repetition": 1.5, "frequency": 0.25}))
    ctx = g_.CtxStore()
    a, d, t = (g_.demand(g, n, ctx_store=ctx) for n in ("a", "d", "t"))
    heads = lambda x, n: x.view(x.shape[0], n, D).transpose(0, 1)[None]
    want = ops.window_attn_fwd(heads(q, H), heads(k, Hkv), heads(v, Hkv), 20, sinks=3, out_dtype=torch.float32)
    assert torch.equal(a, want[0][0].transpose(0, 1).reshape(S, H * D))
    assert torch.equal(g.nodes["default"]["a"].aux_data["flash_l"], want[1][0])
    want = ops.paged_decode_attn(qd.view(2, H, D), kp0, vp0, table, lens, k_new=kn.view(2, Hkv, D),
                                 v_new=vn.view(2, Hkv, D), window=12, sinks=1, out_dtype=torch.float32)
    assert torch.equal(d, want[0].view(2, H * D))
    page_nodes = g.nodes["default"]
    assert torch.equal(page_nodes["kp"].value, kp0) and torch.equal(page_nodes["vp"].value, vp0)
    want = ops.logits_penalty(logits, history=hist, repetition=torch.full((2,), 1.5, device=DEV),
                              frequency=torch.full((2,), 0.25, device=DEV))
    assert torch.equal(t, want[0]) and torch.equal(page_nodes["t"].aux_data["token"], want[1])
    assert set(ctx["a"]) >= {"Q", "K", "V", "out", "l", "m", "window"} and "token" in ctx["t"]
    with pytest.raises(g_.NeuroDSLError):
        g_.addrule(g, g_.GraphRule("bad", ["q", "k", "v"], "window_attention", {"n_heads": 3, "window": 4}))
        g_.demand(g, "bad")


def test_operator_graph_captured_before_its_first_run():
    """A node first demanded inside a capture keeps no workspace from there: its
    zeros are only written when the captured graph runs."""
    from neurodsl_b200 import graph as g_
    ops = _ops()
    gen = torch.Generator(device=DEV)
    gen.manual_seed(4)
    rn = lambda *s: torch.randn(s, generator=gen, device=DEV).to(torch.bfloat16)
    B, H, page, max_pages = 2, 2, 16, 400
    q, kp, vp = rn(B, H * D), rn(B * max_pages, H, page, D), rn(B * max_pages, H, page, D)
    table = torch.arange(B * max_pages, dtype=torch.int32, device=DEV).view(B, max_pages)
    lens = torch.tensor([6400, 5000], dtype=torch.int32, device=DEV)
    want, _ = ops.paged_decode_attn(q.view(B, H, D), kp, vp, table, lens, out_dtype=torch.float32)
    g = g_.NeuroGraph()
    for n, x in (("q", q), ("kp", kp), ("vp", vp), ("table", table), ("lens", lens)):
        g_.set_(g, n, x)
    g_.addrule(g, g_.GraphRule("d", ["q", "kp", "vp", "table", "lens"], "paged_decode_attn", {"n_heads": H}))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = g_.demand(g, "d")
    node = g.nodes["default"]["d"]
    for x in node.aux_data.values():      # what the capture alone has "written" may hold anything
        if isinstance(x, torch.Tensor):
            x.fill_(1)
    g_.set_(g, "q", q)
    assert torch.equal(g_.demand(g, "d").view(B, H, D), want)
    for _ in range(3):
        graph.replay()
        assert torch.equal(captured.view(B, H, D), want)
    assert ops.device_error() == 0
