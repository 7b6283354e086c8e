"""Cases that measure the serving operators: sliding-window prefill attention,
decode attention over a paged cache, the paged cache's store and eviction, and
the penalties on logits.

Each operator has a plain form (elementary torch operations in 32 bits, one
rounding at the end) and the library's form; `own` chooses which one run()
computes.  exact() gives the same results from the definitions in 64 bits.
"""
import math

import torch

own = False

D = 64   # head dimension of every attention entry point


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one chat turn: Q, K and V read in place from the fused projection of a 12-head layer
        {"name": "window short prompt", "op": "window", "B": 1, "H": 12, "Hkv": 12, "Sq": 213,
         "Sk": 213, "window": 64, "sinks": 4, "layout": "token"},
        # the next chunk of a long prompt against the head-major cache that the earlier chunks filled
        {"name": "window prompt chunk", "op": "window", "B": 2, "H": 16, "Hkv": 4, "Sq": 509,
         "Sk": 4099, "window": 1024, "sinks": 4, "layout": "cache"},
        # whole long prompts, contiguous head-major
        {"name": "window long prompt", "op": "window", "B": 2, "H": 16, "Hkv": 16, "Sq": 8192,
         "Sk": 8192, "window": 1024, "sinks": 4, "layout": "head"},
        # one user, one token: latency; window and sinks as in the prefill
        {"name": "decode one user", "op": "decode", "B": 1, "H": 12, "Hkv": 12, "page": 16,
         "max_len": 700, "ragged": False, "append": True, "window": 256, "sinks": 4,
         "weights": False, "out": "bf16"},
        # a serving batch whose sequences have every length
        {"name": "decode ragged batch", "op": "decode", "B": 64, "H": 12, "Hkv": 12, "page": 64,
         "max_len": 2048, "ragged": True, "append": True, "window": 0, "sinks": 0,
         "weights": False, "out": "bf16"},
        # few sequences with long caches, shared K/V heads, weights accumulated for eviction
        {"name": "decode long weights", "op": "decode", "B": 8, "H": 16, "Hkv": 4, "page": 128,
         "max_len": 32768, "ragged": False, "append": False, "window": 0, "sinks": 0,
         "weights": True, "out": "f32"},
        # a short prompt's keys and values into the pages
        {"name": "store short prompt", "op": "store", "B": 1, "Hkv": 12, "S": 37, "page": 16,
         "ragged": False},
        # a padded batch of long prompts
        {"name": "store batch", "op": "store", "B": 32, "Hkv": 12, "S": 2048, "page": 64,
         "ragged": True},
        # one user's cache at its limit
        {"name": "evict one user", "op": "evict", "B": 1, "Hkv": 12, "page": 16, "max_len": 500,
         "ragged": False, "budget": 256, "sinks": 4, "recent": 32},
        # a batch of long caches cut to a quarter
        {"name": "evict batch", "op": "evict", "B": 16, "Hkv": 16, "page": 64, "max_len": 8192,
         "ragged": True, "budget": 2048, "sinks": 4, "recent": 256},
        # one user's next token under a grammar
        {"name": "logits one user", "op": "logits", "rows": 1, "V": 50257, "hist": 300,
         "n_bias": 8, "mask": True, "dtype": "f32", "out": "f32"},
        # a large serving batch
        {"name": "logits batch", "op": "logits", "rows": 512, "V": 50257, "hist": 1024,
         "n_bias": 16, "mask": True, "dtype": "bf16", "out": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "decode", "decode", "store", "evict", "logits"])
    Hkv = rng.choice([1, 2, 4, 8, 12, 16])
    G = rng.choice([1, 1, 2, 3, 4, 8])
    page = rng.choice([1, 16, 16, 24, 64, 100, 128])
    if op == "window":
        H = Hkv * G
        B = _log(rng, 1, 8)
        Sk = _log(rng, 1, 8192)
        while B * H * Sk > 32 * 8192:
            B, Sk = max(1, B // 2), (Sk if B > 1 else Sk // 2)
        Sq = rng.choice([Sk, Sk, max(1, Sk // 7), 1])
        return {"op": op, "B": B, "H": H, "Hkv": Hkv, "Sq": Sq, "Sk": Sk,
                "window": _log(rng, 1, 1024), "sinks": rng.choice([0, 1, 4, 17, 130]),
                "layout": rng.choice(["head", "token", "cache"])}
    if op == "decode":
        B = _log(rng, 1, 128)
        max_len = _log(rng, 1, 32768)
        while B * Hkv * max_len > 8 * 4 * 32768 or B * Hkv * G * max_len > 8 * 16 * 32768:
            B, max_len = max(1, B // 2), (max_len if B > 1 else max_len // 2)
        window = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
        return {"op": op, "B": B, "H": Hkv * G, "Hkv": Hkv, "page": page, "max_len": max_len,
                "ragged": rng.random() < 0.7, "append": rng.random() < 0.5, "window": window,
                "sinks": rng.choice([0, 4, 40]) if window else 0, "weights": rng.random() < 0.3,
                "out": rng.choice(["bf16", "bf16", "f32"])}
    if op == "store":
        B, S = _log(rng, 1, 32), _log(rng, 1, 2048)
        while B * S * Hkv > 32 * 1024 * 12:
            B //= 2
        return {"op": op, "B": B, "Hkv": Hkv, "S": S, "page": page, "ragged": rng.random() < 0.7}
    if op == "evict":
        B, max_len = _log(rng, 1, 12), _log(rng, 16, 8192)
        budget = max(1, int(max_len * rng.uniform(0.1, 0.9)))
        budget = min(budget, 2048)
        sinks = min(rng.choice([0, 1, 4]), budget)
        return {"op": op, "B": B, "Hkv": Hkv, "page": page, "max_len": max_len,
                "ragged": rng.random() < 0.7, "budget": budget, "sinks": sinks,
                "recent": int((budget - sinks) * rng.uniform(0.0, 0.6))}
    rows, V = _log(rng, 1, 512), _log(rng, 100, 150000)
    while rows * V > 256 * 50257:
        rows //= 2
    return {"op": op, "rows": rows, "V": V, "hist": _log(rng, 1, 4096),
            "n_bias": rng.choice([0, 3, 16, 100]), "mask": rng.random() < 0.5,
            "dtype": rng.choice(["f32", "bf16"]), "out": rng.choice(["f32", "bf16"])}


def _lengths(B, max_len, ragged, least=1):
    """The lengths of a batch: one is the longest, a ragged batch's others go down evenly."""
    if not ragged:
        return [max_len] * B
    return [max(least, max_len - (max_len * b) // B) for b in range(B)]


def _visible(L, window, sinks):
    """Keys that the token at position L - 1 attends to."""
    if window <= 0 or window >= L:
        return L
    return window + min(sinks, L - window)


def work(case):
    c = case
    if c["op"] == "window":
        off = c["Sk"] - c["Sq"]
        pairs = sum(_visible(off + i + 1, c["window"], c["sinks"]) for i in range(c["Sq"]))
        first = max(0, off - c["window"] + 1)
        keys = c["Sk"] - first + min(c["sinks"], first)
        rows = c["B"] * c["H"] * c["Sq"]
        return {"bytes": rows * (4 * D + 8) + 4 * D * c["B"] * c["Hkv"] * keys,
                "flops": 4.0 * D * c["B"] * c["H"] * pairs}
    if c["op"] == "decode":
        n = sum(_visible(L, c["window"], c["sinks"])
                for L in _lengths(c["B"], c["max_len"], c["ragged"]))
        rows = c["B"] * c["H"]
        b = 4 * D * c["Hkv"] * n + rows * (2 * D + (2 if c["out"] == "bf16" else 4) * D + 4)
        b += 4 * c["B"] * (1 + -(-c["max_len"] // c["page"]))
        if c["append"]:
            b += 2 * 4 * D * c["B"] * c["Hkv"]
        if c["weights"]:
            b += 8 * c["Hkv"] * n
        return {"bytes": b, "flops": 4.0 * D * c["H"] * n}
    if c["op"] == "store":
        n = sum(_lengths(c["B"], c["S"], c["ragged"]))
        return {"bytes": 8 * D * c["Hkv"] * n, "flops": 0}
    if c["op"] == "evict":
        L = _lengths(c["B"], c["max_len"], c["ragged"])
        kept = sum(min(x, c["budget"]) for x in L)
        return {"bytes": c["Hkv"] * (4 * sum(L) + kept * (8 * D + 4) + 4 * c["B"] * c["max_len"]),
                "flops": 0}
    rows, V = c["rows"], c["V"]
    size = {"f32": 4, "bf16": 2}
    b = rows * V * (size[c["dtype"]] + size[c["out"]])
    b += 4 * rows * c["hist"] + 8 * rows * c["n_bias"] + (rows * V // 8 if c["mask"] else 0)
    return {"bytes": b, "flops": 0}


# -------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(torch.bfloat16)


def _perm(g, n):
    return torch.randperm(n, generator=g, device="cuda")


def _pool(g, B, Hkv, page, max_pages, spare):
    """A pool with pages in no order: K, V [n_pages][Hkv][page][64] and a table [B][max_pages]."""
    n_pages = B * max_pages + spare
    k = _randn(g, n_pages, Hkv, page, D)
    v = _randn(g, n_pages, Hkv, page, D)
    order = _perm(g, n_pages).to(torch.int32)
    table = order[:B * max_pages].view(B, max_pages).contiguous()
    return k, v, table, order[B * max_pages:]


def _shuffled_lengths(g, case, key):
    L = torch.tensor(_lengths(case["B"], case[key], case["ragged"]), dtype=torch.int32,
                     device="cuda")
    return L[_perm(g, case["B"])].contiguous()


def _drop_unused(table, lens, page):
    """Table entries past a sequence's last page are -1, as a page manager leaves them."""
    used = (torch.arange(table.shape[1], device="cuda")[None, :] * page) < lens[:, None]
    return torch.where(used, table, torch.full_like(table, -1)).contiguous()


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    if c["op"] == "window":
        B, H, Hkv, Sq, Sk = c["B"], c["H"], c["Hkv"], c["Sq"], c["Sk"]
        if c["layout"] == "head":
            s["Q"] = _randn(g, B, H, Sq, D)
            s["K"], s["V"] = _randn(g, B, Hkv, Sk, D), _randn(g, B, Hkv, Sk, D)
            s["O"] = torch.empty((B, H, Sq, D), dtype=torch.bfloat16, device="cuda")
        else:
            heads = lambda x, n: x.unflatten(-1, (n, D)).transpose(1, 2)
            s["O"] = heads(torch.empty((B, Sq, H * D), dtype=torch.bfloat16, device="cuda"), H)
            if c["layout"] == "token":   # the fused projection; a chunk's rows are its last ones
                qkv = _randn(g, B, Sk, (H + 2 * Hkv) * D)
                s["Q"] = heads(qkv[:, Sk - Sq:, :H * D], H)
                s["K"] = heads(qkv[..., H * D:(H + Hkv) * D], Hkv)
                s["V"] = heads(qkv[..., (H + Hkv) * D:], Hkv)
            else:                        # caches with room for more tokens
                s["Q"] = heads(_randn(g, B, Sq, H * D), H)
                s["K"] = _randn(g, B, Hkv, Sk + 61, D)[:, :, :Sk]
                s["V"] = _randn(g, B, Hkv, Sk + 61, D)[:, :, :Sk]
        s["lse"] = torch.empty((B, H, Sq), dtype=torch.float32, device="cuda")
        s["m"] = torch.empty((B, H, Sq), dtype=torch.float32, device="cuda")
    elif c["op"] == "decode":
        B, H, Hkv, page = c["B"], c["H"], c["Hkv"], c["page"]
        max_pages = -(-c["max_len"] // page) + 1
        s["k"], s["v"], table, _ = _pool(g, B, Hkv, page, max_pages, 3)
        s["lens"] = _shuffled_lengths(g, c, "max_len")
        s["table"] = _drop_unused(table, s["lens"], page)
        s["q"] = _randn(g, B, H, D)
        s["k_new"] = _randn(g, B, Hkv, D) if c["append"] else None
        s["v_new"] = _randn(g, B, Hkv, D) if c["append"] else None
        s["weights"] = None
        if c["weights"]:
            s["weights"] = torch.rand((B, Hkv, max_pages * page), generator=g, device="cuda")
        dt = torch.bfloat16 if c["out"] == "bf16" else torch.float32
        s["out"] = torch.empty((B, H, D), dtype=dt, device="cuda")
        s["lse"] = torch.empty((B, H), dtype=torch.float32, device="cuda")
        s["workspace"] = None
        if own:
            from neurodsl_b200 import ops
            s["workspace"] = ops.paged_decode_workspace(B, H, Hkv, max_pages * page,
                                                        weights=c["weights"])
    elif c["op"] == "store":
        B, Hkv, S, page = c["B"], c["Hkv"], c["S"], c["page"]
        lens = _shuffled_lengths(g, c, "S")
        pos0 = torch.randint(0, 2 * page + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        max_pages = -(-(S + 2 * page) // page)
        s["k"], s["v"], table, _ = _pool(g, B, Hkv, page, max_pages, 3)
        s["table"] = _drop_unused(table, pos0 + lens, page)
        s["src"] = _randn(g, B * S, 3 * Hkv * D)
        s["pos0"], s["lens"] = pos0, lens
    elif c["op"] == "evict":
        B, Hkv, page, budget = c["B"], c["Hkv"], c["page"], c["budget"]
        max_pages, out_pages = -(-c["max_len"] // page), -(-budget // page)
        s["k"], s["v"], table, spare = _pool(g, B, Hkv, page, max_pages, B * out_pages)
        s["lens"] = _shuffled_lengths(g, c, "max_len")
        s["table"] = _drop_unused(table, s["lens"], page)
        s["out_table"] = spare.view(B, out_pages).contiguous()
        # a few keys take most of the weight; many of the small ones are equal
        w = torch.rand((B, Hkv, max_pages * page), generator=g, device="cuda") ** 6
        s["weights"] = torch.where(w < 0.01, torch.floor(w * 1024) / 1024, w)
        s["weights_out"] = torch.empty_like(s["weights"])
        s["kept"] = torch.empty((B, Hkv, budget), dtype=torch.int32, device="cuda")
        s["new_lens"] = torch.empty((B,), dtype=torch.int32, device="cuda")
        s["workspace"] = None
    else:
        rows, V = c["rows"], c["V"]
        dts = {"f32": torch.float32, "bf16": torch.bfloat16}
        x = 4.0 * torch.randn((rows, V), generator=g, device="cuda")
        s["logits"] = x.to(dts[c["dtype"]])
        # half of a history is common tokens, which repeat; short histories are padded with -1
        n = c["hist"]
        common = torch.randint(0, max(1, min(V, 1 + n // 4)), (rows, n), generator=g, device="cuda")
        rare = torch.randint(0, V, (rows, n), generator=g, device="cuda")
        pick = torch.rand((rows, n), generator=g, device="cuda") < 0.5
        at = torch.arange(n, device="cuda")[None, :]
        lens = torch.randint(1, n + 1, (rows, 1), generator=g, device="cuda")
        lens[0] = n
        hist = torch.where(pick, common, rare)
        s["history"] = torch.where(at < lens, hist, torch.full_like(hist, -1)).to(torch.int32)
        u = lambda lo, hi: lo + (hi - lo) * torch.rand((rows,), generator=g, device="cuda")
        s["repetition"], s["presence"], s["frequency"] = u(1.0, 1.5), u(0.0, 1.0), u(0.0, 0.5)
        s["bias_ids"] = s["bias"] = None
        if c["n_bias"]:
            nb = min(c["n_bias"], V)
            s["bias_ids"] = torch.rand((rows, V), generator=g, device="cuda").topk(
                nb, dim=1).indices.to(torch.int32).contiguous()
            s["bias"] = 3.0 * torch.randn((rows, nb), generator=g, device="cuda")
        s["mask"] = None
        if c["mask"]:
            words = -(-V // 32)
            s["mask"] = torch.randint(-2**31, 2**31, (rows, words), generator=g, device="cuda",
                                      dtype=torch.int64).to(torch.int32)
        s["out"] = torch.empty((rows, V), dtype=dts[c["out"]], device="cuda")
        s["idx"] = torch.empty((rows,), dtype=torch.int32, device="cuda")
    return s


# --------------------------------------------------------------- plain forms
def _window_plain(s, c):
    B, H, Hkv, Sq, Sk = c["B"], c["H"], c["Hkv"], c["Sq"], c["Sk"]
    q = s["Q"].float().reshape(B, Hkv, H // Hkv, Sq, D)
    k, v = s["K"].float().unsqueeze(2), s["V"].float().unsqueeze(2)
    x = (q @ k.transpose(-1, -2)).mul_(1.0 / math.sqrt(D))
    p = torch.arange(Sk - Sq, Sk, device="cuda")[:, None]
    j = torch.arange(Sk, device="cuda")[None, :]
    seen = (j <= p) & ((j > p - c["window"]) | (j < c["sinks"]))
    x.masked_fill_(~seen, -math.inf)
    m = x.amax(-1, keepdim=True)
    e = x.sub_(m).exp_()
    total = e.sum(-1, keepdim=True)
    out = (e @ v) / total
    s["O"].copy_(out.reshape(B, H, Sq, D))
    s["m"].copy_(m.reshape(B, H, Sq))
    s["lse"].copy_((m + total.log()).reshape(B, H, Sq))
    return s["O"], s["lse"], s["m"]


def _decode_plain(s, c):
    B, H, Hkv, page = c["B"], c["H"], c["Hkv"], c["page"]
    L = s["lens"].long()
    table = s["table"].clamp(min=0).long()
    if c["append"]:
        at = table.gather(1, ((L - 1) // page)[:, None])[:, 0]
        s["k"][at, :, (L - 1) % page] = s["k_new"]
        s["v"][at, :, (L - 1) % page] = s["v_new"]
    k = s["k"][table].transpose(1, 2).reshape(B, Hkv, -1, D)
    v = s["v"][table].transpose(1, 2).reshape(B, Hkv, -1, D)
    q = s["q"].float().view(B, Hkv, H // Hkv, D)
    x = (q @ k.float().transpose(-1, -2)) * (1.0 / math.sqrt(D))
    j = torch.arange(k.shape[2], device="cuda")[None, :]
    seen = j < L[:, None]
    if c["window"]:
        seen = seen & ((j >= L[:, None] - c["window"]) | (j < c["sinks"]))
    seen = seen[:, None, None, :]
    x = x.masked_fill(~seen, -math.inf)
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(-1, keepdim=True)
    out = (e @ v.float()) / total
    s["out"].copy_(out.view(B, H, D))
    s["lse"].copy_((m + total.log()).view(B, H))
    got = [s["out"], s["lse"]]
    if c["weights"]:
        s["weights"] += (e / total).sum(2)
        got.append(s["weights"])
    if c["append"]:
        got += [s["k"], s["v"]]
    return got


def _store_plain(s, c):
    B, Hkv, S, page = c["B"], c["Hkv"], c["S"], c["page"]
    x = s["src"].view(B, S, 3, Hkv, D)
    tok = torch.arange(S, device="cuda")[None, :]
    # padding repeats the sequence's last token, so that every row has a place
    last = torch.minimum(tok, s["lens"].long()[:, None] - 1)
    pos = s["pos0"].long()[:, None] + last
    at = s["table"].long().gather(1, pos // page)
    rows = x.gather(1, last[:, :, None, None, None].expand(B, S, 3, Hkv, D))
    s["k"][at, :, pos % page] = rows[:, :, 1]
    s["v"][at, :, pos % page] = rows[:, :, 2]
    return s["k"], s["v"]


def _evict_plain(s, c):
    B, Hkv, page, budget = c["B"], c["Hkv"], c["page"], c["budget"]
    w = s["weights"]
    n = w.shape[2]
    L = s["lens"].long()[:, None, None]
    j = torch.arange(n, device="cuda")[None, None, :]
    held = (j < c["sinks"]) | (j >= L - c["recent"])
    rank = torch.where(held, torch.full_like(w, math.inf), w)
    rank = torch.where(j < L, rank, torch.full_like(w, -math.inf))
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    keep = torch.minimum(L, torch.full_like(L, budget))
    slot = torch.arange(budget, device="cuda")[None, None, :]
    order = torch.where(slot < keep, order, torch.full_like(order, n)).sort(-1).values
    there = order < n
    src = order.clamp(max=n - 1)
    head = torch.arange(Hkv, device="cuda")[None, :, None]
    table = s["table"].clamp(min=0).long()[:, None, :].expand(B, Hkv, -1)
    from_page = table.gather(2, src // page)
    to_page = s["out_table"].long()[:, None, :].expand(B, Hkv, -1).gather(
        2, (slot // page).expand(B, Hkv, budget))
    to_row = slot % page
    for pool in (s["k"], s["v"]):
        got = torch.where(there[..., None], pool[from_page, head, src % page],
                          pool[to_page, head, to_row])
        pool[to_page, head, to_row] = got
    s["weights_out"].zero_()
    s["weights_out"][..., :budget] = torch.where(there, w.gather(2, src),
                                                 torch.zeros_like(w[..., :1]))
    s["kept"].copy_(torch.where(there, order, torch.full_like(order, -1)))
    s["new_lens"].copy_(keep[:, 0, 0])
    return s["k"], s["v"], s["weights_out"], s["kept"], s["new_lens"]


def _logits_plain(s, c):
    V = c["V"]
    x = s["logits"].float()
    hist = s["history"].long()
    count = torch.zeros_like(x).scatter_add_(1, hist.clamp(min=0), (hist >= 0).float())
    seen = count > 0
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = torch.where(seen, x - s["presence"][:, None], x)
    x = torch.where(seen, x - s["frequency"][:, None] * count, x)
    if s["bias"] is not None:
        x = x.scatter_add(1, s["bias_ids"].long(), s["bias"])
    if s["mask"] is not None:
        v = torch.arange(V, device="cuda")
        bit = (s["mask"][:, v >> 5] >> (v & 31)) & 1
        x = x.masked_fill(bit == 0, -math.inf)
    s["out"].copy_(x)
    s["idx"].copy_(s["out"].argmax(-1))
    return s["out"], s["idx"]


def run(state):
    s, c = state, state["case"]
    if own:
        return _run_own(s, c)
    return {"window": _window_plain, "decode": _decode_plain, "store": _store_plain,
            "evict": _evict_plain, "logits": _logits_plain}[c["op"]](s, c)


def _run_own(s, c):
    from neurodsl_b200 import ops
    if c["op"] == "window":
        return ops.window_attn_fwd(s["Q"], s["K"], s["V"], c["window"], sinks=c["sinks"],
                                   out=s["O"], lse=s["lse"], row_max=s["m"])
    if c["op"] == "decode":
        out, lse = ops.paged_decode_attn(s["q"], s["k"], s["v"], s["table"], s["lens"],
                                         k_new=s["k_new"], v_new=s["v_new"], window=c["window"],
                                         sinks=c["sinks"], out=s["out"], lse=s["lse"],
                                         weights=s["weights"], workspace=s["workspace"])
        got = [out, lse]
        if c["weights"]:
            got.append(s["weights"])
        if c["append"]:
            got += [s["k"], s["v"]]
        return got
    if c["op"] == "store":
        n = c["Hkv"] * D
        ops.paged_kv_store(s["src"], n, 2 * n, s["k"], s["v"], s["table"], c["B"], c["S"],
                           pos0=s["pos0"], lens=s["lens"])
        return s["k"], s["v"]
    if c["op"] == "evict":
        ops.paged_kv_evict(s["k"], s["v"], s["table"], s["lens"], s["weights"], s["out_table"],
                           c["budget"], sinks=c["sinks"], recent=c["recent"],
                           weights_out=s["weights_out"], kept=s["kept"], new_lens=s["new_lens"])
        return s["k"], s["v"], s["weights_out"], s["kept"], s["new_lens"]
    return ops.logits_penalty(s["logits"], history=s["history"], repetition=s["repetition"],
                              presence=s["presence"], frequency=s["frequency"],
                              bias_ids=s["bias_ids"], bias=s["bias"], mask=s["mask"],
                              out=s["out"], idx=s["idx"])


# ------------------------------------------------------- 64-bit definitions
def _softmax_rows(x):
    m = x.max(-1, keepdim=True).values
    lse = torch.logsumexp(x, -1)
    return torch.exp(x - lse[..., None]), lse, m[..., 0]


def _rows_of(pool, table, b, h, L, page):
    """Keys or values 0 .. L-1 of one sequence and head, in order."""
    used = table[b, :-(-L // page)].long()
    return pool[used, h].reshape(-1, D)[:L].double()


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "window":
        B, H, Hkv, Sq, Sk = c["B"], c["H"], c["Hkv"], c["Sq"], c["Sk"]
        O = torch.empty((B, H, Sq, D), dtype=torch.float64, device="cuda")
        lse = torch.empty((B, H, Sq), dtype=torch.float64, device="cuda")
        m = torch.empty_like(lse)
        step = 512
        for i0 in range(0, Sq, step):
            i1 = min(Sq, i0 + step)
            pos = torch.arange(Sk - Sq + i0, Sk - Sq + i1, device="cuda")
            lo = max(0, Sk - Sq + i0 - c["window"] + 1)
            head = min(c["sinks"], lo)
            keys = torch.cat([torch.arange(head, device="cuda"),
                              torch.arange(lo, Sk - Sq + i1, device="cuda")])
            near = pos[:, None] - keys[None, :]
            ok = (near >= 0) & ((near < c["window"]) | (keys < c["sinks"])[None, :])
            for b in range(B):
                k = s["K"][b][:, keys].double().repeat_interleave(H // Hkv, 0)
                v = s["V"][b][:, keys].double().repeat_interleave(H // Hkv, 0)
                x = torch.einsum("hqd,hkd->hqk", s["Q"][b, :, i0:i1].double(), k) / math.sqrt(D)
                x[:, ~ok] = -math.inf
                p, lse[b, :, i0:i1], m[b, :, i0:i1] = _softmax_rows(x)
                O[b, :, i0:i1] = torch.einsum("hqk,hkd->hqd", p, v)
        return O, lse, m
    if c["op"] == "decode":
        B, H, Hkv, page = c["B"], c["H"], c["Hkv"], c["page"]
        G = H // Hkv
        k, v = s["k"].clone(), s["v"].clone()
        out = torch.empty((B, H, D), dtype=torch.float64, device="cuda")
        lse = torch.empty((B, H), dtype=torch.float64, device="cuda")
        w = s["weights"].double() if c["weights"] else None
        for b, L in enumerate(s["lens"].tolist()):
            if c["append"]:
                at = int(s["table"][b, (L - 1) // page])
                k[at, :, (L - 1) % page] = s["k_new"][b]
                v[at, :, (L - 1) % page] = s["v_new"][b]
            keys = torch.arange(L, device="cuda")
            if c["window"]:
                keys = keys[(keys >= L - c["window"]) | (keys < c["sinks"])]
            for h in range(Hkv):
                q = s["q"][b, h * G:(h + 1) * G].double()
                x = q @ _rows_of(k, s["table"], b, h, L, page)[keys].T / math.sqrt(D)
                p, lse[b, h * G:(h + 1) * G], _ = _softmax_rows(x)
                out[b, h * G:(h + 1) * G] = p @ _rows_of(v, s["table"], b, h, L, page)[keys]
                if w is not None:
                    w[b, h, keys] += p.sum(0)
        return [out, lse] + ([w] if w is not None else []) + ([k, v] if c["append"] else [])
    if c["op"] == "store":
        B, Hkv, S, page = c["B"], c["Hkv"], c["S"], c["page"]
        n = Hkv * D
        k, v = s["k"], s["v"]
        for b, (L, p0) in enumerate(zip(s["lens"].tolist(), s["pos0"].tolist())):
            pos = torch.arange(p0, p0 + L, device="cuda")
            at = s["table"][b].long()[pos // page]
            src = s["src"][b * S:b * S + L]
            k[at, :, pos % page] = src[:, n:2 * n].view(L, Hkv, D)
            v[at, :, pos % page] = src[:, 2 * n:].view(L, Hkv, D)
        return k, v
    if c["op"] == "evict":
        B, Hkv, page, budget = c["B"], c["Hkv"], c["page"], c["budget"]
        k, v = s["k"], s["v"]
        kept = torch.full((B, Hkv, budget), -1, dtype=torch.int32, device="cuda")
        new_lens = torch.empty((B,), dtype=torch.int32, device="cuda")
        w_out = torch.zeros_like(s["weights"])
        for b, L in enumerate(s["lens"].tolist()):
            n = min(L, budget)
            new_lens[b] = n
            for h in range(Hkv):
                w = s["weights"][b, h, :L]
                if L > budget:
                    a, z = c["sinks"], L - c["recent"]
                    mid = w[a:z].cpu().numpy()
                    best = (-mid).argsort(kind="stable")[:budget - c["sinks"] - c["recent"]]
                    mid_keep = torch.from_numpy(best.copy()).cuda() + a
                    rows = torch.cat([torch.arange(a, device="cuda"), mid_keep.sort().values,
                                      torch.arange(z, L, device="cuda")])
                else:
                    rows = torch.arange(L, device="cuda")
                slot = torch.arange(n, device="cuda")
                src, dst = s["table"][b].long()[rows // page], s["out_table"][b].long()[slot // page]
                k[dst, h, slot % page] = k[src, h, rows % page]
                v[dst, h, slot % page] = v[src, h, rows % page]
                kept[b, h, :n] = rows.to(torch.int32)
                w_out[b, h, :n] = w[rows]
        return k, v, w_out, kept, new_lens
    x = s["logits"].double()
    for r in range(c["rows"]):
        hist = s["history"][r]
        tok, count = hist[hist >= 0].long().unique(return_counts=True)
        y = x[r, tok]
        rep = s["repetition"][r].double()
        y = torch.where(y > 0, y / rep, y * rep)
        x[r, tok] = y - s["presence"][r].double() - s["frequency"][r].double() * count
        if s["bias"] is not None:
            x[r, s["bias_ids"][r].long()] += s["bias"][r].double()
        if s["mask"] is not None:
            words = s["mask"][r].long() & 0xFFFFFFFF
            bits = (words[:, None] >> torch.arange(32, device="cuda")) & 1
            x[r, bits.flatten()[:c["V"]] == 0] = -math.inf
    return x, None
