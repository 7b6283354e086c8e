"""The serving operators' calls made by the extension (csrc/py_calls.cpp) and
by the foreign-function interface: one entry point behind both, so for any
arguments both give the same bits or both refuse in the same words."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _ops():
    from neurodsl_b200 import _lib, ops
    assert _lib.load_calls(), "the extension is built and loads"
    return ops, _lib


def _bf(g, *shape):
    return torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)


def arguments(name):
    """A valid call's arguments by name; what it writes."""
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    i32 = dict(dtype=torch.int32, device=DEV)
    f32 = dict(dtype=torch.float32, device=DEV)
    B, H, Hkv, page, mp, D = 3, 4, 2, 8, 5, 64
    n = 2 * B * mp
    pool = lambda: dict(k_pages=_bf(g, n, Hkv, page, D), v_pages=_bf(g, n, Hkv, page, D))  # noqa: E731
    table = torch.arange(B * mp, **i32).view(B, mp)
    lens = torch.tensor([1, 17, 40], **i32)
    if name == "window_attn_fwd":
        Sq, Sk = 9, 21
        return dict(Q=_bf(g, B, H, Sq, D), K=_bf(g, B, Hkv, Sk, D), V=_bf(g, B, Hkv, Sk, D), window=7, sinks=2,
                    scale=0.25, out=torch.zeros((B, H, Sq, D), dtype=torch.bfloat16, device=DEV),
                    lse=torch.zeros((B, H, Sq), **f32), row_max=torch.zeros((B, H, Sq), **f32))
    if name == "paged_decode_attn":
        ops, _ = _ops()
        return dict(q=_bf(g, B, H, D), **pool(), block_table=table, lens=lens, k_new=_bf(g, B, Hkv, D),
                    v_new=_bf(g, B, Hkv, D), window=11, sinks=1, scale=0.125, out=torch.zeros((B, H, D), **f32),
                    lse=torch.zeros((B, H), **f32), weights=torch.zeros((B, Hkv, mp * page), **f32),
                    workspace=ops.paged_decode_workspace(B, H, Hkv, mp * page, weights=True))
    if name == "paged_kv_store":
        S = 6
        return dict(src=_bf(g, B * S, 2 * Hkv * D), k_col=0, v_col=Hkv * D, **pool(), block_table=table, B=B, S=S,
                    pos0=torch.tensor([0, 3, 30], **i32), lens=torch.tensor([6, 0, 5], **i32))
    if name == "paged_kv_evict":
        return dict(**pool(), block_table=table, lens=lens, weights=torch.rand((B, Hkv, mp * page), generator=g, **f32),
                    out_table=table + B * mp, budget=16, sinks=2, recent=4,
                    weights_out=torch.zeros((B, Hkv, mp * page), **f32), kept=torch.zeros((B, Hkv, 16), **i32),
                    new_lens=torch.zeros((B,), **i32))
    V = 300
    return dict(logits=torch.randn((B, V), generator=g, **f32),
                history=torch.randint(0, V, (B, 20), generator=g, **i32),
                history_lens=torch.tensor([20, 3, 0], **i32), repetition=torch.full((B,), 1.5, **f32),
                presence=torch.full((B,), 0.5, **f32), frequency=torch.full((B,), 0.25, **f32),
                bias_ids=torch.randint(0, V, (B, 4), generator=g, **i32), bias=torch.ones((B, 4), **f32),
                mask=torch.randint(-2**31, 2**31 - 1, (B, 10), generator=g, **i32),
                out=torch.zeros((B, V), **f32), idx=torch.zeros((B,), **i32))


NAMES = ["window_attn_fwd", "paged_decode_attn", "paged_kv_store", "paged_kv_evict", "logits_penalty"]


def outcome(monkeypatch, name, direct, change):
    """The bits of every tensor after the call, or the refusal's words."""
    ops, lib = _ops()
    args = arguments(name)
    change(args)
    made = []
    if direct:
        def quick(op, *a):
            made.append(real(op, *a))
            return made[-1]
        real = ops._quick
        monkeypatch.setattr(ops, "_quick", quick)
    else:
        monkeypatch.setattr(lib, "calls", False)
    try:
        ret = getattr(ops, name)(**args)
    except Exception as e:  # noqa: BLE001
        return (type(e), str(e)), made
    finally:
        monkeypatch.undo()
    torch.cuda.synchronize()
    ops.device_error()  # a table cut short is reported there: not this module's matter
    args.pop("workspace", None)
    ret = ret if isinstance(ret, tuple) else (ret,)
    tensors = list(args.values()) + list(ret)
    return [None if t is None else t.contiguous().view(torch.uint8).cpu() for t in tensors
            if t is None or (isinstance(t, torch.Tensor) and t.is_cuda and t.numel())], made


def same(a, b):
    if isinstance(a, tuple) or isinstance(b, tuple):
        return a == b
    return len(a) == len(b) and all((x is None and y is None) or torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("name", NAMES)
def test_common_calls_are_direct_and_the_same(monkeypatch, name):
    optional = {"window_attn_fwd": ["scale"], "paged_decode_attn": ["scale", "weights"],
                "paged_kv_store": ["lens"], "paged_kv_evict": [],
                "logits_penalty": ["history_lens", "repetition", "presence", "frequency", "mask"]}
    for gone in [None] + optional[name]:
        def change(args):
            if gone is not None:
                args[gone] = None
        direct, made = outcome(monkeypatch, name, True, change)
        checked, _ = outcome(monkeypatch, name, False, change)
        assert made == [True], gone
        assert same(direct, checked), gone


def test_pairs_left_out(monkeypatch):
    for name, pair in [("paged_decode_attn", ("k_new", "v_new")), ("logits_penalty", ("bias_ids", "bias"))]:
        def change(args):
            args.update(dict.fromkeys(pair))
        direct, made = outcome(monkeypatch, name, True, change)
        assert made == [True] and same(direct, outcome(monkeypatch, name, False, change)[0])


def variants(value):
    """Other values for an argument: missing, on the host, of another type,
    shape or layout; none of them an index that a kernel would follow."""
    yield "none", None
    yield "text", "x"
    if isinstance(value, torch.Tensor):
        yield "host", value.cpu()
        yield "double", value.double()
        yield "short", value[:-1]
        yield "half", value[..., :value.shape[-1] // 2]
        yield "empty", value[:0]
        yield "deeper", value.unsqueeze(0)
        yield "turned", value.transpose(0, -1)
        yield "spread", torch.stack([value, value], -1)[..., 0]
        yield "rows", torch.cat([value, value], -1)[..., :value.shape[-1]]
    elif isinstance(value, int):
        for v in (0, -1, 2**31 - 1, 2**31, 2**40, -2**40, float(value), True):
            yield repr(v), v
    else:
        for v in (1, 2.0, "x"):
            yield repr(v), v


@pytest.mark.parametrize("name", NAMES)
def test_the_same_answer_or_the_same_refusal(monkeypatch, name):
    for key, value in arguments(name).items():
        for what, other in variants(value):
            def change(args):
                args[key] = other.clone(memory_format=torch.preserve_format) if (
                    isinstance(other, torch.Tensor) and what in ("double", "host")) else other
            a, _ = outcome(monkeypatch, name, True, change)
            b, _ = outcome(monkeypatch, name, False, change)
            assert same(a, b), (key, what, a if isinstance(a, tuple) else "ran", b if isinstance(b, tuple) else "ran")


def test_integers_past_32_bits(monkeypatch):
    """They are refused, or as good as unlimited, and never cut to their low bits."""
    def refused(name, **change):
        got, _ = outcome(monkeypatch, name, True, lambda args: args.update(change))
        return isinstance(got, tuple)
    for v in (2**32, -2**32):
        assert refused("paged_kv_evict", recent=v)
        assert refused("paged_kv_evict", sinks=v)
        assert refused("paged_kv_evict", budget=v)
        assert refused("paged_kv_store", pos0=v, lens=None)
        assert refused("paged_kv_store", k_col=v)
    wide = outcome(monkeypatch, "window_attn_fwd", True, lambda a: a.update(window=2**32))[0]
    assert same(wide[3:], outcome(monkeypatch, "window_attn_fwd", True, lambda a: a.update(window=1000))[0][3:])


def test_memory_errors_do_not_outlive_a_refusal(monkeypatch):
    """A status of the entry point itself (here: a small workspace) comes out as
    the library's error through both, and the next call is fine."""
    def change(args):
        args["workspace"] = args["workspace"][:64]
    a, _ = outcome(monkeypatch, "paged_decode_attn", True, change)
    b, _ = outcome(monkeypatch, "paged_decode_attn", False, change)
    assert isinstance(a, tuple) and a == b
    assert outcome(monkeypatch, "paged_decode_attn", True, lambda args: None)[1] == [True]


def test_current_stream_and_capture():
    ops, _ = _ops()
    args = arguments("logits_penalty")
    want, idx = ops.logits_penalty(**args)
    torch.cuda.synchronize()
    want, idx = want.clone(), idx.clone()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    args["out"].zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        ops.logits_penalty(**args)
    torch.cuda.synchronize()
    assert not args["out"].any()  # captured, not run
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(args["out"], want) and torch.equal(args["idx"], idx)
    args["out"].zero_()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.logits_penalty(**args)
    s.synchronize()
    assert torch.equal(args["out"], want)


@pytest.mark.parametrize("name, made", [("window_attn_fwd", ("out", "lse", "row_max")),
                                        ("paged_decode_attn", ("out", "lse", "workspace")),
                                        ("paged_kv_evict", ("weights_out", "kept", "new_lens")),
                                        ("logits_penalty", ("out", "idx"))])
def test_outputs_are_made_on_the_calls_stream(monkeypatch, name, made):
    """Memory from another stream's pool may still be in use there."""
    ops, _ = _ops()
    args = arguments(name)
    want = getattr(ops, name)(**args)
    torch.cuda.synchronize()
    args = arguments(name)      # weights and pages as they were
    args.update(dict.fromkeys(made))
    if "out" in made:
        args["out_dtype"] = want[0].dtype
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    streams = []
    for fn in ("empty", "zeros", "empty_like"):
        def note(*a, real=getattr(torch, fn), **k):
            streams.append(torch.cuda.current_stream())
            return real(*a, **k)
        monkeypatch.setattr(torch, fn, note)
    got = getattr(ops, name)(**args, stream=s)
    monkeypatch.undo()
    assert len(streams) == len(made) and all(x == s for x in streams)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_two_threads_at_once():
    """Each with a stream, a workspace and buffers of its own."""
    import threading
    ops, _ = _ops()
    names = ["paged_decode_attn", "logits_penalty", "window_attn_fwd"]
    want = {}
    for name in names:
        args = arguments(name)
        args.pop("weights", None)
        want[name] = [t.clone() for t in getattr(ops, name)(**args)]
    torch.cuda.synchronize()
    wrong = []

    def work():
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                sets = {}
                for name in names:
                    sets[name] = arguments(name)
                    sets[name].pop("weights", None)
                for _ in range(40):
                    for name in names:
                        got = getattr(ops, name)(**sets[name])
                        if not all(torch.equal(a, b) for a, b in zip(got, want[name])):
                            wrong.append(name)
        except Exception as e:  # noqa: BLE001
            wrong.append(e)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong
