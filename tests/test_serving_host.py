"""Argument checks of the window, paged-cache and logits entry points, on the
host: each refuses a bad call with its status and message before any device
work, and accepts empty ones."""
import ctypes

import pytest


def _lib():
    from neurodsl_b200 import _lib
    return _lib, _lib.load()


P = ctypes.c_void_p(0x10000)      # a 16-byte aligned address that is never read
ODD = ctypes.c_void_p(0x10004)
ST = (ctypes.c_int64 * 3)(64, 64 * 100, 64 * 400)


def window(lib, **kw):
    a = dict(q=P, k=P, v=P, o=P, qs=ST, o_dtype=1, B=1, H=4, Hkv=2, Sq=10, Sk=20, D=64,
             scale=0.125, window=8, sinks=2)
    a.update(kw)
    return lib.nd_window_attn_fwd(None, a["q"], a["qs"], a["k"], ST, a["v"], ST, a["o"], ST,
                                  a["o_dtype"], None, None, a["B"], a["H"], a["Hkv"], a["Sq"],
                                  a["Sk"], a["D"], a["scale"], a["window"], a["sinks"])


@pytest.mark.parametrize("kw, status", [
    (dict(D=32), "ND_ERR_UNSUPPORTED"), (dict(Hkv=3), "ND_ERR_SHAPE"), (dict(Hkv=0), "ND_ERR_SHAPE"),
    (dict(Sq=21), "ND_ERR_SHAPE"), (dict(window=0), "ND_ERR_INVALID_ARG"),
    (dict(sinks=-1), "ND_ERR_INVALID_ARG"), (dict(scale=0.0), "ND_ERR_INVALID_ARG"),
    (dict(scale=float("nan")), "ND_ERR_INVALID_ARG"), (dict(o_dtype=2), "ND_ERR_UNSUPPORTED"),
    (dict(B=-1), "ND_ERR_INVALID_ARG"), (dict(q=None), "ND_ERR_INVALID_ARG"),
    (dict(o=ODD), "ND_ERR_ALIGNMENT"), (dict(qs=None), "ND_ERR_INVALID_ARG"),
    (dict(qs=(ctypes.c_int64 * 3)(60, 6400, 25600)), "ND_ERR_SHAPE"),
    (dict(qs=(ctypes.c_int64 * 3)(64, 6400, 0), B=2), "ND_ERR_SHAPE"),
    (dict(B=0), "ND_OK"), (dict(Sq=0), "ND_OK"), (dict(H=0, Hkv=0), "ND_OK"),
])
def test_window_attn_checks(kw, status):
    m, lib = _lib()
    assert window(lib, **kw) == getattr(m, status), lib.nd_last_error_string()


def decode(lib, **kw):
    a = dict(q=P, kn=None, vn=None, k=P, v=P, n_pages=8, page=16, table=P, ld=4, max_pages=4,
             lens=P, out=P, o_dtype=1, weights=None, w_ld=0, B=2, H=4, Hkv=2, D=64, window=0,
             sinks=0, scale=0.125, ws=P, ws_bytes=1 << 40)
    a.update(kw)
    return lib.nd_paged_decode_attn(None, a["q"], a["kn"], a["vn"], a["k"], a["v"], a["n_pages"],
                                    a["page"], a["table"], a["ld"], a["max_pages"], a["lens"],
                                    a["out"], a["o_dtype"], None, a["weights"], a["w_ld"], a["B"],
                                    a["H"], a["Hkv"], a["D"], a["window"], a["sinks"], a["scale"],
                                    a["ws"], a["ws_bytes"])


@pytest.mark.parametrize("kw, status", [
    (dict(D=128), "ND_ERR_UNSUPPORTED"), (dict(page=0), "ND_ERR_SHAPE"),
    (dict(max_pages=1 << 26, ld=1 << 26), "ND_ERR_SHAPE"), (dict(ld=3), "ND_ERR_SHAPE"),
    (dict(n_pages=0), "ND_ERR_SHAPE"), (dict(H=5), "ND_ERR_SHAPE"), (dict(Hkv=0), "ND_ERR_SHAPE"),
    (dict(kn=P), "ND_ERR_INVALID_ARG"), (dict(window=-1), "ND_ERR_INVALID_ARG"),
    (dict(sinks=-1), "ND_ERR_INVALID_ARG"), (dict(scale=float("inf")), "ND_ERR_INVALID_ARG"),
    (dict(weights=P, w_ld=63), "ND_ERR_SHAPE"), (dict(lens=None), "ND_ERR_INVALID_ARG"),
    (dict(table=None), "ND_ERR_INVALID_ARG"), (dict(k=ODD), "ND_ERR_ALIGNMENT"),
    (dict(q=ODD), "ND_ERR_ALIGNMENT"), (dict(ws=None), "ND_ERR_WORKSPACE"),
    (dict(ws_bytes=64), "ND_ERR_WORKSPACE"), (dict(ws=ODD), "ND_ERR_ALIGNMENT"),
    (dict(B=70000, H=2), "ND_ERR_SHAPE"), (dict(o_dtype=3), "ND_ERR_UNSUPPORTED"),
    (dict(B=-2), "ND_ERR_INVALID_ARG"), (dict(B=0, q=None, k=None, lens=None), "ND_OK"),
    (dict(H=0, Hkv=0), "ND_OK"),
])
def test_paged_decode_checks(kw, status):
    m, lib = _lib()
    assert decode(lib, **kw) == getattr(m, status), lib.nd_last_error_string()


def test_paged_workspace_size():
    m, lib = _lib()
    n, w = ctypes.c_size_t(0), ctypes.c_size_t(0)
    f = lib.nd_paged_decode_workspace_size
    assert f(2, 8, 2, 1000, 64, 0, ctypes.byref(n)) == m.ND_OK
    assert f(2, 8, 2, 1000, 64, 1, ctypes.byref(w)) == m.ND_OK
    assert w.value >= n.value + 2 * 8 * 1000 * 4
    # sizes do not depend on the batch or the length without weights
    assert f(64, 8, 2, 1 << 20, 64, 0, ctypes.byref(w)) == m.ND_OK and w.value == n.value
    assert f(2, 8, 3, 1000, 64, 0, ctypes.byref(n)) == m.ND_ERR_SHAPE
    assert f(2, 8, 2, -1, 64, 0, ctypes.byref(n)) == m.ND_ERR_INVALID_ARG
    assert f(2, 8, 2, 1 << 30, 64, 0, ctypes.byref(n)) == m.ND_ERR_SHAPE
    assert f(2, 8, 2, 8, 32, 0, ctypes.byref(n)) == m.ND_ERR_UNSUPPORTED
    assert f(2, 8, 2, 8, 64, 0, None) == m.ND_ERR_INVALID_ARG


def store(lib, **kw):
    a = dict(src=P, ld=384, k_col=128, v_col=256, k=P, v=P, n_pages=8, page=16, table=P, t_ld=4,
             max_pages=4, B=2, S=30, Hkv=2, pos0=10, pos_dev=None, lens=None, D=64)
    a.update(kw)
    return lib.nd_paged_kv_store(None, a["src"], a["ld"], a["k_col"], a["v_col"], a["k"], a["v"],
                                 a["n_pages"], a["page"], a["table"], a["t_ld"], a["max_pages"],
                                 a["B"], a["S"], a["Hkv"], a["pos0"], a["pos_dev"], a["lens"],
                                 a["D"])


@pytest.mark.parametrize("kw, status", [
    (dict(pos0=35), "ND_ERR_SHAPE"), (dict(pos0=-1), "ND_ERR_INVALID_ARG"),
    (dict(ld=380), "ND_ERR_SHAPE"), (dict(k_col=4), "ND_ERR_SHAPE"), (dict(v_col=264), "ND_ERR_SHAPE"),
    (dict(src=None), "ND_ERR_INVALID_ARG"), (dict(src=ODD), "ND_ERR_ALIGNMENT"),
    (dict(D=32), "ND_ERR_UNSUPPORTED"), (dict(S=-1), "ND_ERR_INVALID_ARG"),
    (dict(n_pages=0), "ND_ERR_SHAPE"), (dict(S=0, src=None), "ND_OK"), (dict(B=0), "ND_OK"),
])
def test_paged_store_checks(kw, status):
    m, lib = _lib()
    assert store(lib, **kw) == getattr(m, status), lib.nd_last_error_string()


def evict(lib, **kw):
    a = dict(k=P, v=P, n_pages=8, page=16, table=P, t_ld=4, max_pages=4, lens=P,
             w=ctypes.c_void_p(0x100000), w_ld=64, ot=P, ot_ld=2, out_pages=2,
             wo=ctypes.c_void_p(0x200000), wo_ld=64, kept=P, new_lens=P, B=2, Hkv=2, D=64,
             budget=32, sinks=4, recent=8)
    a.update(kw)
    return lib.nd_paged_kv_evict(None, a["k"], a["v"], a["n_pages"], a["page"], a["table"],
                                 a["t_ld"], a["max_pages"], a["lens"], a["w"], a["w_ld"], a["ot"],
                                 a["ot_ld"], a["out_pages"], a["wo"], a["wo_ld"], a["kept"],
                                 a["new_lens"], a["B"], a["Hkv"], a["D"], a["budget"], a["sinks"],
                                 a["recent"])


@pytest.mark.parametrize("kw, status", [
    (dict(budget=0, sinks=0, recent=0), "ND_ERR_INVALID_ARG"), (dict(sinks=25), "ND_ERR_INVALID_ARG"),
    (dict(sinks=-1), "ND_ERR_INVALID_ARG"), (dict(budget=33), "ND_ERR_SHAPE"),
    (dict(ot_ld=1), "ND_ERR_SHAPE"), (dict(w_ld=63), "ND_ERR_SHAPE"), (dict(wo_ld=31), "ND_ERR_SHAPE"),
    (dict(wo=ctypes.c_void_p(0x100100)), "ND_ERR_INVALID_ARG"), (dict(kept=None), "ND_ERR_INVALID_ARG"),
    (dict(D=8), "ND_ERR_UNSUPPORTED"), (dict(B=0, lens=None), "ND_OK"),
])
def test_paged_evict_checks(kw, status):
    m, lib = _lib()
    assert evict(lib, **kw) == getattr(m, status), lib.nd_last_error_string()


def logits(lib, **kw):
    a = dict(x=ctypes.c_void_p(0x100000), dt=0, ld=100, rows=2, V=100, hist=P, h_ld=8, n=8,
             h_lens=None, rep=P, pres=None, freq=None, ids=None, bias=None, nb=0, mask=None,
             m_ld=0, out=ctypes.c_void_p(0x200000), odt=0, o_ld=100, idx=None)
    a.update(kw)
    return lib.nd_logits_penalty(None, a["x"], a["dt"], a["ld"], a["rows"], a["V"], a["hist"],
                                 a["h_ld"], a["n"], a["h_lens"], a["rep"], a["pres"], a["freq"],
                                 a["ids"], a["bias"], a["nb"], a["mask"], a["m_ld"], a["out"],
                                 a["odt"], a["o_ld"], a["idx"])


@pytest.mark.parametrize("kw, status", [
    (dict(dt=2), "ND_ERR_UNSUPPORTED"), (dict(ld=99), "ND_ERR_SHAPE"), (dict(o_ld=99), "ND_ERR_SHAPE"),
    (dict(h_ld=7), "ND_ERR_SHAPE"), (dict(hist=None), "ND_ERR_INVALID_ARG"),
    (dict(ids=P), "ND_ERR_INVALID_ARG"), (dict(mask=P, m_ld=3), "ND_ERR_SHAPE"),
    (dict(x=None), "ND_ERR_INVALID_ARG"), (dict(n=-1), "ND_ERR_INVALID_ARG"),
    (dict(V=0, ld=0, o_ld=0), "ND_ERR_SHAPE"), (dict(out=ctypes.c_void_p(0x100000), odt=1), "ND_ERR_INVALID_ARG"),
    (dict(out=ctypes.c_void_p(0x100010)), "ND_ERR_INVALID_ARG"),
    (dict(x=ctypes.c_void_p(0x100002)), "ND_ERR_ALIGNMENT"), (dict(rows=0, x=None, out=None), "ND_OK"),
])
def test_logits_penalty_checks(kw, status):
    m, lib = _lib()
    assert logits(lib, **kw) == getattr(m, status), lib.nd_last_error_string()


def test_python_front_end_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    from neurodsl_b200 import ops
    bf = torch.zeros((1, 1, 4, 64), dtype=torch.bfloat16)
    i32 = torch.zeros((1, 2), dtype=torch.int32)
    with pytest.raises(TypeError):
        ops.window_attn_fwd(bf, bf, bf, 4)
    with pytest.raises(TypeError):
        ops.paged_decode_attn(bf[0], bf, bf, i32, i32[:, 0])
    with pytest.raises(TypeError):
        ops.paged_kv_store(bf[0, 0], 0, 0, bf, bf, i32, 1, 4)
    with pytest.raises(TypeError):
        ops.paged_kv_evict(bf, bf, i32, i32[:, 0], torch.zeros(1, 1, 8), i32, 4)
    with pytest.raises(TypeError):
        ops.logits_penalty(torch.zeros(1, 10))


def test_the_calls_extension_leaves_everything_uncommon_to_the_checks():
    """It is built and loads; it answers None, never a status, to tensors that
    are not on a GPU, to things that are no tensors and to a wrong count."""
    torch = pytest.importorskip("torch")
    lib, _ = _lib()
    calls = lib.load_calls()
    assert calls, "python -m neurodsl_b200.build makes it"
    host = torch.zeros(2, 3)
    for name, n in [("window_attn_fwd", 9), ("paged_decode_attn", 14), ("paged_kv_store", 10),
                    ("paged_kv_evict", 12), ("logits_penalty", 11)]:
        fn = getattr(calls, name)
        for value in (None, host, "x", 3, 2**70, 1.5, object()):
            assert fn(*[value] * n) is None
            assert fn(host, *[value] * (n - 1)) is None
        assert fn() is None and fn(*[host] * (n + 1)) is None
    with pytest.raises(TypeError):
        calls.bind(1, 2)


def test_paged_evict_refuses_lengths_that_overlap():
    """Lengths written over others that are still to be read; the same lengths in
    place are fine (here: as far as the missing device)."""
    m, lib = _lib()
    at = lambda i: ctypes.c_void_p(0x300000 + 4 * i)  # noqa: E731
    for i in (1, -1):
        assert evict(lib, lens=at(0), new_lens=at(i)) == m.ND_ERR_INVALID_ARG
        assert b"new_lens" in lib.nd_last_error_string()
    for i in (0, 2, -2):
        evict(lib, lens=at(0), new_lens=at(i), D=64, kept=None)      # refused for kept alone
        assert b"new_lens" not in lib.nd_last_error_string()


def test_ops_imports_where_torch_was_built_without_cuda():
    """As before the serving operators: only the calls need a GPU."""
    import os
    import subprocess
    import sys
    pytest.importorskip("torch")
    program = """
import torch
for name in dir(torch._C):
    if name.startswith("_cuda_"):
        delattr(torch._C, name)
import neurodsl_b200.ops as ops, neurodsl_b200.graph
try:
    ops.logits_penalty(torch.zeros(1, 4))
except TypeError as e:
    print("refused:", e)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", program], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert "refused: logits must be a CUDA tensor" in r.stdout


def test_the_calls_extension_is_of_this_interpreter_and_torch(monkeypatch, tmp_path):
    """One built for another torch is neither taken for fresh nor loaded; the calls
    then go through ctypes."""
    import sys
    torch = pytest.importorskip("torch")
    from neurodsl_b200 import build
    m, lib = _lib()
    assert m.load_calls()
    mine = m.calls_path()
    assert build.build_calls() == mine
    monkeypatch.setattr(torch, "__version__", "1.13.0")
    assert m.calls_path() != mine
    monkeypatch.setattr(m, "calls", None)
    assert m.load_calls() is False
    made = []
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: made.append(cmd) or type("R", (), dict(returncode=0)))
    assert build.build_calls() == m.calls_path()
    assert len(made) == 1 and m.calls_path() in made[0]
    monkeypatch.setattr(torch, "__version__", mine.split("torch-")[1][:-3])
    monkeypatch.setattr(sys.implementation, "cache_tag", "cpython-27")
    assert m.calls_path() != mine


def test_a_build_without_a_compiler_or_headers(monkeypatch):
    """The library alone is enough: a warning, no error."""
    pytest.importorskip("torch")
    import torch.utils.cpp_extension as ext
    from neurodsl_b200 import build
    with monkeypatch.context() as c:
        c.setenv("CXX", "/nowhere/c++")
        with pytest.warns(UserWarning, match="no C.. compiler"):
            assert build.build_calls(force=True) is None
    monkeypatch.setattr(ext, "include_paths", lambda *a, **k: ["/nowhere"])
    with pytest.warns(UserWarning, match="python_variable.h"):
        assert build.build_calls(force=True) is None
