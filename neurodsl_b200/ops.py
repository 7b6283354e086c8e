"""Torch-tensor front end of the C ABI: one function per hot-path kernel.

Tensors are CUDA tensors (torch is used only to own device memory and to
name the current stream); each call validates dtype/shape/contiguity here
and then calls the corresponding nd_* entry point, which validates again.
Outputs are allocated here when the caller passes none.
"""
from __future__ import annotations

import ctypes
import math
import operator

import torch

from . import _lib
from ._lib import check

_DT = {torch.float32: _lib.ND_F32, torch.bfloat16: _lib.ND_BF16}
ACT = {"none": _lib.ND_ACT_NONE, "sigmoid": _lib.ND_ACT_GELU_SIGMOID,
       "tanh": _lib.ND_ACT_GELU_TANH, "erf": _lib.ND_ACT_GELU_ERF}


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(stream=None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _need(t, name, dtype=None, dims=None, contiguous=True):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if dims is not None and t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dims, got shape {tuple(t.shape)}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _row_strides(t, name):
    """{row, head, batch} element strides of a [B][H][S][64] view, D contiguous."""
    if t.stride(3) != 1:
        raise ValueError(f"{name}: the 64 head dims of a row must be contiguous")
    return (ctypes.c_int64 * 3)(t.stride(2), t.stride(1), t.stride(0))


def flash_attn_fwd(Q, K, V, causal=True, scale=None, out=None, out_dtype=torch.bfloat16,
                   lse=None, row_max=None, stream=None):
    """O = softmax(Q·Kᵀ·scale [causal]) · V for [B][H][S][64] bf16 tensors.

    Mirrors flash_attn_fwd!(dev, out, Q, K, V, d_head; causal)
    (src/flash_attention.jl:113-134); returns (O, lse, row_max) like the
    reference's (out, l, m).  Q, K, V and `out` may be strided views, e.g.
    token-major slices of an (S, 3·H·64) QKV projection viewed as
    [B][H][S][64]; they are then read and written in place
    (nd_flash_attn_fwd_strided) instead of being copied per head.
    """
    for n, t in (("Q", Q), ("K", K), ("V", V)):
        _need(t, n, torch.bfloat16, 4, contiguous=False)
    B, H, Sq, D = Q.shape
    Sk = K.shape[2]
    if K.shape != (B, H, Sk, D) or V.shape != K.shape:
        raise ValueError(f"shape mismatch Q{tuple(Q.shape)} K{tuple(K.shape)} V{tuple(V.shape)}")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty((B, H, Sq, D), dtype=out_dtype, device=Q.device)
    _need(out, "out", None, 4, contiguous=False)
    if tuple(out.shape) != (B, H, Sq, D):
        raise ValueError(f"out{tuple(out.shape)} != {(B, H, Sq, D)}")
    if lse is None:
        lse = torch.empty((B, H, Sq), dtype=torch.float32, device=Q.device)
    if row_max is None:
        row_max = torch.empty((B, H, Sq), dtype=torch.float32, device=Q.device)
    lib = _lib.load()
    if all(t.is_contiguous() for t in (Q, K, V, out)):
        check(lib.nd_flash_attn_fwd(_stream(stream), _ptr(Q), _ptr(K), _ptr(V), _ptr(out),
                                    _DT[out.dtype], _ptr(lse), _ptr(row_max), B, H, Sq, Sk,
                                    D, float(scale), int(bool(causal))))
    else:
        check(lib.nd_flash_attn_fwd_strided(
            _stream(stream), _ptr(Q), _row_strides(Q, "Q"), _ptr(K), _row_strides(K, "K"),
            _ptr(V), _row_strides(V, "V"), _ptr(out), _row_strides(out, "out"), _DT[out.dtype],
            _ptr(lse), _ptr(row_max), B, H, Sq, Sk, D, float(scale), int(bool(causal))))
    return out, lse, row_max


def kv_decode_workspace_size(B, H, L, D=64):
    n = ctypes.c_size_t(0)
    check(_lib.load().nd_kv_decode_workspace_size(B, H, L, D, ctypes.byref(n)))
    return n.value


def kv_decode_attn(q, k_cache, v_cache, L, k_new=None, v_new=None, scale=None, out=None,
                   out_dtype=torch.bfloat16, lse=None, workspace=None, want_lse=True,
                   stream=None):
    """Single-token decode over keys [0, L) of [B][H][L_max][64] bf16 caches.

    With k_new/v_new the token at L-1 is appended to the caches in the same
    pass.  Returns (out [B][H][64], lse [B][H]).
    """
    _need(q, "q", torch.bfloat16, 3)
    _need(k_cache, "k_cache", torch.bfloat16, 4)
    _need(v_cache, "v_cache", torch.bfloat16, 4)
    B, H, D = q.shape
    L_max = k_cache.shape[2]
    if k_cache.shape != (B, H, L_max, D) or v_cache.shape != k_cache.shape:
        raise ValueError("cache shape mismatch")
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new go together")
    if k_new is not None:
        _need(k_new, "k_new", torch.bfloat16, 3)
        _need(v_new, "v_new", torch.bfloat16, 3)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty((B, H, D), dtype=out_dtype, device=q.device)
    if lse is None and want_lse:
        lse = torch.empty((B, H), dtype=torch.float32, device=q.device)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    check(_lib.load().nd_kv_decode_attn(_stream(stream), _ptr(q), _ptr(k_new), _ptr(v_new),
                                        _ptr(k_cache), _ptr(v_cache), _ptr(out), _DT[out.dtype],
                                        _ptr(lse), B, H, int(L), L_max, D, float(scale),
                                        _ptr(workspace), ws_bytes))
    return out, lse


def kv_decode_attn_qkv(qkv, k_cache, v_cache, L, scale=None, out=None, out_dtype=torch.bfloat16,
                       lse=None, workspace=None, want_lse=False, stream=None):
    """Decode attention from a fused QKV projection qkv [B][3*H*64] (bf16,
    unit column stride; rows may be padded): q, k_new and v_new are its three
    column blocks, and k_new / v_new are appended at position L-1.
    Returns (out [B][H][64], lse [B][H] or None)."""
    if not isinstance(qkv, torch.Tensor) or qkv.dtype != torch.bfloat16 or qkv.dim() != 2:
        raise ValueError("qkv must be a 2-D bf16 tensor")
    if not qkv.is_cuda or qkv.stride(1) != 1:
        raise ValueError("qkv must be a CUDA tensor with unit column stride")
    _need(k_cache, "k_cache", torch.bfloat16, 4)
    _need(v_cache, "v_cache", torch.bfloat16, 4)
    B = qkv.shape[0]
    _, H, L_max, D = k_cache.shape
    if k_cache.shape[0] != B or v_cache.shape != k_cache.shape or qkv.shape[1] != 3 * H * D:
        raise ValueError("qkv / cache shape mismatch")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if out is None:
        out = torch.empty((B, H, D), dtype=out_dtype, device=qkv.device)
    if lse is None and want_lse:
        lse = torch.empty((B, H), dtype=torch.float32, device=qkv.device)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    check(_lib.load().nd_kv_decode_attn_qkv(_stream(stream), _ptr(qkv), qkv.stride(0),
                                            _ptr(k_cache), _ptr(v_cache), _ptr(out),
                                            _DT[out.dtype], _ptr(lse), B, H, int(L), L_max, D,
                                            float(scale), _ptr(workspace), ws_bytes))
    return out, lse


def set_pdl(enable):
    """Programmatic dependent launch for this thread's decode-step kernels
    (nd_set_pdl); returns the previous setting."""
    prev = ctypes.c_int(0)
    check(_lib.load().nd_set_pdl(1 if enable else 0, ctypes.byref(prev)))
    return bool(prev.value)


class pdl:
    """Context manager: launches inside run with programmatic dependent
    launch on (or off), restoring the previous setting on exit."""

    def __init__(self, enable=True):
        self.enable = enable

    def __enter__(self):
        self.prev = set_pdl(self.enable)
        return self

    def __exit__(self, *exc):
        set_pdl(self.prev)
        return False


def set_sm_limit(sms):
    """Cap the SMs this thread's persistent GEMM / prefill-attention launches
    occupy (nd_set_sm_limit; 0 = all); returns the previous setting."""
    prev = ctypes.c_int(0)
    check(_lib.load().nd_set_sm_limit(int(sms), ctypes.byref(prev)))
    return prev.value


class sm_limit:
    """Context manager: launches inside leave all but `sms` SMs to other
    streams' kernels (0 = no cap), restoring the previous cap on exit."""

    def __init__(self, sms):
        self.sms = sms

    def __enter__(self):
        self.prev = set_sm_limit(self.sms)
        return self

    def __exit__(self, *exc):
        set_sm_limit(self.prev)
        return False


def kv_append(k_new, v_new, k_cache, v_cache, pos, stream=None):
    _need(k_new, "k_new", torch.bfloat16, 3)
    _need(v_new, "v_new", torch.bfloat16, 3)
    B, H, D = k_new.shape
    L_max = k_cache.shape[2]
    check(_lib.load().nd_kv_append(_stream(stream), _ptr(k_new), _ptr(v_new), _ptr(k_cache),
                                   _ptr(v_cache), B, H, int(pos), L_max, D))


def linear(A, W, bias=None, residual=None, act="none", out=None, out_dtype=torch.bfloat16,
           stream=None):
    """Y = act(A·Wᵀ + bias) + residual with A [M][K], W [N][K] bf16.

    :linear (src/dispatch.jl:363-384) / fused_linear_gelu
    (notebook/compiler.ipynb cell 15) with the GELU variant `act`.
    """
    _need(A, "A", torch.bfloat16, 2)
    _need(W, "W", torch.bfloat16, 2)
    M, K = A.shape
    N = W.shape[0]
    if W.shape[1] != K:
        raise ValueError(f"A{tuple(A.shape)} and W{tuple(W.shape)} disagree on K")
    if bias is not None:
        _need(bias, "bias", torch.float32)
        if bias.numel() != N:
            raise ValueError("bias length != N")
    rdt = _lib.ND_F32
    if residual is not None:
        _need(residual, "residual", None, 2)
        if tuple(residual.shape) != (M, N):
            raise ValueError("residual shape != (M, N)")
        rdt = _DT[residual.dtype]
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=A.device)
    _need(out, "out", None, 2)
    check(_lib.load().nd_gemm_bias_act(_stream(stream), _ptr(A), _ptr(W), _ptr(bias),
                                       _ptr(residual), rdt, _ptr(out), _DT[out.dtype], M, N, K,
                                       ACT[act] if isinstance(act, str) else int(act)))
    return out


def linear_qkv_cache(A, W, bias, out, k_cache, v_cache, B, S, pos0=0, stream=None):
    """The QKV projection out = A·Wᵀ + bias (A [B*S][K], W [3*H*64][K], bf16
    out) that also writes its K and V column blocks into the head-major
    caches [B][H][L_max][64] at positions pos0.. (nd_gemm_qkv_cache)."""
    _need(A, "A", torch.bfloat16, 2)
    _need(W, "W", torch.bfloat16, 2)
    _need(out, "out", torch.bfloat16, 2)
    _need(k_cache, "k_cache", torch.bfloat16, 4)
    _need(v_cache, "v_cache", torch.bfloat16, 4)
    M, K = A.shape
    _, H, L_max, D = k_cache.shape
    if D != 64 or W.shape != (3 * H * 64, K) or tuple(out.shape) != (M, 3 * H * 64):
        raise ValueError("QKV projection / cache shape mismatch")
    if v_cache.shape != k_cache.shape or k_cache.shape[0] != B:
        raise ValueError("cache shape mismatch")
    if bias is not None:
        _need(bias, "bias", torch.float32)
    check(_lib.load().nd_gemm_qkv_cache(_stream(stream), _ptr(A), _ptr(W), _ptr(bias), _ptr(out),
                                        M, K, _ptr(k_cache), _ptr(v_cache), int(B), int(S), H,
                                        L_max, int(pos0)))
    return out


def linear_qkv_cache_peers(A, W, bias, out, k_caches, v_caches, H, L_max, B, b0, S, pos0=0,
                           stream=None):
    """The full-head QKV projection of this rank's B prompts (sequences b0..)
    writing the K/V columns of head h into the cache of rank h // H
    (nd_gemm_qkv_cache_peers); k_caches / v_caches: every rank's cache base
    pointer (ints, [..][H][L_max][64] bf16), this rank's own included."""
    _need(A, "A", torch.bfloat16, 2)
    _need(W, "W", torch.bfloat16, 2)
    _need(out, "out", torch.bfloat16, 2)
    _need(bias, "bias", torch.float32, 1)
    tp = len(k_caches)
    M, K = A.shape
    if W.shape != (3 * tp * H * 64, K) or tuple(out.shape) != (M, 3 * tp * H * 64) or M != B * S:
        raise ValueError("QKV projection / cache shape mismatch")
    kc = (ctypes.c_void_p * tp)(*k_caches)
    vc = (ctypes.c_void_p * tp)(*v_caches)
    check(_lib.load().nd_gemm_qkv_cache_peers(_stream(stream), _ptr(A), _ptr(W), _ptr(bias),
                                              _ptr(out), M, K, kc, vc, tp, int(B), int(b0),
                                              int(S), int(H), int(L_max), int(pos0)))
    return out


def ln_linear(x, W, p=None, p_bias=None, gamma=None, beta=None, eps=1e-5, s_out=None, bias=None,
              act="none", out=None, out_dtype=torch.bfloat16, stream=None):
    """Y = act(LayerNorm(x + p + p_bias)·Wᵀ + bias) for at most 32 rows, with
    the residual sum s = bf16(x + p + p_bias) written to s_out if given
    (nd_ln_gemm: residual :add + :layernorm + :linear in one launch)."""
    _need(x, "x", torch.bfloat16, 2)
    _need(W, "W", torch.bfloat16, 2)
    M, K = x.shape
    N = W.shape[0]
    if W.shape[1] != K:
        raise ValueError(f"x{tuple(x.shape)} and W{tuple(W.shape)} disagree on K")
    for name, t in (("p", p), ("s_out", s_out)):
        if t is not None:
            _need(t, name, torch.bfloat16, 2)
            if tuple(t.shape) != (M, K):
                raise ValueError(f"{name} shape != x shape")
    for name, t, n in (("p_bias", p_bias, K), ("gamma", gamma, K), ("beta", beta, K),
                       ("bias", bias, N)):
        if t is not None:
            _need(t, name, torch.float32)
            if t.numel() != n:
                raise ValueError(f"{name} length != {n}")
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=x.device)
    _need(out, "out", None, 2)
    check(_lib.load().nd_ln_gemm(_stream(stream), _ptr(x), _ptr(p), _ptr(p_bias), _ptr(gamma),
                                 _ptr(beta), float(eps), _ptr(s_out), _ptr(W), _ptr(bias),
                                 _ptr(out), _DT[out.dtype], M, N, K,
                                 ACT[act] if isinstance(act, str) else int(act)))
    return out


def gelu(x, act="sigmoid", out=None, stream=None):
    """Elementwise GELU of a float32 tensor (nd_gelu, the unfused :gelu op)."""
    _need(x, "x", torch.float32)
    if out is None:
        out = torch.empty_like(x)
    _need(out, "out", torch.float32)
    check(_lib.load().nd_gelu(_stream(stream), _ptr(x), _ptr(out), x.numel(),
                              ACT[act] if isinstance(act, str) else int(act)))
    return out


def scale_mask(scores, d_head, out=None, stream=None):
    """scores / sqrt(d_head) with the causal mask (-Inf above the diagonal) of
    one float32 [rows][cols] block (nd_scale_mask, the :scale_mask op)."""
    _need(scores, "scores", torch.float32, 2)
    if out is None:
        out = torch.empty_like(scores)
    _need(out, "out", torch.float32, 2)
    check(_lib.load().nd_scale_mask(_stream(stream), _ptr(scores), _ptr(out), scores.shape[0],
                                    scores.shape[1], int(d_head)))
    return out


def add(a, b, out=None, stream=None):
    """a + b for float32 tensors (nd_add, the :add op): b of a's shape; a
    vector of one value per column, else per row, of a 2-D a (the
    reference's vector cases, columns preferred); or, as its general
    broadcast does, a (1, cols) row, a (rows, 1) column or a single value."""
    _need(a, "a", torch.float32)
    _need(b, "b", torch.float32)
    rows, cols = (a.shape[0], a.shape[1]) if a.dim() == 2 else (1, a.numel())
    if tuple(b.shape) == tuple(a.shape):
        mode = 0
    elif a.dim() == 2 and b.dim() == 1 and b.numel() == cols:
        mode = 1
    elif a.dim() == 2 and b.dim() == 1 and b.numel() == rows:
        mode = 2
    elif a.dim() == 2 and b.dim() == 2 and tuple(b.shape) == (1, cols):
        mode = 1
    elif a.dim() == 2 and b.dim() == 2 and tuple(b.shape) == (rows, 1):
        mode = 2
    elif b.numel() == 1 and b.dim() <= a.dim():
        mode = 3
    else:
        raise ValueError(f"add: shapes {tuple(a.shape)} and {tuple(b.shape)} do not broadcast")
    if out is None:
        out = torch.empty_like(a)
    _need(out, "out", torch.float32)
    check(_lib.load().nd_add(_stream(stream), _ptr(a), _ptr(b), _ptr(out), rows, cols, mode))
    return out


def softmax(x, out=None, stream=None):
    """Row softmax of a float32 [rows][cols] matrix (nd_softmax, the :softmax op)."""
    _need(x, "x", torch.float32, 2)
    if out is None:
        out = torch.empty_like(x)
    _need(out, "out", torch.float32, 2)
    check(_lib.load().nd_softmax(_stream(stream), _ptr(x), _ptr(out), x.shape[0], x.shape[1]))
    return out


def layernorm(x, gamma=None, beta=None, eps=1e-5, out=None, out_dtype=None, mean=None,
              rstd=None, stats=True, stream=None):
    """Row LayerNorm of x [rows][d]; returns (y, mean, rstd).  With
    stats=False and no mean/rstd buffers the statistics are not written
    (mean and rstd come back as None)."""
    _need(x, "x", None, 2)
    rows, d = x.shape
    if out is None:
        out = torch.empty((rows, d), dtype=out_dtype or x.dtype, device=x.device)
    if mean is None and stats:
        mean = torch.empty(rows, dtype=torch.float32, device=x.device)
    if rstd is None and stats:
        rstd = torch.empty(rows, dtype=torch.float32, device=x.device)
    for n, t in (("gamma", gamma), ("beta", beta)):
        if t is not None:
            _need(t, n, torch.float32)
    check(_lib.load().nd_layernorm(_stream(stream), _ptr(x), _DT[x.dtype], _ptr(gamma),
                                   _ptr(beta), _ptr(out), _DT[out.dtype], _ptr(mean), _ptr(rstd),
                                   rows, d, float(eps)))
    return out, mean, rstd


def convert_2d(src, rows, cols, src_col_major, dst_dtype, out=None, stream=None):
    """Column-major (Julia) or row-major 2-D matrix -> row-major [rows][cols]."""
    _need(src, "src")
    if src.numel() != rows * cols:
        raise ValueError("src size != rows*cols")
    if out is None:
        out = torch.empty((rows, cols), dtype=dst_dtype, device=src.device)
    check(_lib.load().nd_convert_2d(_stream(stream), _ptr(src), _DT[src.dtype],
                                    int(bool(src_col_major)), _ptr(out), _DT[out.dtype], rows,
                                    cols))
    return out


def convert_2d_padded(src, rows, cols, src_col_major, dst_dtype, ld_dst, out=None, stream=None):
    """convert_2d into rows of ld_dst >= cols elements, the columns past cols
    zero (nd_convert_2d_padded): [rows][ld_dst]."""
    _need(src, "src")
    if src.numel() != rows * cols:
        raise ValueError("src size != rows*cols")
    if out is None:
        out = torch.empty((rows, ld_dst), dtype=dst_dtype, device=src.device)
    if tuple(out.shape) != (rows, ld_dst) or not out.is_contiguous():
        raise ValueError("out must be a contiguous [rows][ld_dst] matrix")
    check(_lib.load().nd_convert_2d_padded(_stream(stream), _ptr(src), _DT[src.dtype],
                                           int(bool(src_col_major)), _ptr(out), _DT[out.dtype],
                                           rows, cols, ld_dst))
    return out


_IDX_DT = {torch.float32: _lib.ND_F32, torch.int32: _lib.ND_I32, torch.int64: _lib.ND_I64}


def gather_rows(table, idx, index_base=1, out=None, stream=None):
    """out[i] = table[idx[i] - index_base] on the device (nd_gather_rows: the
    :embedding op).  table [vocab][d] fp32 or bf16 with unit column stride;
    idx any shape of float32 / int32 / int64 indices on the device.  A bad
    index gives a zero row and sets the device error word (device_error()),
    without a host synchronisation."""
    if table.dim() != 2 or table.stride(1) != 1:
        raise ValueError("table must be 2-D with contiguous rows")
    if table.dtype not in _DT:
        raise ValueError(f"table dtype {table.dtype} not supported")
    if idx.dtype not in _IDX_DT:
        raise ValueError(f"index dtype {idx.dtype} not supported")
    if idx.device != table.device:
        raise ValueError("indices and table must be on the same device")
    idx = idx.reshape(-1).contiguous()
    n = idx.numel()
    vocab, d = table.shape
    if out is None:
        out = torch.empty((n, d), dtype=table.dtype, device=table.device)
    if out.dim() != 2 or tuple(out.shape) != (n, d) or out.stride(1) != 1 or out.dtype != table.dtype:
        raise ValueError("out must be an [n][d] matrix of the table's dtype with contiguous rows")
    check(_lib.load().nd_gather_rows(_stream(stream), _ptr(table), _DT[table.dtype],
                                     table.stride(0), vocab, _ptr(idx), _IDX_DT[idx.dtype],
                                     int(index_base), n, d, _ptr(out), out.stride(0)))
    return out


def copy_2d(src, dst, stream=None):
    """dst[:, :] = src[:, :] for 2-D views with unit column strides
    (nd_copy_2d: the :slice_cols, :hcat_heads and :identity copies)."""
    for name, t in (("src", src), ("dst", dst)):
        if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
            raise ValueError(f"{name} must be 2-D with contiguous rows")
    if tuple(src.shape) != tuple(dst.shape) or src.dtype != dst.dtype:
        raise ValueError("src and dst differ in shape or dtype")
    rows, cols = src.shape
    ld = lambda t: t.stride(0) if rows > 1 else cols
    check(_lib.load().nd_copy_2d(_stream(stream), _ptr(src), ld(src), _ptr(dst), ld(dst), rows,
                                 cols, src.element_size()))
    return dst


def copy_2d_batched(src, dst, stream=None):
    """dst[b, :, :] = src[b, :, :] for 3-D views whose rows are contiguous
    (nd_copy_2d_batched: any batch and row strides)."""
    for name, t in (("src", src), ("dst", dst)):
        if not t.is_cuda or t.dim() != 3 or (t.shape[2] > 1 and t.stride(2) != 1):
            raise ValueError(f"{name} must be a 3-D CUDA view with contiguous rows")
    if tuple(src.shape) != tuple(dst.shape) or src.dtype != dst.dtype:
        raise ValueError("src and dst differ in shape or dtype")
    batch, rows, cols = src.shape
    check(_lib.load().nd_copy_2d_batched(_stream(stream), _ptr(src), src.stride(1), src.stride(0),
                                         _ptr(dst), dst.stride(1), dst.stride(0), batch, rows,
                                         cols, src.element_size()))
    return dst


def device_error():
    """Read and clear the device error word (non-zero after a timed-out wait)."""
    c = ctypes.c_int(0)
    check(_lib.load().nd_device_error(ctypes.byref(c)))
    return c.value


def embed(ids, wte, wpe=None, pos=None, out=None, stream=None):
    """y[t] = wte[ids[t]] + wpe[pos[t]] (bf16 [T][d]); ids/pos int32 [T]."""
    _need(ids, "ids", torch.int32, 1)
    _need(wte, "wte", torch.bfloat16, 2)
    T = ids.numel()
    vocab, d = wte.shape
    n_pos = 0
    if pos is not None:
        _need(pos, "pos", torch.int32, 1)
        _need(wpe, "wpe", torch.bfloat16, 2)
        n_pos = wpe.shape[0]
    if out is None:
        out = torch.empty((T, d), dtype=torch.bfloat16, device=wte.device)
    _need(out, "out", torch.bfloat16, 2)
    check(_lib.load().nd_embed(_stream(stream), _ptr(ids), _ptr(pos), _ptr(wte), _ptr(wpe),
                               _ptr(out), T, d, vocab, n_pos))
    return out


def argmax(logits, idx=None, val=None, stream=None):
    """First index of the largest value of each row of logits [rows][V]."""
    _need(logits, "logits", None, 2, contiguous=False)
    if logits.stride(1) != 1:
        raise ValueError("logits rows must be contiguous")
    rows, V = logits.shape
    if idx is None:
        idx = torch.empty(rows, dtype=torch.int32, device=logits.device)
    check(_lib.load().nd_argmax(_stream(stream), _ptr(logits), _DT[logits.dtype],
                                logits.stride(0), rows, V, _ptr(idx), _ptr(val)))
    return idx


def kv_store(src, k_col, v_col, k_cache, v_cache, B, S, pos0=0, stream=None):
    """K/V rows of a [B·S][ld] bf16 projection into [B][H][L_max][64] caches."""
    _need(src, "src", torch.bfloat16, 2, contiguous=False)
    if src.stride(1) != 1:
        raise ValueError("src rows must be contiguous")
    _need(k_cache, "k_cache", torch.bfloat16, 4)
    _need(v_cache, "v_cache", torch.bfloat16, 4)
    _, H, L_max, D = k_cache.shape
    check(_lib.load().nd_kv_store(_stream(stream), _ptr(src), src.stride(0), k_col, v_col,
                                  _ptr(k_cache), _ptr(v_cache), B, S, H, L_max, pos0, D))


def add_layernorm(x, p, bias=None, gamma=None, beta=None, eps=1e-5, s_out=None, out=None,
                  stream=None):
    """s = x + p (+ bias) (bf16, s_out may be x), y = LayerNorm(s); returns (s, y)."""
    _need(x, "x", torch.bfloat16, 2)
    _need(p, "p", None, 2)
    rows, d = x.shape
    if s_out is None:
        s_out = torch.empty_like(x)
    if out is None:
        out = torch.empty_like(x)
    check(_lib.load().nd_add_layernorm(_stream(stream), _ptr(x), _ptr(p), _DT[p.dtype],
                                       _ptr(bias), _ptr(gamma), _ptr(beta), _ptr(s_out),
                                       _ptr(out), rows, d, float(eps)))
    return s_out, out


# ---- sliding window, paged cache and logits penalties -------------------------
# A serving step makes these calls once a layer, so their checks are written to
# cost little: plain attribute reads, one device number for all tensors.
_BF16, _F32, _INT32 = torch.bfloat16, torch.float32, torch.int32
_I64x3 = ctypes.c_int64 * 3
_INT_MAX = 2**31 - 1
# the current device's number, a device's current stream as an int (a torch built
# without CUDA has neither, and no tensor that a call would take)
_cuda_device = getattr(torch._C, "_cuda_getDevice", None)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _device_of(t, name):
    """The device number of a call's first tensor."""
    dev = t.get_device() if isinstance(t, torch.Tensor) else -1
    if dev < 0:
        raise TypeError(f"{name} must be a CUDA tensor")
    return dev


def _tensor(t, name, dtype, dims, dev, contiguous=True):
    """Checks one tensor (dtype None: float32 or bfloat16; dims None: any)."""
    if (isinstance(t, torch.Tensor) and t.get_device() == dev and t.dtype is dtype
            and (dims is None or t.dim() == dims) and (not contiguous or t.is_contiguous())):
        return
    d = t.get_device() if isinstance(t, torch.Tensor) else -1
    if d < 0:
        raise TypeError(f"{name} must be a CUDA tensor")
    if d != dev:
        raise ValueError(f"{name} is on cuda:{d}, the call's first tensor on cuda:{dev}")
    if dtype is None:
        if t.dtype not in _DT:
            raise ValueError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    elif t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if dims is not None and t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dims, got shape {tuple(t.shape)}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _vector(t, name, dtype, n, dev):
    _tensor(t, name, dtype, None, dev)
    if t.numel() != n:
        raise ValueError(f"{name} must have {n} values, got {t.numel()}")


def _matrix(t, name, dtype, rows, dev):
    """Checks a [rows][cols] matrix with contiguous rows; returns (cols, row stride)."""
    _tensor(t, name, dtype, 2, dev, contiguous=False)
    r, cols = t.shape
    if r != rows or (cols > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} must be [{rows}][cols] with contiguous rows, got {tuple(t.shape)}")
    ld = t.stride(0) if r > 1 else cols
    if ld < cols:
        raise ValueError(f"{name} rows overlap")
    return cols, ld


def _stream_of(dev, stream):
    """The raw stream of a call: the caller's, which must be one of the
    tensors' device, or that device's current one."""
    if stream is None:
        return _raw_stream(dev)
    if stream.device.index != dev:
        raise ValueError(f"stream is on {stream.device}, the tensors on cuda:{dev}")
    return stream.cuda_stream


def _call(fn, dev, *args):
    """fn(*args) with the tensors' device current."""
    if _cuda_device() == dev:
        rc = fn(*args)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args)
    if rc:
        check(rc)


def _quick(name, *args):
    """The call as the extension makes it (csrc/py_calls.cpp), where its
    arguments are the common kind; whether it was made.  Otherwise the caller's
    own checks follow, which refuse the call or carry it out."""
    calls = _lib.calls
    if calls is None:
        calls = _lib.load_calls()
    rc = getattr(calls, name)(*args) if calls else None
    if rc:
        check(rc)
    return rc is not None


def _int(v):
    """v as a C int that is refused, or unlimited, just as v would be (the
    foreign-function call would drop the high bits)."""
    v = operator.index(v)
    return v if -_INT_MAX <= v <= _INT_MAX else (_INT_MAX if v > 0 else -1)


def _empty(shape, dtype, device, stream):
    """An output made for a call: on the call's stream, so that its memory is
    free of work that other streams still have with it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _addr(t):
    return None if t is None else t.data_ptr()


def _strides4(t, name):
    """{row, head, batch} strides of a [B][H][S][64] view, D contiguous."""
    b, h, s, d = t.stride()
    if d != 1:
        raise ValueError(f"{name}: the 64 head dims of a row must be contiguous")
    return _I64x3(s, h, b)


def window_attn_fwd(Q, K, V, window, sinks=0, scale=None, out=None, out_dtype=torch.bfloat16,
                    lse=None, row_max=None, stream=None):
    """Causal attention with a sliding window and sinks (nd_window_attn_fwd):
    Q [B][H][Sq][64], K and V [B][Hkv][Sk][64] bf16, H a multiple of Hkv,
    Sq <= Sk; the queries are the last Sq positions, and the query at position
    p sees key j when j <= p and (j > p - window or j < sinks).

    Returns (O, lse, row_max) like flash_attn_fwd, and like there Q, K, V and
    `out` may be strided views (a fused projection, a longer cache).  All Sk keys and
    values have to be finite, padding too: a masked value weighs 0, and 0 times an
    infinity is NaN."""
    if out is not None and stream is None and _quick(
            "window_attn_fwd", Q, K, V, window, sinks, scale, out, lse, row_max):
        return out, lse, row_max
    dev = _device_of(Q, "Q")
    _tensor(Q, "Q", _BF16, 4, dev, False)
    _tensor(K, "K", _BF16, 4, dev, False)
    _tensor(V, "V", _BF16, 4, dev, False)
    B, H, Sq, D = q_shape = Q.shape
    Bk, Hkv, Sk, Dk = k_shape = K.shape
    if Bk != B or Dk != D or V.shape != k_shape:
        raise ValueError(f"shape mismatch Q{tuple(Q.shape)} K{tuple(K.shape)} V{tuple(V.shape)}")
    if out is None:
        out = _empty(q_shape, out_dtype, Q.device, stream)
    _tensor(out, "out", None, 4, dev, False)
    if out.shape != q_shape:
        raise ValueError(f"out must be {tuple(q_shape)}, got {tuple(out.shape)}")
    if lse is None:
        lse = _empty((B, H, Sq), _F32, Q.device, stream)
    if row_max is None:
        row_max = _empty((B, H, Sq), _F32, Q.device, stream)
    _vector(lse, "lse", _F32, B * H * Sq, dev)
    _vector(row_max, "row_max", _F32, B * H * Sq, dev)
    _call(_lib.load().nd_window_attn_fwd, dev, _stream_of(dev, stream), Q.data_ptr(),
          _strides4(Q, "Q"), K.data_ptr(), _strides4(K, "K"), V.data_ptr(), _strides4(V, "V"),
          out.data_ptr(), _strides4(out, "out"), _DT[out.dtype], lse.data_ptr(),
          row_max.data_ptr(), B, H, Hkv, Sq, Sk, D, 1.0 / math.sqrt(D) if scale is None else scale,
          _int(window), _int(sinks))
    return out, lse, row_max


def _pool(k_pages, v_pages, dev):
    """Checks a pool; returns (n_pages, Hkv, page_size, D)."""
    _tensor(k_pages, "k_pages", _BF16, 4, dev)
    _tensor(v_pages, "v_pages", _BF16, 4, dev)
    shape = k_pages.shape
    if v_pages.shape != shape:
        raise ValueError("k_pages and v_pages differ in shape")
    return shape


def paged_decode_workspace_size(B, H, Hkv, max_len, weights=False, D=64):
    n = ctypes.c_size_t(0)
    check(_lib.load().nd_paged_decode_workspace_size(B, H, Hkv, int(max_len), D,
                                                     int(bool(weights)), ctypes.byref(n)))
    return n.value


def paged_decode_workspace(B, H, Hkv, max_len, weights=False, device=None):
    """A zero-filled workspace for paged_decode_attn calls of up to these
    sizes (max_len: pages a sequence times page_size; weights: for calls that
    accumulate them, 4 bytes more for every query head and key of the table).  Every call leaves it ready for the next; calls that may
    run at the same time, two captured graphs' among them, need one each."""
    n = paged_decode_workspace_size(B, H, Hkv, max_len, weights)
    return torch.zeros(n, dtype=torch.uint8, device=device if device is not None else "cuda")


def paged_decode_attn(q, k_pages, v_pages, block_table, lens, k_new=None, v_new=None, window=0,
                      sinks=0, scale=None, out=None, out_dtype=torch.bfloat16, lse=None,
                      want_lse=True, weights=None, workspace=None, stream=None):
    """Decode attention of one new token per sequence over a paged cache
    (nd_paged_decode_attn): q [B][H][64], pages [n_pages][Hkv][page_size][64]
    bf16, block_table [B][max_pages] and lens [B] int32 on the device.

    With k_new / v_new [B][Hkv][64] the token at lens - 1 is appended in the
    same pass.  window > 0 sees the last `window` keys and the first `sinks`.
    weights [B][Hkv][>= max_pages * page_size] fp32 gains every visible key's
    attention weight, summed over its group's query heads.  workspace: from
    paged_decode_workspace, kept by the caller from call to call; without one
    each call makes its own.  Returns (out [B][H][64], lse [B][H] or None)."""
    if (out is not None and stream is None and (lse is not None or not want_lse) and _quick(
            "paged_decode_attn", q, k_pages, v_pages, block_table, lens, k_new, v_new, window, sinks,
            scale, out, lse, weights, workspace)):
        return out, lse
    dev = _device_of(q, "q")
    _tensor(q, "q", _BF16, 3, dev)
    B, H, D = q_shape = q.shape
    n_pages, Hkv, page_size, Dk = _pool(k_pages, v_pages, dev)
    max_pages, table_ld = _matrix(block_table, "block_table", _INT32, B, dev)
    if Dk != D:
        raise ValueError(f"q has head_dim {D}, the pages {Dk}")
    _vector(lens, "lens", _INT32, B, dev)
    if (k_new is None) != (v_new is None):
        raise ValueError("k_new and v_new go together")
    if k_new is not None:
        _tensor(k_new, "k_new", _BF16, 3, dev)
        _tensor(v_new, "v_new", _BF16, 3, dev)
        if k_new.shape != (B, Hkv, D) or v_new.shape != (B, Hkv, D):
            raise ValueError(f"k_new and v_new must be {(B, Hkv, D)}")
    if out is None:
        out = _empty(q_shape, out_dtype, q.device, stream)
    _tensor(out, "out", None, 3, dev)
    if out.shape != q_shape:
        raise ValueError(f"out must be {tuple(q_shape)}, got {tuple(out.shape)}")
    if lse is None and want_lse:
        lse = _empty((B, H), _F32, q.device, stream)
    if lse is not None:
        _vector(lse, "lse", _F32, B * H, dev)
    weights_ld = 0
    if weights is not None:
        _tensor(weights, "weights", _F32, 3, dev)
        if weights.shape[:2] != (B, Hkv):
            raise ValueError(f"weights must be [{B}][{Hkv}][keys], got {tuple(weights.shape)}")
        weights_ld = weights.shape[2]
    if workspace is None:
        # made on the call's stream, so that its memory is reused only after the call
        with torch.cuda.stream(stream if stream is not None else torch.cuda.current_stream(dev)):
            workspace = paged_decode_workspace(B, H, Hkv, max_pages * page_size,
                                               weights is not None, device=q.device)
    else:
        _tensor(workspace, "workspace", workspace.dtype, None, dev)
    _call(_lib.load().nd_paged_decode_attn, dev, _stream_of(dev, stream), q.data_ptr(),
          _addr(k_new), _addr(v_new), k_pages.data_ptr(), v_pages.data_ptr(), n_pages, page_size,
          block_table.data_ptr(), table_ld, max_pages, lens.data_ptr(), out.data_ptr(),
          _DT[out.dtype], _addr(lse), _addr(weights), weights_ld, B, H, Hkv, D,
          _int(window), _int(sinks),
          1.0 / math.sqrt(D) if scale is None else scale, workspace.data_ptr(), workspace.nbytes)
    return out, lse


def paged_kv_store(src, k_col, v_col, k_pages, v_pages, block_table, B, S, pos0=0, lens=None,
                   stream=None):
    """K/V rows of a [B*S][ld] bf16 projection into a paged cache
    (nd_paged_kv_store): token (b, s) goes to position pos0 + s of sequence b.
    pos0: an int, or int32 [B] on the device; lens: int32 [B] tokens of each
    sequence, the rest being padding (None: all S)."""
    if stream is None and _quick("paged_kv_store", src, k_col, v_col, k_pages, v_pages, block_table,
                                 B, S, pos0, lens):
        return
    dev = _device_of(src, "src")
    cols, ld = _matrix(src, "src", _BF16, B * S, dev)
    n_pages, Hkv, page_size, D = _pool(k_pages, v_pages, dev)
    max_pages, table_ld = _matrix(block_table, "block_table", _INT32, B, dev)
    pos_dev = None
    if isinstance(pos0, torch.Tensor):
        _vector(pos0, "pos0", _INT32, B, dev)
        pos_dev, pos0 = pos0.data_ptr(), 0
    if lens is not None:
        _vector(lens, "lens", _INT32, B, dev)
    if max(k_col, v_col) + Hkv * D > cols:
        raise ValueError("k_col / v_col: the heads' columns do not fit src")
    _call(_lib.load().nd_paged_kv_store, dev, _stream_of(dev, stream), src.data_ptr(), ld,
          _int(k_col), _int(v_col), k_pages.data_ptr(), v_pages.data_ptr(), n_pages, page_size,
          block_table.data_ptr(), table_ld, max_pages, B, S, Hkv, _int(pos0), pos_dev,
          _addr(lens), D)


def paged_kv_evict(k_pages, v_pages, block_table, lens, weights, out_table, budget, sinks=0,
                   recent=0, weights_out=None, kept=None, new_lens=None, stream=None):
    """Cut every (sequence, kv head) of a paged cache to `budget` keys by
    accumulated attention weight (nd_paged_kv_evict): the first `sinks`, the
    last `recent` and the largest weights between stay, copied in order to
    out_table's pages, which must be none of the source pages.

    weights [B][Hkv][keys] fp32 as paged_decode_attn accumulates them.
    new_lens may be `lens` itself.

    Returns (kept [B][Hkv][budget] int32 positions, -1 past the last;
    new_lens [B]; weights_out [B][Hkv][keys], the kept keys' weights first,
    zeros behind them)."""
    if kept is not None and stream is None and _quick(
            "paged_kv_evict", k_pages, v_pages, block_table, lens, weights, out_table, budget, sinks,
            recent, weights_out, kept, new_lens):
        return kept, new_lens, weights_out
    dev = _device_of(k_pages, "k_pages")
    n_pages, Hkv, page_size, D = _pool(k_pages, v_pages, dev)
    _tensor(lens, "lens", _INT32, 1, dev)
    B = lens.numel()
    max_pages, table_ld = _matrix(block_table, "block_table", _INT32, B, dev)
    out_pages, out_ld = _matrix(out_table, "out_table", _INT32, B, dev)
    _tensor(weights, "weights", _F32, 3, dev)
    if weights_out is None:
        weights_out = _empty(weights.shape, _F32, weights.device, stream)
    _tensor(weights_out, "weights_out", _F32, 3, dev)
    if weights.shape[:2] != (B, Hkv) or weights_out.shape[:2] != (B, Hkv):
        raise ValueError(f"weights and weights_out must be [{B}][{Hkv}][keys]")
    if kept is None:
        kept = _empty((B, Hkv, max(0, int(budget))), _INT32, lens.device, stream)
    _vector(kept, "kept", _INT32, B * Hkv * max(0, budget), dev)
    if new_lens is None:
        new_lens = _empty((B,), _INT32, lens.device, stream)
    _vector(new_lens, "new_lens", _INT32, B, dev)
    _call(_lib.load().nd_paged_kv_evict, dev, _stream_of(dev, stream), k_pages.data_ptr(),
          v_pages.data_ptr(), n_pages, page_size, block_table.data_ptr(), table_ld, max_pages,
          lens.data_ptr(), weights.data_ptr(), weights.shape[2], out_table.data_ptr(), out_ld,
          out_pages, weights_out.data_ptr(), weights_out.shape[2], kept.data_ptr(),
          new_lens.data_ptr(), B, Hkv, D, _int(budget), _int(sinks), _int(recent))
    return kept, new_lens, weights_out


def logits_penalty(logits, history=None, history_lens=None, repetition=None, presence=None,
                   frequency=None, bias_ids=None, bias=None, mask=None, out=None, out_dtype=None,
                   idx=None, greedy=True, stream=None):
    """Penalties, biases and a grammar mask on logits [rows][V], and the greedy
    token (nd_logits_penalty, which gives the order of the operations).

    history int32 [rows][n] (negative: no token), of which the first
    history_lens [rows] count; repetition, presence, frequency fp32 [rows];
    bias_ids int32 / bias fp32 [rows][n_bias]; mask int32 [rows][>= V/32] or
    [>= V/32] for all rows, bit v % 32 of word v / 32 allowing token v.  `out`
    may be `logits` itself.  Returns (out, idx int32 [rows], or None with
    greedy=False)."""
    if out is not None and stream is None and (idx is not None or not greedy) and _quick(
            "logits_penalty", logits, history, history_lens, repetition, presence, frequency,
            bias_ids, bias, mask, out, idx):
        return out, idx
    dev = _device_of(logits, "logits")
    rows = logits.shape[0]
    V, ld = _matrix(logits, "logits", None, rows, dev)
    if out is None:
        out = _empty((rows, V), out_dtype or logits.dtype, logits.device, stream)
    out_V, out_ld = _matrix(out, "out", None, rows, dev)
    if out_V != V:
        raise ValueError(f"out must be {(rows, V)}, got {tuple(out.shape)}")
    n_hist = hist_ld = 0
    hist_addr = None
    if history is not None:
        n_hist, hist_ld = _matrix(history, "history", _INT32, rows, dev)
        # a history without entries has no memory; it is still a history, and not read
        hist_addr = history.data_ptr() if n_hist else logits.data_ptr()
    if history_lens is not None:
        _vector(history_lens, "history_lens", _INT32, rows, dev)
    if repetition is not None:
        _vector(repetition, "repetition", _F32, rows, dev)
    if presence is not None:
        _vector(presence, "presence", _F32, rows, dev)
    if frequency is not None:
        _vector(frequency, "frequency", _F32, rows, dev)
    n_bias = 0
    if (bias_ids is None) != (bias is None):
        raise ValueError("bias_ids and bias go together")
    if bias is not None:
        _tensor(bias_ids, "bias_ids", _INT32, 2, dev)
        _tensor(bias, "bias", _F32, 2, dev)
        if bias_ids.shape != bias.shape or bias.shape[0] != rows:
            raise ValueError(f"bias_ids and bias must be [{rows}][n]")
        n_bias = bias.shape[1]
    mask_ld = 0
    if mask is not None:
        _tensor(mask, "mask", torch.uint32 if mask.dtype is torch.uint32 else _INT32, None, dev, False)
        words = mask.shape[-1] if mask.dim() in (1, 2) else 0
        if words < (V + 31) // 32 or (words > 1 and mask.stride(-1) != 1) or (
                mask.dim() == 2 and mask.shape[0] != rows):
            raise ValueError(f"mask must be [{rows}][words] or [words] of at least "
                             f"{(V + 31) // 32} contiguous words")
        if mask.dim() == 2:
            mask_ld = mask.stride(0) if rows > 1 else words
    if idx is None and greedy:
        idx = _empty((rows,), _INT32, logits.device, stream)
    if idx is not None:
        _vector(idx, "idx", _INT32, rows, dev)
    _call(_lib.load().nd_logits_penalty, dev, _stream_of(dev, stream), logits.data_ptr(),
          _DT[logits.dtype], ld, rows, V, hist_addr, hist_ld, n_hist, _addr(history_lens),
          _addr(repetition), _addr(presence), _addr(frequency), _addr(bias_ids), _addr(bias),
          n_bias, _addr(mask), mask_ld, out.data_ptr(), _DT[out.dtype], out_ld, _addr(idx))
    return out, idx


# ---- tensor-parallel reduction over NVLink peer memory ----------------------
def comm_region_bytes(rows_max, d):
    n = ctypes.c_size_t(0)
    check(_lib.load().nd_comm_region_bytes(rows_max, d, ctypes.byref(n)))
    return n.value


def comm_slot_offset(slot, rows_max, d):
    n = ctypes.c_size_t(0)
    check(_lib.load().nd_comm_slot_offset(slot, rows_max, d, ctypes.byref(n)))
    return n.value


def comm_alloc(nbytes):
    """A zero-filled region on the current device; returns (pointer, 64-byte IPC handle)."""
    p = ctypes.c_void_p()
    h = ctypes.create_string_buffer(64)
    check(_lib.load().nd_comm_alloc(nbytes, ctypes.byref(p), h))
    return p.value, h.raw


def comm_open(handle):
    p = ctypes.c_void_p()
    check(_lib.load().nd_comm_open(ctypes.create_string_buffer(handle, 64), ctypes.byref(p)))
    return p.value


def comm_close(ptr):
    check(_lib.load().nd_comm_close(ctypes.c_void_p(ptr)))


def comm_free(ptr):
    check(_lib.load().nd_comm_free(ctypes.c_void_p(ptr)))


def allreduce_add_layernorm(regions, rank, region_bytes, rows_max, slot, x, bias, gamma, beta,
                            s_out, out, eps=1e-5, stream=None):
    """s_out = x + Σ_r (rank r's partial in `slot`) + bias, out = LayerNorm(s_out)."""
    _need(x, "x", torch.bfloat16, 2)
    rows, d = x.shape
    arr = (ctypes.c_void_p * len(regions))(*regions)
    check(_lib.load().nd_allreduce_add_layernorm(
        _stream(stream), arr, len(regions), rank, region_bytes, rows_max, slot, _ptr(x),
        _ptr(bias), _ptr(gamma), _ptr(beta), _ptr(s_out), _ptr(out), rows, d, float(eps)))
    return s_out, out


def gemm_allreduce_add_layernorm(a, w, regions, rank, region_bytes, rows_max, slot, x, bias, gamma,
                                 beta, s_out, out, eps=1e-5, stream=None):
    """s_out = x + Σ_r bf16(a_r · w_rᵀ) + bias, out = LayerNorm(s_out): this rank's projection
    tile and the cross-rank reduction in one launch (a [rows, K], w [d, K], both bf16)."""
    _need(a, "a", torch.bfloat16, 2)
    _need(w, "w", torch.bfloat16, 2)
    _need(x, "x", torch.bfloat16, 2)
    rows, d = x.shape
    if a.shape[0] != rows or w.shape[0] != d or a.shape[1] != w.shape[1]:
        raise ValueError(f"gemm_allreduce_add_layernorm: a {tuple(a.shape)} w {tuple(w.shape)} "
                         f"x {tuple(x.shape)}")
    arr = (ctypes.c_void_p * len(regions))(*regions)
    check(_lib.load().nd_gemm_allreduce_add_layernorm(
        _stream(stream), _ptr(a), _ptr(w), a.shape[1], arr, len(regions), rank, region_bytes,
        rows_max, slot, _ptr(x), _ptr(bias), _ptr(gamma), _ptr(beta), _ptr(s_out), _ptr(out),
        rows, d, float(eps)))
    return s_out, out
