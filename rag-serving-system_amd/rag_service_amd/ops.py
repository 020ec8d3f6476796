"""The embedding encoder's operators on torch tensors: 8-bit rows and products, block norms, cross attention.

Thin wrappers of the C-ABI's handle-free calls (``rr_quantize_rows``, ``rr_linear_i8``, ``rr_block_norm``,
``rr_cross_attention`` in ``include/rag_retrieval.h``, which states the arithmetic). They stand for the forward pass of the
reference's embedding half (``batch_processor.py:88-91``), for inference only: tensors that ask for gradients are refused.

Every call runs on the current stream of its tensors' device, allocates its results and scratch memory there through torch
(so calls can be captured into a graph and run on several streams at once), and returns without waiting. Arguments that do
not fit raise ``ValueError`` / ``TypeError`` here or ``HipRetrievalError`` from the C side, before anything is enqueued.
There is no CPU form.
"""
from __future__ import annotations

import sys
from typing import NamedTuple, Optional

from ._lib import (RR_ACT_GELU, RR_ACT_NONE, RR_NORM_LAYER, RR_NORM_NONE, RR_NORM_RMS, RR_TYPE_BF16, RR_TYPE_F16,
                   RR_TYPE_F32, RR_TYPE_I8, HipRetrievalError, _check, load_library)

__all__ = ["quantize_rows", "linear_int8", "block_norm", "cross_attention", "NormedBlock"]

ACTS = {"none": RR_ACT_NONE, "gelu": RR_ACT_GELU}
NORMS = {"none": RR_NORM_NONE, "layer": RR_NORM_LAYER, "rms": RR_NORM_RMS}


def _torch():
    torch = sys.modules.get("torch")      # whoever holds a tensor has it loaded; this package does not load it itself
    if torch is None:
        raise TypeError("rag_service_amd.ops works on torch tensors; torch is not loaded")
    return torch


_FLOAT_CODES: dict = {}
_RAW_STREAM = None


def _float_codes():
    if not _FLOAT_CODES:
        global _RAW_STREAM
        torch = _torch()
        # the current stream's handle without a Stream object (0.1 instead of 2 us a call), where this torch has it
        _RAW_STREAM = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda index: torch.cuda.current_stream(index).cuda_stream)
        _FLOAT_CODES.update({torch.float32: RR_TYPE_F32, torch.bfloat16: RR_TYPE_BF16, torch.float16: RR_TYPE_F16})
    return _FLOAT_CODES


def _tensor(name: str, t, dtypes, device=None, shape=None):
    """t is a torch tensor on a GPU (on `device`), of one of `dtypes` and of `shape`, and asks for no gradient."""
    try:
        if (t.dtype in dtypes and t.is_cuda and not t.requires_grad and (device is None or t.device == device)
                and (shape is None or t.shape == shape)):
            return t
    except AttributeError:
        pass
    torch = _torch()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, not {type(t).__name__}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} has type {t.dtype}; expected one of {sorted(str(d) for d in dtypes)}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}; expected {tuple(shape)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient; these operators are for inference (torch.no_grad())")
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}; these operators run on the GPU only")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}; expected {device}")
    return t


def _rows(name: str, t):
    """t as (rows, cols) without a copy: its last dimension contiguous, its rows evenly spaced."""
    if t.dim() == 2 and t.is_contiguous() and t.shape[1] > 0:
        return t
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} has shape {tuple(t.shape)}; expected (..., columns)")
    if t.dim() != 2:
        try:
            t = t.view(-1, t.shape[-1]) if t.numel() else t.reshape(0, t.shape[-1])
        except RuntimeError:
            raise ValueError(f"{name}: rows of shape {tuple(t.shape)}, strides {t.stride()} are not evenly spaced") from None
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous (strides {t.stride()})")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{name}: rows overlap (strides {t.stride()})")
    return t


def _ld(t) -> int:
    rows, cols = t.shape
    return t.stride(0) if rows > 1 else cols


def _vector(name: str, t, dtypes, device, n: int):
    """t as a contiguous vector of n values, or None."""
    if t is None:
        return None
    _tensor(name, t, dtypes, device, (n,))
    return t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _place(t):
    """(device index, stream handle) that a call on t's device uses."""
    index = t.get_device()
    return index, _RAW_STREAM(index)


def _scratch(nbytes: int, like):
    if nbytes < 0:
        raise HipRetrievalError(nbytes, load_library().rr_last_error().decode(errors="replace"))
    return like.new_empty(nbytes, dtype=_torch().uint8) if nbytes else None


def quantize_rows(x):
    """8-bit rows of x (..., cols): int8 values of the same shape and fp32 scales (...), with
    scale = max|row| / 127 and value = rint(x / scale). A row that holds a NaN or an infinity gets scale NaN and zeros."""
    torch = _torch()
    codes = _float_codes()
    _tensor("x", x, codes)
    x2 = _rows("x", x)
    rows, cols = x2.shape
    q = x.new_empty(x.shape, dtype=torch.int8)
    scale = x.new_empty(x.shape[:-1], dtype=torch.float32)
    device, stream = _place(x)
    _check(load_library().rr_quantize_rows(device, stream, codes[x.dtype], x2.data_ptr(), _ld(x2), rows, cols,
                                           q.data_ptr(), cols, scale.data_ptr()))
    return q, scale


def linear_int8(x, w, w_scale, *, x_scale=None, bias=None, act: str = "none", out_dtype=None):
    """act(x8 @ w.T * (x_scale * w_scale) + bias): a linear layer with int8 weights w (n, k), a scale for each output
    channel (n), and 8-bit rows with a scale each.

    x (..., k) is int8 with x_scale (...), or floating point, whose rows are then made as ``quantize_rows`` makes them.
    act: "none" or "gelu" (erf). The integer sum is exact; the result is rounded once, to out_dtype (x's own type by
    default, fp32 for int8 rows). bias: (n) fp32 or None."""
    torch = _torch()
    codes = _float_codes()
    if act not in ACTS:
        raise ValueError(f"act must be one of {sorted(ACTS)}")
    _tensor("x", x, (torch.int8,) if x_scale is not None else tuple(codes))
    dev = x.device
    if out_dtype is None:
        out_dtype = torch.float32 if x_scale is not None else x.dtype
    if out_dtype not in codes:
        raise ValueError(f"out_dtype must be one of {sorted(str(d) for d in codes)}")
    x2 = _rows("x", x)
    m, k = x2.shape
    _tensor("w", w, (torch.int8,), dev)
    if w.dim() != 2 or w.shape[1] != k:
        raise ValueError(f"w has shape {tuple(w.shape)}; expected (n, {k})")
    w = _rows("w", w)
    n = w.shape[0]
    w_scale = _vector("w_scale", w_scale, (torch.float32,), dev, n)
    bias = _vector("bias", bias, (torch.float32,), dev, n)
    if x_scale is not None:
        _tensor("x_scale", x_scale, (torch.float32,), dev, x.shape[:-1])
        x_scale = x_scale.contiguous()
        x_type = RR_TYPE_I8
    else:
        x_type = codes[x.dtype]
    lib = load_library()
    need = 0 if x_type == RR_TYPE_I8 else lib.rr_linear_i8_workspace(x_type, m, n, k)
    ws = _scratch(need, x)
    out = x.new_empty(x.shape[:-1] + (n,), dtype=out_dtype)
    device, stream = _place(x)
    _check(lib.rr_linear_i8(device, stream, x_type, x2.data_ptr(), _ld(x2), _ptr(x_scale), w.data_ptr(), _ld(w),
                            w_scale.data_ptr(), _ptr(bias), ACTS[act], codes[out_dtype], out.data_ptr(), n, m, n, k,
                            _ptr(ws), need))
    return out


class NormedBlock(NamedTuple):
    """What ``block_norm`` returns: None for what was not asked for."""
    stream: Optional[object]     # residual_scale * residual + gate * post_norm(y)
    normed: Optional[object]     # next_norm(stream)
    rows8: Optional[object]      # int8 rows of normed ...
    scale: Optional[object]      # ... and their fp32 scales


def block_norm(y, residual=None, *, residual_scale: float = 1.0, gate=None, rows_per_gate: int = 1,
               post_norm: str = "none", post_weight=None, post_bias=None, next_norm: str = "layer", next_weight=None,
               next_bias=None, eps: float = 1e-5, stream: bool = True, normed: bool = True, rows8: bool = False):
    """The norms around a block, fused with what joins the block's output y (..., cols) to the residual stream:

        stream = residual_scale * residual + gate * post_norm(y);  normed = next_norm(stream);  rows8, scale of normed

    post_norm, next_norm: "none", "layer" or "rms". gate: (cols) for all rows, or (gate_rows, cols), of which row r takes
    row r // rows_per_gate. Everything is fp32 from the inputs on and rounded once per output. ``stream``, ``normed`` and
    ``rows8`` say which results are wanted. An encoder's LayerNorm(x + y) is
    ``block_norm(y, x, next_weight=w, next_bias=b, stream=False).normed``."""
    torch = _torch()
    codes = _float_codes()
    for kind in (post_norm, next_norm):
        if kind not in NORMS:
            raise ValueError(f"a norm must be one of {sorted(NORMS)}")
    _tensor("y", y, codes)
    dt, dev = (y.dtype,), y.device
    y2 = _rows("y", y)
    rows, cols = y2.shape
    x2 = g2 = None
    if residual is not None:
        _tensor("residual", residual, dt, dev, y.shape)
        x2 = _rows("residual", residual)
    if gate is not None:
        _tensor("gate", gate, dt, dev)
        if gate.dim() == 1:
            gate, rows_per_gate = gate[None], max(1, rows)
        if gate.dim() != 2 or gate.shape[1] != cols:
            raise ValueError(f"gate has shape {tuple(gate.shape)}; expected ({cols},) or (gate_rows, {cols})")
        g2 = _rows("gate", gate)
    pw, pb = _vector("post_weight", post_weight, dt, dev, cols), _vector("post_bias", post_bias, dt, dev, cols)
    nw, nb = _vector("next_weight", next_weight, dt, dev, cols), _vector("next_bias", next_bias, dt, dev, cols)
    if next_norm == "none":
        if rows8:
            raise ValueError("rows8 needs a next norm")
        normed = False
    h = y.new_empty(y.shape) if stream else None
    o = y.new_empty(y.shape) if normed else None
    q = y.new_empty(y.shape, dtype=torch.int8) if rows8 else None
    s = y.new_empty(y.shape[:-1], dtype=torch.float32) if rows8 else None
    device, on = _place(y)
    _check(load_library().rr_block_norm(
        device, on, codes[y.dtype], rows, cols, y2.data_ptr(), _ld(y2), _ptr(x2), _ld(x2) if x2 is not None else 0,
        float(residual_scale), _ptr(g2), _ld(g2) if g2 is not None else 0, g2.shape[0] if g2 is not None else 0,
        int(rows_per_gate), NORMS[post_norm], _ptr(pw), _ptr(pb), NORMS[next_norm], _ptr(nw), _ptr(nb), float(eps),
        _ptr(h), cols, _ptr(o), cols, _ptr(q), cols, _ptr(s)))
    return NormedBlock(h, o, q, s)


def cross_attention(q, k, v, *, scale: Optional[float] = None, key_lengths=None, key_mask=None, q_offsets=None,
                    k_offsets=None, max_q: Optional[int] = None, max_k: Optional[int] = None):
    """Attention of queries to an encoder's states of another length (or their own: self-attention without causality).

    Dense: q (batch, queries, heads, d), k and v (batch, keys, kv_heads, d); packed: q (rows, heads, d) with q_offsets,
    k and v (rows, kv_heads, d) with k_offsets (int32, batch + 1, on the device: sequence b holds rows
    [offsets[b], offsets[b + 1])); the two sides may differ in form. For a packed side max_q / max_k is the longest
    sequence (the results hold for longer ones too; it sizes the launch). heads is a multiple of kv_heads.
    key_lengths: (batch) int32, the sequence's first keys that take part. key_mask: (batch, keys) bool or uint8, dense keys
    only. Keys left out may hold anything. A query without keys gets zeros; packed rows that no sequence holds are
    undefined. scale: d ** -0.5 by default. Returns q's shape and type."""
    torch = _torch()
    codes = _float_codes()
    _tensor("q", q, codes)
    dt, dev = (q.dtype,), q.device
    _tensor("k", k, dt, dev)
    _tensor("v", v, dt, dev)
    q_dense, k_dense = q_offsets is None, k_offsets is None
    if q.dim() != (4 if q_dense else 3):
        raise ValueError(f"q has shape {tuple(q.shape)}; expected (batch, queries, heads, d), or (rows, heads, d) with q_offsets")
    if k.dim() != (4 if k_dense else 3):
        raise ValueError(f"k has shape {tuple(k.shape)}; expected (batch, keys, kv_heads, d), or (rows, kv_heads, d) with k_offsets")
    if v.shape != k.shape:
        raise ValueError(f"v has shape {tuple(v.shape)}, k {tuple(k.shape)}")
    heads, d = q.shape[-2:]
    kv_heads = k.shape[-2]
    if k.shape[-1] != d:
        raise ValueError(f"q has head size {d}, k {k.shape[-1]}")
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name}: the last dimension must be contiguous (strides {t.stride()})")
    for name, t, longest in (("q_offsets", q_offsets, max_q), ("k_offsets", k_offsets, max_k)):
        if t is None:
            continue
        _tensor(name, t, (torch.int32,), dev)
        if t.dim() != 1 or t.shape[0] < 1 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous vector of batch + 1 row numbers")
        if longest is None or longest < 0:
            raise ValueError(f"{name} goes with max_q / max_k, the longest sequence")
    batch = q.shape[0] if q_dense else q_offsets.shape[0] - 1
    if (k.shape[0] if k_dense else k_offsets.shape[0] - 1) != batch:
        raise ValueError("queries and keys have different batch sizes")
    max_q = q.shape[1] if q_dense else int(max_q)
    max_k = k.shape[1] if k_dense else int(max_k)
    key_lengths = _vector("key_lengths", key_lengths, (torch.int32,), dev, batch)
    stride = 0
    if key_mask is not None:
        if not k_dense:
            raise ValueError("key_mask goes with dense keys")
        _tensor("key_mask", key_mask, (torch.bool, torch.uint8), dev, (batch, max_k))
        if max_k > 1 and key_mask.stride(1) != 1 or batch > 1 and key_mask.stride(0) < max_k:
            key_mask = key_mask.contiguous()
        stride = max(key_mask.stride(0), max_k)
    out = q.new_empty(q.shape)
    lib = load_library()
    code = codes[q.dtype]
    need = lib.rr_cross_attention_workspace(code, batch, heads, kv_heads, d, max_q, max_k)
    ws = _scratch(need, q)
    device, on = _place(q)

    def strides(t, dense):
        return (t.stride(0), t.stride(1), t.stride(2)) if dense else (0, t.stride(0), t.stride(1))

    _check(lib.rr_cross_attention(
        device, on, code, q.data_ptr(), *strides(q, q_dense), k.data_ptr(), *strides(k, k_dense), v.data_ptr(),
        *strides(v, k_dense), out.data_ptr(), *strides(out, q_dense), batch, heads, kv_heads, d, max_q, max_k,
        0 if q_dense else q.shape[0], 0 if k_dense else k.shape[0], _ptr(q_offsets), _ptr(k_offsets), _ptr(key_lengths),
        _ptr(key_mask), stride, float(d ** -0.5 if scale is None else scale), _ptr(ws), need))
    return out
