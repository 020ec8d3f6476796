"""The embedding encoder's operators on torch tensors: 8-bit rows and products, block norms, cross attention.

Thin wrappers of the C-ABI's handle-free calls (``rr_quantize_rows``, ``rr_linear_i8``, ``rr_block_norm``,
``rr_cross_attention`` in ``include/rag_retrieval.h``, which states the arithmetic). They stand for the forward pass of the
reference's embedding half (``batch_processor.py:88-91``), for inference only: tensors that ask for gradients or carry forward-mode
tangents are refused, and so are negated views and calls under a tracer.

Every call runs on the current stream of its tensors' device, allocates its results and scratch memory there through torch
(so calls can be captured into a graph and run on several streams at once), and returns without waiting. Arguments that do
not fit raise ``ValueError`` / ``TypeError``, or ``HipRetrievalError`` from the C-ABI's own checks, before anything is
enqueued. There is no CPU form. Checks and allocations are native code (``_torch_ops.so``, csrc/rr_torch_ops.cpp, built
in-tree against the installed torch); if it is missing every call raises ``HipRetrievalUnavailable``.
"""
from __future__ import annotations

import sys
from typing import NamedTuple, Optional

from ._lib import (LIB_PATH, PKG_ROOT, RR_ACT_GELU, RR_ACT_NONE, RR_NORM_LAYER, RR_NORM_NONE, RR_NORM_RMS,
                   HipRetrievalUnavailable, _check, load_library)

__all__ = ["quantize_rows", "linear_int8", "block_norm", "cross_attention", "NormedBlock"]

ACTS = {"none": RR_ACT_NONE, "gelu": RR_ACT_GELU}
NORMS = {"none": RR_NORM_NONE, "layer": RR_NORM_LAYER, "rms": RR_NORM_RMS}

_native = None


def _load():
    """The native side, bound to the loaded C-ABI library."""
    global _native
    if sys.modules.get("torch") is None:      # whoever holds a tensor has it loaded; this package does not load it itself
        raise TypeError("rag_service_amd.ops works on torch tensors; torch is not loaded")
    load_library()
    try:
        from . import _torch_ops
    except ImportError as e:
        raise HipRetrievalUnavailable(f"cannot load rag_service_amd/_torch_ops.so: {e}; build it with "
                                      f"`make -C {PKG_ROOT}`") from e
    _torch_ops.bind(LIB_PATH)
    _native = _torch_ops
    return _native


def quantize_rows(x):
    """8-bit rows of x (..., cols): int8 values of the same shape and fp32 scales (...), with
    scale = max|row| * (1 / 127) and value = rint(x / scale), all in fp32. A row that holds a NaN or an infinity gets scale NaN and zeros."""
    r = (_native or _load()).quantize_rows(x)
    if type(r) is int:
        _check(r)
    return r


def linear_int8(x, w, w_scale, *, x_scale=None, bias=None, act: str = "none", out_dtype=None):
    """act(x8 @ w.T * (x_scale * w_scale) + bias): a linear layer with int8 weights w (n, k), a scale for each output
    channel (n), and 8-bit rows with a scale each.

    x (..., k) is int8 with x_scale (...), or floating point, whose rows are then made as ``quantize_rows`` makes them.
    act: "none" or "gelu" (erf). The integer sum is exact; the result is rounded once, to out_dtype (x's own type by
    default, fp32 for int8 rows). bias: (n) fp32 or None."""
    if act not in ACTS:
        raise ValueError(f"act must be one of {sorted(ACTS)}")
    r = (_native or _load()).linear_int8(x, w, w_scale, x_scale, bias, ACTS[act], out_dtype)
    if type(r) is int:
        _check(r)
    return r


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
    if post_norm not in NORMS or next_norm not in NORMS:
        raise ValueError(f"a norm must be one of {sorted(NORMS)}")
    if next_norm == "none":
        if rows8:
            raise ValueError("rows8 needs a next norm")
        normed = False
    r = (_native or _load()).block_norm(y, residual, residual_scale, gate, rows_per_gate, NORMS[post_norm], post_weight,
                                        post_bias, NORMS[next_norm], next_weight, next_bias, eps, bool(stream),
                                        bool(normed), bool(rows8))
    if type(r) is int:
        _check(r)
    return NormedBlock._make(r)


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
    r = (_native or _load()).cross_attention(q, k, v, scale, key_lengths, key_mask, q_offsets, k_offsets, max_q, max_k)
    if type(r) is int:
        _check(r)
    return r
