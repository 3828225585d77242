"""Operators either side of the grouped GEMM on CUDA tensors: the router's choice, the
8-bit row quantiser and the whole expert layer for a few tokens.

Thin wrappers of the C entry points (``include/bmoe_b200.h``, section 6). Each allocates the
outputs it is not given, launches on ``stream`` (default: the current stream of the tensors'
device) and does not synchronise. Wrong shapes, types or devices raise ``ValueError``, a
status of the engine raises ``EngineError``. The reference has no counterpart: routed
token counts are its input (agent/search_space.yaml:10-13).
"""

from __future__ import annotations

import contextlib
import ctypes as C

import torch

from . import _capi

_ROW_TYPES = {torch.bfloat16: _capi.TYPE_BF16, torch.float32: _capi.TYPE_FP32}
_WEIGHT_TYPES = {torch.bfloat16: _capi.TYPE_BF16, torch.int8: _capi.TYPE_INT8}
_NO_GUARD = contextlib.nullcontext()


def _require(condition, message: str) -> None:
    if not condition:
        raise ValueError(message)


def _on(device):
    """Context in which ``device`` is the current one."""
    return _NO_GUARD if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(stream, device) -> int | None:
    if stream is None:
        stream = torch.cuda.current_stream(device)
    return int(getattr(stream, "cuda_stream", stream)) or None


def _check_rows(x, name: str) -> None:
    _require(x.is_cuda, f"{name}: the engine has no CPU path, a CUDA tensor is needed")
    _require(x.dim() == 2 and x.dtype in _ROW_TYPES, f"{name}: BF16 or FP32 [rows, columns]")
    _require(x.stride(1) == 1 or x.shape[1] <= 1, f"{name}: columns must be contiguous")


def _check(x, name: str, dtype, shape, device) -> None:
    _require(x.dtype is dtype and x.device == device and tuple(x.shape) == tuple(shape)
             and x.is_contiguous(),
             f"{name}: contiguous {dtype} {list(shape)} on {device} needed")


def route_topk(logits, top_k: int, *, scoring: str = "softmax", renormalize: bool = False,
               bias=None, scale: float = 1.0, expert_ids=None, weights=None, stream=None):
    """The ``top_k`` experts of every token and their weights.

    ``logits`` [tokens, experts] BF16 or FP32 (rows may be strided). Returns ``(expert_ids
    int64, weights float32)``, both [tokens, top_k], largest score first, ties to the
    lower id. ``scoring`` "softmax" or "sigmoid"; ``bias`` [experts] float32 is added to a
    sigmoid score for the choice only; ``renormalize`` divides by the sum over the chosen.
    Experts at -inf or NaN are never chosen; a token left with fewer gets id -1, weight 0."""
    _check_rows(logits, "logits")
    _require(scoring in _capi.SCORINGS, f"unknown scoring: {scoring}")
    tokens, experts = logits.shape
    device = logits.device
    if bias is not None:
        _check(bias, "bias", torch.float32, (experts,), device)
    with _on(device):
        if expert_ids is None:
            expert_ids = torch.empty(tokens, top_k, dtype=torch.int64, device=device)
        else:
            _check(expert_ids, "expert_ids", torch.int64, (tokens, top_k), device)
        if weights is None:
            weights = torch.empty(tokens, top_k, dtype=torch.float32, device=device)
        else:
            _check(weights, "weights", torch.float32, (tokens, top_k), device)
        _require(tokens <= 1 or logits.stride(0) >= experts, "logits: rows must not overlap")
        args = _capi.RouteTopkArgs(
            logits.data_ptr(), None if bias is None else bias.data_ptr(), expert_ids.data_ptr(),
            weights.data_ptr(), tokens, logits.stride(0) if tokens > 1 else 0, experts, top_k,
            _ROW_TYPES[logits.dtype], _capi.SCORINGS[scoring], int(renormalize), scale,
            _stream(stream, device))
        _capi.check(_capi.load().bmoe_route_topk(C.byref(args)), "bmoe_route_topk")
    return expert_ids, weights


def quantize_rows(x, index=None, *, out=None, scale=None, stream=None):
    """Rows of ``x`` [rows, cols] (BF16 or FP32, rows may be strided) in 8 bits.

    Returns ``(q int8, scale float32)`` with ``x[i] ~ q[i] * scale[i]``: the A operand and
    ``row_scale`` of an INT8 product. With ``index`` (int64) output row i is row
    ``index[i]``; an index outside ``x`` leaves its output row untouched."""
    _check_rows(x, "x")
    device = x.device
    src_rows, cols = x.shape
    rows = src_rows
    if index is not None:
        _require(index.dim() == 1, "index: one dimension")
        rows = index.shape[0]
        _check(index, "index", torch.int64, (rows,), device)
    _require(src_rows <= 1 or x.stride(0) >= cols, "x: rows must not overlap")
    with _on(device):
        if out is None:
            out = torch.empty(rows, cols, dtype=torch.int8, device=device)
        else:
            _check(out, "out", torch.int8, (rows, cols), device)
        if scale is None:
            scale = torch.empty(rows, dtype=torch.float32, device=device)
        else:
            _check(scale, "scale", torch.float32, (rows,), device)
        args = _capi.QuantizeRowsArgs(
            x.data_ptr(), None if index is None else index.data_ptr(), out.data_ptr(),
            scale.data_ptr(), rows, src_rows, x.stride(0) if src_rows > 1 else 0, cols,
            _ROW_TYPES[x.dtype], _stream(stream, device))
        _capi.check(_capi.load().bmoe_quantize_rows(C.byref(args)), "bmoe_quantize_rows")
    return out, scale


def moe_decode_workspace(tokens: int, top_k: int, inter: int) -> int:
    """Bytes of workspace ``moe_decode`` needs for these sizes."""
    return int(_capi.load().bmoe_moe_decode_workspace(tokens, top_k, inter))


def moe_decode(x, w_gate_up, w_down, expert_ids, weights, *, gate_up_scale=None,
               down_scale=None, out=None, workspace=None, stream=None):
    """A whole expert layer for up to 64 tokens, in two launches.

    ``x`` BF16 [tokens, hidden]; ``w_gate_up`` [experts, 2 * inter, hidden] (gate rows, then
    up rows) and ``w_down`` [experts, hidden, inter], both BF16, or both INT8 with the
    FP32 ``gate_up_scale`` [experts, 2 * inter] and ``down_scale`` [experts, hidden];
    ``expert_ids`` int64 and ``weights`` float32 [tokens, top_k] as ``route_topk`` returns them
    (ids outside the experts are dropped). Returns BF16 [tokens, hidden]:
    ``out[t] = sum_j weights[t, j] * (silu(x Wgate^T) * (x Wup^T)) Wdown^T``.

    ``workspace``: contiguous uint8 tensor of ``moe_decode_workspace`` bytes, for callers that
    keep one; calls that may overlap need one each."""
    _require(x.is_cuda, "x: the engine has no CPU path, a CUDA tensor is needed")
    device = x.device
    _require(x.dim() == 2 and w_gate_up.dim() == 3 and expert_ids.dim() == 2,
             "x [tokens, hidden], w_gate_up [experts, 2 * inter, hidden], "
             "expert_ids [tokens, top_k] needed")
    tokens, hidden = x.shape
    experts, both = w_gate_up.shape[:2]
    inter, top_k = both // 2, expert_ids.shape[1]
    kind = w_gate_up.dtype
    _require(kind in _WEIGHT_TYPES and both % 2 == 0, "w_gate_up: BF16 or INT8, 2 * inter rows")
    _check(x, "x", torch.bfloat16, (tokens, hidden), device)
    _check(w_gate_up, "w_gate_up", kind, (experts, 2 * inter, hidden), device)
    _check(w_down, "w_down", kind, (experts, hidden, inter), device)
    _check(expert_ids, "expert_ids", torch.int64, (tokens, top_k), device)
    _check(weights, "weights", torch.float32, (tokens, top_k), device)
    if kind is torch.int8:
        _require(gate_up_scale is not None and down_scale is not None,
                 "INT8 weights need gate_up_scale and down_scale")
        _check(gate_up_scale, "gate_up_scale", torch.float32, (experts, 2 * inter), device)
        _check(down_scale, "down_scale", torch.float32, (experts, hidden), device)
    else:
        _require(gate_up_scale is None and down_scale is None, "BF16 weights have no scales")
    lib = _capi.load()
    with _on(device):
        if out is None:
            out = torch.empty(tokens, hidden, dtype=torch.bfloat16, device=device)
        else:
            _check(out, "out", torch.bfloat16, (tokens, hidden), device)
        if workspace is None:
            need = lib.bmoe_moe_decode_workspace(tokens, top_k, inter)
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
        else:
            _require(workspace.dtype is torch.uint8 and workspace.device == device
                     and workspace.is_contiguous(), "workspace: contiguous uint8 tensor")
        args = _capi.MoeDecodeArgs(
            x.data_ptr(), w_gate_up.data_ptr(), w_down.data_ptr(),
            None if gate_up_scale is None else gate_up_scale.data_ptr(),
            None if down_scale is None else down_scale.data_ptr(), expert_ids.data_ptr(),
            weights.data_ptr(), out.data_ptr(), workspace.data_ptr(), workspace.numel(),
            tokens, top_k, experts, hidden, inter, _WEIGHT_TYPES[kind], _stream(stream, device))
        _capi.check(lib.bmoe_moe_decode(C.byref(args)), "bmoe_moe_decode")
    return out
