"""Operators either side of the grouped GEMM on CUDA tensors: the router's choice, the
8-bit row quantiser and the whole expert layer for a few tokens.

Thin wrappers of the C entry points (``include/bmoe_b200.h``, section 6). Each allocates the
outputs it is not given, launches on ``stream`` (default: the current stream of the tensors'
device) and does not synchronise; what it allocates belongs to that stream. Inputs, and outputs
that are given, stay the caller's, who keeps them until the launch has run where they belong to
another stream. There is no backward pass: with gradients enabled, inputs that require one are refused. Wrong shapes, types or
devices raise ``ValueError``, a status of the engine raises ``EngineError``. The reference has
no counterpart: routed token counts are its input (agent/search_space.yaml:10-13).
"""

from __future__ import annotations

import contextlib
import functools

from . import _capi

# PyTorch and what is looked up in it, at the first call: the rest of the package works without
torch = None
_NO_GUARD = contextlib.nullcontext()
_route_topk = _capi.entry("bmoe_route_topk", _capi.RouteTopkArgs)
_quantize_rows = _capi.entry("bmoe_quantize_rows", _capi.QuantizeRowsArgs)
_moe_decode = _capi.entry("bmoe_moe_decode", _capi.MoeDecodeArgs)


def _bind_torch() -> None:
    global torch, _ROW_TYPES, _WEIGHT_TYPES, _current_device, _current_raw_stream
    import torch as module

    _ROW_TYPES = {module.bfloat16: _capi.TYPE_BF16, module.float32: _capi.TYPE_FP32}
    _WEIGHT_TYPES = {module.bfloat16: _capi.TYPE_BF16, module.int8: _capi.TYPE_INT8}
    # the current device, and the raw handle of its current stream without a Stream object (a
    # build of PyTorch without CUDA has neither, nor tensors that get that far)
    _current_device = getattr(module._C, "_cuda_getDevice", None)
    _current_raw_stream = getattr(module._C, "_cuda_getCurrentRawStream", None)
    torch = module


def _on(index: int, stream):
    """Context in which device ``index`` and ``stream`` are the current ones: what is allocated
    in it belongs to the stream that the launch goes to, so the allocator neither hands out
    memory that older work of another stream still reads nor takes it back too early."""
    if stream is None:
        return _NO_GUARD if index == _current_device() else torch.cuda.device(index)
    if not isinstance(stream, torch.cuda.Stream):
        raw = int(getattr(stream, "cuda_stream", stream))
        stream = (torch.cuda.ExternalStream(raw, device=index) if raw
                  else torch.cuda.default_stream(index))
    if stream.device_index != index:
        raise ValueError(f"stream: one of cuda:{index} needed, got {stream.device}")
    return torch.cuda.stream(stream)


def _forward_only(*tensors) -> None:
    """The operators have no backward pass: a result that should carry a gradient is refused."""
    if torch.is_grad_enabled():
        for x in tensors:
            if x is not None and x.requires_grad:
                raise ValueError("no backward pass: detach what requires a gradient, or call "
                                 "under torch.no_grad()")


def _is(x, dtype, shape, index: int) -> bool:
    """``x`` is a contiguous tensor of that type and shape on CUDA device ``index``."""
    return (x.dtype is dtype and x.shape == shape and x.get_device() == index
            and x.is_contiguous())


def _need(x, name: str, dtype, shape, index: int) -> None:
    if not _is(x, dtype, shape, index):
        raise ValueError(f"{name}: contiguous {dtype} {list(shape)} on cuda:{index} needed, got "
                         f"{x.dtype} {list(x.shape)} on {x.device}")


def _rows(x, name: str):
    """Rows, columns, row stride and device of a row matrix with contiguous columns."""
    if not x.is_cuda:
        raise ValueError(f"{name}: the engine has no CPU path, a CUDA tensor is needed")
    if x.dim() != 2 or x.dtype not in _ROW_TYPES:
        raise ValueError(f"{name}: BF16 or FP32 [rows, columns] needed")
    rows, cols = x.shape
    stride, inner = x.stride()
    if inner != 1 and cols > 1:
        raise ValueError(f"{name}: columns must be contiguous")
    if rows > 1 and stride < cols:
        raise ValueError(f"{name}: rows must not overlap")
    return rows, cols, stride if rows > 1 else 0, x.get_device()


def route_topk(logits, top_k: int, *, scoring: str = "softmax", renormalize: bool = False,
               bias=None, scale: float = 1.0, expert_ids=None, weights=None, stream=None):
    """The ``top_k`` experts of every token and their weights.

    ``logits`` [tokens, experts] BF16 or FP32 (rows may be strided). Returns ``(expert_ids
    int64, weights float32)``, both [tokens, top_k], largest score first, ties to the
    lower id. ``scoring`` "softmax" or "sigmoid"; ``bias`` [experts] float32 is added to a
    sigmoid score for the choice only; ``renormalize`` divides by the sum over the chosen.
    Experts at -inf or NaN are never chosen; a token left with fewer gets id -1, weight 0."""
    if torch is None:
        _bind_torch()
    _forward_only(logits, bias)
    tokens, experts, row_stride, index = _rows(logits, "logits")
    if scoring not in _capi.SCORINGS:
        raise ValueError(f"unknown scoring: {scoring}")
    if bias is not None:
        _need(bias, "bias", torch.float32, (experts,), index)
    with _on(index, stream):
        if expert_ids is None:
            expert_ids = torch.empty(tokens, top_k, dtype=torch.int64, device=logits.device)
        else:
            _need(expert_ids, "expert_ids", torch.int64, (tokens, top_k), index)
        if weights is None:
            weights = torch.empty(tokens, top_k, dtype=torch.float32, device=logits.device)
        else:
            _need(weights, "weights", torch.float32, (tokens, top_k), index)
        status = _route_topk(
            logits.data_ptr(), 0 if bias is None else bias.data_ptr(), expert_ids.data_ptr(),
            weights.data_ptr(), tokens, row_stride, experts, top_k, _ROW_TYPES[logits.dtype],
            _capi.SCORINGS[scoring], 1 if renormalize else 0, scale, _current_raw_stream(index))
        _capi.check(status, "bmoe_route_topk")
    return expert_ids, weights


def quantize_rows(x, index=None, *, out=None, scale=None, stream=None):
    """Rows of ``x`` [rows, cols] (BF16 or FP32, rows may be strided) in 8 bits.

    Returns ``(q int8, scale float32)`` with ``x[i] ~ q[i] * scale[i]``: the A operand and
    ``row_scale`` of an INT8 product. With ``index`` (int64) output row i is row
    ``index[i]``; an index outside ``x`` leaves its output row untouched."""
    if torch is None:
        _bind_torch()
    _forward_only(x)
    src_rows, cols, row_stride, device = _rows(x, "x")
    rows = src_rows
    if index is not None:
        rows = index.numel()
        _need(index, "index", torch.int64, (rows,), device)
    with _on(device, stream):
        if out is None:
            out = torch.empty(rows, cols, dtype=torch.int8, device=x.device)
        else:
            _need(out, "out", torch.int8, (rows, cols), device)
        if scale is None:
            scale = torch.empty(rows, dtype=torch.float32, device=x.device)
        else:
            _need(scale, "scale", torch.float32, (rows,), device)
        status = _quantize_rows(
            x.data_ptr(), 0 if index is None else index.data_ptr(), out.data_ptr(),
            scale.data_ptr(), rows, src_rows, row_stride, cols, _ROW_TYPES[x.dtype],
            _current_raw_stream(device))
        _capi.check(status, "bmoe_quantize_rows")
    return out, scale


@functools.lru_cache(maxsize=256)
def moe_decode_workspace(tokens: int, top_k: int, inter: int) -> int:
    """Bytes of workspace ``moe_decode`` needs for these sizes."""
    return int(_capi.load().bmoe_moe_decode_workspace(tokens, top_k, inter))


def moe_decode(x, w_gate_up, w_down, expert_ids, weights, *, gate_up_scale=None,
               down_scale=None, out=None, workspace=None, status=None, stream=None):
    """A whole expert layer for up to 64 tokens.

    ``x`` BF16 [tokens, hidden]; ``w_gate_up`` [experts, 2 * inter, hidden] (gate rows, then
    up rows) and ``w_down`` [experts, hidden, inter], both BF16, or both INT8 with the
    FP32 ``gate_up_scale`` [experts, 2 * inter] and ``down_scale`` [experts, hidden];
    ``expert_ids`` int64 and ``weights`` float32 [tokens, top_k] as ``route_topk`` returns them
    (ids outside the experts are dropped). Returns BF16 [tokens, hidden]:
    ``out[t] = sum_j weights[t, j] * (silu(x Wgate^T) * (x Wup^T)) Wdown^T``.

    ``workspace``: contiguous uint8 tensor of ``moe_decode_workspace`` bytes, for callers that
    keep one; calls that may overlap need one each.

    ``status``: int32 tensor [1] that starts at zero and may serve many calls. Every wait inside
    the kernels is bounded (one second); one that runs out leaves a non-zero word there, and NaN
    in what could not be computed. A call that finds the word set makes all of ``out`` NaN."""
    if torch is None:
        _bind_torch()
    _forward_only(x, w_gate_up, w_down, weights, gate_up_scale, down_scale)
    if not x.is_cuda:
        raise ValueError("x: the engine has no CPU path, a CUDA tensor is needed")
    if x.dim() != 2 or w_gate_up.dim() != 3 or expert_ids.dim() != 2:
        raise ValueError("x [tokens, hidden], w_gate_up [experts, 2 * inter, hidden] and "
                         "expert_ids [tokens, top_k] needed")
    kind = w_gate_up.dtype
    if kind not in _WEIGHT_TYPES:
        raise ValueError("w_gate_up: BF16 or INT8 weights")
    int8 = kind is torch.int8
    if int8 != (gate_up_scale is not None) or int8 != (down_scale is not None):
        raise ValueError("INT8 weights have gate_up_scale and down_scale, BF16 weights none")
    index = x.get_device()
    tokens, hidden = x.shape
    experts, both, _ = w_gate_up.shape
    inter, top_k = both // 2, expert_ids.shape[1]
    _need(x, "x", torch.bfloat16, (tokens, hidden), index)
    _need(w_gate_up, "w_gate_up", kind, (experts, 2 * inter, hidden), index)
    _need(w_down, "w_down", kind, (experts, hidden, inter), index)
    _need(expert_ids, "expert_ids", torch.int64, (tokens, top_k), index)
    _need(weights, "weights", torch.float32, (tokens, top_k), index)
    if int8:
        _need(gate_up_scale, "gate_up_scale", torch.float32, (experts, 2 * inter), index)
        _need(down_scale, "down_scale", torch.float32, (experts, hidden), index)
    with _on(index, stream):
        if out is None:
            out = torch.empty_like(x)
        else:
            _need(out, "out", torch.bfloat16, (tokens, hidden), index)
        if workspace is None:
            workspace = torch.empty(moe_decode_workspace(tokens, top_k, inter),
                                    dtype=torch.uint8, device=x.device)
        else:
            _need(workspace, "workspace", torch.uint8, (workspace.numel(),), index)
        if status is not None:
            _need(status, "status", torch.int32, (1,), index)
        result = _moe_decode(
            x.data_ptr(), w_gate_up.data_ptr(), w_down.data_ptr(),
            gate_up_scale.data_ptr() if int8 else 0, down_scale.data_ptr() if int8 else 0,
            expert_ids.data_ptr(), weights.data_ptr(), out.data_ptr(), workspace.data_ptr(),
            workspace.numel(), tokens, top_k, experts, hidden, inter, _WEIGHT_TYPES[kind],
            _current_raw_stream(index), 0 if status is None else status.data_ptr())
        _capi.check(result, "bmoe_moe_decode")
    return out
