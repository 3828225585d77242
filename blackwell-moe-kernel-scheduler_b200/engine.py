"""Python face of the sm_100a engine: plan, device worklist builder, probe.

Everything here calls the C interface (``include/bmoe_b200.h``); PyTorch is
used only to own device memory and streams. Names follow the reference's C++
boundary (``Bf16GroupedGemmPlan``: ``initialize`` / ``run`` / ``stats``,
include/blackwell_moe/kernels/grouped_gemm.cuh:51-69) and return the same
status codes instead of raising.
"""

from __future__ import annotations

import ctypes as C
from typing import Sequence

import numpy as np

from . import _capi

TILE_DTYPE = np.dtype(
    [("expert_id", "<u4"), ("tile_m", "<u4"), ("tile_n", "<u4"),
     ("valid_m", "<u4"), ("valid_n", "<u4")]
)


def _scheduler_id(scheduler) -> int:
    if isinstance(scheduler, str):
        if scheduler not in _capi.SCHEDULER_NAMES:
            raise ValueError(f"unknown scheduler: {scheduler}")
        return _capi.SCHEDULER_NAMES[scheduler]
    return int(scheduler)


def _stream_ptr(stream) -> int | None:
    if stream is None:
        return None
    if hasattr(stream, "cuda_stream"):
        return int(stream.cuda_stream) or None
    return int(stream) or None


def tiles_to_numpy(tiles, count: int) -> np.ndarray:
    """ctypes ``Tile`` array -> structured numpy array (copy)."""
    raw = np.frombuffer(tiles, dtype=TILE_DTYPE, count=count)
    return raw.copy()


def _address(arr: np.ndarray) -> int:
    return arr.__array_interface__["data"][0]


def _byte_type(a, w, scaled: bool) -> int:
    """Operand type of one-byte tensors: with scales INT8 (both ``torch.int8``, else -1), without
    FP8 E4M3 bytes."""
    import torch

    if not scaled:
        return _capi.TYPE_FP8_E4M3
    return _capi.TYPE_INT8 if a.dtype is w.dtype is torch.int8 else -1


def _scales_fit(data_type, a, w, row_scale, col_scale) -> bool:
    """Scales are there exactly for INT8 operands: FP32, one per row of ``a`` and one per
    (expert, output channel)."""
    import torch

    if data_type != _capi.TYPE_INT8:
        return data_type != -1 and row_scale is None and col_scale is None
    return (a.dtype is w.dtype is torch.int8
            and row_scale is not None and col_scale is not None
            and row_scale.dtype is torch.float32 and col_scale.dtype is torch.float32
            and row_scale.device == a.device and col_scale.device == a.device
            and row_scale.is_contiguous() and col_scale.is_contiguous()
            and row_scale.numel() >= int(a.shape[0])
            and tuple(col_scale.shape) == tuple(w.shape[:2]))


def _table(index: np.ndarray, columns) -> np.ndarray:
    """One line ``base + index * size`` per (base, size); addresses are whole uint64 values."""
    spec = np.array(columns, dtype=np.uint64)
    return spec[:, :1] + spec[:, 1:] * index


def _expert_pointers(per_expert) -> np.ndarray:
    """Address of every expert's slice of a contiguous FP32 tensor [experts, n]."""
    experts, n = int(per_expert.shape[0]), int(per_expert.shape[1])
    return per_expert.data_ptr() + np.arange(experts, dtype=np.uint64) * (n * 4)


class GroupedGemmPlan:
    """Reusable launch plan for ``D_e = A_e @ B_e^T`` over routed experts.

    Set-ups and launches take effect in the order of the calls, on any streams, and can be
    captured into CUDA graphs; a graph keeps what it refers to, until the plan is closed, and
    the plan can be set up again meanwhile. The tensors of a captured set-up are the caller's
    to keep."""

    def __init__(self) -> None:
        self._lib = _capi.load()
        self._handle = self._lib.bmoe_plan_create()
        if not self._handle:
            raise MemoryError("bmoe_plan_create failed")
        self._keep = None  # argument arrays / tensors kept alive for the plan

    def close(self) -> None:
        if getattr(self, "_handle", None):
            self._lib.bmoe_plan_destroy(self._handle)
            self._handle = None

    def __del__(self) -> None:  # pragma: no cover - interpreter shutdown order
        try:
            self.close()
        except Exception:
            pass

    # ------------------------------------------------------------ set-up --
    def initialize(
        self,
        a_ptrs: Sequence[int],
        b_ptrs: Sequence[int],
        d_ptrs: Sequence[int],
        tokens_per_expert: Sequence[int],
        n: int,
        k: int,
        *,
        scheduler="expert_order",
        data_type: int = 0,
        stream=None,
        claim_size: int = 0,
        hybrid_tail_tiles: int = 0,
        cta_count: int = 0,
        tile_n: int = 0,
        cta_group: int = 0,
        raster_along_m: int = -1,
        output_f32: bool = False,
        packed_a: int = 0,
        packed_rows: int = 0,
        results_pushed: bool = False,
        tokens_per_expert_dev: int = 0,
        row_scale_ptrs: Sequence[int] | None = None,
        col_scale_ptrs: Sequence[int] | None = None,
        packed_row_scale: int = 0,
    ) -> int:
        """Pointer-array form of the reference arguments. Returns a status.
        ``packed_a`` / ``packed_rows``: base and row capacity of ONE buffer holding all
        experts' rows back to back (one tensor map instead of one per expert; ``a_ptrs``
        is then ignored). ``results_pushed``: no D descriptors, results leave through
        ``set_push``. ``row_scale_ptrs`` / ``col_scale_ptrs`` / ``packed_row_scale``: scales
        of INT8 operands (``data_type`` 3)."""
        def pointers(values):
            if not isinstance(values, np.ndarray):
                values = np.array([int(p or 0) for p in values], dtype=np.uint64)
            elif values.dtype != np.uint64 or not values.flags.c_contiguous:
                values = np.ascontiguousarray(values, dtype=np.uint64)
            return values if values.size else np.zeros(1, dtype=np.uint64)

        arrays = [None if ptrs is None else pointers(ptrs)
                  for ptrs in (a_ptrs, b_ptrs, d_ptrs, row_scale_ptrs, col_scale_ptrs)]
        return self._initialize(
            *(None if arr is None else _address(arr) for arr in arrays), tokens_per_expert, n, k,
            scheduler=scheduler, data_type=data_type, stream=stream, claim_size=claim_size,
            hybrid_tail_tiles=hybrid_tail_tiles, cta_count=cta_count, tile_n=tile_n,
            cta_group=cta_group, raster_along_m=raster_along_m, output_f32=output_f32,
            packed_a=packed_a, packed_rows=packed_rows, results_pushed=results_pushed,
            tokens_per_expert_dev=tokens_per_expert_dev, packed_row_scale=packed_row_scale)

    def _initialize(self, a, b, d, row_scale, col_scale, tokens_per_expert, n, k, *,
                    scheduler="expert_order", data_type=0, stream=None, claim_size=0,
                    hybrid_tail_tiles=0, cta_count=0, tile_n=0, cta_group=0, raster_along_m=-1,
                    output_f32=False, packed_a=0, packed_rows=0, results_pushed=False,
                    tokens_per_expert_dev=0, packed_row_scale=0) -> int:
        """``initialize`` with the addresses of the pointer arrays, which outlive the call."""
        counts = np.ascontiguousarray(tokens_per_expert, dtype=np.uint32)
        experts = counts.size
        if experts == 0:
            counts = np.zeros(1, dtype=np.uint32)
        args = _capi.GemmArgs(
            a, b, d, _address(counts), experts, n, k, data_type, _scheduler_id(scheduler),
            claim_size, hybrid_tail_tiles, min(int(cta_count), 0xFFFFFFFF), tile_n, cta_group, raster_along_m,
            1 if output_f32 else 0, _stream_ptr(stream), int(packed_a) or None, int(packed_rows),
            1 if results_pushed else 0, 0, int(tokens_per_expert_dev) or None,
            row_scale, col_scale, int(packed_row_scale) or None)
        return int(self._lib.bmoe_plan_initialize(self._handle, C.byref(args)))

    def initialize_packed(self, a, w, d, tokens_per_expert: Sequence[int], *,
                          single_a_map: bool = False, row_scale=None, col_scale=None,
                          **options) -> int:
        """Packed form: ``a`` [sum M, k], ``w`` [E, n, k], ``d`` [sum M, n] CUDA
        tensors, rows of expert 0 first; ``a`` and ``w`` BF16, or both one byte per element
        (FP8 E4M3 bit patterns, or ``torch.int8`` with FP32 ``row_scale`` [rows of a] and
        ``col_scale`` [E, n]; k then a multiple of 16), ``d`` BF16 (FP32 with
        ``output_f32``). Row offsets are the exclusive prefix sum
        of the counts; every expert's slice starts on a 16-byte boundary because
        k and n are multiples of 8. ``single_a_map``: one tensor map over the whole of
        ``a`` instead of one per expert (cheaper to re-plan; tiles at an expert's ragged
        edge then also load the next expert's rows, which costs bandwidth when experts
        have few rows and changes no result)."""
        experts, n, k = w.shape
        d_elem = 4 if options.get("output_f32") else 2
        if d.element_size() != d_elem:
            return _capi.INVALID_ARGUMENT
        if experts != len(tokens_per_expert) or a.shape[1] != k or d.shape[1] != n:
            return _capi.INVALID_ARGUMENT
        if not (a.is_contiguous() and w.is_contiguous() and d.is_contiguous()):
            return _capi.INVALID_ARGUMENT
        counts = np.asarray(tokens_per_expert, dtype=np.int64)
        ends = counts.cumsum()
        total = int(ends[-1]) if experts else 0
        if a.shape[0] < total or d.shape[0] < total:
            return _capi.INVALID_ARGUMENT
        elem = a.element_size()
        if elem != w.element_size() or elem not in (1, 2):
            return _capi.INVALID_ARGUMENT
        if elem == 1:
            options["data_type"] = _byte_type(a, w, row_scale is not None or col_scale is not None)
        if not _scales_fit(options.get("data_type"), a, w, row_scale, col_scale):
            return _capi.INVALID_ARGUMENT
        scaled = row_scale is not None
        # every expert's address: base + first row * bytes of a row, or + id * bytes of a slice
        rows = _table((ends - counts).view(np.uint64), (
            (a.data_ptr(), k * elem), (d.data_ptr(), n * d_elem),
            (row_scale.data_ptr() if scaled else 0, 4)))
        slices = _table(np.arange(experts, dtype=np.uint64), (
            (w.data_ptr(), n * k * elem), (col_scale.data_ptr() if scaled else 0, 4 * n)))
        by_row, by_slice, line = _address(rows), _address(slices), 8 * experts
        if single_a_map:
            options.update(packed_a=a.data_ptr(), packed_rows=a.shape[0])
            if scaled:
                options["packed_row_scale"] = row_scale.data_ptr()
        self._keep = (a, w, d, row_scale, col_scale)
        return self._initialize(
            by_row, by_slice, by_row + line, by_row + 2 * line if scaled else None,
            by_slice + line if scaled else None, counts, n, k, **options)

    def initialize_packed_device_counts(self, a, w, counts_dev_ptr: int, *, row_scale=None,
                                        col_scale=None, **options) -> int:
        """Packed form whose counts exist only on the device: ``counts_dev_ptr`` points at
        uint32 [E] rows per expert, written by work that precedes this call in the stream
        (for example ``bmoe_ep_plan``). Nothing is read back: the worklist is built from
        the device counts, the kernel takes the tile total from device memory, the grid is
        the full persistent grid, and the results leave through ``set_push``. ``a`` is
        the packed row buffer (its row count is the capacity). INT8 operands take
        ``row_scale`` and ``col_scale`` as ``initialize_packed`` does."""
        experts = int(w.shape[0])
        n, k = int(w.shape[1]), int(w.shape[2])
        if experts == 0 or int(a.shape[1]) != k or not (a.is_contiguous() and w.is_contiguous()):
            return _capi.INVALID_ARGUMENT
        elem = int(a.element_size())
        if elem != int(w.element_size()) or elem not in (1, 2):
            return _capi.INVALID_ARGUMENT
        if elem == 1:
            options["data_type"] = _byte_type(a, w, row_scale is not None or col_scale is not None)
        if not _scales_fit(options.get("data_type"), a, w, row_scale, col_scale):
            return _capi.INVALID_ARGUMENT
        if row_scale is not None:
            options["col_scale_ptrs"] = _expert_pointers(col_scale)
            options["packed_row_scale"] = row_scale.data_ptr()
        b_ptrs = (np.uint64(w.data_ptr()) +
                  np.arange(experts, dtype=np.uint64) * np.uint64(n * k * elem))
        zeros = np.zeros(experts, dtype=np.uint64)
        self._keep = (a, w, row_scale, col_scale)
        return self.initialize(zeros, b_ptrs, zeros, np.zeros(experts, dtype=np.uint32), n, k,
                               packed_a=a.data_ptr(), packed_rows=int(a.shape[0]),
                               results_pushed=True, tokens_per_expert_dev=counts_dev_ptr,
                               **options)

    # --------------------------------------------------------------- run --
    def run(self, stream=None) -> int:
        return int(self._lib.bmoe_plan_run(self._handle, _stream_ptr(stream)))

    def set_gate(self, flags_ptr, epoch: int, ranks: int, self_rank: int, group_of_ptr) -> int:
        """Hold back the tiles of an expert group until the other ranks' rows of that
        group have arrived (see ``bmoe_plan_set_gate``); ``flags_ptr`` None removes it."""
        return int(self._lib.bmoe_plan_set_gate(self._handle, flags_ptr, epoch, ranks, self_rank,
                                                group_of_ptr))

    def set_gate_copies(self, copy_mask_ptr) -> int:
        """Also hold a group's tiles back until the sources in ``copy_mask[group]`` have
        raised the flags of their peer copies (``bmoe_plan_set_gate_copies``)."""
        return int(self._lib.bmoe_plan_set_gate_copies(self._handle, copy_mask_ptr or None))

    def set_expand(self, records_ptr, counts_ptr, next_ptr, done_ptr, a_ptr, rows_cap: int,
                   row_bytes: int, record_cap: int, groups: int) -> int:
        """Let the launch copy duplicate rows inside the packed A buffer itself (send-once
        exchange, ``bmoe_plan_set_expand``); ``records_ptr`` None switches it off."""
        return int(self._lib.bmoe_plan_set_expand(self._handle, records_ptr or None, counts_ptr,
                                                  next_ptr, done_ptr, a_ptr, rows_cap, row_bytes,
                                                  record_cap, groups))

    def set_push(self, origin_ptr, expert_row_ptr, y_bases_ptr, ranks: int, y_rows_cap: int) -> int:
        """Send result rows straight to their origin ranks' buffers instead of D (see
        ``bmoe_plan_set_push``); ``origin_ptr`` None switches back."""
        return int(self._lib.bmoe_plan_set_push(self._handle, origin_ptr, expert_row_ptr,
                                                y_bases_ptr, ranks, y_rows_cap))

    def poll(self) -> tuple[int, _capi.DeviceReport]:
        report = _capi.DeviceReport()
        status = int(self._lib.bmoe_plan_poll(self._handle, C.byref(report)))
        return status, report

    def stats(self) -> _capi.PlanStats:
        out = _capi.PlanStats()
        self._lib.bmoe_plan_stats_get(self._handle, C.byref(out))
        return out

    def worklist(self) -> np.ndarray:
        """The device worklist copied back to the host (structured array)."""
        total = self.stats().total_tiles
        tiles = (_capi.Tile * max(1, total))()
        count = C.c_uint32(0)
        _capi.check(
            self._lib.bmoe_plan_read_worklist(self._handle, tiles, total, C.byref(count)),
            "bmoe_plan_read_worklist",
        )
        return tiles_to_numpy(tiles, int(count.value))

    def set_observers(self, tile_visits=None, cta_tiles=None) -> int:
        self._observers = (tile_visits, cta_tiles)
        return int(self._lib.bmoe_plan_set_observers(
            self._handle,
            tile_visits.data_ptr() if tile_visits is not None else None,
            cta_tiles.data_ptr() if cta_tiles is not None else None,
        ))


    def set_trace(self, trace=None) -> int:
        """``trace``: CUDA int64 tensor [threadblock_count, 16] of wait-cycle counters."""
        self._trace = trace
        return int(self._lib.bmoe_plan_set_trace(
            self._handle, trace.data_ptr() if trace is not None else None))


def grouped_gemm(a, w, d, tokens_per_expert: Sequence[int], **options) -> None:
    """One-shot packed grouped GEMM on the current CUDA device; raises on error."""
    plan = GroupedGemmPlan()
    try:
        _capi.check(plan.initialize_packed(a, w, d, tokens_per_expert, **options),
                    "bmoe_plan_initialize")
        _capi.check(plan.run(options.get("stream")), "bmoe_plan_run")
        status, report = plan.poll()
        if status != _capi.OK:
            raise _capi.EngineError(status, f"grouped_gemm (site {report.code}, cta {report.cta})")
    finally:
        plan.close()


# ------------------------------------------------------- device worklist --


def worklist_layout(experts: int) -> _capi.WorklistLayout:
    out = _capi.WorklistLayout()
    _capi.check(_capi.load().bmoe_worklist_layout_for(experts, C.byref(out)),
                "bmoe_worklist_layout_for")
    return out


def build_worklist_on_device(counts_dev, n: int, tile_m: int, tile_n: int, *,
                             order: int = _capi.ORDER_EXPERT,
                             raster: int = _capi.RASTER_N_FASTEST,
                             tile_capacity: int, stream=None):
    """Runs the integer worklist kernels on ``counts_dev`` (CUDA int32 tensor).

    Returns ``(tiles, workspace, layout)``: ``tiles`` is a CUDA uint8 tensor of
    ``tile_capacity * 20`` bytes holding the records, ``workspace`` a CUDA uint8
    tensor whose regions ``layout`` describes. Nothing is synchronised.
    """
    import torch

    experts = int(counts_dev.numel())
    layout = worklist_layout(experts)
    device = counts_dev.device
    tiles = torch.empty(max(1, tile_capacity) * 20, dtype=torch.uint8, device=device)
    workspace = torch.empty(layout.bytes + 256, dtype=torch.uint8, device=device)
    base = (workspace.data_ptr() + 255) // 256 * 256
    request = _capi.WorklistRequest(experts=experts, n=n, tile_m=tile_m, tile_n=tile_n,
                                    order=order, raster=raster)
    _capi.check(
        _capi.load().bmoe_worklist_build(
            counts_dev.data_ptr(), C.byref(request), tiles.data_ptr(), tile_capacity,
            base, _stream_ptr(stream)),
        "bmoe_worklist_build",
    )
    offset = base - workspace.data_ptr()
    return tiles, workspace[offset:], layout


def read_worklist_arrays(workspace, layout: _capi.WorklistLayout, experts: int) -> dict:
    """Copies the builder's auxiliary arrays to the host as numpy arrays."""
    raw = workspace.cpu().numpy()

    def view(off: int, dtype: str, count: int) -> np.ndarray:
        width = np.dtype(dtype).itemsize
        return raw[off:off + width * count].view(dtype).copy()

    totals = view(layout.off_totals, "<u4", 8)
    return {
        "total_tiles": int(totals[0]),
        "active_experts": int(totals[1]),
        "total_rows": int(totals[2]) | (int(totals[3]) << 32),
        "total_valid_elements": int(totals[4]) | (int(totals[5]) << 32),
        "overflow": int(totals[6]),
        "row_offsets": view(layout.off_row_offsets, "<u8", experts + 1),
        "expert_m_tiles": view(layout.off_expert_m_tiles, "<u4", experts),
        "expert_tiles": view(layout.off_expert_tiles, "<u4", experts),
        "tile_offsets": view(layout.off_tile_offsets, "<u4", experts + 1),
        "active_ids": view(layout.off_active_ids, "<u4", experts),
        "visit_order": view(layout.off_visit_order, "<u4", experts),
        "visit_tile_offsets": view(layout.off_visit_tile_offsets, "<u4", experts + 1),
    }


# ----------------------------------------------------------------- probe --


def launch_scheduler_probe(scheduler: int, tiles_dev, tile_count: int, cta_count: int, *,
                           claim_size: int = 1, work_scale: int = 1, next_tile=None,
                           tile_visits=None, tile_checksums=None, cta_tile_counts=None,
                           cta_valid_elements=None, stream=None) -> int:
    """``launch_scheduler_probe`` of the reference; tensors are CUDA tensors."""

    def ptr(t):
        return t.data_ptr() if t is not None else None

    args = _capi.ProbeArgs(
        tiles=ptr(tiles_dev), tile_count=tile_count, cta_count=cta_count,
        claim_size=claim_size, work_scale=work_scale, next_tile=ptr(next_tile),
        tile_visits=ptr(tile_visits), tile_checksums=ptr(tile_checksums),
        cta_tile_counts=ptr(cta_tile_counts), cta_valid_elements=ptr(cta_valid_elements),
        stream=_stream_ptr(stream),
    )
    return int(_capi.load().bmoe_probe_launch(scheduler, C.byref(args)))
