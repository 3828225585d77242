"""Calls of the layer operators (section 6 of bmoe_b200.h) and of INT8 plans that are refused:
argument checks come before any CUDA call, so they run without a GPU. Pointers are
numbers that are never read."""

import ctypes as C

import pytest

P = 4096          # an aligned, never dereferenced "device pointer"


def route_args(cap, **change):
    fields = dict(logits_dev=P, bias_dev=None, expert_ids_dev=P, weights_dev=P, tokens=4,
                  row_stride=0, experts=16, top_k=2, logits_type=cap.TYPE_FP32, scoring=0,
                  renormalize=0, scale=1.0, stream=None)
    fields.update(change)
    return cap.RouteTopkArgs(**fields)


@pytest.mark.parametrize("change,want", [
    (dict(logits_type=3), "UNSUPPORTED_DATA_TYPE"),
    (dict(logits_type=1), "UNSUPPORTED_DATA_TYPE"),
    (dict(experts=0), "INVALID_ARGUMENT"),
    (dict(experts=1025, top_k=1), "INVALID_ARGUMENT"),
    (dict(top_k=0), "INVALID_ARGUMENT"),
    (dict(top_k=17), "INVALID_ARGUMENT"),              # more than the experts
    (dict(experts=64, top_k=33), "INVALID_ARGUMENT"),
    (dict(scoring=2), "INVALID_ARGUMENT"),
    (dict(bias_dev=P), "INVALID_ARGUMENT"),            # bias goes with sigmoid scores
    (dict(row_stride=15), "INVALID_ARGUMENT"),
    (dict(tokens=1 << 31), "INVALID_ARGUMENT"),
    (dict(logits_dev=None), "INVALID_ARGUMENT"),
    (dict(logits_dev=P + 2), "INVALID_ARGUMENT"),
    (dict(expert_ids_dev=None), "INVALID_ARGUMENT"),
    (dict(weights_dev=None), "INVALID_ARGUMENT"),
    (dict(expert_ids_dev=P + 4), "INVALID_ARGUMENT"),
    (dict(weights_dev=P + 2), "INVALID_ARGUMENT"),
    (dict(scoring=1, bias_dev=P + 2), "INVALID_ARGUMENT"),
    (dict(tokens=0, logits_dev=None), "OK"),
])
def test_route_topk_checks(engine, change, want):
    cap = engine._capi
    args = route_args(cap, **change)
    assert cap.load().bmoe_route_topk(C.byref(args)) == getattr(cap, want)


def quantize_args(cap, **change):
    fields = dict(src_dev=P, index_dev=None, dst_dev=P, scale_dev=P, rows=4, src_rows=4,
                  src_stride=0, cols=32, src_type=cap.TYPE_BF16, stream=None)
    fields.update(change)
    return cap.QuantizeRowsArgs(**fields)


@pytest.mark.parametrize("change,want", [
    (dict(src_type=3), "UNSUPPORTED_DATA_TYPE"),
    (dict(cols=0), "INVALID_ARGUMENT"),
    (dict(cols=24), "INVALID_ARGUMENT"),
    (dict(src_stride=16), "INVALID_ARGUMENT"),
    (dict(src_stride=36), "INVALID_ARGUMENT"),         # rows would leave the 16-byte grid
    (dict(src_dev=P + 8), "INVALID_ARGUMENT"),
    (dict(dst_dev=P + 8), "INVALID_ARGUMENT"),
    (dict(src_dev=None), "INVALID_ARGUMENT"),
    (dict(dst_dev=None), "INVALID_ARGUMENT"),
    (dict(scale_dev=None), "INVALID_ARGUMENT"),
    (dict(scale_dev=P + 2), "INVALID_ARGUMENT"),
    (dict(index_dev=P + 4), "INVALID_ARGUMENT"),
    (dict(rows=1 << 31, src_rows=1 << 31), "INVALID_ARGUMENT"),
    (dict(rows=5), "INVALID_ARGUMENT"),                # no index: row i is source row i
    (dict(rows=0, src_dev=None), "OK"),
])
def test_quantize_rows_checks(engine, change, want):
    cap = engine._capi
    args = quantize_args(cap, **change)
    assert cap.load().bmoe_quantize_rows(C.byref(args)) == getattr(cap, want)


def decode_args(cap, **change):
    fields = dict(x_dev=P, w_gate_up_dev=P, w_down_dev=P, gate_up_scale_dev=None,
                  down_scale_dev=None, expert_ids_dev=P, weights_dev=P, out_dev=P,
                  workspace_dev=P, workspace_bytes=1 << 40, tokens=4, top_k=2, experts=8,
                  hidden=64, inter=32, data_type=cap.TYPE_BF16, stream=None)
    fields.update(change)
    return cap.MoeDecodeArgs(**fields)


@pytest.mark.parametrize("change,want", [
    (dict(data_type=1), "UNSUPPORTED_DATA_TYPE"),
    (dict(data_type=2), "UNSUPPORTED_DATA_TYPE"),
    (dict(tokens=65), "INVALID_ARGUMENT"),
    (dict(top_k=0), "INVALID_ARGUMENT"),
    (dict(top_k=33), "INVALID_ARGUMENT"),
    (dict(experts=0), "INVALID_ARGUMENT"),
    (dict(experts=1025), "INVALID_ARGUMENT"),
    (dict(hidden=0), "INVALID_ARGUMENT"),
    (dict(hidden=60), "INVALID_ARGUMENT"),
    (dict(hidden=65544), "INVALID_ARGUMENT"),
    (dict(inter=0), "INVALID_ARGUMENT"),
    (dict(inter=65544), "INVALID_ARGUMENT"),
    (dict(inter=12), "INVALID_ARGUMENT"),
    (dict(x_dev=None), "INVALID_ARGUMENT"),
    (dict(x_dev=P + 8), "INVALID_ARGUMENT"),
    (dict(w_gate_up_dev=None), "INVALID_ARGUMENT"),
    (dict(w_down_dev=P + 8), "INVALID_ARGUMENT"),
    (dict(expert_ids_dev=None), "INVALID_ARGUMENT"),
    (dict(weights_dev=None), "INVALID_ARGUMENT"),
    (dict(out_dev=None), "INVALID_ARGUMENT"),
    (dict(workspace_dev=None), "INVALID_ARGUMENT"),
    (dict(workspace_dev=P + 16), "INVALID_ARGUMENT"),
    (dict(workspace_bytes=0), "INVALID_ARGUMENT"),
    (dict(expert_ids_dev=P + 4), "INVALID_ARGUMENT"),
    (dict(weights_dev=P + 1), "INVALID_ARGUMENT"),
    (dict(status_dev=P + 2), "INVALID_ARGUMENT"),
    (dict(data_type=3, gate_up_scale_dev=P + 2, down_scale_dev=P), "INVALID_ARGUMENT"),
    (dict(data_type=3), "INVALID_ARGUMENT"),                       # INT8 without scales
    (dict(data_type=3, gate_up_scale_dev=P), "INVALID_ARGUMENT"),
    (dict(data_type=3, gate_up_scale_dev=P, down_scale_dev=P, hidden=72), "INVALID_ARGUMENT"),
    (dict(data_type=3, gate_up_scale_dev=P, down_scale_dev=P, inter=24), "INVALID_ARGUMENT"),
    (dict(tokens=0, x_dev=None), "OK"),
])
def test_moe_decode_checks(engine, change, want):
    cap = engine._capi
    args = decode_args(cap, **change)
    assert cap.load().bmoe_moe_decode(C.byref(args)) == getattr(cap, want)


def test_moe_decode_workspace_must_hold_the_layer(engine):
    cap = engine._capi
    need = cap.load().bmoe_moe_decode_workspace(4, 2, 32)
    assert need > 0 and need % 256 == 0
    args = decode_args(cap, workspace_bytes=need - 1)
    assert cap.load().bmoe_moe_decode(C.byref(args)) == cap.INVALID_ARGUMENT


def test_null_arguments(engine):
    lib, bad = engine._capi.load(), engine._capi.INVALID_ARGUMENT
    assert lib.bmoe_route_topk(None) == bad
    assert lib.bmoe_quantize_rows(None) == bad
    assert lib.bmoe_moe_decode(None) == bad


def test_int8_plan_checks(engine):
    cap = engine._capi
    plan = engine.GroupedGemmPlan()
    ptr, counts = [4096, 0, 8192], [4, 0, 8]
    scales = dict(row_scale_ptrs=[4096, 0, 4096], col_scale_ptrs=[4096, 0, 4096])
    try:
        def status(n=32, k=32, **options):
            return plan.initialize(ptr, ptr, ptr, counts, n, k, data_type=cap.TYPE_INT8, **options)

        assert status() == cap.INVALID_ARGUMENT                              # no scales
        assert status(row_scale_ptrs=scales["row_scale_ptrs"]) == cap.INVALID_ARGUMENT
        assert status(k=24, **scales) == cap.INVALID_ARGUMENT                # k % 16
        assert status(k=131072, **scales) == cap.INVALID_ARGUMENT            # sums pass 2^31
        assert status(packed_a=4096, packed_rows=12, **scales) == cap.INVALID_ARGUMENT
        assert status(packed_a=4096, packed_rows=12, packed_row_scale=4098,
                      col_scale_ptrs=scales["col_scale_ptrs"]) == cap.INVALID_ARGUMENT
        assert plan.run() == cap.INVALID_ARGUMENT
    finally:
        plan.close()


def test_python_wrappers_refuse_cpu_tensors(engine):
    import torch

    with pytest.raises(ValueError):
        engine.route_topk(torch.zeros(2, 8), 2)
    with pytest.raises(ValueError):
        engine.quantize_rows(torch.zeros(2, 16))
    with pytest.raises(ValueError):
        engine.moe_decode(torch.zeros(2, 16), None, None, None, None)


def test_packed_calls_reach_the_same_checks(engine):
    """The wrappers pass a struct's bytes: the layout is that of the ctypes structure."""
    cap = engine._capi
    for name, layout, args in (("bmoe_route_topk", cap.RouteTopkArgs, route_args(cap)),
                               ("bmoe_quantize_rows", cap.QuantizeRowsArgs, quantize_args(cap)),
                               ("bmoe_moe_decode", cap.MoeDecodeArgs, decode_args(cap))):
        call = cap.entry(name, layout)
        fields = [getattr(args, field) or 0 for field, _ in layout._fields_]
        names = [field for field, _ in layout._fields_]
        tokens = names.index("tokens" if "tokens" in names else "rows")
        assert call(*(0 if i == tokens else v for i, v in enumerate(fields))) == cap.OK
        last = names.index({"bmoe_route_topk": "top_k", "bmoe_quantize_rows": "cols",
                            "bmoe_moe_decode": "inter"}[name])
        assert call(*(7777777 if i == last else v for i, v in enumerate(fields))) == \
            cap.INVALID_ARGUMENT
        with pytest.raises(ValueError):
            call(*(-1 if i == last else v for i, v in enumerate(fields)))
        with pytest.raises(ValueError):
            call(*fields[:-1])


def test_inputs_that_require_a_gradient_are_refused(engine):
    """There is no backward pass, so a result cut off from the graph would be a silent zero."""
    import torch

    def leaf(*shape):
        return torch.zeros(*shape, requires_grad=True)

    x, w1, w2 = torch.zeros(2, 16), torch.zeros(4, 32, 16), torch.zeros(4, 16, 16)
    ids, coef = torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, 2)
    calls = (lambda: engine.route_topk(leaf(2, 8), 2),
             lambda: engine.route_topk(torch.zeros(2, 8), 2, scoring="sigmoid", bias=leaf(8)),
             lambda: engine.quantize_rows(leaf(2, 16)),
             lambda: engine.moe_decode(leaf(2, 16), w1, w2, ids, coef),
             lambda: engine.moe_decode(x, leaf(4, 32, 16), w2, ids, coef),
             lambda: engine.moe_decode(x, w1, leaf(4, 16, 16), ids, coef),
             lambda: engine.moe_decode(x, w1, w2, ids, leaf(2, 2)),
             lambda: engine.moe_decode(x, w1, w2, ids, coef, gate_up_scale=leaf(4, 32)),
             lambda: engine.moe_decode(x, w1, w2, ids, coef, down_scale=leaf(4, 16)))
    for call in calls:
        with pytest.raises(ValueError, match="backward"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="no CPU path"):
            call()


def run_alone(code):
    """``code`` in an interpreter of its own, from the repository's root."""
    import subprocess
    import sys
    from pathlib import Path

    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                          cwd=Path(__file__).resolve().parent.parent, timeout=300)
    assert done.returncode == 0, done.stderr


def test_the_package_imports_without_torch():
    """Planner, C binding and CSV helpers never need it; the layer operators at their first call."""
    run_alone("""
import sys
sys.modules["torch"] = None                      # import torch raises ModuleNotFoundError
import bmoe_b200
assert bmoe_b200.moe_decode_workspace(4, 2, 32) > 0
assert bmoe_b200.host_tiles([5, 0, 9], 256, 128, 256)[1] == 2
try:
    bmoe_b200.route_topk(None, 2)
except ModuleNotFoundError:
    pass
else:
    raise AssertionError("no error")
""")


def test_the_package_imports_beside_a_torch_without_cuda():
    run_alone("""
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
import bmoe_b200
try:
    bmoe_b200.route_topk(torch.zeros(2, 8), 2)
except ValueError:
    pass
else:
    raise AssertionError("no error")
""")
