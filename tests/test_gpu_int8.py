"""INT8 grouped GEMM with a scale per row and per output channel, against exact sums in 64
bits: the integer sums are exact, the result is float(sum) * (row_scale * col_scale) - three
FP32 roundings (2^-24 each, relative) - and one BF16 rounding (2^-8). The reference has no
integer type."""

import numpy as np
import pytest
import torch

from test_gpu_gemm import POLICIES

pytestmark = pytest.mark.gpu

CASES = [
    # counts, n, k
    ([1], 8, 16),
    ([128], 256, 128),
    ([129, 0, 1, 255], 264, 80),
    ([37, 0, 1, 200], 384, 192),
    ([300, 5, 0, 300, 129], 520, 448),
    ([65, 67, 68, 61, 63, 57, 61, 70], 1024, 512),
    ([3] * 40 + [0] * 20 + [500], 256, 1024),
]


def make_int8(counts, n, k, seed=2026):
    g = torch.Generator().manual_seed(seed)
    rows, experts = sum(counts), len(counts)
    a = torch.randint(-127, 128, (rows, k), generator=g).to(torch.int8)
    w = torch.randint(-127, 128, (experts, n, k), generator=g).to(torch.int8)
    row = torch.exp(torch.randn(rows, generator=g) * 2) * 1e-3
    col = torch.exp(torch.randn(experts, n, generator=g) * 2) * 1e-3
    return a, w, row, col


def exact(a, w, row, col, counts):
    out, first = [], 0
    for e, c in enumerate(counts):
        sums = a[first:first + c].double() @ w[e].double().t()     # below 2^53: exact
        out.append(sums * row[first:first + c].double()[:, None] * col[e].double())
        first += c
    return torch.cat(out)


def run_int8(engine, a, w, row, col, counts, policy="expert_order", output_f32=False, **options):
    d = torch.full((max(1, sum(counts)), w.shape[1]), float("nan"),
                   dtype=torch.float32 if output_f32 else torch.bfloat16,
                   device="cuda")[:sum(counts)]
    keep = [t.cuda() for t in (a, w, row, col)]
    plan = engine.GroupedGemmPlan()
    try:
        status = plan.initialize_packed(keep[0], keep[1], d, counts, scheduler=policy,
                                        row_scale=keep[2], col_scale=keep[3],
                                        output_f32=output_f32, **options)
        assert status == 0, engine._capi.status_string(status)
        visits = torch.zeros(plan.stats().total_tiles, dtype=torch.int32, device="cuda")
        assert plan.set_observers(visits, None) == 0
        assert plan.run() == 0
        status, report = plan.poll()
        assert status == 0, (engine._capi.status_string(status), report.code)
        assert torch.all(visits == 1)
        return d.cpu()
    finally:
        plan.close()


def check(got, want, half_steps):
    off = (got.double() - want).abs()
    assert torch.all(off <= want.abs() * half_steps), (off / want.abs().clamp(min=1e-30)).max()


@pytest.mark.parametrize("counts,n,k", CASES)
def test_int8_ragged_cases_all_variants(engine, counts, n, k):
    a, w, row, col = make_int8(counts, n, k)
    want = exact(a, w, row, col, counts)
    base = run_int8(engine, a, w, row, col, counts, raster_along_m=0)
    check(base, want, 2.0 ** -8 + 4 * 2.0 ** -24)
    for tile_n, group in ((64, 1), (128, 1), (256, 1), (256, 2)):
        for raster in (0, 1):
            for policy, opts in POLICIES:
                out = run_int8(engine, a, w, row, col, counts, policy, tile_n=tile_n,
                               cta_group=group, raster_along_m=raster, **opts)
                assert torch.equal(out, base), (policy, opts, tile_n, group, raster)


@pytest.mark.parametrize("group", [1, 2])
@pytest.mark.parametrize("counts,n,k", CASES)
def test_int8_fp32_output(engine, counts, n, k, group):
    a, w, row, col = make_int8(counts, n, k, seed=7)
    out = run_int8(engine, a, w, row, col, counts, output_f32=True, cta_group=group)
    check(out, exact(a, w, row, col, counts), 4 * 2.0 ** -24)


@pytest.mark.parametrize("single", [False, True])
def test_int8_extremes_are_exact(engine, single):
    """-128 included, sums up to 2^30, and a sum that needs all 31 bits."""
    k = 16384
    a = torch.full((5, k), -128, dtype=torch.int8)
    a[1] = 127
    a[2, ::2] = 127
    a[3] = 0
    a[4, : k // 2] = 1
    w = torch.full((1, 16, k), -128, dtype=torch.int8)
    w[0, 1] = 127
    w[0, 2, ::2] = 1
    row, col = torch.ones(5), torch.ones(1, 16)
    out = run_int8(engine, a, w, row, col, [5], output_f32=True, single_a_map=single)
    sums = a.double() @ w[0].double().t()
    assert torch.equal(out, sums.float())              # one rounding, scales of one


def test_int8_largest_k(engine):
    k = 131056                                          # largest multiple of 16 within the limit
    a = torch.full((2, k), -128, dtype=torch.int8)
    w = torch.full((1, 8, k), -128, dtype=torch.int8)
    w[0, 1] = 127
    out = run_int8(engine, a, w, torch.ones(2), torch.ones(1, 8), [2], output_f32=True)
    assert torch.equal(out, (a.double() @ w[0].double().t()).float())


def test_int8_scales_that_are_zero_or_not_finite(engine):
    counts, n, k = [70, 3], 136, 64
    a, w, row, col = make_int8(counts, n, k)
    row[5], row[6], row[71] = float("nan"), float("inf"), 0.0
    col[0, 9], col[1, 0] = 0.0, float("nan")
    out = run_int8(engine, a, w, row, col, counts)
    assert torch.isnan(out[5]).all() and not torch.isfinite(out[6]).any()
    assert torch.all(out[71, 1:] == 0) and torch.isnan(out[70:, 0]).all()
    fine = torch.ones(73, dtype=torch.bool)
    fine[[5, 6]] = False
    assert torch.all(out[:70][fine[:70]][:, 9] == 0)
    assert torch.isfinite(out[fine][:, 1:]).all()


def test_int8_packed_descriptor_replans_and_type_changes(engine):
    """One plan through INT8, BF16 and other counts; the packed form reads one scale array."""
    plan = engine.GroupedGemmPlan()
    try:
        for seed, counts, single in ((1, [40, 0, 131], False), (2, [200, 9, 0], True),
                                     (3, [1, 1, 1], True)):
            n, k = 272, 96
            a, w, row, col = (t.cuda() for t in make_int8(counts, n, k, seed))
            d = torch.empty(sum(counts), n, dtype=torch.bfloat16, device="cuda")
            assert plan.initialize_packed(a, w, d, counts, scheduler="auto", row_scale=row,
                                          col_scale=col, single_a_map=single) == 0
            for _ in range(2):
                d.fill_(float("nan"))
                assert plan.run() == 0 and plan.poll()[0] == 0
                check(d.cpu(), exact(a.cpu(), w.cpu(), row.cpu(), col.cpu(), counts),
                      2.0 ** -8 + 4 * 2.0 ** -24)
            half = torch.randn(sum(counts), k, device="cuda").to(torch.bfloat16)
            full = torch.randn(3, n, k, device="cuda").to(torch.bfloat16)
            assert plan.initialize_packed(half, full, d, counts) == 0
            assert plan.run() == 0 and plan.poll()[0] == 0
            first = 0
            for e, c in enumerate(counts):
                torch.testing.assert_close(d[first:first + c].float(),
                                           half[first:first + c].float() @ full[e].float().t(),
                                           rtol=2.0 ** -7, atol=0.05)
                first += c
    finally:
        plan.close()


def test_int8_counts_on_the_device_and_pushed_results(engine):
    counts, n, k = [33, 0, 190, 7], 264, 128
    a, w, row, col = (t.cuda() for t in make_int8(counts, n, k, seed=4))
    total, cap = sum(counts), sum(counts) + 50
    padded = torch.zeros(cap, k, dtype=torch.int8, device="cuda")
    padded[:total] = a
    scales = torch.full((cap,), float("nan"), device="cuda")
    scales[:total] = row
    counts_dev = torch.tensor(counts, dtype=torch.int32, device="cuda")
    order = torch.randperm(total, generator=torch.Generator().manual_seed(1)).cuda()
    out = torch.full((total, n), float("nan"), dtype=torch.bfloat16, device="cuda")
    bases = torch.tensor([out.data_ptr()], dtype=torch.int64, device="cuda")
    first = torch.tensor([0, 33, 33, 223], dtype=torch.int32, device="cuda")
    plan = engine.GroupedGemmPlan()
    try:
        assert plan.initialize_packed_device_counts(
            padded, w, counts_dev.data_ptr(), row_scale=scales, col_scale=col) == 0
        assert plan.set_push(order.data_ptr(), first.data_ptr(), bases.data_ptr(), 1, total) == 0
        assert plan.run() == 0 and plan.poll()[0] == 0
    finally:
        plan.close()
    want = exact(a.cpu(), w.cpu(), row.cpu(), col.cpu(), counts)
    check(out.cpu()[order.cpu()], want, 2.0 ** -8 + 4 * 2.0 ** -24)


def test_int8_needs_scales_and_matching_types(engine):
    a, w, row, col = (t.cuda() for t in make_int8([4], 32, 32))
    d = torch.empty(4, 32, dtype=torch.bfloat16, device="cuda")
    plan = engine.GroupedGemmPlan()
    bad = engine._capi.INVALID_ARGUMENT
    try:
        assert plan.initialize_packed(a, w, d, [4], row_scale=row) == bad
        assert plan.initialize_packed(a, w, d, [4], col_scale=col) == bad
        assert plan.initialize_packed(a, w, d, [4], row_scale=row, col_scale=col[:, :8]) == bad
        assert plan.initialize_packed(a, w, d, [4], row_scale=row[:2], col_scale=col) == bad
        assert plan.initialize_packed(a, w, d, [4], row_scale=row.double(), col_scale=col) == bad
        assert plan.initialize_packed(a, w.view(torch.uint8), d, [4], row_scale=row,
                                      col_scale=col) == bad
        assert plan.initialize_packed(a.view(torch.uint8), w.view(torch.uint8), d, [4],
                                      row_scale=row, col_scale=col) == bad
        # bytes without scales are FP8 bit patterns, whatever the tensors' type is called
        assert plan.initialize_packed(a, w, d, [4]) == 0
    finally:
        plan.close()


def test_quantised_layer_as_it_is_used(engine):
    """Router, gathered 8-bit rows, INT8 gate-up and down products, top-k combine, against the
    few-token layer on the same 8-bit weights. The two differ by the quantisation of x and of
    h: at most half a step of 1/127 of a row's largest value per element, bounded below with
    the row's absolute sums in 64 bits, plus BF16 roundings of each stage."""
    from bmoe_b200 import ep

    tokens, experts, top_k, hidden, inter = 48, 6, 2, 256, 192
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(tokens, hidden, generator=g, device="cuda").to(torch.bfloat16)
    w1 = torch.randint(-127, 128, (experts, 2 * inter, hidden), generator=g,
                       device="cuda").to(torch.int8)
    w2 = torch.randint(-127, 128, (experts, hidden, inter), generator=g,
                       device="cuda").to(torch.int8)
    s1 = torch.rand(experts, 2 * inter, generator=g, device="cuda") * 1e-3
    s2 = torch.rand(experts, hidden, generator=g, device="cuda") * 1e-3
    ids, coef = engine.route_topk(torch.randn(tokens, experts, generator=g, device="cuda"),
                                  top_k, renormalize=True)
    flat = ids.reshape(-1)
    order = torch.argsort(flat, stable=True)
    counts = torch.bincount(flat, minlength=experts).tolist()
    q, row = engine.quantize_rows(x, order // top_k)
    both = torch.empty(tokens * top_k, 2 * inter, dtype=torch.bfloat16, device="cuda")
    engine.grouped_gemm(q, w1, both, counts, row_scale=row, col_scale=s1)
    gate, up = both.float().chunk(2, 1)
    h = (gate * torch.sigmoid(gate) * up).to(torch.bfloat16)
    hq, hrow = engine.quantize_rows(h)
    part = torch.empty(tokens * top_k, hidden, dtype=torch.bfloat16, device="cuda")
    engine.grouped_gemm(hq, w2, part, counts, row_scale=hrow, col_scale=s2)
    rows = torch.empty_like(order)
    rows[order] = torch.arange(tokens * top_k, device="cuda")
    combined = ep.CudaOps().combine_topk(part, rows.reshape(tokens, top_k), coef)
    torch.cuda.synchronize()
    few = engine.moe_decode(x, w1, w2, ids, coef, gate_up_scale=s1, down_scale=s2)

    bound = torch.zeros(tokens, hidden, dtype=torch.float64)
    half16 = 2.0 ** -8
    for t in range(tokens):
        for j in range(top_k):
            e = int(ids[t, j])
            f1 = w1[e].double().cpu() * s1[e].double().cpu()[:, None]
            f2 = w2[e].double().cpu() * s2[e].double().cpu()[:, None]
            v = x[t].double().cpu()
            y = f1 @ v
            dy = f1.abs().sum(1) * float(v.abs().max()) / 254 + (y.abs() + 1e-9) * half16
            dy = dy * 1.01
            gt, u = y[:inter], y[inter:]
            silu = gt * torch.sigmoid(gt)
            hh = silu * u
            dh = 1.1 * dy[:inter] * (u.abs() + dy[inter:]) + silu.abs() * dy[inter:]
            dh = dh + (hh.abs() + dh) * half16
            dh = dh + (hh.abs() + dh).max() / 254 * 1.01
            c = float(coef[t, j])
            bound[t] += c * (f2.abs() @ dh + (f2 @ hh).abs() * half16 * 1.01
                             + (f2.abs() @ dh) * half16)
    off = (combined.double() - few.double()).abs().cpu()
    assert torch.all(off <= bound + 2 * half16 * (few.double().abs().cpu() + bound)), \
        (off / bound).max()
    # the worst case of both quantisations is wide; each product is checked against exact sums
    # of the very integers it was given, and the combine against the rows it was given
    check(both.cpu(), exact(q.cpu(), w1.cpu(), row.cpu(), s1.cpu(), counts),
          half16 + 4 * 2.0 ** -24)
    check(part.cpu(), exact(hq.cpu(), w2.cpu(), hrow.cpu(), s2.cpu(), counts),
          half16 + 4 * 2.0 ** -24)
    want = (part[rows].reshape(tokens, top_k, hidden).double() * coef.double()[:, :, None])
    size = want.abs().sum(1)
    want = want.sum(1)
    assert torch.all((combined.double() - want).abs() <= want.abs() * half16
                     + size * top_k * 2.0 ** -23)


def test_int8_type_needs_one_byte_operands(engine):
    a = torch.zeros(16, 32, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(1, 8, 32, dtype=torch.bfloat16, device="cuda")
    d = torch.zeros(16, 8, dtype=torch.bfloat16, device="cuda")
    scales = dict(row_scale=torch.ones(16, device="cuda"), col_scale=torch.ones(1, 8, device="cuda"))
    plan = engine.GroupedGemmPlan()
    try:
        assert plan.initialize_packed(a, w, d, [16], data_type=3, **scales) == \
            engine._capi.INVALID_ARGUMENT
    finally:
        plan.close()


def test_plan_recaptured_on_another_stream(engine):
    """A plan that was set up eagerly on one stream is set up again while another stream is
    captured (relaxed mode): the graph holds set-up and launch and replays on new inputs."""
    counts, n, k = [37, 0, 1, 200], 384, 192
    a, w, row, col = make_int8(counts, n, k)
    dev = [t.cuda() for t in (a, w, row, col)]
    d = torch.zeros(sum(counts), n, dtype=torch.bfloat16, device="cuda")
    plan, side = engine.GroupedGemmPlan(), torch.cuda.Stream()
    try:
        for _ in range(2):
            assert plan.initialize_packed(dev[0], dev[1], d, counts, row_scale=dev[2],
                                          col_scale=dev[3], stream=None) == 0
            assert plan.run() == 0
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
            assert plan.initialize_packed(dev[0], dev[1], d, counts, row_scale=dev[2],
                                          col_scale=dev[3], stream=side) == 0
            assert plan.run(side) == 0
        for seed in (5, 6):
            a = make_int8(counts, n, k, seed=seed)[0]
            dev[0].copy_(a)
            d.fill_(float("nan"))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            check(d.cpu(), exact(a, w, row, col, counts), 2.0 ** -8 + 4 * 2.0 ** -24)
        del graph
    finally:
        torch.cuda.synchronize()
        plan.close()
