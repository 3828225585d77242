"""The operators either side of the grouped GEMM on the GPU - router choice, row quantiser,
few-token expert layer - against plain 64-bit forms. Half a step of a type, relative:
FP32 2^-24, BF16 2^-8; every tolerance counts these."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF32, HALF16 = 2.0 ** -24, 2.0 ** -8


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ router --


def route_oracle(logits, top_k, scoring, renormalize, bias, scale):
    """Choice and weights of every row in 64 bits, by a stable sort of (key, id)."""
    x = logits.double().cpu().numpy()
    tokens, experts = x.shape
    ids = np.full((tokens, top_k), -1, dtype=np.int64)
    weights = np.zeros((tokens, top_k))
    for t in range(tokens):
        with np.errstate(over="ignore"):
            sig = 1.0 / (1.0 + np.exp(-x[t]))
        key = x[t] if bias is None else sig + bias.double().cpu().numpy()
        live = ~np.isnan(x[t]) & (x[t] > -np.inf) & ~np.isnan(key) & (key > -np.inf)
        order = sorted(np.nonzero(live)[0], key=lambda e: (-key[e], e))[:top_k]
        if not order:
            continue
        if scoring == "softmax":
            alive = ~np.isnan(x[t]) & (x[t] > -np.inf)
            most = x[t][alive].max()
            part = np.array([1.0 if v == most else math.exp(v - most) for v in x[t][alive]])
            chosen = np.array([1.0 if x[t][e] == most else math.exp(x[t][e] - most)
                               for e in order]) / part.sum()
        else:
            chosen = sig[order]
        if renormalize:
            chosen = chosen / chosen.sum() if chosen.sum() > 0 else chosen * 0.0
        ids[t, :len(order)] = order
        weights[t, :len(order)] = chosen * scale
    return ids, weights


def check_route(engine, logits, top_k, scoring="softmax", renormalize=False, bias=None,
                scale=1.0):
    ids, weights = engine.route_topk(logits.cuda() if not logits.is_cuda else logits, top_k,
                                     scoring=scoring, renormalize=renormalize,
                                     bias=None if bias is None else bias.cuda(), scale=scale)
    want_ids, want = route_oracle(logits, top_k, scoring, renormalize, bias, scale)
    assert ids.dtype is torch.int64 and weights.dtype is torch.float32
    np.testing.assert_array_equal(ids.cpu().numpy(), want_ids)
    # exp of a 32-bit difference d: relative error |d| half steps from rounding d (|d| <= spread
    # of the row) and 2 from the function; as much again for the sum it is divided by, plus
    # the roundings of a sum of E terms (tree: log2 E + E/32), a division, a product
    finite = torch.where(torch.isfinite(logits.double()), logits.double(), 0.0)
    spread = float((finite.amax(1) - finite.amin(1)).max()) if logits.numel() else 0.0
    experts = logits.shape[1]
    tol = (2 * (spread + 2) + experts / 32 + 5 + 8) * HALF32
    got = weights.double().cpu().numpy()
    # below 2^-126 the 32-bit weight has fewer bits
    assert np.all(np.abs(got - want) <= tol * np.abs(want) + 2.0 ** -140), \
        np.abs(got / np.where(want == 0, 1, want) - 1).max()
    return ids, weights


@pytest.mark.parametrize("tokens,experts,top_k", [
    (1, 1, 1), (1, 8, 2), (3, 5, 5), (4, 256, 8), (7, 63, 6), (5, 65, 32), (129, 128, 8),
    (33, 160, 7), (2, 257, 9), (9, 1024, 32), (1000, 33, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scoring,with_bias", [("softmax", False), ("sigmoid", False),
                                               ("sigmoid", True)])
def test_route_topk(engine, tokens, experts, top_k, dtype, scoring, with_bias):
    g = gen(tokens * 1000 + experts)
    logits = (torch.randn(tokens, experts, generator=g) * 2).to(dtype)
    bias = torch.randn(experts, generator=g) * 0.1 if with_bias else None
    for renormalize, scale in ((False, 1.0), (True, 2.5)):
        check_route(engine, logits, top_k, scoring, renormalize, bias, scale)


@pytest.mark.parametrize("experts", [40, 200])
def test_route_topk_ties_go_to_the_lowest_id(engine, experts):
    g = gen(7)
    coarse = torch.randint(-2, 3, (64, experts), generator=g).float()
    coarse[0] = 0.0
    coarse[1, ::2] = -0.0           # both zeros are one value
    coarse[1, 1::2] = 0.0
    coarse[2] = -1.5
    check_route(engine, coarse, 6)
    check_route(engine, coarse.to(torch.bfloat16), 6, renormalize=True)
    check_route(engine, coarse, 6, "sigmoid", bias=torch.zeros(experts))
    check_route(engine, coarse, 6, "sigmoid", bias=torch.randint(0, 2, (experts,),
                                                                 generator=g).float())


def test_route_topk_sums_closer_than_32_bits_tell(engine):
    """sigmoid + bias of neighbours that differ by less than an FP32 step of the sum."""
    experts = 96
    logits = torch.zeros(8, experts)
    # biases step by 2^-26, logits by 2^-24 steps around 0: sums differ in bits 26 and lower
    bias = 1.0 + torch.zeros(experts)
    for t in range(8):
        logits[t] = torch.randperm(experts, generator=gen(t)).float() * 2.0 ** -23
    check_route(engine, logits, 8, "sigmoid", True, bias)
    logits = torch.randn(64, 1, generator=gen(1)).repeat(1, experts)
    logits += torch.randint(-3, 4, (64, experts), generator=gen(2)).float() * 1e-7
    check_route(engine, logits, 8, "sigmoid", False, torch.zeros(experts) + 0.25)


def test_route_topk_switched_off_experts_nan_and_infinities(engine):
    inf, nan = math.inf, math.nan
    logits = torch.randn(12, 20, generator=gen(3))
    logits[:, [0, 7, 19]] = -inf
    logits[1] = -inf                                   # nothing to choose
    logits[2] = nan
    logits[3, 2:] = -inf                               # fewer live experts than top_k
    logits[4, 5] = nan
    logits[5, 4] = inf
    logits[6, [3, 11]] = inf                           # two infinities share the softmax
    logits[7] = torch.finfo(torch.float32).min         # the lowest value is still a value
    logits[8] = torch.finfo(torch.float32).max
    for scoring, bias in (("softmax", None), ("sigmoid", None), ("sigmoid", torch.zeros(20))):
        for renormalize in (False, True):
            row_wise = [check_route(engine, logits[t:t + 1], 4, scoring, renormalize, bias)
                        for t in range(12)]
            ids, weights = engine.route_topk(logits.cuda(), 4, scoring=scoring,
                                             renormalize=renormalize,
                                             bias=None if bias is None else bias.cuda())
            assert torch.equal(ids, torch.cat([r[0] for r in row_wise]))
            assert torch.equal(weights, torch.cat([r[1] for r in row_wise]))
    assert ids[1].tolist() == [-1] * 4 and weights[1].tolist() == [0.0] * 4
    off = torch.zeros(20)
    off[3], off[4] = nan, -inf                         # switched off through the bias
    check_route(engine, torch.randn(9, 20, generator=gen(4)), 18, "sigmoid", True, off)


def test_route_topk_strided_rows_and_given_outputs(engine):
    wide = torch.randn(50, 100, generator=gen(5)).cuda()
    part = wide[:, 3:70]                               # rows 100 apart, first column odd
    ids = torch.full((50, 4), 99, dtype=torch.int64, device="cuda")
    weights = torch.zeros(50, 4, device="cuda")
    out = engine.route_topk(part, 4, expert_ids=ids, weights=weights)
    assert out[0] is ids and out[1] is weights
    want_ids, _ = route_oracle(part, 4, "softmax", False, None, 1.0)
    np.testing.assert_array_equal(ids.cpu().numpy(), want_ids)
    check_route(engine, wide.to(torch.bfloat16)[::3, 1:34], 5)
    empty = engine.route_topk(wide[:0], 4)
    assert empty[0].shape == (0, 4)


def test_wrappers_refuse_what_does_not_fit(engine):
    x = torch.zeros(4, 32, device="cuda")
    for call in (lambda: engine.route_topk(x.double(), 2),
                 lambda: engine.route_topk(x.t(), 2),
                 lambda: engine.route_topk(x, 2, scoring="other"),
                 lambda: engine.route_topk(x, 2, scoring="sigmoid", bias=torch.zeros(32)),
                 lambda: engine.quantize_rows(x.half()),
                 lambda: engine.quantize_rows(x, torch.zeros(4, device="cuda")),
                 lambda: engine.quantize_rows(x, out=torch.zeros(4, 32, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(engine._capi.EngineError):
        engine.route_topk(x, 33)
    with pytest.raises(engine._capi.EngineError):
        engine.quantize_rows(x[:, :24])


# --------------------------------------------------------------- quantiser --


def quantize_oracle(x):
    """The definition, operation by operation in FP32."""
    x = x.float().cpu().numpy()
    largest = np.maximum(np.abs(x).max(1), np.float32(2.0 ** -100)).astype(np.float32)
    inverse = np.float32(127.0) * (np.float32(1.0) / largest).astype(np.float32)
    q = np.rint((x * inverse[:, None]).astype(np.float32))
    return np.clip(q, -127, 127).astype(np.int8), (largest / np.float32(127.0)).astype(np.float32)


@pytest.mark.parametrize("rows,cols", [
    (1, 16), (3, 48), (5, 512), (2, 2048), (300, 272), (7, 7168), (4, 4112), (2, 16384),
    (3, 20000), (2, 40016), (2500, 64), (9, 3008), (2, 70016), (6, 6400)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_rows(engine, rows, cols, dtype):
    g = gen(rows + cols)
    x = torch.randn(rows, cols, generator=g) * torch.exp(3 * torch.randn(rows, 1, generator=g))
    x = x.to(dtype)
    q, scale = engine.quantize_rows(x.cuda())
    want_q, want_scale = quantize_oracle(x)
    np.testing.assert_array_equal(q.cpu().numpy(), want_q)
    np.testing.assert_array_equal(scale.cpu().numpy(), want_scale)
    index = torch.randint(0, rows, (rows + 5,), generator=g)
    q, scale = engine.quantize_rows(x.cuda(), index.cuda())
    np.testing.assert_array_equal(q.cpu().numpy(), want_q[index.numpy()])
    np.testing.assert_array_equal(scale.cpu().numpy(), want_scale[index.numpy()])


def test_quantize_rows_ends_of_the_range(engine):
    x = torch.zeros(10, 64)
    x[1] = 2.0 ** -130                                  # below the floor: zeros
    x[2, 5] = 2.0 ** -100                               # at the floor
    x[3] = torch.finfo(torch.float32).max
    x[4] = torch.linspace(-127, 127, 64) / 127.0
    x[5] = 0.5
    x[5, 0] = 127.0                                     # 0.5 steps: ties go to even
    x[5, 1:8] = torch.tensor([1.5, 2.5, -0.5, -1.5, -2.5, 126.5, -126.5])
    x[6, 63] = -3.0
    x[7, 9] = math.inf
    x[8, 9] = math.nan
    x[9, 0], x[9, 1] = -math.inf, math.nan
    q, scale = engine.quantize_rows(x.cuda())
    fine = slice(0, 7)
    want_q, want_scale = quantize_oracle(x[fine])
    np.testing.assert_array_equal(q[fine].cpu().numpy(), want_q)
    np.testing.assert_array_equal(scale[fine].cpu().numpy(), want_scale)
    assert scale[7].item() == math.inf
    assert math.isnan(scale[8].item()) and math.isnan(scale[9].item())
    assert int(q.abs().max()) <= 127


def test_quantize_rows_bad_indices_leave_rows_alone_and_rows_may_be_strided(engine):
    base = torch.randn(20, 160, generator=gen(1)).to(torch.bfloat16).cuda()
    x = base[:, 32:96]                                  # rows 160 apart
    index = torch.tensor([3, -1, 19, 20, 0, 1 << 40, -(1 << 40)], device="cuda")
    out = torch.full((7, 64), 77, dtype=torch.int8, device="cuda")
    scale = torch.full((7,), 5.0, device="cuda")
    engine.quantize_rows(x, index, out=out, scale=scale)
    want_q, want_scale = quantize_oracle(x)
    for i, src in ((0, 3), (2, 19), (4, 0)):
        np.testing.assert_array_equal(out[i].cpu().numpy(), want_q[src])
        assert scale[i].item() == want_scale[src]
    for i in (1, 3, 5, 6):
        assert torch.all(out[i] == 77) and scale[i].item() == 5.0
    every_other, _ = engine.quantize_rows(base[::2])
    np.testing.assert_array_equal(every_other.cpu().numpy(), quantize_oracle(base[::2])[0])


# ---------------------------------------------------------- few-token layer --


def make_layer(tokens, experts, top_k, hidden, inter, int8, seed, drop=0.0):
    g = gen(seed)
    x = torch.randn(tokens, hidden, generator=g).to(torch.bfloat16)
    w1 = torch.randn(experts, 2 * inter, hidden, generator=g) * hidden ** -0.5
    w2 = torch.randn(experts, hidden, inter, generator=g) * inter ** -0.5
    layer = {"x": x}
    if int8:
        for name, w in (("1", w1), ("2", w2)):
            scale = w.abs().amax(2) / 127
            layer["w" + name] = torch.round(w / scale[..., None]).to(torch.int8)
            layer["s" + name] = scale
    else:
        layer.update(w1=w1.to(torch.bfloat16), w2=w2.to(torch.bfloat16), s1=None, s2=None)
    ids = torch.stack([torch.randperm(max(experts, top_k), generator=g)[:top_k]
                       for _ in range(tokens)])
    ids[torch.rand(tokens, top_k, generator=g) < drop] = -1
    ids[ids >= experts] = experts + 3
    layer["ids"] = ids
    layer["coef"] = torch.rand(tokens, top_k, generator=g) + 0.05
    return layer


def run_layer(engine, layer, **options):
    to = {k: (v.cuda() if v is not None else None) for k, v in layer.items()}
    return engine.moe_decode(to["x"], to["w1"], to["w2"], to["ids"], to["coef"],
                             gate_up_scale=to["s1"], down_scale=to["s2"], **options)


def layer_oracle(layer):
    """out[t] in 64 bits and a bound of the operator's error.

    Sums of K products in FP32: a product of two BF16 (or of a BF16 and an 8-bit integer) is
    exact, a sum's error is at most (additions in a row + 16) steps of its terms' magnitudes;
    one accumulator takes 16 products at a time (K / 16 additions in a row; the joins of
    parallel accumulators and the rounding inside a 16-term sum are in the 16). h keeps 16
    bits, silu and the products around it cost 8 half steps; the slope of silu is below 1.1;
    the result is rounded to BF16 once."""
    x = layer["x"].double()
    tokens, hidden = x.shape
    experts, inter = layer["w1"].shape[0], layer["w2"].shape[2]
    out = torch.zeros(tokens, hidden, dtype=torch.float64)
    err = torch.zeros(tokens, hidden, dtype=torch.float64)
    step = 2 * HALF32
    for t in range(tokens):
        for j, e in enumerate(layer["ids"][t].tolist()):
            if not 0 <= e < experts:
                continue
            w1, w2 = layer["w1"][e].double(), layer["w2"][e].double()
            if layer["s1"] is not None:
                w1 = w1 * layer["s1"][e].double()[:, None]
                w2 = w2 * layer["s2"][e].double()[:, None]
            both, size = w1 @ x[t], w1.abs() @ x[t].abs()
            both_err = size * (hidden / 16 + 16) * step * 2
            gate, up = both[:inter], both[inter:]
            silu = gate / (1 + torch.exp(-gate))
            h = silu * up
            h_err = (1.1 * both_err[:inter] * (up.abs() + both_err[inter:])
                     + silu.abs() * both_err[inter:] + h.abs() * (2.0 ** -16 + 8 * HALF32))
            c = float(layer["coef"][t, j].double())
            out[t] += c * (w2 @ h)
            err[t] += abs(c) * (w2.abs() @ (h_err + h.abs() * (inter / 16 + 24) * step * 2))
    return out, err + out.abs() * HALF16 + 2.0 ** -133


def check_layer(engine, layer, **options):
    got = run_layer(engine, layer, **options)
    want, bound = layer_oracle(layer)
    off = (got.double().cpu() - want).abs()
    assert torch.all(off <= bound), (off / bound.clamp(min=1e-300)).max()
    return got


LAYERS = [
    # tokens, experts, top_k, hidden, inter
    (1, 1, 1, 16, 16), (1, 8, 2, 512, 1024), (2, 3, 3, 48, 16), (3, 5, 2, 80, 176),
    (7, 4, 1, 272, 64), (8, 16, 4, 144, 208), (9, 6, 2, 528, 96), (16, 64, 8, 256, 128),
    (17, 2, 2, 400, 336), (31, 40, 3, 64, 80), (33, 8, 2, 1040, 144), (64, 3, 2, 160, 272),
    (64, 128, 8, 128, 64), (5, 300, 20, 64, 48), (1, 33, 32, 96, 32), (64, 1024, 32, 16, 16),
]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("sizes", LAYERS)
def test_moe_decode(engine, sizes, int8):
    layer = make_layer(*sizes, int8, seed=sum(sizes))
    first = check_layer(engine, layer)
    again = run_layer(engine, layer)
    assert torch.equal(first.view(torch.int16), again.view(torch.int16))


def big_layer(tokens, experts, top_k, hidden, inter, int8, seed):
    """A layer made on the GPU, for weights that do not fit its L2."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def weights(rows, cols):
        w = torch.randn(experts, rows, cols, generator=g, device="cuda") * cols ** -0.5
        if not int8:
            return w.to(torch.bfloat16), None
        scale = w.abs().amax(2) / 127
        return torch.round(w / scale[..., None]).to(torch.int8), scale

    (w1, s1), (w2, s2) = weights(2 * inter, hidden), weights(hidden, inter)
    x = torch.randn(tokens, hidden, generator=g, device="cuda").to(torch.bfloat16)
    ids = torch.rand(tokens, experts, generator=g, device="cuda").argsort(1)[:, :top_k]
    coef = torch.rand(tokens, top_k, generator=g, device="cuda") + 0.05
    return {"x": x, "w1": w1, "w2": w2, "s1": s1, "s2": s2, "ids": ids.contiguous(), "coef": coef}


def big_layer_oracle(layer):
    """``layer_oracle`` with its bound, an expert at a time on the GPU (a token names an expert
    once)."""
    x, ids = layer["x"].double(), layer["ids"]
    (tokens, hidden), (experts, _, inter) = x.shape, layer["w2"].shape
    out = torch.zeros(tokens, hidden, dtype=torch.float64, device="cuda")
    err, step = torch.zeros_like(out), 2 * HALF32
    for e in range(experts):
        token, place = torch.nonzero(ids == e, as_tuple=True)
        if token.numel() == 0:
            continue
        w1, w2 = layer["w1"][e].double(), layer["w2"][e].double()
        if layer["s1"] is not None:
            w1 = w1 * layer["s1"][e].double()[:, None]
            w2 = w2 * layer["s2"][e].double()[:, None]
        both, size = x[token] @ w1.t(), x[token].abs() @ w1.abs().t()
        both_err = size * (hidden / 16 + 16) * step * 2
        gate, up = both.chunk(2, 1)
        gate_err, up_err = both_err.chunk(2, 1)
        silu = gate / (1 + torch.exp(-gate))
        h = silu * up
        h_err = (1.1 * gate_err * (up.abs() + up_err) + silu.abs() * up_err
                 + h.abs() * (2.0 ** -16 + 8 * HALF32))
        c = layer["coef"][token, place].double()[:, None]
        out.index_add_(0, token, c * (h @ w2.t()))
        err.index_add_(0, token, c * ((h_err + h.abs() * (inter / 16 + 24) * step * 2)
                                      @ w2.abs().t()))
    return out, err + out.abs() * HALF16 + 2.0 ** -133


# INT8 weights that are converted (small layers, crowded experts) with rings of three stages, of
# the first or the second kernel or both, and eight k-blocks or more a CTA: the converting warps
# take turns at a slot.
@pytest.mark.parametrize("sizes", [(64, 4, 2, 4096, 4096), (32, 8, 2, 1024, 1024),
                                   (64, 1, 1, 4096, 2048), (48, 2, 1, 2064, 1040),
                                   (28, 6, 3, 1024, 1008), (40, 3, 2, 4096, 1456)])
def test_moe_decode_converted_weights_with_three_stages(engine, sizes):
    layer = big_layer(*sizes, True, seed=sum(sizes))
    want, bound = big_layer_oracle(layer)
    cold = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")

    def call():
        cold.zero_()                                   # weights come from HBM, not from L2
        return engine.moe_decode(layer["x"], layer["w1"], layer["w2"], layer["ids"],
                                 layer["coef"], gate_up_scale=layer["s1"],
                                 down_scale=layer["s2"])

    first = call()
    off = (first.double() - want).abs()
    assert torch.all(off <= bound), (off / bound).max()
    assert all(torch.equal(call(), first) for _ in range(20))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("tokens", [16, 32, 57, 64])
def test_moe_decode_one_of_many_experts_has_every_token(engine, tokens, int8):
    """The lists of about a thousand experts and the columns of all tokens leave the least
    room for stages; the average number of an expert's tokens says nothing of it."""
    layer = big_layer(tokens, 1000, 2, 128, 1040, int8, seed=tokens)
    layer["ids"][:, 0], layer["ids"][:, 1] = 777, -1
    layer["ids"][::16, 1] = 3
    want, bound = big_layer_oracle(layer)
    got = engine.moe_decode(layer["x"], layer["w1"], layer["w2"], layer["ids"], layer["coef"],
                            gate_up_scale=layer["s1"], down_scale=layer["s2"])
    off = (got.double() - want).abs()
    assert torch.all(off <= bound), (off / bound).max()


@pytest.mark.parametrize("hidden,inter", [(8, 8), (24, 40), (72, 8), (1000, 56), (264, 1032)])
def test_moe_decode_odd_multiples_of_eight(engine, hidden, inter):
    for tokens in (1, 6, 20):
        check_layer(engine, make_layer(tokens, 5, 2, hidden, inter, False, seed=hidden))


@pytest.mark.parametrize("int8", [False, True])
def test_moe_decode_dropped_repeated_and_crowded_experts(engine, int8):
    check_layer(engine, make_layer(24, 6, 3, 96, 112, int8, seed=1, drop=0.5))
    none = make_layer(5, 4, 2, 64, 32, int8, seed=2, drop=1.1)
    assert torch.all(run_layer(engine, none) == 0)
    crowd = make_layer(64, 9, 2, 128, 96, int8, seed=3)
    crowd["ids"][:, 0], crowd["ids"][:, 1] = 8, -1     # one expert takes every token
    check_layer(engine, crowd)
    twice = make_layer(11, 4, 4, 96, 64, int8, seed=4)
    twice["ids"][:, 2] = twice["ids"][:, 0]            # the same expert two and four times
    twice["ids"][3] = 2
    twice["ids"][4] = torch.tensor([1, -1, 1, 77])
    check_layer(engine, twice)
    zero = make_layer(3, 4, 2, 64, 64, int8, seed=5)
    zero["coef"][1] = 0.0
    zero["coef"][2] = torch.tensor([-1.5, 2.0])
    check_layer(engine, zero)


@pytest.mark.parametrize("tokens", [4, 30])
def test_moe_decode_bad_values_stay_with_their_tokens(engine, tokens):
    """NaN in an expert's weights or in a token's row reaches the tokens that use it only;
    so does an infinity."""
    layer = make_layer(tokens, 6, 2, 64, 48, False, seed=9)
    layer["ids"] = torch.stack([torch.arange(tokens) % 5, (torch.arange(tokens) + 2) % 5], 1)
    clean = run_layer(engine, layer)
    bad = dict(layer, w1=layer["w1"].clone(), w2=layer["w2"].clone(), x=layer["x"].clone())
    bad["w1"][5], bad["w2"][5] = math.nan, math.inf    # expert 5: chosen by nobody
    assert torch.equal(run_layer(engine, bad), clean)
    bad["w2"][1, :, 3] = math.inf                      # expert 1: some tokens
    bad["w1"][2, 7] = math.nan
    bad["x"][tokens - 1, 11] = math.nan
    got = run_layer(engine, bad)
    hit = ((layer["ids"] == 1) | (layer["ids"] == 2)).any(1)
    hit[tokens - 1] = True
    assert torch.equal(got[~hit.cuda()], clean[~hit.cuda()])
    assert not torch.isfinite(got[hit.cuda()]).all(1).any()


def test_moe_decode_workspace_streams_and_graphs(engine):
    layer = make_layer(13, 10, 4, 320, 160, True, seed=6)
    dev = {k: (v.cuda() if v is not None else None) for k, v in layer.items()}
    need = engine.moe_decode_workspace(13, 4, 160)
    dirty = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")     # NaN everywhere
    want = check_layer(engine, layer, workspace=dirty)

    def call(**options):
        return engine.moe_decode(dev["x"], dev["w1"], dev["w2"], dev["ids"], dev["coef"],
                                 gate_up_scale=dev["s1"], down_scale=dev["s2"], **options)

    with pytest.raises(engine._capi.EngineError):
        call(workspace=dirty[:need - 256])
    # two streams at once, a workspace each; the default is the current stream
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    results = []
    for _ in range(20):
        with torch.cuda.stream(one):
            results.append(call())
        results.append(call(stream=two, workspace=dirty,
                            out=torch.empty_like(want)))
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results)
    # captured with the router in front, replayed on new inputs
    logits = torch.randn(13, 10, device="cuda")
    x = dev["x"].clone()
    with torch.cuda.stream(one):
        def step():
            ids, coef = engine.route_topk(logits, 4, renormalize=True)
            return engine.moe_decode(x, dev["w1"], dev["w2"], ids, coef,
                                     gate_up_scale=dev["s1"], down_scale=dev["s2"])
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=one):
            captured = step()
    for seed in (1, 2, 3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        logits.copy_(torch.randn(13, 10, generator=g, device="cuda"))
        x.copy_(torch.randn(13, 320, generator=g, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, step())


def test_moe_decode_may_write_its_input_and_leaves_the_status_word_alone(engine):
    import ctypes as C

    for int8 in (False, True):
        layer = make_layer(40, 12, 3, 384, 320, int8, seed=8)
        want = run_layer(engine, layer)
        to = {k: (v.cuda() if v is not None else None) for k, v in layer.items()}
        got = engine.moe_decode(to["x"], to["w1"], to["w2"], to["ids"], to["coef"],
                                gate_up_scale=to["s1"], down_scale=to["s2"], out=to["x"])
        assert got is to["x"] and torch.equal(got, want)
    cap = engine._capi
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.empty_like(want)
    workspace = torch.empty(engine.moe_decode_workspace(40, 3, 320), dtype=torch.uint8,
                            device="cuda")
    to["x"].copy_(layer["x"])
    args = cap.MoeDecodeArgs(
        to["x"].data_ptr(), to["w1"].data_ptr(), to["w2"].data_ptr(), to["s1"].data_ptr(),
        to["s2"].data_ptr(), to["ids"].data_ptr(), to["coef"].data_ptr(), out.data_ptr(),
        workspace.data_ptr(), workspace.numel(), 40, 3, 12, 384, 320, cap.TYPE_INT8, None,
        status.data_ptr())
    assert cap.load().bmoe_moe_decode(C.byref(args)) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, want) and status.item() == 0


@pytest.mark.parametrize("sizes,int8", [
    ((1, 8, 2, 512, 1024), False), ((9, 6, 2, 528, 96), True), ((40, 12, 3, 384, 320), False),
    ((64, 3, 2, 160, 272), True), ((16, 8, 4, 1040, 1456), True)])
def test_moe_decode_after_a_wait_that_ran_out(engine, sizes, int8):
    """The status word reaches the caller, and a call that finds it set gives NaN everywhere: the
    way a wait of its own that ran out would, without one."""
    layer = make_layer(*sizes, int8, seed=sum(sizes))
    want = run_layer(engine, layer)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert torch.equal(run_layer(engine, layer, status=status), want) and status.item() == 0
    status.fill_(0x50000004)
    got = run_layer(engine, layer, status=status)
    assert torch.isnan(got).all() and status.item() == 0x50000004
    status.zero_()
    assert torch.equal(run_layer(engine, layer, status=status), want) and status.item() == 0
    for bad in (status.float(), torch.zeros(2, dtype=torch.int32, device="cuda"), status.cpu()):
        with pytest.raises(ValueError):
            run_layer(engine, layer, status=bad)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("tokens", [17, 33, 64])
def test_moe_decode_sparse_and_spread_tokens(engine, tokens, int8):
    """Experts whose few tokens lie far apart, close together, and at both ends."""
    layer = make_layer(tokens, 9, 2, 192, 128, int8, seed=tokens)
    ids = torch.full((tokens, 2), -1, dtype=torch.int64)
    ids[0, 0] = ids[tokens - 1, 0] = 0                 # first and last
    ids[tokens // 2, 1] = 1                            # one in the middle
    ids[::5, 1] = 2
    ids[1:5, 0] = 3
    ids[tokens - 3:, 1] = 4
    ids[::2, 0] = torch.where(ids[::2, 0] < 0, 5, ids[::2, 0])
    ids[3::8, 1] = 6                                   # one of every group of 8
    layer["ids"] = ids
    check_layer(engine, layer)


def test_operators_at_once_from_two_host_threads(engine):
    import threading

    layers = [make_layer(9 + i, 7, 2, 256, 192, bool(i), seed=50 + i) for i in range(2)]
    wants = [run_layer(engine, layer) for layer in layers]
    logits = torch.randn(300, 64, generator=gen(1)).cuda()
    want_ids = engine.route_topk(logits, 4)[0]
    torch.cuda.synchronize()
    failures = []

    def work(i):
        try:
            to = {k: (v.cuda() if v is not None else None) for k, v in layers[i].items()}
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(30):
                    got = engine.moe_decode(to["x"], to["w1"], to["w2"], to["ids"], to["coef"],
                                            gate_up_scale=to["s1"], down_scale=to["s2"])
                    ids = engine.route_topk(logits, 4)[0]
                    stream.synchronize()
                    assert torch.equal(got, wants[i]) and torch.equal(ids, want_ids)
        except Exception as error:   # noqa: BLE001 - reported by the main thread
            failures.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


def test_moe_decode_weights_past_32_bit_offsets(engine):
    """The last expert's weights start beyond 2^32 bytes (and 2^31 elements)."""
    experts, hidden, inter = 70, 4096, 8192
    dev = "cuda"
    w1 = torch.zeros(experts, 2 * inter, hidden, dtype=torch.int8, device=dev)
    w2 = torch.zeros(experts, hidden, inter, dtype=torch.int8, device=dev)
    s1 = torch.full((experts, 2 * inter), 2.0 ** -10, device=dev)
    s2 = torch.full((experts, hidden), 2.0 ** -10, device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    w1[-1] = torch.randint(-127, 128, (2 * inter, hidden), generator=g, device=dev)
    w2[-1] = torch.randint(-127, 128, (hidden, inter), generator=g, device=dev)
    x = torch.randn(2, hidden, generator=g, device=dev).to(torch.bfloat16)
    ids = torch.tensor([[experts - 1], [0]], device=dev)
    out = engine.moe_decode(x, w1, w2, ids, torch.ones(2, 1, device=dev), gate_up_scale=s1,
                            down_scale=s2)
    small = {"x": x[:1].cpu(), "w1": w1[-1:].cpu(), "w2": w2[-1:].cpu(), "s1": s1[-1:].cpu(),
             "s2": s2[-1:].cpu(), "ids": torch.zeros(1, 1, dtype=torch.int64),
             "coef": torch.ones(1, 1)}
    want, bound = layer_oracle(small)
    assert torch.all((out[:1].double().cpu() - want).abs() <= bound)
    assert torch.all(out[1] == 0)


def test_allocations_belong_to_the_stream_of_the_launch(engine, monkeypatch):
    """Memory that a call allocates for a launch on another stream must not be handed out on
    the current stream while the launch has not run yet."""
    layer = make_layer(5, 6, 2, 256, 128, False, seed=3)
    dev = {k: (v.cuda() if v is not None else None) for k, v in layer.items()}
    seen = []
    run = engine.layer._moe_decode
    place = [name for name, _ in engine._capi.MoeDecodeArgs._fields_].index("workspace_dev")
    monkeypatch.setattr(engine.layer, "_moe_decode", lambda *a: seen.append(a[place]) or run(*a))
    side = torch.cuda.Stream()
    need = engine.moe_decode_workspace(5, 2, 128)
    logits, rows = torch.randn(5, 6, device="cuda"), torch.randn(5, 256, device="cuda")
    want = check_layer(engine, layer)
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream):
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
        got = engine.moe_decode(dev["x"], dev["w1"], dev["w2"], dev["ids"], dev["coef"],
                                stream=stream)
        ids, coef = engine.route_topk(logits, 2, stream=stream)
        q, scale = engine.quantize_rows(rows, stream=stream)
        taken = {t.untyped_storage().data_ptr(): t.untyped_storage().nbytes()
                 for t in (ids, coef, q, scale)}
        taken[seen[-1]] = need
        del ids, coef, q, scale
        fresh = [torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
                 for size in taken.values()]
        assert not {t.data_ptr() for t in fresh} & set(taken)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert torch.cuda.current_stream() != side


# INT8 layers with 36 MB of chosen weights or more and at most 24 tokens an expert: activations
# as fixed-point digits (the rule in moe_decode.cu).
DIGIT_LAYERS = [
    # tokens, experts, top_k, hidden, inter
    (1, 1, 1, 3504, 3504), (1, 2, 2, 2064, 3008), (2, 8, 8, 1040, 1456), (5, 3, 2, 2064, 2000),
    (16, 8, 4, 1040, 1456), (17, 8, 4, 1040, 1456), (33, 8, 4, 1040, 1456), (64, 8, 3, 1040, 1456),
    (9, 40, 5, 4000, 80), (24, 1024, 32, 112, 144), (64, 1024, 16, 128, 96), (3, 8, 3, 288, 14336),
]


def digit_bound(layer, bound):
    """The operator's bound plus what the digits lose: an x is off by 2^-22 of its row's largest
    at most, and so is an h (times its weight); the sums of digits are exact."""
    x, extra = layer["x"].double(), torch.zeros_like(bound)
    most = 2.0 ** -22 * x.abs().amax(1)
    for t in range(x.shape[0]):
        for j, e in enumerate(layer["ids"][t].tolist()):
            if not 0 <= e < layer["w1"].shape[0]:
                continue
            inter = layer["w2"].shape[2]
            w1 = layer["w1"][e].double() * layer["s1"][e].double()[:, None]
            w2 = (layer["w2"][e].double() * layer["s2"][e].double()[:, None]).abs()
            both, both_err = w1 @ x[t], w1.abs().sum(1) * most[t]
            gate, up = both[:inter], both[inter:]
            silu = gate / (1 + torch.exp(-gate))
            h_err = (1.1 * both_err[:inter] * (up.abs() + both_err[inter:])
                     + silu.abs() * both_err[inter:])
            h_err = h_err + ((silu * up).abs() + h_err).max() * 2.0 ** -22
            extra[t] += layer["coef"][t, j].double().abs() * (w2 @ h_err)
    return bound + extra


@pytest.mark.parametrize("sizes", DIGIT_LAYERS)
def test_moe_decode_digits(engine, sizes):
    layer = make_layer(*sizes, True, seed=sum(sizes), drop=0.1 if sizes[0] > 2 else 0.0)
    check_layer(engine, layer)


def test_moe_decode_digits_of_rows_with_a_wide_range(engine):
    """One large value in a row, values far below it, a row of zeros, one of subnormals, one
    of the largest numbers; rows that hold a NaN or an infinity stay alone with it."""
    layer = make_layer(8, 8, 8, 1040, 1456, True, seed=77)
    x, g = layer["x"], gen(78)
    x[0, 17] = 4096.0
    x[1] = x[1] * (2.0 ** torch.randint(-40, 1, (1040,), generator=g)).to(torch.bfloat16)
    x[2] = 0.0
    x[3] = x[3].sign() * 2.0 ** -130
    x[4] = x[4] * 2.0 ** 20
    layer["coef"][5] = 2.0 ** -60
    clean = run_layer(engine, layer)
    want, bound = layer_oracle(layer)
    bound = digit_bound(layer, bound)
    assert torch.all((clean.double().cpu() - want).abs() <= bound)
    assert torch.all(clean[2:4] == 0)
    bad = dict(layer, x=x.clone())
    bad["x"][6, 3], bad["x"][7, 1039] = math.nan, math.inf
    got = run_layer(engine, bad)
    assert torch.equal(got[:6], clean[:6])
    assert not torch.isfinite(got[6:]).any()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("tokens", [1, 4, 18])
def test_moe_decode_last_tiles_of_few_channels(engine, tokens, int8):
    """Tiles split over a cluster whose last 16 channels leave whole warps without any."""
    layer = big_layer(tokens, 2, 2, 2064, 3088, int8, seed=tokens)
    want, bound = big_layer_oracle(layer)
    if int8:
        cpu = {name: t.cpu() for name, t in layer.items()}
        bound = digit_bound(cpu, bound.cpu()).cuda()
    got = engine.moe_decode(layer["x"], layer["w1"], layer["w2"], layer["ids"], layer["coef"],
                            gate_up_scale=layer["s1"], down_scale=layer["s2"])
    off = (got.double() - want).abs()
    assert torch.all(off <= bound), (off / bound).max()


def test_moe_decode_digits_that_do_not_fit_beside_h(engine):
    """hidden > top_k * inter: the weights are converted instead."""
    check_layer(engine, make_layer(20, 64, 1, 4000, 160, True, seed=8))


def test_moe_decode_digits_dropped_repeated_streams_and_graphs(engine):
    layer = make_layer(16, 8, 4, 1040, 1456, True, seed=12)
    layer["ids"][3] = 5                                 # four times the same expert
    layer["ids"][4, 2:] = torch.tensor([-1, 90])
    layer["ids"][5] = -1
    need = engine.moe_decode_workspace(16, 4, 1456)
    dirty = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    want = check_layer(engine, layer, workspace=dirty)
    assert torch.all(want[5] == 0)
    dev = {k: v.cuda() for k, v in layer.items()}

    def call(x=dev["x"], ids=dev["ids"], **options):
        return engine.moe_decode(x, dev["w1"], dev["w2"], ids, dev["coef"],
                                 gate_up_scale=dev["s1"], down_scale=dev["s2"], **options)

    assert torch.all(call(ids=torch.full_like(dev["ids"], -1)) == 0)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    results = [call(stream=s) for _ in range(10) for s in streams]
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results)
    x = dev["x"].clone()
    call(x=x, out=x)                                    # in place
    assert torch.equal(x, want)
    x.copy_(dev["x"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(x=x)
    for seed in (1, 2):
        x.copy_(torch.randn(16, 1040, generator=gen(seed)).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(x=x))
    x.copy_(dev["x"])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
