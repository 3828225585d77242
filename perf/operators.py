"""Measured cases of the layer operators either side of the grouped GEMM.

Four operators of one mixture-of-experts layer:

  route     router scores -> the top-k experts of every token and their weights
  quantize  token rows, gathered by index, -> 8-bit integers with one scale per row
  product   8-bit product over routed experts: rows quantised on the way in, a scale per
            token and per output channel, BF16 out
  layer     the whole expert layer for a few tokens: gate and up products, SiLU(gate) * up,
            down product, weighted sum over the token's experts

``run`` computes the plain form (elementary torch operations) unless ``own`` is set; then
it makes the calls a user of the package makes.
"""

import math

import torch

own = False

DEVICE = "cuda"
SMALLEST_ROW_MAX = 2.0 ** -100      # rows below this quantise to zero


# ------------------------------------------------------------------ cases --

def _route(name, tokens, experts, top_k, dtype="fp32", scoring="softmax", renormalize=True,
           bias=False, scale=1.0, off=0):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top_k": top_k,
            "dtype": dtype, "scoring": scoring, "renormalize": renormalize, "bias": bias,
            "scale": scale, "off": off}


def _quantize(name, tokens, copies, cols, dtype="bf16"):
    return {"name": name, "op": "quantize", "tokens": tokens, "copies": copies, "cols": cols,
            "dtype": dtype}


def _product(name, experts, rows, n, k, zipf):
    return {"name": name, "op": "product", "experts": experts, "rows": rows, "n": n, "k": k,
            "zipf": zipf}


def _layer(name, tokens, experts, top_k, hidden, inter, weights, ranks=1, padded=0):
    return {"name": name, "op": "layer", "tokens": tokens, "experts": experts, "top_k": top_k,
            "hidden": hidden, "inter": inter, "weights": weights, "ranks": ranks,
            "padded": padded}


def listed():
    return [
        # a decode step of four sequences, DeepSeek-shaped: 256 experts, top-8, sigmoid scores
        # with a balancing bias that takes part in the choice and not in the weight
        _route("route_decode_e256", 4, 256, 8, "fp32", "sigmoid", True, True, 2.5),
        # prefill of the skew sweep (E=128, top-8); BF16 scores tie often; 3 experts switched off
        _route("route_prefill_e128", 16384, 128, 8, "bf16", off=3),
        # rows of one decode batch, one copy per routed expert (decode configuration's k)
        _quantize("quantize_decode_k7168", 64, 8, 7168),
        # dispatch of the Mixtral-shaped configuration: T=4096, top-2, K=4096
        _quantize("quantize_dispatch_k4096", 4096, 2, 4096),
        # dense 8-bit product of one small batch (N=7168, K=2048 of the dense M-sweep)
        _product("product_dense_m16", 1, 16, 7168, 2048, 0.0),
        # skew sweep: E=128, N=768, K=2048, Zipf 1.0, ragged experts, some of a few rows
        _product("product_sweep_e128", 128, 16384, 768, 2048, 1.0),
        # Mixtral-shaped up-projection: E=8, 8192 routed rows, K=4096, N=14336, Zipf 1.0
        _product("product_mixtral", 8, 8192, 14336, 4096, 1.0),
        # smallest layer: the CPU-runnable configuration's experts, one token
        _layer("layer_small_t1", 1, 8, 2, 512, 1024, "bf16"),
        # one sequence decoding, Mixtral-shaped experts: latency of the weight stream
        _layer("layer_mixtral_t1", 1, 8, 2, 4096, 14336, "bf16"),
        # a batch of 32 sequences over the skew sweep's experts: most of the 128 are active
        _layer("layer_sweep_t32", 32, 128, 8, 2048, 768, "bf16"),
        # 8-bit weights, 64 slots of which 9 are padding, Mixtral-shaped: every expert active
        _layer("layer_mixtral_t64_int8", 64, 8, 2, 4096, 14336, "int8", padded=9),
        # one of 8 expert-parallel ranks, decode configuration's experts (32 of 256 here):
        # assignments to other ranks' experts are dropped
        _layer("layer_rank_t16_int8", 16, 32, 8, 7168, 2048, "int8", ranks=8),
    ]


def _log(rng, low, high, step=1):
    """A multiple of ``step`` in [low, high], uniform over its logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["route", "quantize", "product", "product", "layer", "layer", "layer"])
    if op == "route":
        experts = _log(rng, 4, 512)
        scoring = rng.choice(["softmax", "sigmoid"])
        top_k = rng.randint(1, min(16, experts))
        case = _route("", _log(rng, 1, 16384), experts, top_k, rng.choice(["fp32", "bf16"]),
                      scoring, rng.random() < 0.6,
                      scoring == "sigmoid" and rng.random() < 0.7,
                      rng.choice([1.0, 1.0, 2.5]),
                      rng.choice([0, 0, 1, experts // 2, experts - top_k // 2 - 1]))
    elif op == "quantize":
        cols = _log(rng, 16, 16384, 16)
        tokens = _log(rng, 1, max(1, min(16384, (1 << 24) // cols)))
        case = _quantize("", tokens, rng.randint(0, 4), cols, rng.choice(["bf16", "fp32"]))
    elif op == "product":
        experts = _log(rng, 1, 128)
        n, k = _log(rng, 64, 14336, 8), _log(rng, 64, 7168, 16)
        rows = _log(rng, 1, 16384)
        while 2 * rows * n * k > 4e11 or experts * n * k > 2e9:
            rows, n = max(1, rows // 2), max(64, n // 2 // 8 * 8)
        case = _product("", experts, rows, n, k, rng.choice([0.0, 0.5, 1.0, 1.5]))
    else:
        weights = rng.choice(["bf16", "int8"])
        step = 16 if weights == "int8" else 8
        tokens = _log(rng, 1, 64)
        hidden, inter = _log(rng, 256, 7168, step), _log(rng, 64, 14336, step)
        experts = _log(rng, 2, 256)
        while experts * 3 * hidden * inter * (1 if weights == "int8" else 2) > 1.4e9:
            experts, inter = max(2, experts // 2), max(64, inter * 3 // 4 // step * step)
        ranks = rng.choice([1, 1, 4])
        case = _layer("", tokens, experts, rng.randint(1, min(8, experts)), hidden, inter,
                      weights, ranks, rng.choice([0, 0, tokens // 3]))
    del case["name"]
    return case


def _counts(case):
    """Rows per expert: Zipf shares of the rows, largest first, remainders to the front."""
    share = [(e + 1.0) ** -case["zipf"] for e in range(case["experts"])]
    total = sum(share)
    counts = [int(case["rows"] * s / total) for s in share]
    for i in range(case["rows"] - sum(counts)):
        counts[i % len(counts)] += 1
    return counts


# ----------------------------------------------------------------- inputs --

def _int8_weights(experts, n, k, gen):
    """Weights ~ N(0, 1/sqrt(k)) in 8 bits with one scale per output channel."""
    w = torch.empty(experts, n, k, dtype=torch.int8, device=DEVICE)
    scale = torch.empty(experts, n, dtype=torch.float32, device=DEVICE)
    for e in range(experts):
        full = torch.randn(n, k, generator=gen, device=DEVICE) * k ** -0.5
        scale[e] = full.abs().amax(1) / 127.0
        w[e] = torch.round(full / scale[e][:, None]).to(torch.int8)
    return w, scale


def _bf16_weights(experts, n, k, gen):
    w = torch.empty(experts, n, k, dtype=torch.bfloat16, device=DEVICE)
    for e in range(experts):
        w[e] = torch.randn(n, k, generator=gen, device=DEVICE) * k ** -0.5
    return w


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"case": case}
    op = case["op"]
    if op == "route":
        tokens, experts = case["tokens"], case["experts"]
        logits = torch.randn(tokens, experts, generator=gen, device=DEVICE) * 1.5
        logits += torch.randn(experts, generator=gen, device=DEVICE) * 0.5
        if case["off"]:     # experts out of service
            gone = torch.randperm(experts, generator=gen, device=DEVICE)[:case["off"]]
            logits[:, gone] = -math.inf
        state["logits"] = logits.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        state["bias"] = (torch.randn(experts, generator=gen, device=DEVICE) * 0.05
                         if case["bias"] else None)
    elif op == "quantize":
        tokens, cols = case["tokens"], case["cols"]
        x = torch.randn(tokens, cols, generator=gen, device=DEVICE)
        x *= torch.exp(torch.randn(tokens, 1, generator=gen, device=DEVICE))
        x[:, torch.randint(cols, (max(1, cols // 500),), generator=gen, device=DEVICE)] *= 8.0
        state["x"] = x.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32)
        # 0 copies: no gather, every row once in order
        state["index"] = (torch.randperm(tokens * case["copies"], generator=gen, device=DEVICE)
                          // case["copies"] if case["copies"] else None)
    elif op == "product":
        counts = _counts(case)
        state["counts"] = counts
        state["x"] = torch.randn(case["rows"], case["k"], generator=gen,
                                 device=DEVICE).to(torch.bfloat16)
        state["w"], state["w_scale"] = _int8_weights(case["experts"], case["n"], case["k"], gen)
        # buffers a serving program keeps
        state["q"] = torch.empty(case["rows"], case["k"], dtype=torch.int8, device=DEVICE)
        state["scale"] = torch.empty(case["rows"], dtype=torch.float32, device=DEVICE)
        state["out"] = torch.empty(case["rows"], case["n"], dtype=torch.bfloat16, device=DEVICE)
        if own:
            # The plan's storage is kept; with one expert its row count is fixed and the
            # whole plan is, with routed experts every pass has counts of its own.
            import bmoe_b200

            state["plan"] = bmoe_b200.GroupedGemmPlan()
            if case["experts"] == 1:
                _plan_product(state)
    else:
        tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
        total = experts * case["ranks"]
        state["x"] = torch.randn(tokens, case["hidden"], generator=gen,
                                 device=DEVICE).to(torch.bfloat16)
        scores = torch.randn(tokens, total, generator=gen, device=DEVICE)
        scores -= torch.log(1.0 + torch.randperm(total, generator=gen, device=DEVICE)) * 0.5
        best, ids = torch.topk(scores, top_k, dim=1)
        weights = torch.softmax(best, 1)
        if case["padded"]:
            ids[tokens - case["padded"]:] = -1
        ids[ids >= experts] = -1
        state["ids"], state["weights"] = ids, weights.contiguous()
        make = _int8_weights if case["weights"] == "int8" else \
            (lambda *a: (_bf16_weights(*a), None))
        state["w_gate_up"], state["gate_up_scale"] = make(experts, 2 * case["inter"],
                                                          case["hidden"], gen)
        state["w_down"], state["down_scale"] = make(experts, case["hidden"], case["inter"], gen)
    return state


# ---------------------------------------------------- the framework's calls --

def _plan_product(state):
    status = state["plan"].initialize_packed(
        state["q"], state["w"], state["out"], state["counts"], scheduler="auto",
        row_scale=state["scale"], col_scale=state["w_scale"],
        stream=torch.cuda.current_stream().cuda_stream)
    if status:
        raise RuntimeError(f"plan: status {status}")


def _own(state):
    import bmoe_b200

    case = state["case"]
    if case["op"] == "route":
        return bmoe_b200.route_topk(state["logits"], case["top_k"], scoring=case["scoring"],
                                    renormalize=case["renormalize"], bias=state["bias"],
                                    scale=case["scale"])
    if case["op"] == "quantize":
        q, scale = bmoe_b200.quantize_rows(state["x"], state["index"])
        return q, scale
    if case["op"] == "product":
        bmoe_b200.quantize_rows(state["x"], out=state["q"], scale=state["scale"])
        if case["experts"] > 1:
            _plan_product(state)
        status = state["plan"].run(torch.cuda.current_stream().cuda_stream)
        if status:
            raise RuntimeError(f"run: status {status}")
        return state["out"]
    return bmoe_b200.moe_decode(state["x"], state["w_gate_up"], state["w_down"], state["ids"],
                                state["weights"], gate_up_scale=state["gate_up_scale"],
                                down_scale=state["down_scale"])


# ------------------------------------------------------------- plain forms --

def _plain_route(state):
    case = state["case"]
    logits = state["logits"].float()
    live = logits > -math.inf                       # NaN and -inf are never chosen
    if case["scoring"] == "softmax":
        key = logits
        e = torch.exp(logits - logits.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        # chosen by the sum, in 64 bits: neighbours in it may be closer than 32 bits tell
        key = 1.0 / (1.0 + torch.exp(-logits.double()))
        if state["bias"] is not None:
            key = key + state["bias"].double()
        score = 1.0 / (1.0 + torch.exp(-logits))
    key = torch.where(live, key, -math.inf)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
    chosen = torch.gather(live, 1, order)
    weights = torch.where(chosen, torch.gather(score, 1, order), 0.0)
    if case["renormalize"]:
        total = weights.sum(1, keepdim=True)
        weights = torch.where(total > 0, weights / total, 0.0)
    return torch.where(chosen, order, -1), weights * case["scale"]


def _plain_quantize(x, index=None):
    x = x.float()
    if index is not None:
        x = x[index]
    largest = x.abs().amax(1, keepdim=True).clamp(min=SMALLEST_ROW_MAX)
    q = torch.round(x * (127.0 / largest)).clamp(-127, 127)
    return q.to(torch.int8), (largest / 127.0).squeeze(1)


def _plain_product(state):
    q, scale = _plain_quantize(state["x"])
    rows = torch.split(q.float(), state["counts"])
    sums = torch.cat([a @ w.float().t() for a, w in zip(rows, state["w"])])
    counts = torch.tensor(state["counts"])
    col = torch.cat([s.expand(c, -1) for c, s in zip(counts.tolist(), state["w_scale"])])
    return (sums * scale[:, None] * col).to(torch.bfloat16)


def _plain_layer(state):
    case = state["case"]
    x, ids, coef = state["x"].float(), state["ids"], state["weights"]
    experts, (tokens, top_k) = case["experts"], ids.shape
    valid = (ids >= 0) & (ids < experts)
    if tokens * top_k < experts:
        # few assignments: the chosen experts' weights, one product per assignment
        pick = torch.where(valid, ids, 0).reshape(-1)
        w1, w2 = state["w_gate_up"][pick].float(), state["w_down"][pick].float()
        if state["gate_up_scale"] is not None:
            w1 *= state["gate_up_scale"][pick][:, :, None]
            w2 *= state["down_scale"][pick][:, :, None]
        both = torch.bmm(w1, x.repeat_interleave(top_k, 0)[:, :, None])
        gate, up = both[:, :case["inter"]], both[:, case["inter"]:]
        out = torch.bmm(w2, gate / (1.0 + torch.exp(-gate)) * up)[:, :, 0]
        out = out * torch.where(valid, coef, 0.0).reshape(-1, 1)
        return out.reshape(tokens, top_k, -1).sum(1).to(torch.bfloat16)
    # many: every expert on every token, weighted by what the router gave it
    w1, w2 = state["w_gate_up"].float(), state["w_down"].float()
    if state["gate_up_scale"] is not None:
        w1 *= state["gate_up_scale"][:, :, None]
        w2 *= state["down_scale"][:, :, None]
    both = torch.matmul(w1, x.t())
    gate, up = both[:, :case["inter"]], both[:, case["inter"]:]
    out = torch.matmul(w2, gate / (1.0 + torch.exp(-gate)) * up)
    share = torch.zeros(tokens, experts, device=x.device)
    share.scatter_add_(1, torch.where(valid, ids, 0), torch.where(valid, coef, 0.0))
    return (out * share.t()[:, None, :]).sum(0).t().to(torch.bfloat16)


def run(state):
    op = state["case"]["op"]
    if own:
        result = _own(state)
    elif op == "route":
        result = _plain_route(state)
    elif op == "quantize":
        result = _plain_quantize(state["x"], state["index"])
    elif op == "product":
        result = _plain_product(state)
    else:
        result = _plain_layer(state)
    if op == "quantize":        # the values that the 8 bits stand for
        q, scale = result
        return {"values": q.float() * scale[:, None], "scale": scale}
    if op == "route":
        return {"ids": result[0], "weights": result[1]}
    return {"out": result}


# ------------------------------------------------------------------- work --

def _active(case):
    """Experts that hold weights of a pass: expected number of distinct ones."""
    draws = (case["tokens"] - case["padded"]) * case["top_k"]
    total = case["experts"] * case["ranks"]
    return case["experts"] * (1.0 - (1.0 - 1.0 / total) ** draws)


def work(case):
    op = case["op"]
    if op == "route":
        cells, picks = case["tokens"] * case["experts"], case["tokens"] * case["top_k"]
        return {"bytes": cells * (2 if case["dtype"] == "bf16" else 4) + picks * 12,
                "flops": cells * 4}
    if op == "quantize":
        rows = case["tokens"] * max(1, case["copies"])
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": case["tokens"] * case["cols"] * size + rows * (case["cols"] + 4)
                + (rows * 8 if case["copies"] else 0),
                "flops": 3 * rows * case["cols"]}
    if op == "product":
        m, n, k = case["rows"], case["n"], case["k"]
        active = sum(1 for c in _counts(case) if c)
        return {"bytes": 2 * m * k + active * n * (k + 4) + 2 * m * n, "flops": 2 * m * n * k}
    size = 1 if case["weights"] == "int8" else 2
    pairs = (case["tokens"] - case["padded"]) * case["top_k"] / case["ranks"]
    weights = 3 * case["hidden"] * case["inter"]
    scales = 4 * (2 * case["inter"] + case["hidden"]) if size == 1 else 0
    return {"bytes": _active(case) * (weights * size + scales)
            + 4 * case["tokens"] * case["hidden"] + 12 * case["tokens"] * case["top_k"],
            "flops": 2 * pairs * weights}


# ------------------------------------------------------ results in 64 bits --

def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "route":
        x = state["logits"].double()
        alive = torch.isfinite(x) | (x == math.inf)
        if case["scoring"] == "softmax":
            score = torch.softmax(torch.where(alive, x, -math.inf), 1)
            key = x
        else:
            score = torch.sigmoid(x)
            key = score + (0.0 if state["bias"] is None else state["bias"].double())
        key = torch.where(alive, key, -math.inf)
        ids = torch.argsort(key, dim=1, descending=True, stable=True)[:, :case["top_k"]]
        weights = score.gather(1, ids) * alive.gather(1, ids)
        if case["renormalize"]:
            weights = weights / weights.sum(1, keepdim=True).clamp(min=1e-300)
        return {"ids": torch.where(alive.gather(1, ids), ids, -1),
                "weights": weights * case["scale"]}
    if op == "quantize" or op == "product":
        x = state["x"].double()
        if op == "quantize" and state["index"] is not None:
            x = x.index_select(0, state["index"])
        largest = x.abs().max(dim=1).values.clamp(min=SMALLEST_ROW_MAX)
        if op == "quantize":
            # which step a value next to a border goes to is the operator's choice
            return {"values": None, "scale": largest / 127.0}
        # the product of what the operator quantised: rounding the rows is part of it and is
        # defined in 32 bits, x * (127 / largest) with one rounding each
        inv = (127.0 / largest.float()).double()
        q = torch.round((x * inv[:, None]).float().double())
        out = torch.empty(case["rows"], case["n"], dtype=torch.float64, device=DEVICE)
        first = 0
        for e, count in enumerate(state["counts"]):
            piece = slice(first, first + count)
            out[piece] = torch.matmul(q[piece], state["w"][e].double().t())
            out[piece] *= (largest[piece] / 127.0)[:, None] * state["w_scale"][e].double()
            first += count
        return {"out": out}
    tokens = case["tokens"]
    out = torch.zeros(tokens, case["hidden"], dtype=torch.float64, device=DEVICE)
    for e in range(case["experts"]):
        token, place = torch.nonzero(state["ids"] == e, as_tuple=True)
        if token.numel() == 0:
            continue
        w1, w2 = state["w_gate_up"][e].double(), state["w_down"][e].double()
        if state["gate_up_scale"] is not None:
            w1 = w1 * state["gate_up_scale"][e].double()[:, None]
            w2 = w2 * state["down_scale"][e].double()[:, None]
        both = state["x"][token].double() @ w1.t()
        gate, up = both.chunk(2, dim=1)
        part = (gate * torch.sigmoid(gate) * up) @ w2.t()
        out.index_add_(0, token, part * state["weights"][token, place].double()[:, None])
    return {"out": out}
