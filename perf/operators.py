"""The integer and routing operators, measured over the range of sizes they are used at.

A case is a dict of plain values; `op` says which public entry points one pass goes through:

    quantize   quantize_int8 + dequantize_int8: activations -> codes and token scales -> the values they stand for
    gemm       int8_gemm: codes and scales of both operands -> C
    linear     int8_linear: 16/32-bit activations, quantised token by token, times int8 weights -> C
    experts    gather_tokens_int8 + int8_grouped_gemm: tokens to their experts' rows, each expert's product
    sort       sort_routes: a router's choices -> the order of the rows by expert, and back
    exchange   gather_tokens and combine_tokens, with their gradients where `grad` is set

Where `own` is false, `run` computes the same in elementary torch operations.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # A decode step of sixteen sequences: the call itself is the cost.
        {"name": "quantize_decode_16", "op": "quantize", "rows": 16, "k": 8192, "x": "bf16"},
        # The activations of a large prefill, or a weight matrix at load time.
        {"name": "quantize_prefill_8192", "op": "quantize", "rows": 8192, "k": 8192, "x": "bf16"},
        # One token through an 8192 x 8192 projection: the weights stream once.
        {"name": "linear_token_1", "op": "linear", "m": 1, "n": 8192, "k": 8192, "x": "bf16", "out": "bf16"},
        # The wide decode projection of the benchmark: 128 rows of activations against 28672 x 8192 weights.
        {"name": "linear_batch_128", "op": "linear", "m": 128, "n": 28672, "k": 8192, "x": "bf16", "out": "bf16"},
        # A prefill chunk of an odd number of tokens in half precision.
        {"name": "linear_prefill_1000", "op": "linear", "m": 1000, "n": 8192, "k": 8192, "x": "f16", "out": "f16"},
        # The square product of the benchmark.
        {"name": "gemm_8192", "op": "gemm", "m": 8192, "n": 8192, "k": 8192, "out": "bf16"},
        # The first product of the benchmark's expert layer (256 experts, gate and up of 2048, six experts a token): decode.
        {"name": "experts_tokens_64", "op": "experts", "tokens": 64, "topk": 6, "experts": 256, "n": 4096, "k": 4096,
         "x": "bf16", "out": "bf16", "skew": 0.0},
        # The same for a prefill batch, with experts of unequal popularity.
        {"name": "experts_tokens_4096", "op": "experts", "tokens": 4096, "topk": 6, "experts": 256, "n": 4096, "k": 4096,
         "x": "bf16", "out": "bf16", "skew": 0.5},
        # The routing of one decoded token: latency alone.
        {"name": "sort_token_1", "op": "sort", "tokens": 1, "topk": 6, "experts": 256, "skew": 0.0, "dropped": 0.0},
        # The routing of a training batch, a few of whose routes the router dropped.
        {"name": "sort_tokens_16384", "op": "sort", "tokens": 16384, "topk": 8, "experts": 256, "skew": 0.5, "dropped": 0.02},
        # Decode: rows out to the experts and back.
        {"name": "exchange_decode_64", "op": "exchange", "tokens": 64, "topk": 6, "experts": 256, "hidden": 4096, "x": "bf16",
         "grad": False, "skew": 0.0, "dropped": 0.0},
        # A training step's rows out and back, forward and backward.
        {"name": "exchange_train_4096", "op": "exchange", "tokens": 4096, "topk": 6, "experts": 256, "hidden": 4096, "x": "bf16",
         "grad": True, "skew": 0.5, "dropped": 0.02},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _multiple(rng, lo, hi, of):
    return _log_int(rng, max(1, lo // of), hi // of) * of


def draw(rng):
    op = rng.choice(("quantize", "gemm", "linear", "linear", "experts", "sort", "exchange"))
    x = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "quantize":
        k = _log_int(rng, 16, 28672)
        return {"op": op, "rows": _log_int(rng, 1, min(28672, (1 << 25) // k)), "k": k, "x": x}
    if op in ("gemm", "linear"):
        # any number of rows (decode to prefill), layer widths that need not be whole tiles
        k = _multiple(rng, 256, 16384, rng.choice((16, 64, 128)))
        n = _multiple(rng, 64, 28672, rng.choice((8, 64, 256)))
        m = _log_int(rng, 1, max(1, min(8192, (1 << 38) // (n * k))))
        case = {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(("bf16", "f16", "f32"))}
        return {**case, "x": x} if op == "linear" else case
    experts = rng.choice((4, 8, 16, 32, 64, 128, 160, 256))
    topk = min(rng.randint(1, 8), experts)
    tokens = _log_int(rng, 1, 4096)
    skew = rng.choice((0.0, 0.5, 1.0))
    if op == "sort":
        return {"op": op, "tokens": _log_int(rng, 1, 16384), "topk": topk, "experts": experts, "skew": skew,
                "dropped": rng.choice((0.0, 0.05))}
    if op == "experts":
        return {"op": op, "tokens": _log_int(rng, 1, 2048), "topk": min(4, topk), "experts": min(experts, 128),
                "n": _multiple(rng, 256, 4096, 8), "k": _multiple(rng, 256, 4096, 16), "x": x,
                "out": rng.choice(("bf16", "f16", "f32")), "skew": skew}
    return {"op": op, "tokens": min(tokens, 2048 if x == "f32" else 4096), "topk": min(topk, 6), "experts": experts,
            "hidden": _log_int(rng, 64, 4096), "x": x, "grad": rng.random() < 0.6, "skew": skew,
            "dropped": rng.choice((0.0, 0.05))}


# ---- inputs -------------------------------------------------------------------------------------------------------


def _normal(gen, shape, sigma, dtype):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, sigma, generator=gen).to(dtype)


def _activations(gen, rows, k, dtype):
    """Normal values with a few channels far above the others, as the residual stream of a trained model has them."""
    x = torch.empty((rows, k), dtype=torch.float32, device="cuda").normal_(0.0, 1.0, generator=gen)
    x[:, torch.randint(0, k, (max(1, k // 512),), generator=gen, device="cuda")] *= 8.0
    return x.to(dtype)


def _weights(gen, experts, n, k):
    """Layers of normal weights, stored as int8 codes with a scale for each output channel."""
    codes = torch.empty((experts, n, k), dtype=torch.int8, device="cuda")
    scales = torch.empty((experts, n), dtype=torch.float32, device="cuda")
    for e in range(experts):
        w = torch.empty((n, k), dtype=torch.float32, device="cuda").normal_(0.0, 0.02, generator=gen)
        scales[e] = w.abs().amax(1) / 127.0
        codes[e] = torch.round(w / scales[e][:, None]).clamp_(-127.0, 127.0).to(torch.int8)
    return codes, scales


def _router(case, gen):
    """The router's choices: the topk experts of each token by its logits, and weights that sum to one."""
    t, e, topk = case["tokens"], case["experts"], case["topk"]
    logits = torch.randn((t, e), generator=gen, device="cuda")
    if case["skew"]:
        logits += case["skew"] * torch.randn((1, e), generator=gen, device="cuda")
    weights, ids = torch.softmax(logits, -1).topk(topk, -1)
    weights = weights / weights.sum(-1, keepdim=True)
    if case.get("dropped"):
        ids = torch.where(torch.rand((t, topk), generator=gen, device="cuda") < case["dropped"], -1, ids)
    return ids.contiguous(), weights.contiguous()


def _order(ids, experts):
    """Stable order of the routes by expert: (offsets, position, source). Routes of no expert come last."""
    flat = ids.reshape(-1)
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    source = torch.argsort(key, stable=True)
    position = torch.empty_like(source)
    position[source] = torch.arange(source.numel(), device=ids.device)
    offsets = torch.searchsorted(key[source], torch.arange(experts + 1, device=ids.device))
    return offsets.int(), position.int().reshape(ids.shape), source.int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op = case["op"]
    state = {"op": op}
    if op == "quantize":
        return {**state, "x": _activations(gen, case["rows"], case["k"], DTYPES[case["x"]])}
    if op in ("gemm", "linear"):
        weights, scales = _weights(gen, 1, case["n"], case["k"])
        state |= {"b": weights[0], "sb": scales[0], "out": DTYPES[case["out"]]}
        x = _activations(gen, case["m"], case["k"], DTYPES[case.get("x", "bf16")])
        if op == "linear":
            return {**state, "x": x}
        scales = x.float().abs().amax(1) / 127.0
        return {**state, "a": torch.round(x.float() / scales[:, None]).to(torch.int8), "sa": scales}
    ids, weights = _router(case, gen)
    if op == "sort":
        return {**state, "ids": ids, "experts": case["experts"]}
    # the order of the rows, as the router's part of the program left it
    state |= dict(zip(("offsets", "position", "source"), _order(ids, case["experts"])))
    rows, dtype = ids.numel(), DTYPES[case["x"]]
    if op == "experts":
        state["w"], state["sw"] = _weights(gen, case["experts"], case["n"], case["k"])
        # what a program with a fixed number of rows for each expert would know: the most rows that one of them gets
        capacity = int((state["offsets"][1:] - state["offsets"][:-1]).max())
        return {**state, "x": _activations(gen, case["tokens"], case["k"], dtype), "out": DTYPES[case["out"]], "capacity": capacity}
    h = case["hidden"]
    state |= {"grad": case["grad"], "x": _activations(gen, case["tokens"], h, dtype), "weights": weights,
              "expert_out": _normal(gen, (rows, h), 1.0, dtype)}
    if case["grad"]:
        state |= {"d_rows": _normal(gen, (rows, h), 1.0, dtype), "d_y": _normal(gen, (case["tokens"], h), 1.0, dtype)}
        for name in ("x", "weights", "expert_out"):
            state[name].requires_grad_()
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------


def _plain_codes(x):
    """Codes and scales of each row. The quotients in 64 bits: in 32 a value next to a border gets its neighbour's code."""
    amax = x.abs().amax(1).float()
    fine = torch.isfinite(amax)
    quotient = 127.0 * x.double() / amax.double()[:, None]
    codes = torch.where((fine & (amax > 0.0))[:, None], torch.round(quotient), 0.0).to(torch.int8)
    return codes, torch.where(fine, amax / 127.0, torch.nan)


def _plain_product(a, sa, b, sb, out):
    return ((a.float() @ b.float().T) * sa[:, None] * sb).to(out)


def _plain_experts(s):
    offsets, source, topk = s["offsets"].long(), s["source"].long(), s["position"].shape[1]
    codes, scales = _plain_codes(s["x"])
    rows, experts = source.numel(), offsets.numel() - 1
    token = source // topk
    # every expert's rows in a block of the same length, one batched product
    place = offsets[:-1, None] + torch.arange(s["capacity"], device=source.device)
    filled = place < offsets[1:, None]
    blocks = torch.where(filled[..., None], codes[token[place.clamp(max=rows - 1)]].float(), 0.0)
    product = torch.bmm(blocks, s["w"].float().transpose(1, 2))
    row = torch.arange(rows, device=source.device)
    expert = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    live, expert = (expert < experts)[:, None], expert.clamp(max=experts - 1)
    c = product[expert, (row - offsets[expert]).clamp(max=s["capacity"] - 1)] * scales[token][:, None] * s["sw"][expert]
    return torch.where(live, c, 0.0).to(s["out"])


def _plain_exchange(s):
    x, w, expert_out = (s[name].detach() for name in ("x", "weights", "expert_out"))
    position, source = s["position"].long(), s["source"].long()
    topk, live_rows = position.shape[1], s["offsets"][-1].long()
    row_live = (torch.arange(source.numel(), device=source.device) < live_rows)[:, None]
    route_live = (position < live_rows)[..., None]
    token = source // topk
    rows = torch.where(row_live, x[token], 0.0)
    returned = torch.where(route_live, expert_out[position].float(), 0.0)              # [tokens, topk, hidden]
    y = (returned * w[..., None]).sum(1).to(x.dtype)
    if not s["grad"]:
        return {"rows": rows, "y": y}
    d_x = torch.where(route_live, s["d_rows"][position].float(), 0.0).sum(1).to(x.dtype)
    d_expert = torch.where(row_live, s["d_y"].float()[token] * w.reshape(-1)[source][:, None], 0.0).to(x.dtype)
    d_w = (returned * s["d_y"].float()[:, None]).sum(-1)
    return {"rows": rows, "y": y, "d_x": d_x, "d_expert_out": d_expert, "d_weights": d_w}


def _run_own(s):
    import gpu_kernels_b200 as g
    op = s["op"]
    if op == "quantize":
        codes, scales = g.quantize_int8(s["x"])
        return {"values": g.dequantize_int8(codes, scales), "scales": scales}
    if op == "gemm":
        return g.int8_gemm(s["a"], s["b"], s["sa"], s["sb"], out_dtype=s["out"])
    if op == "linear":
        return g.int8_linear(s["x"], s["b"], s["sb"], out_dtype=s["out"])
    if op == "sort":
        return tuple(g.sort_routes(s["ids"], s["experts"]))
    routes = g.Routes(s["offsets"], s["position"], s["source"])
    if op == "experts":
        codes, scales = g.gather_tokens_int8(s["x"], routes)
        return g.int8_grouped_gemm(codes, s["w"], scales, s["sw"], routes.offsets, out_dtype=s["out"])
    rows = g.gather_tokens(s["x"], routes)
    y = g.combine_tokens(s["expert_out"], routes, s["weights"])
    if not s["grad"]:
        return {"rows": rows, "y": y}
    d_x, = torch.autograd.grad(rows, s["x"], s["d_rows"])
    d_expert, d_w = torch.autograd.grad(y, (s["expert_out"], s["weights"]), s["d_y"])
    return {"rows": rows.detach(), "y": y.detach(), "d_x": d_x, "d_expert_out": d_expert, "d_weights": d_w}


def run(state):
    if own:
        return _run_own(state)
    op = state["op"]
    if op == "quantize":
        codes, scales = _plain_codes(state["x"])
        return {"values": codes.float() * scales[:, None], "scales": scales}
    if op == "gemm":
        return _plain_product(state["a"], state["sa"], state["b"], state["sb"], state["out"])
    if op == "linear":
        codes, scales = _plain_codes(state["x"])
        return _plain_product(codes, scales, state["b"], state["sb"], state["out"])
    if op == "sort":
        return _order(state["ids"], state["experts"])
    return _plain_experts(state) if op == "experts" else _plain_exchange(state)


SIZES = {"bf16": 2, "f16": 2, "f32": 4}


def work(case):
    op = case["op"]
    if op == "quantize":
        n = case["rows"] * case["k"]
        return {"bytes": n * (SIZES[case["x"]] + 1 + 1 + 4) + 8 * case["rows"], "flops": 0}
    if op in ("gemm", "linear"):
        m, n, k = case["m"], case["n"], case["k"]
        a = 1 if op == "gemm" else SIZES[case["x"]]
        return {"bytes": m * k * a + n * k + 4 * n + m * n * SIZES[case["out"]] + (4 * m if op == "gemm" else 0), "flops": 2.0 * m * n * k}
    t, topk, e = case["tokens"], case["topk"], case["experts"]
    routes = t * topk
    if op == "sort":
        return {"bytes": routes * 16 + 4 * (e + 1), "flops": 0}
    if op == "experts":
        n, k = case["n"], case["k"]
        live = e * (1.0 - (1.0 - topk / e) ** t) if topk < e else e        # experts that some token is sent to (equal popularity)
        return {"bytes": live * n * (k + 4) + t * k * SIZES[case["x"]] + routes * (4 + n * SIZES[case["out"]]),
                "flops": 2.0 * routes * n * k}
    token, row = t * case["hidden"] * SIZES[case["x"]], routes * case["hidden"] * SIZES[case["x"]]
    # out: a token's row read, its rows written; back: the rows read, the token's written; the gradients the other way round,
    # that of the weighted sum reading the rows again for the weights' gradient
    forward, backward = 2 * (token + row) + 12 * routes, 2 * token + 3 * row + 16 * routes
    return {"bytes": forward + (backward if case["grad"] else 0), "flops": 0}


# ---- the same results from the definitions, in 64 bits ------------------------------------------------------------


def _exact_codes(x):
    """The integers nearest to 127 x / max|x| of each row (an even one between two), and max|x| / 127."""
    top = x.double().abs().max(1, keepdim=True).values
    ratio = torch.where(top > 0.0, x.double() * 127.0 / top, 0.0)
    low = torch.floor(ratio)
    up = (ratio - low > 0.5) | ((ratio - low == 0.5) & (low.remainder(2.0) == 1.0))
    return low + up, (top / 127.0).squeeze(1)


def exact(case, seed):
    op = case["op"]
    if op == "sort":
        return None                                               # whole numbers
    s = prepare(case, seed)
    if op == "quantize":
        codes, scales = _exact_codes(s["x"])
        return {"values": codes * scales[:, None], "scales": scales}
    if op == "gemm":
        return (s["a"].double() * s["sa"].double()[:, None]) @ (s["b"].double() * s["sb"].double()[:, None]).T
    if op == "linear":
        codes, scales = _exact_codes(s["x"])
        return (codes * scales[:, None]) @ (s["b"].double() * s["sb"].double()[:, None]).T
    offsets = s["offsets"].tolist()
    token = s["source"].long() // case["topk"]
    if op == "experts":
        codes, scales = _exact_codes(s["x"])
        c = torch.zeros((token.numel(), case["n"]), dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            own_rows = slice(offsets[e], offsets[e + 1])
            if offsets[e] < offsets[e + 1]:
                a = (codes * scales[:, None])[token[own_rows]]
                c[own_rows] = a @ (s["w"][e].double() * s["sw"][e].double()[:, None]).T
        return c
    live = offsets[-1]
    x, w, expert_out = (s[name].detach().double() for name in ("x", "weights", "expert_out"))
    route = s["source"].long()[:live]
    token = token[:live]
    rows = torch.zeros_like(expert_out)
    rows[:live] = x[token]
    y = torch.zeros_like(x).index_add_(0, token, w.reshape(-1)[route][:, None] * expert_out[:live])
    if not case["grad"]:
        return {"rows": rows, "y": y}
    d_y = s["d_y"].double()
    d_x = torch.zeros_like(x).index_add_(0, token, s["d_rows"].double()[:live])
    d_expert = torch.zeros_like(expert_out)
    d_expert[:live] = w.reshape(-1)[route][:, None] * d_y[token]
    d_w = torch.zeros(w.numel(), dtype=torch.float64, device="cuda")
    d_w[route] = (expert_out[:live] * d_y[token]).sum(-1)
    return {"rows": rows, "y": y, "d_x": d_x, "d_expert_out": d_expert, "d_weights": d_w.reshape(w.shape)}
