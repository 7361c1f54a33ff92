"""The bucketed ("grouped by expert") matrix products and what belongs to them, as workloads.

Five operators of the framework: the grouping of a batch's rows by bucket (`GroupPlan`), the grouped linear layer with
its gradients (`grouped_linear`), the quantisation to 8-bit floating point with one scale per row block of 128 and per
tile of 128 x 128 (`quantize_fp8_rows`, `quantize_fp8_tiles`), and the 8-bit linear layer, grouped or dense (`linear_fp8`).

`run` computes them in plain torch operations in 32 bits where `own` is false and through the framework's entry points
where it is true; `exact` restates the definitions in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FORMATS = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}


def listed():
    return [
        # one training batch routed to the eight piece-count buckets
        {"name": "plan-batch", "op": "plan", "T": 16384, "E": 8, "routing": "pieces", "wide_ids": True},
        # a large batch over many experts, ids as a router's argmax leaves them
        {"name": "plan-many", "op": "plan", "T": 262143, "E": 256, "routing": "zipf", "wide_ids": False},
        # first layer of the layer stack in mixed precision: fp32 parameters, 16-bit activations, 32 outputs per bucket
        {"name": "train-stack", "op": "train", "T": 16384, "E": 8, "K": 1024, "N": 32, "dtype": "bf16", "weights": "fp32",
         "routing": "pieces"},
        # the largest step: wide layers in bf16, forward and all three gradients
        {"name": "train-wide", "op": "train", "T": 16384, "E": 8, "K": 4096, "N": 2048, "dtype": "bf16", "weights": "bf16",
         "routing": "pieces"},
        # many experts of very different sizes, some empty, padding rows, sizes that no tile divides, fp16
        {"name": "train-ragged", "op": "train", "T": 6001, "E": 64, "K": 1000, "N": 200, "dtype": "fp16", "weights": "fp16",
         "routing": "zipf"},
        # one position evaluated at a time: latency
        {"name": "eval-one", "op": "eval", "T": 1, "E": 8, "K": 1024, "N": 1024, "dtype": "bf16", "weights": "bf16",
         "routing": "pieces"},
        # a few positions over many experts: every expert's weights are read for a row or two
        {"name": "eval-few", "op": "eval", "T": 96, "E": 64, "K": 2048, "N": 1024, "dtype": "bf16", "weights": "bf16",
         "routing": "even"},
        # activations of a large batch on their way into an 8-bit layer
        {"name": "quantize-rows", "op": "rows8", "T": 16384, "K": 4096, "dtype": "bf16", "format": "e4m3"},
        # fp32 parameters of a bucketed layer, quantised once per export; sizes that 128 does not divide
        {"name": "quantize-tiles", "op": "tiles8", "E": 8, "N": 1000, "K": 2040, "dtype": "fp32", "format": "e4m3"},
        # single position through an 8-bit bucketed layer
        {"name": "fp8-one", "op": "fp8", "T": 1, "E": 8, "K": 2048, "N": 1024, "dtype": "bf16", "format": "e4m3",
         "routing": "pieces"},
        # evaluation of a large batch through an 8-bit bucketed layer
        {"name": "fp8-wide", "op": "fp8", "T": 16384, "E": 8, "K": 4096, "N": 2048, "dtype": "bf16", "format": "e4m3",
         "routing": "pieces"},
        # a dense 8-bit layer of odd sizes in the wide-range format
        {"name": "fp8-dense", "op": "fp8", "T": 4099, "E": 1, "K": 2000, "N": 1500, "dtype": "fp16", "format": "e5m2",
         "routing": "dense"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm, odd ones among them."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "train", "train", "eval", "rows8", "tiles8", "fp8", "fp8"])
    routing = rng.choice(["pieces", "zipf", "even"])
    if op == "plan":
        return {"op": op, "T": _spread(rng, 1, 1 << 18), "E": _spread(rng, 1, 512), "routing": routing,
                "wide_ids": rng.random() < 0.5}
    if op == "rows8":
        return {"op": op, "T": _spread(rng, 1, 16384), "K": _spread(rng, 16, 4096), "dtype": rng.choice(sorted(DTYPES)),
                "format": rng.choice(sorted(FORMATS))}
    if op == "tiles8":
        return {"op": op, "E": _spread(rng, 1, 16), "N": _spread(rng, 1, 2048), "K": _spread(rng, 16, 4096),
                "dtype": rng.choice(sorted(DTYPES)), "format": rng.choice(sorted(FORMATS))}
    case = {"op": op, "T": _spread(rng, 1, 16384), "E": _spread(rng, 1, 64), "K": _spread(rng, 16, 4096),
            "N": _spread(rng, 1, 2048), "dtype": rng.choice(["bf16", "fp16"])}
    if op == "eval":
        case["T"] = _spread(rng, 1, 512)
    case["E"] = max(1, min(case["E"], (1 << 26) // (case["N"] * case["K"])))  # the listed cases' number of weights at most
    if op == "fp8":
        if rng.random() < 0.3:
            return {**case, "E": 1, "format": rng.choice(sorted(FORMATS)), "routing": "dense"}
        return {**case, "format": rng.choice(sorted(FORMATS)), "routing": routing}
    return {**case, "weights": rng.choice([case["dtype"], "fp32"]), "routing": routing}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _buckets(case, g):
    """Bucket ids as the batch brings them; -1 marks a padding row."""
    T, E = case["T"], case["E"]
    if case["routing"] == "pieces":  # piece counts of real games: most positions in the middle buckets
        u = (torch.rand(T, generator=g, device="cuda") + torch.rand(T, generator=g, device="cuda")) / 2
        b = (u * E).to(torch.int64).clamp_(max=E - 1)
    elif case["routing"] == "zipf":  # a few large experts, a long tail, some empty; one row in 16 is padding
        u = torch.rand(T, generator=g, device="cuda")
        b = (torch.exp(u * math.log(E + 1.0)) - 1.0).to(torch.int64).clamp_(max=E - 1)
        if T > 1:
            b = torch.where(torch.rand(T, generator=g, device="cuda") < 1 / 16, torch.full_like(b, -1), b)
    else:
        b = torch.randint(0, E, (T,), generator=g, device="cuda")
    return b if case.get("wide_ids", True) else b.to(torch.int32)


def _activations(T, K, g, dtype):
    """Clipped activations times a scale of their own for each row; about half of them are zero."""
    x = torch.randn(T, K, generator=g, device="cuda").clamp_(min=0)
    return (x * torch.exp(0.5 * torch.randn(T, 1, generator=g, device="cuda"))).to(dtype)


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "plan":
        return {"case": case, "bucket": _buckets(case, g)}
    if op == "rows8":
        return {"case": case, "x": _activations(case["T"], case["K"], g, DTYPES[case["dtype"]])}
    if op == "tiles8":
        w = torch.randn(case["E"] * case["N"], case["K"], generator=g, device="cuda") * 0.02
        return {"case": case, "w": w.to(DTYPES[case["dtype"]])}
    T, E, K, N, dtype = case["T"], case["E"], case["K"], case["N"], DTYPES[case["dtype"]]
    bucket = None if case["routing"] == "dense" else _buckets(case, g)
    x = _activations(T, K, g, dtype)
    w = torch.randn(E * N, K, generator=g, device="cuda") / math.sqrt(K)
    bias = torch.randn(E * N, generator=g, device="cuda") * 0.1
    if op == "fp8":
        q, scale = _tiles8(w, E, case["format"])
        pitch = -(-K // 16) * 16  # rows of 8-bit weights start at multiples of 16 bytes, as the quantiser leaves them
        rows = torch.zeros(E * N, pitch, dtype=torch.uint8, device="cuda")
        rows[:, :K] = q.view(torch.uint8)
        q = rows.view(q.dtype)[:, :K]
        return {"case": case, "bucket": bucket, "x": x, "q": q, "scale": scale, "bias": bias}
    w, bias = w.to(DTYPES[case["weights"]]), bias.to(DTYPES[case["weights"]])
    state = {"case": case, "bucket": bucket, "x": x, "w": w, "bias": bias}
    if op == "train":
        state["dy"] = (torch.randn(T, N, generator=g, device="cuda") / math.sqrt(N)).to(dtype)
        for name in ("x", "w", "bias"):
            state[name].requires_grad_(True)
    return state


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _plan(bucket, E):
    """(order, offsets): rows by bucket in their own order, padding rows last; offsets[e] is the first place of bucket e."""
    key = torch.where(bucket < 0, torch.full_like(bucket, E), bucket)
    order = torch.sort(key, stable=True).indices
    sizes = (key.view(-1, 1) == torch.arange(E, device=key.device)).sum(0) if key.numel() * E <= 1 << 27 else \
        torch.bincount(key, minlength=E + 1)[:E]
    return order.to(torch.int32), torch.cat([sizes.new_zeros(1), sizes.cumsum(0)]).to(torch.int32)


def _padded(bucket, E, T):
    """Rows laid out as [E, capacity] (T where a place is empty): the ragged product becomes one batched product."""
    if bucket is None:
        return torch.arange(T, device="cuda").view(1, T)
    order, offsets = (t.to(torch.int64) for t in _plan(bucket, E))
    sizes = offsets[1:] - offsets[:-1]
    capacity = max(1, int(sizes.max()))
    place = torch.arange(capacity, device="cuda")
    rows = order[(offsets[:-1, None] + place).clamp_(max=T - 1)]
    return torch.where(place < sizes[:, None], rows, torch.full_like(rows, T))


def _gathered(x, rows):
    """x[rows] with a row of zeros behind the last one."""
    return torch.cat([x, x.new_zeros(1, x.shape[1])])[rows]


def _scattered(y, rows, T):
    out = y.new_zeros(T + 1, y.shape[-1])
    out[rows.reshape(-1)] = y.reshape(-1, y.shape[-1])
    return out[:T]


def _product(x, w, bias, rows):
    E, T = rows.shape[0], x.shape[0]
    w = w.view(E, -1, w.shape[-1])
    y = torch.matmul(_gathered(x, rows), w.transpose(1, 2)) + bias.view(E, 1, -1)
    return _scattered(y, rows, T)


def _block_scale(largest, format):
    """2^ceil(log2(largest / MAX)); 1 for an empty block.  Both formats' MAX is 7/8 of a power of two."""
    m, e = torch.frexp(largest)
    top = {"e4m3": 9, "e5m2": 16}[format]
    e = torch.where(m > 0.875, e + 1, e) - top
    return torch.where(largest > 0, torch.ldexp(torch.ones_like(largest), e.clamp(min=-126)), torch.ones_like(largest))


def _rows8(x, format):
    T, K = x.shape
    C = -(-K // 128)
    p = torch.nn.functional.pad(x.float(), (0, C * 128 - K)).view(T, C, 128)
    scale = _block_scale(p.abs().amax(2), format)
    return (p / scale[:, :, None]).to(FORMATS[format]).view(T, C * 128)[:, :K], scale


def _tiles8(w, E, format):
    K = w.shape[-1]
    N = w.shape[0] // E
    R, C = -(-N // 128), -(-K // 128)
    p = torch.nn.functional.pad(w.float().view(E, N, K), (0, C * 128 - K, 0, R * 128 - N)).view(E, R, 128, C, 128)
    scale = _block_scale(p.abs().amax((2, 4)), format)
    q = (p / scale[:, :, None, :, None]).to(FORMATS[format]).view(E, R * 128, C * 128)
    return q[:, :N, :K].reshape(E * N, K), scale


def _rows_values(q, scale):
    return q.to(scale.dtype) * scale.repeat_interleave(128, 1)[:, : q.shape[1]]


def _tiles_values(q, scale, E):
    N = q.shape[0] // E
    s = scale.repeat_interleave(128, 1)[:, :N].repeat_interleave(128, 2)[:, :, : q.shape[1]]
    return q.to(scale.dtype) * s.reshape(E * N, -1)


def _run_plain(state):
    case = state["case"]
    op = case["op"]
    if op == "plan":
        order, offsets = _plan(state["bucket"], case["E"])
        return {"order": order, "offsets": offsets}
    if op == "rows8":
        q, scale = _rows8(state["x"], case["format"])
        return {"q": q, "scale": scale}
    if op == "tiles8":
        q, scale = _tiles8(state["w"], case["E"], case["format"])
        return {"q": q, "scale": scale}
    E, dtype = case["E"], DTYPES[case["dtype"]]
    rows = _padded(state["bucket"], E, case["T"])
    if op == "fp8":
        x = _rows_values(*_rows8(state["x"], case["format"]))
        w = _tiles_values(state["q"], state["scale"], E)
        return _product(x, w, state["bias"], rows).to(dtype)
    x, w = state["x"].float(), state["w"].to(dtype).float()  # fp32 parameters are rounded to the activations' type
    y = _product(x, w, state["bias"].float(), rows).to(dtype)
    if op == "eval":
        return y
    dy = _gathered(state["dy"].float(), rows)
    dx = _scattered(torch.matmul(dy, w.view(E, -1, w.shape[1])), rows, case["T"])
    dw = torch.matmul(dy.transpose(1, 2), _gathered(x, rows))
    out = DTYPES[case["weights"]]
    return {"y": y, "dx": dx.to(dtype), "dw": dw.view_as(w).to(out), "dbias": dy.sum(1).view(-1).to(out)}


def run(state):
    if not own:
        with torch.no_grad():
            return _run_plain(state)
    from nnue_pytorch_b200 import fp8_functions as f8
    from nnue_pytorch_b200 import grouped_linear_functions as gl

    case = state["case"]
    op = case["op"]
    if op == "plan":
        plan = gl.GroupPlan(state["bucket"], case["E"])
        return {"order": plan.order, "offsets": plan.offsets}
    if op == "rows8":
        blocks = f8.quantize_fp8_rows(state["x"], FORMATS[case["format"]])
        return {"q": blocks.q, "scale": blocks.scale}
    if op == "tiles8":
        blocks = f8.quantize_fp8_tiles(state["w"], case["E"], FORMATS[case["format"]])
        return {"q": blocks.q, "scale": blocks.scale}
    plan = None if state["bucket"] is None else gl.GroupPlan(state["bucket"], case["E"])
    if op == "fp8":
        return f8.linear_fp8(state["x"], f8.Fp8Blocks(state["q"], state["scale"]), state["bias"], plan)
    if op == "eval":
        with torch.no_grad():
            return gl.grouped_linear(state["x"], state["w"], state["bias"], plan)
    y = gl.grouped_linear(state["x"], state["w"], state["bias"], plan)
    dx, dw, dbias = torch.autograd.grad(y, (state["x"], state["w"], state["bias"]), state["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "dbias": dbias}


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    op = case["op"]
    if op == "plan":
        return {"bytes": case["T"] * ((8 if case["wide_ids"] else 4) + 4) + 4 * (case["E"] + 1), "flops": 0}
    if op == "rows8":
        T, K = case["T"], case["K"]
        return {"bytes": T * K * (size[case["dtype"]] + 1) + 4 * T * -(-K // 128), "flops": 0}
    if op == "tiles8":
        E, N, K = case["E"], case["N"], case["K"]
        return {"bytes": E * N * K * (size[case["dtype"]] + 1) + 4 * E * -(-N // 128) * -(-K // 128), "flops": 0}
    T, E, K, N = case["T"], case["E"], case["K"], case["N"]
    ids = 0 if case["routing"] == "dense" else 8 * T
    read = min(E, T)  # buckets whose weights can be needed
    if op == "fp8":
        return {"bytes": 2 * T * (K + N) + read * N * (K + 4) + ids, "flops": 2 * T * N * K}
    weights = size[case["weights"]]
    forward = 2 * T * (K + N) + read * N * (K + 1) * weights + ids
    if op == "eval":
        return {"bytes": forward, "flops": 2 * T * N * K}
    # backward: dy once; x and w are in hand, but a pass of their own reads them again; dx, dw and dbias are written
    return {"bytes": forward + 2 * T * (N + K) + E * N * (K + 1) * weights, "flops": 6 * T * N * K}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def _exact_scale(block, format):
    largest = block.abs().amax(-1)
    power = torch.ceil(torch.log2(largest / LARGEST[format]))
    # log2 of a number next to a power of two may land on either side: settle it by comparison
    power = torch.where(torch.exp2(power - 1) * LARGEST[format] >= largest, power - 1, power)
    power = torch.where(torch.exp2(power) * LARGEST[format] < largest, power + 1, power)
    return torch.where(largest > 0, torch.exp2(power.clamp(min=-126)), torch.ones_like(largest))


def _exact_round8(v, format):
    """v, at most MAX in size, to the nearest number of the format, ties to even."""
    bits, lowest = {"e4m3": (3, -6), "e5m2": (2, -14)}[format]
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0**-60)))
    exponent = torch.where(torch.exp2(exponent) > v.abs(), exponent - 1, exponent)
    exponent = torch.where(torch.exp2(exponent + 1) <= v.abs(), exponent + 1, exponent)
    step = torch.exp2(exponent.clamp(min=lowest) - bits)
    return torch.round(v / step) * step


def _exact_rows8(x, format):
    q, scales = torch.empty_like(x), []
    for k in range(0, x.shape[1], 128):
        s = _exact_scale(x[:, k : k + 128], format)
        q[:, k : k + 128] = _exact_round8(x[:, k : k + 128] / s[:, None], format)
        scales.append(s)
    return q, torch.stack(scales, 1)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op == "plan":
            return None  # whole numbers
        if op == "rows8":
            q, scale = _exact_rows8(state["x"].double(), case["format"])
            return {"q": q, "scale": scale}
        if op == "tiles8":
            E, N, K = case["E"], case["N"], case["K"]
            w = state["w"].double().view(E, N, K)
            q = torch.empty_like(w)
            scale = torch.empty(E, -(-N // 128), -(-K // 128), dtype=torch.float64, device="cuda")
            for n in range(0, N, 128):
                for k in range(0, K, 128):
                    block = w[:, n : n + 128, k : k + 128]
                    s = _exact_scale(block.reshape(E, -1), case["format"])
                    scale[:, n // 128, k // 128] = s
                    q[:, n : n + 128, k : k + 128] = _exact_round8(block / s.view(E, 1, 1), case["format"])
            return {"q": q.view(E * N, K), "scale": scale}
        T, E, K, N = case["T"], case["E"], case["K"], case["N"]
        x, bias = state["x"].double(), state["bias"].double().view(E, N)
        if op == "fp8":
            q, scale = _exact_rows8(x, case["format"])
            x = q * scale.repeat_interleave(128, 1)[:, :K]
            w = _tiles_values(state["q"], state["scale"].double(), E).view(E, N, K)
        else:
            w = state["w"].to(DTYPES[case["dtype"]]).double().view(E, N, K)
        bucket = torch.zeros(T, dtype=torch.int64, device="cuda") if state["bucket"] is None else state["bucket"]
        y = torch.zeros(T, N, dtype=torch.float64, device="cuda")
        dx, dw, dbias = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(bias)
        for e in range(E):
            rows = torch.nonzero(bucket == e).view(-1)
            y[rows] = x[rows] @ w[e].T + bias[e]
            if op == "train":
                dy = state["dy"].double()[rows]
                dx[rows] = dy @ w[e]
                dw[e] = dy.T @ x[rows]
                dbias[e] = dy.sum(0)
        if op != "train":
            return y
        return {"y": y, "dx": dx, "dw": dw.view(E * N, K), "dbias": dbias.view(-1)}
