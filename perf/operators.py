"""Matrix products in 8-bit integers and the routing of tokens to experts, as cases that can be timed and compared.

The operators: weights held as int8 with a scale per output channel (`Int8Tensor`), their product with activations that get a scale per
token (`Int8MatMul`), tokens sorted by expert and back with weights applied, and the gradients of both (`TokenRouting`), and the experts'
products between the two (`Int8Experts`). The plain forms below say what each computes:

* a row of values x becomes s = max|x| / 127, held in 32 bits, and q = the integer next to x / s, ties to the even one;
* a product is the exact integer sum of q_x q_w, times the token's scale, times the channel's;
* the experts' hidden values act(gate) * up are held in the activations' type and become int8 rows again;
* a slot whose expert is -1 goes nowhere: no row, no weight, no gradient.
"""
from __future__ import annotations

import math

import torch

own = False

ELEMS = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# the largest listed products and passes over memory: nothing drawn costs more
MAX_LINEAR = 8192 * 28672 * 4096
MAX_QUANTIZE = 14336 * 4096
MAX_EXPERTS = 2048 * 2 * 3 * 14336 * 4096
MAX_EXPERT_WEIGHTS = 8 * 3 * 14336 * 4096
MAX_ROUTE = 4096 * 2 * 4096


def _linear(name, rows, k, n, dtype):
    return {"name": name, "kind": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype}


def _experts(name, tokens, experts, topk, hidden, ffn, dtype):
    return {"name": name, "kind": "experts", "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden, "ffn": ffn,
            "act": "silu", "dropped": 0.0, "dtype": dtype}


def _route(name, tokens, experts, topk, hidden, dropped, train, dtype):
    return {"name": name, "kind": "route", "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden, "dropped": dropped,
            "train": train, "dtype": dtype}


def listed():
    return [
        # One decoded token through a small projection (attn_k of the 8B model): latency is all there is.
        _linear("linear_1_small", 1, 4096, 1024, "bf16"),
        # Sixteen sequences decoded together through the deep projection, ffn_down.
        _linear("linear_16_deep", 16, 14336, 4096, "bf16"),
        # A short prompt of a ragged length through the fused q/k/v shape.
        _linear("linear_333", 333, 4096, 6144, "f16"),
        # A long prompt through gate + up: the largest product.
        _linear("linear_8192_wide", 8192, 4096, 28672, "bf16"),
        # A weight matrix becomes int8 while a model is loaded, and what it then stands for.
        {"name": "quantize_load", "kind": "quantize", "rows": 14336, "k": 4096, "dtype": "f32"},
        # The same for a small matrix of odd width, out of a 16-bit checkpoint.
        {"name": "quantize_small", "kind": "quantize", "rows": 257, "k": 1001, "dtype": "bf16"},
        # One decoded token through a layer of eight wide experts, two of which it uses.
        _experts("experts_1", 1, 8, 2, 4096, 14336, "bf16"),
        # Forty-eight sequences decoded together through a layer of many narrow experts.
        _experts("experts_48_narrow", 48, 64, 6, 2048, 1408, "bf16"),
        # A prompt through a layer of eight wide experts: the largest.
        _experts("experts_2048", 2048, 8, 2, 4096, 14336, "bf16"),
        # Seven tokens of a decode batch to 128 experts and back: the smallest routing, forward only.
        _route("route_7", 7, 128, 8, 2048, 0.0, False, "f16"),
        # A training step's routing of a batch of 4096 tokens: forward and gradients.
        _route("route_train_4096", 4096, 8, 2, 4096, 0.0, True, "bf16"),
        # The same on a rank that holds a part of the experts (a third of the slots belongs elsewhere), odd sizes, in 32 bits.
        _route("route_train_777", 777, 60, 4, 1037, 0.33, True, "f32"),
    ]


# ---- the ranges the listed cases stand for -------------------------------------------------------------------------------

def _log_int(rng, lo, hi, step=1):
    return max(lo, int(round(lo * (hi / lo) ** rng.random() / step)) * step)


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "quantize", "experts", "experts", "route", "route"])
    step = rng.choice([1, 2, 8, 64, 128])
    if kind == "linear":
        while True:
            case = {"kind": kind, "rows": _log_int(rng, 1, 8192), "k": _log_int(rng, 256, 14336, step), "n": _log_int(rng, 64, 28672, step),
                    "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
            if case["rows"] * case["k"] * case["n"] <= MAX_LINEAR:
                return case
    if kind == "quantize":
        while True:
            case = {"kind": kind, "rows": _log_int(rng, 64, 28672), "k": _log_int(rng, 64, 14336, step), "dtype": rng.choice(list(ELEMS))}
            if case["rows"] * case["k"] <= MAX_QUANTIZE:
                return case
    while True:
        experts = rng.choice([2, 4, 8, 16, 60, 64, 128])
        case = {"kind": kind, "tokens": _log_int(rng, 1, 4096), "experts": experts, "topk": rng.randint(1, min(8, experts)),
                "hidden": _log_int(rng, 256, 6144, step), "dropped": rng.choice([0.0, 0.0, 0.1, 0.5])}
        slots = case["tokens"] * case["topk"]
        if kind == "route":
            case |= {"train": rng.random() < 0.7, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
            if slots * case["hidden"] <= MAX_ROUTE:
                return case
            continue
        # 16-bit activations, as models with experts run: the hidden values between the two products have that type
        case |= {"ffn": _log_int(rng, 128, 14336, step), "act": rng.choice(["silu", "silu", "gelu"]), "dtype": rng.choice(["bf16", "f16"])}
        values = 3 * case["hidden"] * case["ffn"]
        if slots * values <= MAX_EXPERTS and experts * values <= MAX_EXPERT_WEIGHTS:
            return case


# ---- inputs --------------------------------------------------------------------------------------------------------------

def _channels(experts, n, k, gen):
    """N(0, 0.02) weights as int8 and a scale per output channel, as a checkpoint in this form holds them."""
    data = torch.empty(experts, n, k, dtype=torch.int8, device="cuda")
    scales = torch.empty(experts, n, device="cuda")
    for e in range(experts):
        w = torch.randn(n, k, device="cuda", generator=gen).mul_(0.02)
        scales[e] = w.abs().amax(1) / 127
        data[e] = torch.round(w / scales[e][:, None]).to(torch.int8)
    return data, scales


def _acts(rows, k, dtype, gen):
    """N(0, 1) activations with the few large features that hidden states have."""
    x = torch.randn(rows, k, device="cuda", generator=gen)
    x[:, torch.randperm(k, device="cuda", generator=gen)[: max(1, k // 512)]] *= 6
    return x.to(ELEMS[dtype])


def _router(case, gen):
    """A router's choice: the highest of logits that prefer some experts, with the softmax of the chosen ones."""
    logits = torch.randn(case["tokens"], case["experts"], device="cuda", generator=gen)
    logits += 0.5 * torch.randn(case["experts"], device="cuda", generator=gen)
    top, ids = logits.topk(case["topk"], dim=1)
    ids = ids.to(torch.int32)
    if case["dropped"]:
        ids[torch.rand(ids.shape, device="cuda", generator=gen) < case["dropped"]] = -1
    return ids, top.softmax(1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if own:
        import inference_rs_b200 as pkg
    if kind == "linear":
        data, scales = _channels(1, case["n"], case["k"], gen)
        s = {"kind": kind, "x": _acts(case["rows"], case["k"], case["dtype"], gen)}
        if own:
            s["linear"] = pkg.Int8MatMul(pkg.Int8Tensor(data[0], scales[0]))
        else:
            s["w"] = (data[0], scales[0])
        return s
    if kind == "quantize":
        w = torch.randn(case["rows"], case["k"], device="cuda", generator=gen).mul_(0.02)
        return {"kind": kind, "w": w.to(ELEMS[case["dtype"]])}
    tokens, hidden = case["tokens"], case["hidden"]
    ids, weights = _router(case, gen)
    s = {"kind": kind, "ids": ids, "weights": weights, "experts": case["experts"], "x": _acts(tokens, hidden, case["dtype"], gen)}
    if kind == "experts":
        parts = [_channels(case["experts"], n, k, gen) for n, k in ((case["ffn"], hidden), (case["ffn"], hidden), (hidden, case["ffn"]))]
        if own:
            s["layer"] = pkg.Int8Experts(*(pkg.Int8Tensor(*p) for p in parts), activation=case["act"])
        else:
            s |= {"parts": parts, "act": case["act"]}
        return s
    s["y"] = torch.randn(ids.numel(), hidden, device="cuda", generator=gen).to(ELEMS[case["dtype"]])
    s["train"] = case["train"]
    if case["train"]:
        s["grad_rows"] = torch.randn(ids.numel(), hidden, device="cuda", generator=gen).to(ELEMS[case["dtype"]])
        s["grad_out"] = torch.randn(tokens, hidden, device="cuda", generator=gen).to(ELEMS[case["dtype"]])
        for name in ("x", "y", "weights"):
            s[name].requires_grad_()
    return s


# ---- one pass, plain form ------------------------------------------------------------------------------------------------

def _rows_to_int8(x):
    """The quotients in 64 bits: in 32 a value next to the border between two integers could fall on either side. The scale, too, is
    the rounded quotient, not a product with 1 / 127."""
    amax = x.float().abs().amax(1)
    scales = torch.where(torch.isfinite(amax), (amax.double() / 127).float(), torch.nan)
    q = torch.round(x.double() / scales.double()[:, None])
    return torch.nan_to_num(q, 0.0), scales


def _product(q, scales, data, channel_scales):
    """Sums of up to 2^31 do not fit into the 24 bits of a float: the product is made of 64-bit values."""
    return (q @ data.double().T).float() * scales[:, None] * channel_scales


def _activate(name, g):
    if name == "silu":
        return g / (1 + torch.exp(-g))
    return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))


def _sorted_slots(ids, experts):
    """Slots in the order of their experts (those of one expert in their own order), where each expert's rows start, and each slot's
    row. Slots that go nowhere come last and count as -1."""
    flat = torch.where((ids >= 0) & (ids < experts), ids, experts).flatten().long()
    order = torch.argsort(flat, stable=True)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device).index_add_(0, flat, torch.ones_like(flat))
    offsets = torch.cat([counts.new_zeros(1), counts[:experts].cumsum(0)])
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=ids.device)
    position = torch.where(flat < experts, position, -1)
    order = torch.where(torch.arange(order.numel(), device=ids.device) < offsets[-1], order, -1)
    return order.int(), offsets.int(), position.int().view(ids.shape)


def _to_rows(values, order, topk):
    """Row r: the token of slot order[r]; zeros where there is none."""
    rows = values[order.clamp(min=0).long() // topk]
    return torch.where(order[:, None] >= 0, rows, 0)


def _from_rows(rows, position, weights):
    """Token t: sum over its slots of weight * row."""
    picked = torch.where(position[..., None] >= 0, rows.float()[position.clamp(min=0).long()], 0)
    return (picked * torch.where(position >= 0, weights, 0)[..., None]).sum(1)


@torch.no_grad()
def _plain(s):
    kind = s["kind"]
    if kind == "linear":
        return _product(*_rows_to_int8(s["x"]), *s["w"]).to(s["x"].dtype)
    if kind == "quantize":
        q, scales = _rows_to_int8(s["w"])
        return {"values": q.float() * scales[:, None], "scales": scales}
    x, ids, weights = s["x"], s["ids"], s["weights"]
    order, offsets, position = _sorted_slots(ids, s["experts"])
    topk = ids.shape[1]
    if kind == "experts":
        (gate, gate_s), (up, up_s), (down, down_s) = s["parts"]
        q, scales = _rows_to_int8(x)
        y = torch.zeros(ids.numel(), x.shape[1], device=x.device)
        starts = offsets.tolist()
        for e in range(s["experts"]):
            slots = order[starts[e]:starts[e + 1]].long()
            if slots.numel() == 0:
                continue
            qe, se = q[slots // topk], scales[slots // topk]
            hidden = _activate(s["act"], _product(qe, se, gate[e], gate_s[e])) * _product(qe, se, up[e], up_s[e])
            y[starts[e]:starts[e + 1]] = _product(*_rows_to_int8(hidden.to(x.dtype)), down[e], down_s[e])
        return _from_rows(y, position, weights).to(x.dtype)
    y = s["y"]
    out = {"order": order, "offsets": offsets, "position": position, "rows": _to_rows(x, order, topk),
           "out": _from_rows(y, position, weights).to(x.dtype)}
    if s["train"]:
        grad_out = s["grad_out"].float()
        slot_weights = torch.where(order >= 0, weights.flatten()[order.clamp(min=0).long()], 0)
        picked = y.float()[position.clamp(min=0).long()]
        out["grad_x"] = _from_rows(s["grad_rows"], position, torch.ones_like(weights)).to(x.dtype)
        out["grad_y"] = (_to_rows(grad_out, order, topk) * slot_weights[:, None]).to(y.dtype)
        out["grad_weights"] = torch.where(position >= 0, (picked * grad_out[:, None, :]).sum(2), 0)
    return out


# ---- one pass, the framework's operators ---------------------------------------------------------------------------------

def _own(s):
    kind = s["kind"]
    if kind == "linear":
        return s["linear"].forward(s["x"])
    import inference_rs_b200 as pkg
    if kind == "quantize":
        t = pkg.Int8Tensor.quantize(s["w"])
        return {"values": t.dequantize(), "scales": t.scales}
    if kind == "experts":
        return s["layer"].forward(s["x"], s["ids"], s["weights"])
    routing = pkg.TokenRouting(s["ids"], s["experts"])
    rows = routing.dispatch(s["x"])
    out = routing.combine(s["y"], s["weights"])
    result = {"order": routing.order, "offsets": routing.offsets, "position": routing.position, "rows": rows.detach(), "out": out.detach()}
    if s["train"]:
        grads = torch.autograd.grad([rows, out], [s["x"], s["y"], s["weights"]], [s["grad_rows"], s["grad_out"]])
        result |= dict(zip(("grad_x", "grad_y", "grad_weights"), grads))
    return result


def run(s):
    return _own(s) if own else _plain(s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------

def work(case):
    kind, es = case["kind"], ELEMS[case["dtype"]].itemsize
    if kind == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": n * k + 4 * n + es * rows * (k + n), "flops": 2 * rows * n * k}
    if kind == "quantize":
        return {"bytes": case["rows"] * (case["k"] * (es + 4) + 4), "flops": 0}
    tokens, experts, topk, hidden = case["tokens"], case["experts"], case["topk"], case["hidden"]
    slots = round(tokens * topk * (1 - case["dropped"]))
    if kind == "experts":
        used = experts * (1 - (1 - topk * (1 - case["dropped"]) / experts) ** tokens)
        weights = case["ffn"] * (3 * hidden + 8) + 4 * hidden
        return {"bytes": int(used * weights) + 2 * es * tokens * hidden + 8 * tokens * topk, "flops": 6 * slots * hidden * case["ffn"]}
    total = tokens * topk
    ints = 4 * (3 * total + experts + 1)
    moved = es * hidden * (tokens + total + slots + tokens) + 4 * total  # forward: x, rows, y, out, weights
    if case["train"]:
        moved += es * hidden * (slots + tokens + tokens + total) + 4 * total  # grad_rows, grad_x, grad_out, grad_y, grad_weights
    return {"bytes": ints + moved, "flops": 0}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------

def _exact_int8(x):
    """Integers and scales of one matrix's rows, from the definition."""
    x = x.double()
    scales = (x.abs().max(dim=1).values / 127).float().double()  # the scale itself is held in 32 bits
    q = torch.where(scales[:, None] > 0, torch.round(x / scales[:, None].clamp(min=1e-300)), 0.0)
    return q, scales


def _exact_linear(x, data, channel_scales):
    q, s = _exact_int8(x)
    return torch.einsum("rk,nk->rn", q, data.double()) * torch.outer(s, channel_scales.double())


def _exact_act(name, g):
    return g * torch.sigmoid(g) if name == "silu" else 0.5 * g * (1 + torch.tanh((2 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3)))


@torch.no_grad()
def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    kind = case["kind"]
    if kind == "linear":
        return _exact_linear(s["x"], *s["w"])
    if kind == "quantize":
        q, scales = _exact_int8(s["w"])
        return {"values": q * scales[:, None], "scales": scales}
    x, ids, w = s["x"].double(), s["ids"], s["weights"].double()
    tokens, topk = ids.shape
    if kind == "experts":
        (gate, gate_s), (up, up_s), (down, down_s) = s["parts"]
        out = torch.zeros_like(x)
        for e in range(case["experts"]):
            t, j = torch.where(ids == e)
            if t.numel():
                hidden = _exact_act(case["act"], _exact_linear(x[t], gate[e], gate_s[e])) * _exact_linear(x[t], up[e], up_s[e])
                # the hidden values have the activations' type by definition, as they are integers by definition afterwards
                y = _exact_linear(hidden.to(ELEMS[case["dtype"]]), down[e], down_s[e])
                out.index_add_(0, t, y * w[t, j][:, None])
        return out
    chosen = ids.flatten().tolist()
    slots = sorted((i for i, e in enumerate(chosen) if e >= 0), key=lambda i: chosen[i])  # sorted() keeps equal ones in order
    rows_of = torch.tensor(slots, dtype=torch.int64, device=x.device)
    count = rows_of.numel()

    def padded(rows):
        full = torch.zeros(tokens * topk, case["hidden"], dtype=torch.float64, device=x.device)
        full[:count] = rows
        return full

    order = torch.full((tokens * topk,), -1, dtype=torch.int32, device=x.device)
    order[:count] = rows_of.int()
    position = torch.full((tokens * topk,), -1, dtype=torch.int32, device=x.device)
    position[rows_of] = torch.arange(count, dtype=torch.int32, device=x.device)
    offsets = torch.tensor([sum(1 for e in chosen if 0 <= e < b) for b in range(case["experts"] + 1)], dtype=torch.int32, device=x.device)
    token, weight, y = rows_of // topk, w.flatten()[rows_of], s["y"].double()[:count]
    result = {"order": order, "offsets": offsets, "position": position.view(tokens, topk), "rows": padded(x[token]),
              "out": torch.zeros_like(x).index_add_(0, token, y * weight[:, None])}
    if case["train"]:
        grad_out = s["grad_out"].double()
        grad_weights = torch.zeros(tokens * topk, dtype=torch.float64, device=x.device)
        grad_weights[rows_of] = (grad_out[token] * y).sum(1)
        result |= {"grad_x": torch.zeros_like(x).index_add_(0, token, s["grad_rows"].double()[:count]),
                   "grad_y": padded(grad_out[token] * weight[:, None]), "grad_weights": grad_weights.view(tokens, topk)}
    return result
