"""The work of the 4-bit weight operators, as sizes, inputs, plain forms and definitions.

Four operators that sit beside the Q4 KV-cache attention in a decoder layer whose weights are
held in the same 4-bit format as the cache (codes packed 8 per 32-bit word along the input
dimension, one scale and one bias per 64 inputs):

* linear:  y = x W^T, or with two matrices y = silu(x G^T) * (x U^T);
* experts: the same with one matrix (pair) per expert, over rows sorted by expert;
* route:   top-k of a router's logits per token, its softmax weights, and the counting sort
           of the (token, slot) pairs by expert;
* combine: the weighted sum of each token's expert rows, added to a residual.

With ``own`` false, ``run`` computes them from elementary tensor operations in 32 bits; with
``own`` true it calls this repository's kernels.
"""

import math

import torch

own = False

GROUP = 64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
# No drawn case costs more than the largest listed one.
MOST_FLOPS = 2.0 * 4096 * 4096 * 14336 * 2
MOST_WEIGHTS = 128256 * 4096
# Groups of 64 inputs: the widths of the models named below and odd counts between them.
GROUPS = [4, 5, 7, 8, 11, 13, 16, 19, 22, 27, 32, 37, 45, 51, 60, 64, 77, 91, 112, 139, 171, 224]


def _linear(name, tokens, inputs, outputs, gated, dtype):
    return {"name": name, "op": "linear", "tokens": tokens, "inputs": inputs, "outputs": outputs,
            "gated": gated, "dtype": dtype}


def _experts(name, tokens, experts, top_k, inputs, outputs, gated, dtype):
    return {"name": name, "op": "experts", "tokens": tokens, "experts": experts, "top_k": top_k,
            "inputs": inputs, "outputs": outputs, "gated": gated, "dtype": dtype}


def _route(name, tokens, experts, top_k, normalize):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top_k": top_k,
            "normalize": normalize}


def _combine(name, tokens, top_k, width, dtype):
    return {"name": name, "op": "combine", "tokens": tokens, "top_k": top_k, "width": width,
            "dtype": dtype}


def listed():
    return [
        # one agent decodes a token: the attention output projection of a Llama-3.1-8B layer
        _linear("linear-1-token", 1, 4096, 4096, False, "bf16"),
        # eight agents decode: the vocabulary projection, the largest matrix of the model
        _linear("linear-8-tokens-vocabulary", 8, 4096, 128256, False, "bf16"),
        # an odd batch of agents: the gated half of a Gemma-3-12B MLP
        _linear("gated-37-tokens", 37, 3840, 15360, True, "bf16"),
        # one 512-token prefill chunk: the MLP's down projection of a Llama-3.1-8B layer
        _linear("linear-512-token-chunk", 512, 14336, 4096, False, "f16"),
        # several agents' chunks at once: the gated half of the same MLP, the most arithmetic
        _linear("gated-4096-tokens", 4096, 4096, 14336, True, "bf16"),
        # one agent decodes: the six routed experts of a DeepSeek-Coder-V2-Lite layer
        _experts("experts-1-token-gated", 1, 64, 6, 2048, 1408, True, "bf16"),
        # 256 agents decode: the down projection of the same layer, about 24 rows an expert
        _experts("experts-256-tokens-down", 256, 64, 6, 1408, 2048, False, "bf16"),
        # a batch of prefill chunks: the gated experts of a GPT-OSS-20B shaped layer (width
        # 2880 is 45 groups, no multiple of 128)
        _experts("experts-4096-tokens-gated", 4096, 32, 4, 2880, 2880, True, "bf16"),
        # routing of one decoded token (weights from the softmax over all 64 experts)
        _route("route-1-token", 1, 64, 6, False),
        # routing of a batch of prefill chunks (weights over the chosen four)
        _route("route-4096-tokens", 4096, 32, 4, True),
        # 16 agents decode: six expert rows a token
        _combine("combine-16-tokens", 16, 6, 2048, "bf16"),
        # a batch of prefill chunks: four expert rows a token
        _combine("combine-4096-tokens", 4096, 4, 2880, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "experts", "experts", "route", "combine"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    gated = rng.random() < 0.5
    while True:
        tokens = _log_int(rng, 1, 4096)
        if op == "linear":
            c = _linear("", tokens, GROUP * rng.choice(GROUPS),
                        _log_int(rng, 256, 32768), gated, dtype)
            weights = c["inputs"] * c["outputs"] * (2 if gated else 1)
        elif op == "experts":
            experts = _log_int(rng, 4, 128)
            c = _experts("", tokens, experts, rng.randint(1, min(8, experts)),
                         GROUP * rng.choice(GROUPS[4:16]), _log_int(rng, 256, 4096), gated, dtype)
            weights = c["inputs"] * c["outputs"] * (2 if gated else 1) * experts
        elif op == "route":
            experts = _log_int(rng, 4, 256)
            c = _route("", tokens, experts, rng.randint(1, min(8, experts)), rng.random() < 0.5)
            weights = 0
        else:
            c = _combine("", tokens, rng.randint(1, 8), _log_int(rng, 256, 8192), dtype)
            weights = 0
        if weights <= MOST_WEIGHTS and work(c)["flops"] <= MOST_FLOPS:
            del c["name"]
            return c


# ----------------------------------------------------------------------------- inputs


def _quantized(shape, gen, dtype):
    """Normal weights of a trained matrix's size in the cache's 4-bit format: per group the
    larger edge is an exact code, code = round((w - bias) / scale)."""
    lead, k = shape[:-1], shape[-1]
    w = torch.randn(*lead, k // GROUP, GROUP, generator=gen, device="cuda") * (1.0 / math.sqrt(k))
    lo, hi = w.amin(-1), w.amax(-1)
    side = lo.abs() > hi.abs()
    scale = ((hi - lo) / 15).clamp_min(1e-7)
    scale = torch.where(side, scale, -scale)
    bias = torch.where(side, lo, hi)
    scale = bias / torch.round(bias / scale)
    codes = torch.round((w - bias[..., None]) / scale[..., None]).clamp_(0, 15).to(torch.int32)
    del w
    codes = codes.view(*lead, k // 8, 8) << (4 * torch.arange(8, dtype=torch.int32, device="cuda"))
    return codes.sum(-1, dtype=torch.int32), scale.to(dtype), bias.to(dtype)


def _router_logits(tokens, experts, gen):
    """Logits of a trained router: some experts are liked more by all tokens."""
    liked = torch.randn(experts, generator=gen, device="cuda") * 0.5
    return torch.randn(tokens, experts, generator=gen, device="cuda") + liked


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": dict(case)}
    if case["op"] == "route":
        s["logits"] = _router_logits(case["tokens"], case["experts"], gen)
        return s
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "combine":
        t, k, d = case["tokens"], case["top_k"], case["width"]
        s["y"] = torch.randn(t * k, d, generator=gen, device="cuda").to(dtype)
        s["residual"] = torch.randn(t, d, generator=gen, device="cuda").to(dtype)
        s["weights"] = torch.softmax(torch.randn(t, k, generator=gen, device="cuda"), -1)
        s["positions"] = torch.randperm(t * k, generator=gen, device="cuda").to(torch.int32).view(t, k)
        return s
    lead = (case["experts"],) if case["op"] == "experts" else ()
    shape = (*lead, case["outputs"], case["inputs"])
    s["x"] = torch.randn(case["tokens"], case["inputs"], generator=gen, device="cuda").to(dtype)
    s["w"] = [_quantized(shape, gen, dtype) for _ in range(2 if case["gated"] else 1)]
    if case["op"] == "experts":
        logits = _router_logits(case["tokens"], case["experts"], gen)
        s["routing"] = _plain_route(logits, case["top_k"], True)
        if not case["gated"]:  # the down projection takes the gated rows, sorted by expert
            rows = case["tokens"] * case["top_k"]
            s["x"] = torch.randn(rows, case["inputs"], generator=gen, device="cuda").to(dtype)
    if own:  # a program lays its weights out once, when it loads them
        s["w"] = [_package().Q4Weight(*w) for w in s["w"]]
    return s


# ----------------------------------------------------------------------------- plain forms


def _dequantized(w):
    codes, scales, biases = w
    shifts = 4 * torch.arange(8, dtype=torch.int32, device=codes.device)
    n = ((codes[..., None] >> shifts) & 15).to(torch.float32)
    n = n.view(*scales.shape, GROUP)
    return (n * scales.float()[..., None] + biases.float()[..., None]).flatten(-2)


def _gated(parts):
    if len(parts) == 1:
        return parts[0]
    return parts[0] / (1 + torch.exp(-parts[0])) * parts[1]


def _plain_linear(x, w):
    xf = x.float()
    return _gated([xf @ _dequantized(m).t() for m in w]).to(x.dtype)


def _plain_experts(x, w, routing, case):
    """Rows sorted by expert, in blocks of one expert each: a block's matrix is dequantized
    and multiplied with the block's rows."""
    offsets, order = routing[2].long(), routing[3].long()
    n_experts, rows = offsets.numel() - 1, order.numel()
    xs = x[order // case["top_k"]] if case["gated"] else x
    size = max(1, rows // n_experts)
    counts = offsets[1:] - offsets[:-1]
    blocks = -(-counts // size)
    ends = blocks.cumsum(0)
    n_blocks = min(rows, rows // size + n_experts)
    block = torch.arange(n_blocks, device=x.device)
    expert = torch.searchsorted(ends, block, right=True).clamp_max(n_experts - 1)
    first = offsets[expert] + (block - ends[expert] + blocks[expert]) * size
    row = first[:, None] + torch.arange(size, device=x.device)
    live = (row < offsets[expert + 1][:, None]) & (block < ends[-1])[:, None]
    xb = xs.float()[row.clamp_max(rows - 1)]
    yb = _gated([xb @ _dequantized([p[expert] for p in m]).transpose(1, 2) for m in w]).to(x.dtype)
    out = torch.empty(rows + 1, yb.shape[-1], dtype=x.dtype, device=x.device)
    out[torch.where(live, row, rows)] = yb
    return out[:rows]


def _plain_route(logits, top_k, normalize):
    tokens, n_experts = logits.shape
    ranked = torch.argsort(logits, dim=-1, descending=True, stable=True)
    experts = ranked[:, :top_k]
    chosen = torch.gather(logits, 1, experts)
    top = logits.amax(-1, keepdim=True)
    over = chosen if normalize else logits
    weights = torch.exp(chosen - top) / torch.exp(over - top).sum(-1, keepdim=True)
    flat = experts.reshape(-1)
    order = torch.argsort(flat, stable=True)
    positions = torch.empty_like(order)
    positions[order] = torch.arange(order.numel(), device=order.device)
    ids = torch.arange(n_experts + 1, device=flat.device)
    offsets = torch.searchsorted(flat[order], ids)
    as32 = [t.to(torch.int32) for t in (experts, offsets, order, positions.view(tokens, top_k))]
    return [as32[0], weights, as32[1], as32[2], as32[3]]


def _plain_combine(y, weights, positions, residual):
    rows = y.float()[positions.long()]
    return ((rows * weights[..., None]).sum(1) + residual.float()).to(y.dtype)


def _package():
    from __graft_entry__ import load_package

    return load_package()


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        am = _package()
        if op == "linear":
            if case["gated"]:
                return am.quantized_swiglu(state["x"], *state["w"])
            return am.quantized_matmul(state["x"], *state["w"])
        if op == "experts":
            routing = am.ExpertRouting(*state["routing"])
            if case["gated"]:
                return am.expert_swiglu(state["x"], *state["w"], routing)
            return am.expert_matmul(state["x"], *state["w"], routing)
        if op == "route":
            r = am.route_experts(state["logits"], case["top_k"], normalize=case["normalize"])
            return [r.experts, r.weights, r.offsets, r.order, r.positions]
        return am.combine_experts(state["y"], state["weights"], state["positions"],
                                  residual=state["residual"])
    if op == "linear":
        return _plain_linear(state["x"], state["w"])
    if op == "experts":
        return _plain_experts(state["x"], state["w"], state["routing"], case)
    if op == "route":
        return _plain_route(state["logits"], case["top_k"], case["normalize"])
    return _plain_combine(state["y"], state["weights"], state["positions"], state["residual"])


# ----------------------------------------------------------------------------- work


def work(case):
    """Bytes that a pass has to read and write once, and its products and sums.  A matrix of n
    weights is n / 2 bytes of codes and n / 16 bytes of scales and biases; of the experts only
    those that at least one token chose are read (their expected number)."""
    op, tokens = case["op"], case["tokens"]
    if op == "route":
        e, k = case["experts"], case["top_k"]
        return {"bytes": tokens * (4 * e + 16 * k) + 4 * (e + 1), "flops": 3 * tokens * e}
    if op == "combine":
        k, d = case["top_k"], case["width"]
        return {"bytes": tokens * (2 * d * (k + 2) + 8 * k), "flops": 2 * tokens * k * d}
    matrices = 2 if case["gated"] else 1
    weights = case["inputs"] * case["outputs"] * matrices
    rows, read, index = tokens, tokens, 0
    if op == "experts":
        e, k = case["experts"], case["top_k"]
        rows = tokens * k
        read = tokens if case["gated"] else rows
        index = 4 * (e + 1 + (rows if case["gated"] else 0))
        weights *= e * (1 - (1 - k / e) ** tokens)
    return {"bytes": weights * 9 / 16 + 2 * (read * case["inputs"] + rows * case["outputs"]) + index,
            "flops": 2.0 * rows * case["inputs"] * case["outputs"] * matrices}


# ----------------------------------------------------------------------------- definition


def _exact_matrix(w):
    codes, scales, biases = w
    n = torch.empty(codes.shape[0], codes.shape[1] * 8, dtype=torch.float64, device=codes.device)
    for i in range(8):
        n[:, i::8] = (codes.to(torch.int64) >> (4 * i)).bitwise_and(15)
    return (n * scales.double().repeat_interleave(GROUP, 1) + biases.double().repeat_interleave(GROUP, 1))


def _exact_product(x, w):
    x = x.double()
    cut = max(1, (1 << 27) // w[0].shape[1] // 8)  # output columns at a time
    cols = []
    for n in range(0, w[0].shape[0], cut):
        cols.append(x @ _exact_matrix([p[n:n + cut] for p in w]).mT)
    return torch.cat(cols, 1)


def _exact_mlp(x, w):
    y = _exact_product(x, w[0])
    if len(w) == 2:
        y = y * torch.special.expit(y) * _exact_product(x, w[1])
    return y


def exact(case, seed):
    """The operators' definitions in 64 bits (the route's whole numbers have no such value)."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "linear":
        return _exact_mlp(s["x"], s["w"])
    if op == "experts":
        bounds, order = s["routing"][2].tolist(), s["routing"][3].long()
        y = torch.zeros(order.numel(), case["outputs"], dtype=torch.float64, device="cuda")
        for e, (a, b) in enumerate(zip(bounds[:-1], bounds[1:])):
            if a < b:
                x = s["x"][order[a:b] // case["top_k"]] if case["gated"] else s["x"][a:b]
                y[a:b] = _exact_mlp(x, [[p[e] for p in m] for m in s["w"]])
        return y
    if op == "route":
        p = s["logits"].double()
        p = torch.sort(p, -1, descending=True).values
        e = torch.exp(p - p[:, :1])
        k = case["top_k"]
        whole = e[:, :k] if case["normalize"] else e
        return [None, e[:, :k] / whole.sum(-1, keepdim=True), None, None, None]
    y, w, at = s["y"].double(), s["weights"].double(), s["positions"].long()
    out = s["residual"].double()
    for j in range(case["top_k"]):
        out = out + w[:, j:j + 1] * y[at[:, j]]
    return out
