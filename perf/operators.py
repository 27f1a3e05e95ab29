"""Products of 8-bit weights with a scale for each block of 128 x 128, as the calls that a program makes which serves such weights.

A case names an operator and its sizes:

  quantize  rows of activations to e4m3 codes with a power of two for each run of 128 columns
  linear    rows times a projection stored as e4m3 codes with a 32-bit scale for each block of 128 x 128
  gated     the same with a gate and an up matrix, and silu(gate) * up of the two products
  experts   one product of a routed feed-forward: the rows are sorted by expert, every expert has a matrix of its own

The definition, for rows x [M, K] and a matrix with codes C [N, K] and scales S [ceil(N / 128), ceil(K / 128)]: with a the largest
absolute value of a run b of 128 columns of a row, the run's scale is s = 2^p, p the smallest integer (at least -126) with
a 2^-p <= 448, or 1 where a is 0; its codes are x / s rounded to e4m3; and

    y[m, n] = sum over b of s[m, b] S[n // 128, b] (sum over the run of code[m, k] C[n, k]).
"""
import math
import random

import torch

own = False
DEVICE = "cuda"
BLOCK = 128
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # The normed rows of a decode step of eight requests, ahead of a projection (the 8B sizes).
        {"name": "quantize_decode", "kind": "quantize", "dtype": "bf16", "rows": 8, "k": 4096},
        # The activations of two long prompts, ahead of the down projection.
        {"name": "quantize_prompt", "kind": "quantize", "dtype": "bf16", "rows": 8192, "k": 14336},
        # 32-bit rows whose last run is short.
        {"name": "quantize_odd", "kind": "quantize", "dtype": "f32", "rows": 1001, "k": 2000},
        # One request's output projection: the smallest product, where latency counts.
        {"name": "linear_single", "kind": "linear", "rows": 1, "k": 4096, "n": 4096, "out": "bf16"},
        # The down projection of a decode step of eight requests.
        {"name": "linear_decode", "kind": "linear", "rows": 8, "k": 14336, "n": 4096, "out": "bf16"},
        # Short portions of several prompts in one step, on a projection with odd sizes; 32-bit rows come back.
        {"name": "linear_odd", "kind": "linear", "rows": 333, "k": 1000, "n": 1302, "out": "f32"},
        # The query, key and value projection of a prompt.
        {"name": "linear_prompt", "kind": "linear", "rows": 2048, "k": 4096, "n": 6144, "out": "bf16"},
        # Gate and up of a decode step: the largest weights of a layer.
        {"name": "gated_decode", "kind": "gated", "rows": 8, "k": 4096, "n": 14336, "out": "bf16"},
        # The same on four prompts at once: the largest product.
        {"name": "gated_prompt", "kind": "gated", "rows": 8192, "k": 4096, "n": 14336, "out": "bf16"},
        # Gated experts on a decode step of eight requests with four choices each: the chosen experts' weights are the work.
        {"name": "experts_decode", "kind": "experts", "tokens": 8, "top": 4, "experts": 32, "k": 2048, "n": 1024, "act": "swiglu",
         "by_pair": True, "skew": 1.0, "out": "bf16"},
        # The first product of routed experts on a prompt.
        {"name": "experts_prompt", "kind": "experts", "tokens": 2048, "top": 4, "experts": 32, "k": 2048, "n": 1024, "act": "relu2",
         "by_pair": True, "skew": 1.0, "out": "bf16"},
        # The second product on a short prompt with odd sizes, where some experts get many rows and some none; 32-bit rows come back.
        {"name": "experts_odd", "kind": "experts", "tokens": 301, "top": 3, "experts": 28, "k": 1200, "n": 1416, "act": "none",
         "by_pair": False, "skew": 4.0, "out": "f32"},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "linear", "gated", "gated", "experts", "experts"])
    step = rng.choice([1, 8, 64, 128, 128])           # (sizes of real matrices are mostly multiples of 128, not all)
    k, n = (max(step, _spread(rng, 200, 8192) // step * step) for _ in range(2))
    rows = _spread(rng, 1, 64) if rng.random() < 0.5 else _spread(rng, 65, 4096)
    out = rng.choice(["bf16", "bf16", "f32"])
    if kind == "quantize":
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f32"]), "rows": rows, "k": k}
    if kind in ("linear", "gated"):
        return {"kind": kind, "rows": rows, "k": k, "n": n, "out": out}
    act = rng.choice(["none", "relu2", "silu", "gelu", "swiglu", "glu_clamp"])
    experts = rng.choice([8, 16, 28, 32, 60])
    return {"kind": kind, "tokens": rows, "top": rng.randint(1, 6), "experts": experts, "k": min(k, 2560), "n": min(n, 2048), "act": act,
            "by_pair": act != "none" or rng.random() < 0.3, "skew": rng.choice([1.0, 1.0, 4.0]), "out": out}


def _gated(case):
    return case["kind"] == "gated" or case.get("act") in ("swiglu", "glu_clamp")


# ------------------------------------------------------------------ inputs
def _generator(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(random.Random(f"{seed} {sorted((k, str(v)) for k, v in case.items() if k != 'name')}").getrandbits(62))
    return g


def _normal(shape, g):
    return torch.randn(shape, generator=g, device=DEVICE, dtype=torch.float32)


def _activations(rows, k, dtype, g):
    """Rows as a norm leaves them: about unit size, a few columns far larger than the others, every row of a size of its own."""
    size = torch.where(torch.rand(k, generator=g, device=DEVICE) < 0.01, 20.0, 1.0) * (0.3 * _normal((k,), g)).exp()
    return (_normal((rows, k), g) * size * (0.5 * _normal((rows, 1), g)).exp()).to(TYPES[dtype])


def _blocks(count):
    return -(-count // BLOCK)


def _matrix(count, n, k, g):
    """``count`` matrices as a checkpoint stores them: e4m3 codes [count, n, k] and a 32-bit scale for each block."""
    w = _normal((count, n, k), g) * (k ** -0.5)
    padded = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK)).view(count, _blocks(n), BLOCK, _blocks(k), BLOCK)
    scales = padded.abs().amax((2, 4)) / 448.0
    codes = (padded / scales[:, :, None, :, None]).view(count, _blocks(n) * BLOCK, -1)[:, :n, :k]
    return codes.to(torch.float8_e4m3fn).contiguous(), scales.contiguous()


def _routing(case, g):
    """Pairs (token, choice) sorted by expert: offsets [experts + 1] and order [pairs], as the router leaves them."""
    tokens, top, experts = case["tokens"], min(case["top"], case["experts"]), case["experts"]
    liking = case["skew"] * _normal((experts,), g)      # (with a skew a few experts are chosen by most tokens, some by none)
    ids = (_normal((tokens, experts), g) + liking).topk(top, dim=1).indices.reshape(-1)
    order = torch.sort(ids, stable=True).indices.to(torch.int32)
    counts = torch.bincount(ids, minlength=experts)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    return offsets, order, top, int(counts.max())


def prepare(case, seed):
    g = _generator(case, seed)
    state = {"case": case}
    if case["kind"] == "quantize":
        state["x"] = _activations(case["rows"], case["k"], case["dtype"], g)
        return state
    count = case.get("experts", 1)
    state["w"] = [_matrix(count, case["n"], case["k"], g) for _ in range(2 if _gated(case) else 1)]
    if case["kind"] == "experts":
        offsets, order, top, most = _routing(case, g)
        state.update(offsets=offsets, order=order, top=top, most=most)
        rows = case["tokens"] if case["by_pair"] else len(order)
    else:
        rows = case["rows"]
    state["x"] = _activations(rows, case["k"], "bf16", g)
    if own:
        from torchinferno_b200.kernels.block_scaled import BlockScaledExperts, BlockScaledMatrix, BlockScaledWeight
        stacks = [[BlockScaledMatrix(c, s) for c, s in zip(codes, scales)] for codes, scales in state.pop("w")]
        if case["kind"] == "experts":
            state["weight"] = BlockScaledExperts(*stacks)
        else:
            state["weight"] = BlockScaledWeight(*(stack[0] for stack in stacks), epilogue="swiglu" if _gated(case) else "none")
    return state


# ------------------------------------------------------------------ plain form
def _quantized(x):
    """Codes (e4m3) and scales (32 bits) of rows."""
    rows, k = x.shape
    runs = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).view(rows, -1, BLOCK)
    largest = runs.abs().amax(-1)
    part, power = torch.frexp(largest)                # largest = part * 2^power, part in [1/2, 1); 448 = 7/8 * 2^9
    power = (power - 9 + (part > 0.875)).clamp(min=-126)
    scales = torch.where(largest == 0, 1.0, ((power + 127) << 23).view(torch.float32))
    codes = (runs / scales[..., None]).view(rows, -1)[:, :k].to(torch.float8_e4m3fn)
    return codes, scales


def _widened_rows(x):
    codes, scales = _quantized(x)
    return codes.float() * scales.repeat_interleave(BLOCK, 1)[:, :x.shape[1]]


def _widened(codes, scales):
    n, k = codes.shape[-2:]
    return codes.float() * scales.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]


def _act(name, sums):
    if name == "swiglu":
        gate, up = sums
        return gate * torch.sigmoid(gate) * up
    if name == "glu_clamp":
        gate, up = sums[0].clamp(max=LIMIT), sums[1].clamp(-LIMIT, LIMIT)
        return gate * torch.sigmoid(ALPHA * gate) * (up + 1)
    v = sums[0]
    if name == "relu2":
        return v.clamp(min=0).square()
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return v


LIMIT, ALPHA = 7.0, 1.702      # (of the clamped gated unit)


def run(state):
    case, x = state["case"], state["x"]
    if case["kind"] == "quantize":
        if own:
            from torchinferno_b200.kernels.block_scaled import quantize_rows
            codes, scales = quantize_rows(x)
        else:
            codes, scales = _quantized(x)
        return {"codes": codes, "scales": scales}
    dtype = TYPES[case["out"]]
    if case["kind"] == "experts":
        offsets, order, top = state["offsets"], state["order"], state["top"]
        if own:
            from torchinferno_b200.kernels import ops
            y = torch.empty((len(order), case["n"]), dtype=dtype, device=x.device)
            return ops.moe_expert_product(x, state["weight"], y, offsets, order, top, x_by_pair=case["by_pair"], act=case["act"],
                                          limit=LIMIT, alpha=ALPHA)
        # (the experts' rows side by side, each expert's padded to the longest)
        at = offsets[:-1, None].long() + torch.arange(state["most"], device=x.device)
        there = at < offsets[1:, None]
        rows = _widened_rows(x)
        source = (order // top).long() if case["by_pair"] else torch.arange(len(order), device=x.device)
        padded = rows[source[at.clamp(max=len(order) - 1)]] * there[..., None]
        sums = [torch.bmm(padded, _widened(codes, scales).transpose(1, 2)) for codes, scales in state["w"]]
        return _act(case["act"], sums)[there].to(dtype)
    if own:
        from torchinferno_b200.kernels import gemm
        product = gemm.linear_swiglu if _gated(case) else gemm.linear
        return product(x, state["weight"], out_dtype=dtype)
    rows = _widened_rows(x)
    sums = [rows @ _widened(codes[0], scales[0]).t() for codes, scales in state["w"]]
    return _act("swiglu" if _gated(case) else "none", sums).to(dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = {"bf16": 2, "f32": 4}
    if case["kind"] == "quantize":
        numbers = case["rows"] * case["k"]
        return {"bytes": numbers * (size[case["dtype"]] + 1) + case["rows"] * _blocks(case["k"]) * 4, "flops": 2 * numbers}
    matrices, n, k = 2 if _gated(case) else 1, case["n"], case["k"]
    weight = matrices * (n * k + 4 * _blocks(n) * _blocks(k))
    if case["kind"] != "experts":
        rows = case["rows"]
        return {"bytes": weight + 2 * rows * k + size[case["out"]] * rows * n, "flops": 2 * matrices * rows * n * k}
    # (which experts have a row is known when the inputs are: in the mean over even choices)
    top, experts = min(case["top"], case["experts"]), case["experts"]
    pairs = case["tokens"] * top
    read = experts * (1 - (1 - top / experts) ** case["tokens"]) if case["skew"] == 1.0 else min(experts, pairs) * 0.75
    rows_read = case["tokens"] if case["by_pair"] else pairs
    return {"bytes": int(read * weight) + 2 * rows_read * k + pairs * (4 + size[case["out"]] * n), "flops": 2 * matrices * pairs * n * k}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_rows(x):
    """(codes, scales) by the definition, all in 64 bits; e4m3 has steps of an eighth of a binade, and of 2^-9 below 2^-6."""
    rows, k = x.shape
    x = x.double()
    powers = torch.tensor([2.0 ** p for p in range(-126, 129)], dtype=torch.float64, device=x.device)
    binades = torch.tensor([2.0 ** p for p in range(-6, 10)], dtype=torch.float64, device=x.device)
    codes, scales = torch.empty_like(x), torch.empty(rows, _blocks(k), dtype=torch.float64, device=x.device)
    for b in range(_blocks(k)):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        largest = part.abs().max(1).values
        scales[:, b] = torch.where(largest == 0, 1.0, powers[torch.searchsorted(448.0 * powers, largest)])      # the first that is large enough
        v = part / scales[:, b:b + 1]
        step = binades[(torch.searchsorted(binades, v.abs(), right=True) - 1).clamp(min=0)] / 8
        codes[:, b * BLOCK:(b + 1) * BLOCK] = torch.round(v / step) * step          # (to even among the two nearest)
    return codes, scales


def _exact_product(x, codes, scales):
    """x [M, K] (codes times scales already) times one matrix, in 64 bits."""
    n, k = codes.shape
    at_n, at_k = torch.arange(n, device=x.device) // BLOCK, torch.arange(k, device=x.device) // BLOCK
    return x @ (codes.double() * scales.double()[at_n][:, at_k]).t()


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = kept
    x = state["x"]
    if case["kind"] == "quantize":
        if x.numel() > 1 << 25:      # (the largest would take 64-bit copies of several times its size)
            return None
        codes, scales = _exact_rows(x)
        return {"codes": codes, "scales": scales}
    if case["kind"] != "experts":
        codes, scales = _exact_rows(x)
        rows = codes * scales[:, torch.arange(x.shape[1], device=x.device) // BLOCK]
        return _act("swiglu" if _gated(case) else "none", [_exact_product(rows, c[0], s[0]) for c, s in state["w"]])
    codes, scales = _exact_rows(x)
    rows = codes * scales[:, torch.arange(x.shape[1], device=x.device) // BLOCK]
    offsets, order = state["offsets"].tolist(), state["order"].long()
    y = torch.empty(len(order), case["n"], dtype=torch.float64, device=x.device)
    for e in range(case["experts"]):
        at = torch.arange(offsets[e], offsets[e + 1], device=x.device)
        if len(at):
            taken = rows[order[at] // state["top"]] if case["by_pair"] else rows[at]
            y[at] = _act(case["act"], [_exact_product(taken, c[e], s[e]) for c, s in state["w"]])
    return y
