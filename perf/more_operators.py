"""4-bit microscaled weights and rows, and the norm that leaves quantised rows, as the calls that a program makes which serves such weights.

A case names an operator and its sizes:

  quantize  rows of activations to 4-bit codes with an 8-bit scale for each run of 16 columns, and back to the numbers these stand for
  norm      residual + delta, root-mean-square norm, and the normed rows in 4 bits, or in 8 bits with a scale for each run of 128 columns
  linear    rows times a projection of 4-bit codes
  gated     the same with a gate and an up matrix, and silu(gate) * up of the two products
  experts   one product of a routed feed-forward: the rows are sorted by expert, every expert has a matrix of its own

The definition.  A code is one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 with a sign (e2m1), a scale an e4m3 number, to nearest and ties to even both.
Rows x [M, K], with a the largest absolute value of a row: r = 2^p, p the smallest integer (at least -126) with a 2^-p <= 2688 = 6 * 448, or 1 where a
is 0; for a run b of 16 columns with largest absolute value a_b: s = e4m3(a_b / (6 r)); codes c = e2m1(x / (s r)), 0 where s is 0; the row
stands for c s r.  A matrix [N, K] is codes C, scales S [N, ceil(K / 16)] and a 32-bit factor f.  With quantised rows

    y[m, n] = r[m] f (sum over b of s[m, b] S[n, b] (sum over the run of c[m, k] C[n, k])).

8-bit rows: e4m3 codes of x / s, s = 2^p for each run of 128 columns, p the smallest integer (at least -126) with a_b 2^-p <= 448, or 1 where a_b is 0.  A
norm's rows are rounded to the type of delta before they are quantised.
"""
import math
import random

import torch

own = False
DEVICE = "cuda"
RUN = 16
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # The rows of a decode step of eight requests ahead of the output projection (the 8B sizes): the smallest call, where latency counts.
        {"name": "quantize_decode", "kind": "quantize", "dtype": "bf16", "rows": 8, "k": 4096},
        # The activations of two long prompts, ahead of the down projection.
        {"name": "quantize_prompt", "kind": "quantize", "dtype": "bf16", "rows": 8192, "k": 14336},
        # The norm ahead of a decode step's projections.
        {"name": "norm_decode", "kind": "norm", "form": "4bit", "dtype": "bf16", "rows": 8, "k": 4096},
        # The same on two long prompts.
        {"name": "norm_prompt", "kind": "norm", "form": "4bit", "dtype": "bf16", "rows": 8192, "k": 4096},
        # The norm ahead of 8-bit weights, at a width that is no whole number of runs and row by row in 32 bits.
        {"name": "norm_bytes_odd", "kind": "norm", "form": "8bit", "dtype": "f32", "rows": 1001, "k": 2000},
        # One request's output projection: the smallest product.
        {"name": "linear_single", "kind": "linear", "rows": 1, "k": 4096, "n": 4096, "out": "bf16"},
        # Short portions of several prompts in one step, on a projection with odd sizes; 32-bit rows come back.
        {"name": "linear_odd", "kind": "linear", "rows": 333, "k": 1000, "n": 1302, "out": "f32"},
        # Gate and up of a decode step of eight requests: the largest weights of a layer.
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
    kind = rng.choice(["quantize", "norm", "norm", "linear", "linear", "linear", "gated", "gated", "experts", "experts"])
    step = rng.choice([1, 8, 16, 128, 128])           # (sizes of real matrices are mostly multiples of 128, not all)
    k, n = (max(step, _spread(rng, 200, 8192) // step * step) for _ in range(2))
    rows = _spread(rng, 1, 64) if rng.random() < 0.5 else _spread(rng, 65, 4096)
    out = rng.choice(["bf16", "bf16", "f32"])
    if kind == "quantize":
        return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f32"]), "rows": rows, "k": k}
    if kind == "norm":
        return {"kind": kind, "form": rng.choice(["4bit", "4bit", "8bit"]), "dtype": rng.choice(["bf16", "bf16", "f32"]), "rows": rows, "k": k}
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


def _runs(count, run=RUN):
    return -(-count // run)


def _matrix(count, n, k, g):
    """``count`` matrices as a checkpoint stores them: codes [count, n, ceil(k / 2)], two in a byte (the even column in the lower half), scales
    [count, n, ceil(k / 16)] in e4m3 and factors [count]."""
    w = torch.nn.functional.pad(_normal((count, n, k), g) * (k ** -0.5), (0, -k % RUN)).view(count, n, -1, RUN)
    factors = w.abs().amax((1, 2, 3)) / 2688.0
    scales = (w.abs().amax(3) / (6.0 * factors[:, None, None])).clamp(2.0 ** -6, 448.0).to(torch.float8_e4m3fn)
    v = (w / (scales.float() * factors[:, None, None])[..., None]).view(count, n, -1)
    a = v.abs()
    codes = sum((a > border).to(torch.uint8) for border in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)) + 8 * (v < 0).to(torch.uint8)
    return (codes[..., 0::2] | (codes[..., 1::2] << 4))[..., :(k + 1) // 2].contiguous(), scales.contiguous(), factors


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
    if case["kind"] == "norm":
        rows, k = case["rows"], case["k"]
        state["delta"] = _activations(rows, k, case["dtype"], g)
        state["residual"] = 4.0 * _normal((rows, k), g)
        state["weight"] = 1.0 + 0.2 * _normal((k,), g)
        state["sum"] = torch.empty_like(state["residual"])      # (where the next residual goes)
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
        from torchinferno_b200.kernels.microscaled import MicroscaledExperts, MicroscaledMatrix, MicroscaledWeight
        stacks = [[MicroscaledMatrix(c, s, f, columns=case["k"]) for c, s, f in zip(*stack)] for stack in state.pop("w")]
        if case["kind"] == "experts":
            state["weight"] = MicroscaledExperts(*stacks)
        else:
            state["weight"] = MicroscaledWeight(*(stack[0] for stack in stacks), epilogue="swiglu" if _gated(case) else "none")
    return state


# ------------------------------------------------------------------ plain form
def _e4m3(v):
    """To the nearest of 0, 2^-9, ..., 448 (v at least 0)."""
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v).exponent - 1).clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(max=448.0)


def _e2m1(v):
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).to(v.dtype)
    return (torch.round(v / step) * step).clamp(-6.0, 6.0)


def _power(largest, most, bits):
    """2^p, p the smallest integer (at least -126) with largest 2^-p <= most 2^bits, most in (1/2, 1]; 1 where largest is 0."""
    part, exponent = torch.frexp(largest)
    p = (exponent - bits + (part > most)).clamp(min=-126)
    return torch.ldexp(torch.ones_like(largest), torch.where(largest == 0, torch.zeros_like(p), p))


def _wide(x):      # (numbers in 32 bits may lie nearer to a border than a quotient in 32 bits can tell)
    return x.double() if x.dtype == torch.float32 else x.float()


def _quantized(x):
    """The numbers that rows in 4 bits stand for."""
    rows, k = x.shape
    v = _wide(x)
    r = _power(v.abs().amax(1), 2688.0 / 4096.0, 12)
    t = torch.nn.functional.pad(v / r[:, None], (0, -k % RUN)).view(rows, -1, RUN)
    s = _e4m3(t.abs().amax(-1) / 6.0)[..., None]
    codes = _e2m1(t / torch.where(s == 0, 1.0, s)) * (s != 0)
    return ((codes * s).view(rows, -1)[:, :k] * r[:, None]).float()


def _quantized_bytes(x):
    """The same in 8 bits."""
    rows, k = x.shape
    t = torch.nn.functional.pad(_wide(x), (0, -k % 128)).view(rows, -1, 128)
    s = _power(t.abs().amax(-1), 448.0 / 512.0, 9)[..., None]
    v = t / s
    return (torch.sign(v) * _e4m3(v.abs()) * s).view(rows, -1)[:, :k].float()


def _widened(codes, scales, factors, k):
    values = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    halves = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., :k].long()
    numbers = values[halves & 7] * torch.where(halves > 7, -1.0, 1.0)
    return numbers * scales.float().repeat_interleave(RUN, -1)[..., :k] * factors[:, None, None]


LIMIT, ALPHA = 7.0, 1.702      # (of the clamped gated unit)


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


def run(state):
    case = state["case"]
    if case["kind"] == "quantize":
        if own:
            from torchinferno_b200.kernels.microscaled import quantize_rows
            return quantize_rows(state["x"]).widened(torch.bfloat16)
        return _quantized(state["x"]).to(torch.bfloat16)
    if case["kind"] == "norm":
        delta, residual, weight = state["delta"], state["residual"], state["weight"]
        if own:
            from torchinferno_b200.kernels import block_scaled, microscaled
            form = microscaled if case["form"] == "4bit" else block_scaled
            rows = form.add_rmsnorm(delta, residual, weight, EPS, new_residual=state["sum"])
            return {"residual": state["sum"], "rows": rows.widened(torch.bfloat16)}
        h = residual + delta.float()
        normed = (h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * weight).to(delta.dtype)
        rows = _quantized(normed) if case["form"] == "4bit" else _quantized_bytes(normed)
        return {"residual": h, "rows": rows.to(torch.bfloat16)}
    x, dtype, k = state["x"], TYPES[case["out"]], case["k"]
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
        rows = _quantized(x)
        source = (order // top).long() if case["by_pair"] else torch.arange(len(order), device=x.device)
        padded = rows[source[at.clamp(max=len(order) - 1)]] * there[..., None]
        sums = [torch.bmm(padded, _widened(*stack, k).transpose(1, 2)) for stack in state["w"]]
        return _act(case["act"], sums)[there].to(dtype)
    if own:
        from torchinferno_b200.kernels import gemm
        product = gemm.linear_swiglu if _gated(case) else gemm.linear
        return product(x, state["weight"], out_dtype=dtype)
    rows = _quantized(x)
    sums = [rows @ _widened(*stack, k)[0].t() for stack in state["w"]]
    return _act("swiglu" if _gated(case) else "none", sums).to(dtype)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size, k = {"bf16": 2, "f32": 4}, case["k"]
    if case["kind"] == "quantize":
        numbers = case["rows"] * k
        return {"bytes": numbers * (size[case["dtype"]] + 2), "flops": 3 * numbers}
    if case["kind"] == "norm":
        numbers = case["rows"] * k
        return {"bytes": numbers * (size[case["dtype"]] + 4 + 4 + 2) + 4 * k, "flops": 8 * numbers}
    matrices, n = 2 if _gated(case) else 1, case["n"]
    weight = matrices * (n * _runs(k, 2) + n * _runs(k) + 4)
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
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)]


def _nearest(v, values):
    """The nearest of ``values`` (ascending, from 0) to each v >= 0, of two the one with the even index."""
    table = torch.tensor(values, dtype=torch.float64, device=v.device)
    low = (torch.searchsorted(table, v, right=True) - 1).clamp(max=len(values) - 1)
    high = (low + 1).clamp(max=len(values) - 1)
    below, above = v - table[low], table[high] - v
    return table[torch.where((above < below) | ((above == below) & (low % 2 == 1)), high, low)]


def _first_power(largest, most):
    powers = torch.tensor([2.0 ** p for p in range(-126, 129)], dtype=torch.float64, device=largest.device)
    return torch.where(largest == 0, 1.0, powers[torch.searchsorted(most * powers, largest)])      # (the first that is large enough)


def _exact_rows(x, form="4bit"):
    """The numbers that quantised rows stand for, some rows at a time."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for first in range(0, x.shape[0], 512):
        part = x[first:first + 512].double()
        to = out[first:first + 512]
        if form == "4bit":
            r = _first_power(part.abs().max(1).values, 2688.0)
            part = part / r[:, None]
        for b in range(0, x.shape[1], 2048):
            v = part[:, b:b + 2048]
            width, run = v.shape[1], RUN if form == "4bit" else 128
            at = torch.arange(width, device=x.device) // run
            largest = torch.zeros(v.shape[0], _runs(width, run), dtype=torch.float64, device=x.device).scatter_reduce(
                1, at.expand_as(v), v.abs(), "amax")
            if form == "4bit":
                s = _nearest(largest / 6.0, E4M3)[:, at]
                q = _nearest((v / torch.where(s == 0, math.inf, s)).abs(), E2M1) * s * r[:, None]
            else:
                s = _first_power(largest, 448.0)[:, at]
                q = _nearest((v / s).abs(), E4M3) * s
            to[:, b:b + 2048] = torch.copysign(q, v)
    return out


def _exact_matrix(codes, scales, factor, k):
    table = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=codes.device)
    numbers = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    numbers[:, 0::2], numbers[:, 1::2] = table[(codes % 16).long()], table[(codes // 16).long()]
    return numbers[:, :k] * scales.to(torch.float64)[:, torch.arange(k, device=codes.device) // RUN] * factor.double()


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = kept
    if case["kind"] == "quantize":
        return _exact_rows(state["x"])
    if case["kind"] == "norm":
        h = (state["residual"].double() + state["delta"].double()).float().double()      # (the residual is held in 32 bits)
        normed = h / ((h * h).mean(1) + EPS).sqrt()[:, None] * state["weight"].double()
        return {"residual": h, "rows": _exact_rows(normed.to(state["delta"].dtype), case["form"])}
    rows, k = _exact_rows(state["x"]), case["k"]
    if case["kind"] != "experts":
        return _act("swiglu" if _gated(case) else "none", [rows @ _exact_matrix(*(part[0] for part in stack), k).t() for stack in state["w"]])
    offsets, order = state["offsets"].tolist(), state["order"].long()
    y = torch.empty(len(order), case["n"], dtype=torch.float64, device=rows.device)
    for e in range(case["experts"]):
        at = torch.arange(offsets[e], offsets[e + 1], device=rows.device)
        if len(at):
            taken = rows[order[at] // state["top"]] if case["by_pair"] else rows[at]
            y[at] = _act(case["act"], [taken @ _exact_matrix(*(part[e] for part in stack), k).t() for stack in state["w"]])
    return y
