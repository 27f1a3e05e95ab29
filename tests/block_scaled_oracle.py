"""The definition of 8-bit block-scaled rows and products in 64 bits, for the tests (any device)."""
from __future__ import annotations

import torch

BLOCK = 128


def random_matrix(n, k, seed, device="cpu", sizes=(0.02, 3.0)):
    """Codes over the whole range of e4m3 (zeros and its subnormal numbers among them) and scales of different sizes."""
    from torchinferno_b200.kernels.block_scaled import BlockScaledMatrix
    g = torch.Generator().manual_seed(seed)
    codes = (torch.randn(n, k, generator=g) * 60).clamp(-448, 448)
    codes[torch.rand(n, k, generator=g) < 0.05] *= 1e-4
    scales = torch.empty(-(-n // BLOCK), -(-k // BLOCK)).uniform_(*sizes, generator=g) / 60
    return BlockScaledMatrix(codes.to(torch.float8_e4m3fn).to(device), scales.to(device))


# Products that between them take every way through the kernels: (rows, columns, features, (rows of a tile, blocks that share it, steps of a block, stages of its
# ring)).  Rings wrap where a block has more steps than stages, the ring of scales of tiles of up to 128 rows from 17 steps on; features that are no whole
# blocks, columns that are no whole runs, more tiles than blocks among them.
PLAIN_PATHS = [
    (8, 4096, 9600, (16, 2, 16, 5)), (8, 4096, 19200, (16, 1, 32, 5)), (7, 600, 38530, (16, 1, 10, 5)), (8, 8320, 500, (16, 8, 9, 5)), (3, 4000, 3201, (16, 4, 8, 5)),
    (20, 2500, 19200, (32, 1, 20, 4)), (31, 300, 38530, (32, 1, 6, 4)), (20, 8320, 500, (32, 8, 9, 4)), (9, 4096, 3001, (32, 4, 8, 4)), (17, 4096, 9100, (32, 2, 16, 4)),
    (64, 8320, 500, (64, 8, 9, 7)), (64, 8320, 3200, (64, 4, 17, 7)), (50, 8320, 9001, (64, 2, 33, 7)), (520, 4096, 1280, (64, 1, 32, 7)), (50, 1100, 19300, (64, 1, 18, 7)),
    (100, 2500, 19200, (128, 1, 40, 4)), (128, 1100, 9601, (128, 1, 9, 4)), (1000, 1100, 2300, (128, 1, 9, 4)),
    (1100, 1100, 4001, (256, 1, 18, 6)), (700, 2600, 4001, (256, 1, 21, 6)), (2000, 128, 5000, (256, 1, 3, 6))]
# The same with a gate and an up matrix of half the features each.
GATED_PATHS = [
    (8, 4096, 19200, (16, 1, 32, 5)), (5, 8320, 500, (16, 8, 9, 5)), (20, 2500, 19206, (32, 1, 20, 4)), (50, 8320, 9002, (64, 2, 33, 7)), (520, 4096, 1280, (64, 1, 32, 7)),
    (100, 2500, 19202, (128, 1, 40, 4)), (1100, 1100, 4006, (256, 1, 18, 6)), (700, 2600, 4002, (256, 1, 21, 6))]
# Rows sorted by expert: (pairs, experts, columns, features, ...); steps are those of the most tiles that so many pairs may be.
EXPERT_PATHS = [
    (250, 32, 2100, 2050, (16, 1, 51, 5)), (840, 28, 1200, 1416, (32, 1, 30, 4)), (31200, 240, 1100, 200, (128, 1, 63, 4)), (2400, 6, 1200, 2001, (256, 1, 20, 6)),
    (22300, 223, 300, 130, (256, 1, 15, 6))]


def plan(rows, columns, features, experts=0):
    """The library's own account of how such a product runs."""
    import ctypes
    from torchinferno_b200.kernels import block_scaled, ops
    few = rows <= (block_scaled.FEW_EXPERT_ROWS * experts if experts else block_scaled.FEW_ROWS)
    found = (ctypes.c_int * 4)()
    assert ops.lib().tib_block_scaled_plan(int(not few), rows, features, columns, experts, ctypes.addressof(found)) == 0
    return tuple(found)


def matrix64(matrix):
    n, k = matrix.shape
    at_n, at_k = torch.arange(n, device=matrix.device) // BLOCK, torch.arange(k, device=matrix.device) // BLOCK
    return matrix.codes.to(torch.float32).double() * matrix.scales.double()[at_n][:, at_k]


def rows64(x):
    """(codes, scales) of rows by the definition; every power of two comes from a table, every border from a comparison."""
    rows, k = x.shape
    x = x.double()
    powers = torch.tensor([2.0 ** p for p in range(-126, 129)], dtype=torch.float64, device=x.device)
    binades = torch.tensor([2.0 ** p for p in range(-6, 10)], dtype=torch.float64, device=x.device)
    codes, scales = torch.empty_like(x), torch.empty(rows, -(-k // BLOCK), dtype=torch.float64, device=x.device)
    for b in range(scales.shape[1]):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        largest = part.abs().max(1).values
        at = (448.0 * powers[None] < largest[:, None]).sum(1).clamp(max=len(powers) - 1)
        s = torch.where(largest == 0, 1.0, powers[at])
        s = torch.where(torch.isfinite(part).all(1), s, torch.nan)
        scales[:, b] = s
        v = part / s[:, None]
        step = binades[((binades[None, None] <= v.abs()[..., None]).sum(-1) - 1).clamp(min=0)] / 8
        codes[:, b * BLOCK:(b + 1) * BLOCK] = torch.round(v / step) * step
    return codes, scales


def widened_rows64(x):
    codes, scales = rows64(x)
    return codes * scales[:, torch.arange(x.shape[1], device=x.device) // BLOCK]


def product64(x, matrix):
    """(the product in 64 bits, a bound of what 32-bit sums may be off by).  A sum of 128 products of codes (each exact in 32 bits) and of the
    runs' shares rounds at most 128 + 2 runs + 2 times, each time by at most a step of 2^-23 of what has been summed."""
    rows, w = widened_rows64(x), matrix64(matrix)
    runs = -(-x.shape[1] // BLOCK)
    return rows @ w.t(), (BLOCK + 2 * runs + 2) * 2.0 ** -23 * (rows.abs() @ w.abs().t())


def gated64(gate, up, act="swiglu", limit=7.0, alpha=1.702):
    """(value, bound) of a gated unit of two (value, bound) pairs; g sigmoid(g) and its clamped form have slopes of at most 1.1."""
    (g, eg), (u, eu) = gate, up
    if act == "glu_clamp":
        g, u = g.clamp(max=limit), u.clamp(-limit, limit) + 1
    else:
        alpha = 1.0
    s = g * torch.sigmoid(alpha * g)
    y = s * u
    # (the exponential, the quotient and two products in 32 bits: 8 roundings, the exponential's argument among them)
    return y, 1.1 * eg * (u.abs() + eu) + s.abs() * eu + 8 * 2.0 ** -23 * (1 + (alpha * g).abs()) * y.abs() + 2.0 ** -126


def act64(value, act):
    v, e = value
    if act == "relu2":
        r = v.clamp(min=0)
        return r * r, 2 * r * e + e * e + 2.0 ** -23 * r * r
    if act == "silu":
        return gated64(value, (torch.ones_like(v), torch.zeros_like(v)))
    if act == "gelu":
        y = 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
        return y, 1.2 * e + 8 * 2.0 ** -23 * v.abs() + 2.0 ** -126
    return v, e


def check(got, value, out_dtype, what=""):
    """``got`` within the bound of the sums and half a step of its own type (bf16: 2^-8 of the value)."""
    want, bound = value
    bound = bound + (2.0 ** -8 * (want.abs() + bound) if out_dtype == torch.bfloat16 else 0.0)
    assert got.dtype == out_dtype and got.shape == want.shape
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound.clamp(min=1e-300)).nan_to_num(9e9).max()):.2f} of the bound"


def requantised64(value, bf16=True):
    """Rows known within a bound, as a product reads them: (the widened codes of the value, how far those of the true rows may be off).  Rounding is
    monotonic for a given scale; the run's scale may be that of the largest number less or plus its bound, too."""
    h, e = value
    if bf16:
        e = e + 2.0 ** -8 * (h.abs() + e)
    want = widened_rows64(h)
    lo, hi = (h.abs() - e).clamp(min=0), h.abs() + e
    off = torch.zeros_like(h)
    for scales in (rows64(lo)[1], rows64(hi)[1], rows64(h)[1]):
        s = scales[:, torch.arange(h.shape[1], device=h.device) // BLOCK]
        for v in (h - e, h, h + e):
            # (a run's largest as it is for this scale, so that the codes are made with it)
            c = (v / s).clamp(-448, 448)
            step = 2.0 ** (torch.floor(torch.log2(c.abs().clamp(min=2.0 ** -6))) - 3)
            off = torch.maximum(off, (torch.round(c / step) * step * s - want).abs())
    return want, off


def product_of_known64(known, matrix):
    """A product of rows of :func:`requantised64`."""
    rows, off = known
    w = matrix64(matrix)
    runs = -(-rows.shape[1] // BLOCK)
    return rows @ w.t(), off @ w.abs().t() + (BLOCK + 2 * runs + 2) * 2.0 ** -23 * ((rows.abs() + off) @ w.abs().t())
