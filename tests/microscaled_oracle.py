"""The definition of 4-bit microscaled rows, matrices and products in 64 bits, for the tests (any device): every number comes from a table, every rounding from
comparisons."""
from __future__ import annotations

import math

import torch

CODES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
SCALES = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)]


def nearest(v, values):
    """Index of the nearest of ``values`` (ascending, from 0) to each v >= 0; of two as near the even one."""
    table = torch.tensor(values, dtype=torch.float64, device=v.device)
    low = (torch.searchsorted(table, v, right=True) - 1).clamp(max=len(values) - 1)
    high = (low + 1).clamp(max=len(values) - 1)
    below, above = v - table[low], table[high] - v
    return torch.where((above < below) | ((above == below) & (low % 2 == 1)), high, low)


def table(values, index):
    return torch.tensor(values, dtype=torch.float64, device=index.device)[index]


def row_powers(largest):
    powers = torch.tensor([2.0 ** p for p in range(-126, 129)], dtype=torch.float64, device=largest.device)
    finite = torch.isfinite(largest)
    found = powers[torch.searchsorted(2688.0 * powers, torch.where(finite, largest, 0.0))]
    return torch.where(largest == 0, 1.0, torch.where(finite, found, math.nan))


def rows64(x):
    """The numbers [rows, columns] that the rows ``x`` stand for, quantised; NaN throughout a row that is not finite."""
    rows, k = x.shape
    x = x.double()
    r = row_powers(x.abs().nan_to_num(math.inf, math.inf).amax(1))
    fine = ~r.isnan()
    t = torch.nn.functional.pad(torch.where(fine[:, None], x, 0.0) / torch.where(fine, r, 1.0)[:, None], (0, -k % 16)).view(rows, -1, 16)
    s = table(SCALES, nearest(t.abs().amax(2) / 6.0, SCALES))[..., None]
    size = table(CODES, nearest(torch.where(s == 0, 0.0, (t / torch.where(s == 0, 1.0, s)).abs()), CODES))
    return (torch.copysign(size, t) * s).view(rows, -1)[:, :k] * r[:, None]


def matrix64(matrix):
    n, k = matrix.shape
    signed = CODES + [-v for v in CODES]
    codes = torch.stack([matrix.codes % 16, matrix.codes // 16], 2).view(n, -1)[:, :k].long()
    scales = matrix.scales.to(torch.float32).double()[:, torch.arange(k, device=codes.device) // 16]
    return table(signed, codes) * scales * matrix.factor.double().reshape(())


def random_matrix(n, k, seed, device="cpu", factor=1e-3):
    """Codes of every kind (both zeros among them) and scales over the whole range of e4m3, zero and its subnormal numbers among them."""
    from torchinferno_b200.kernels.microscaled import MicroscaledMatrix
    g = torch.Generator().manual_seed(seed)
    halves = torch.randint(0, 16, (n, k + k % 2), generator=g, dtype=torch.uint8)
    scales = (4.0 * torch.randn(n, -(-k // 16), generator=g).exp()).clamp(max=448.0)
    scales[torch.rand(scales.shape, generator=g) < 0.03] = 0.0
    scales[torch.rand(scales.shape, generator=g) < 0.03] = 2.0 ** -8
    codes = (halves[:, 0::2] | (halves[:, 1::2] << 4)).contiguous()
    return MicroscaledMatrix(codes.to(device), scales.to(torch.float8_e4m3fn).to(device), torch.tensor(factor, dtype=torch.float32, device=device), k)
