"""4-bit microscaled weights and rows: e2m1 codes with an e4m3 scale for each run of 16 columns, and the products of such rows with such weights.

A code is one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 with a sign.  A matrix [N, K] has one fp32 factor f beside its scales S: number (n, k) stands for
code(n, k) * S[n, k // 16] * f.  The rows x [M, K] of a product are quantised on the way, or come as :class:`MicroscaledRows` from
:func:`quantize_rows` or from a norm that leaves them so (:func:`add_rmsnorm`).  With a the largest absolute value of a row, and a_b that of a run b:

    r = 2^p, p the smallest integer (at least -126) with a * 2^-p <= 2688 = 6 * 448 (1 where a is 0)
    s = a_b / (6 r) rounded to e4m3        codes = x / (s r) rounded to e2m1, at most 6 (0 where s is 0)
    y[m, n] = r[m] f sum over b of s[m, b] S[n, b] (sum over run b of code_x[m, k] code_w[n, k])

All rounding is to nearest, ties to even, of the exact quotient: codes are the same on any machine.  Sums have 32 bits, y is rounded once, and whatever f and r
are it is lost only where it is beyond 32 bits itself (with a factor for each pair too, :func:`ops.moe_expert_product`, from 2^-50 to 2^50 in size or 0).  A row
that holds an infinity or a NaN makes its whole output row NaN.  A row's codes are its own: they do not depend on the rows beside it.

There is no backward pass: this is an inference engine's weight format.
"""
from __future__ import annotations

import functools
import math
from dataclasses import dataclass
from typing import Sequence

import torch

from torchinferno_b200.kernels import ops

RUN = 16                # columns of a scale
STEP = 256              # columns are padded to whole steps
TILE = 128              # rows of a tile of scales
GROUP = 8               # rows whose codes lie together
SCALE_DTYPE = torch.float8_e4m3fn
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
BORDERS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)       # (on a border the even code is taken: the one above 0.75, 1.75 and 3.5)
LARGEST = 6.0 * 448.0
ORDINARY = (2.0 ** -100, 2.0 ** 70)      # factors of matrices that every kernel takes; others' products run on pairs of SMs,
FAR_EXPERTS = 223                        # which take so many experts
_OUT_DTYPES = (torch.bfloat16, torch.float32)


def _count(columns: int, each: int) -> int:
    return -(-columns // each)


@dataclass(frozen=True)
class MicroscaledMatrix:
    """A matrix as a checkpoint stores it: ``codes`` [N, ceil(K / 2)] (uint8, two codes a byte, the even column in the lower half), ``scales``
    [N, ceil(K / 16)] in e4m3 (none negative) and ``factor``, one fp32 number.  ``columns``: K where it is odd (else twice the bytes)."""
    codes: torch.Tensor
    scales: torch.Tensor
    factor: torch.Tensor
    columns: int | None = None

    def __post_init__(self) -> None:
        if self.codes.dtype != torch.uint8 or self.codes.dim() != 2 or 0 in self.codes.shape:
            raise ValueError(f"codes must be a non-empty 2-D tensor of uint8, got {self.codes.dtype} {tuple(self.codes.shape)}")
        if self.columns is None:
            object.__setattr__(self, "columns", 2 * self.codes.shape[1])
        if _count(self.columns, 2) != self.codes.shape[1]:
            raise ValueError(f"{self.columns} columns do not have {self.codes.shape[1]} bytes of codes")
        wanted = (self.codes.shape[0], _count(self.columns, RUN))
        if self.scales.dtype != SCALE_DTYPE or tuple(self.scales.shape) != wanted:
            raise ValueError(f"scales of a {tuple(self.shape)} matrix must be {SCALE_DTYPE} {wanted}, got {self.scales.dtype} {tuple(self.scales.shape)}")
        if self.factor.dtype != torch.float32 or self.factor.numel() != 1:
            raise ValueError(f"the factor must be one float32 number, got {self.factor.dtype} {tuple(self.factor.shape)}")
        if len({self.codes.device, self.scales.device, self.factor.device}) != 1:
            raise ValueError(f"codes are on {self.codes.device}, scales on {self.scales.device}, the factor on {self.factor.device}")

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.codes.shape[0], self.columns))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def to(self, device: torch.device | str) -> "MicroscaledMatrix":
        return MicroscaledMatrix(self.codes.to(device), self.scales.to(device), self.factor.to(device), self.columns)

    def widened(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The numbers the matrix stands for (on any device)."""
        n, k = self.shape
        signed = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float32, device=self.device)
        halves = torch.stack([self.codes & 15, self.codes >> 4], dim=2).view(n, -1)[:, :k]
        scales = self.scales.to(torch.float32).repeat_interleave(RUN, 1)[:, :k]
        return (signed[halves.long()] * scales * self.factor.reshape(())).to(dtype)


def _nearest_scales(v: torch.Tensor) -> torch.Tensor:
    """The e4m3 numbers nearest to ``v`` (64 bits, none negative), ties to even, at most 448."""
    steps = torch.tensor([2.0 ** (binade - 3) for binade in range(-6, 9)], dtype=v.dtype, device=v.device)
    step = steps[(torch.frexp(v).exponent.long() - 1).clamp(-6, 8) + 6]
    return (torch.round(v / step) * step).clamp(max=448.0).to(torch.float32).to(SCALE_DTYPE)


def quantize_matrix(matrix: torch.Tensor) -> MicroscaledMatrix:
    """The 4-bit form of ``matrix`` [N, K]: f = (its largest absolute value) / 2688, S = e4m3(a run's largest / (6 f)), codes the nearest ones; ties to even.

    Quotients are taken in 64 bits, of products that are exact there: a quotient that is not on a border, a number of few bits, is off it by 2^-32 of it or more."""
    if matrix.dim() != 2 or 0 in matrix.shape:
        raise ValueError(f"quantize_matrix takes a non-empty matrix, got {tuple(matrix.shape)}")
    n, k = matrix.shape
    matrix = matrix.detach()
    largest = matrix.abs().amax().to(torch.float32)
    factor = (largest / torch.full_like(largest, LARGEST)).clamp(min=torch.finfo(torch.float32).tiny)      # (a number of Python's would be a product with its inverse on a GPU)
    codes = torch.empty((n, _count(k, 2)), dtype=torch.uint8, device=matrix.device)
    scales = torch.empty((n, _count(k, RUN)), dtype=SCALE_DTYPE, device=matrix.device)
    wide_factor, rows = factor.to(torch.float64), max(1, (1 << 24) // k)
    for first in range(0, n, rows):
        at = slice(first, first + rows)
        runs = torch.nn.functional.pad(matrix[at].to(torch.float64), (0, -k % RUN)).view(-1, scales.shape[1], RUN)
        scales[at] = _nearest_scales(runs.abs().amax(2) / (6.0 * wide_factor))
        wide = scales[at].to(torch.float64)[..., None]
        size = torch.where(wide == 0, 0.0, runs.abs() / torch.where(wide == 0, 1.0, wide * wide_factor))
        part = torch.zeros(runs.shape, dtype=torch.uint8, device=matrix.device)
        for i, border in enumerate(BORDERS):
            part += size >= border if i % 2 else size > border
        part += 8 * ((runs < 0) & (part > 0)).to(torch.uint8)
        part = part.view(len(part), -1)
        codes[at] = (part[:, 0::2] | (part[:, 1::2] << 4))[:, :codes.shape[1]]
    return MicroscaledMatrix(codes, scales, factor, k)


# ------------------------------------------------------------------------------------------------ rows
@functools.lru_cache(maxsize=4096)
def _sizes(rows: int, columns: int, experts: int) -> tuple[int, int, int, torch.Size]:
    """(where in a buffer for so many rows' codes, scales and factors the scales begin, where the factors, its bytes, the rows' shape); see
    csrc/microscaled.cuh.  (experts: 0 for rows that are not sorted.)"""
    steps = _count(columns, STEP)
    codes, scales = (_count(rows, GROUP) + experts) * steps * (GROUP * STEP // 2), (_count(rows, TILE) + experts) * steps * (TILE * STEP // RUN)
    return codes, codes + scales, codes + scales + 4 * rows, torch.Size((rows, columns))


_makes = functools.lru_cache(maxsize=4096)(ops.microscaled_makes)


class MicroscaledRows:
    """Quantised rows [rows, columns], as the kernels read them.  ``dtype``: the type of what they were made from."""
    __slots__ = ("buffer", "shape", "dtype", "codes_at", "scales_at", "factors_at")

    def __init__(self, like: torch.Tensor, rows: int, columns: int, dtype: torch.dtype) -> None:
        scales, factors, size, self.shape = _sizes(rows, columns, 0)
        self.buffer = buffer = ops.new_bytes(like, size)
        self.dtype, self.codes_at = dtype, (at := buffer.data_ptr())
        self.scales_at, self.factors_at = at + scales, at + factors

    @property
    def device(self) -> torch.device:
        return self.buffer.device

    def get_device(self) -> int:
        return self.buffer.get_device()

    def __len__(self) -> int:
        return self.shape[0]

    def widened(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The numbers the rows stand for, in ``dtype`` (bfloat16, which holds them all but where they underflow, or float32; left out: the rows' own)."""
        rows, columns = self.shape
        dtype = self.dtype if dtype is None else dtype
        ops.need_rows(self, None, None, "widened")
        if dtype not in _OUT_DTYPES:
            raise ops.KernelError(f"widened: unsupported dtype {dtype}")
        out = ops.new_rows(self.buffer, rows, columns, dtype)
        ops.microscaled_widen(self.codes_at, self.scales_at, self.factors_at, out, rows, columns)
        return out


def quantize_rows(x: torch.Tensor) -> MicroscaledRows:
    """The rows ``x`` [M, K] (bfloat16 or float32, any row stride) in 4 bits; see the module's text."""
    count = ops.need_rows(x, None, None, "quantize_rows")
    rows = MicroscaledRows(x, count, x.shape[1], x.dtype)
    ops.microscaled_rows(x, rows.codes_at, rows.scales_at, rows.factors_at)
    return rows


def add_rmsnorm(delta: torch.Tensor | None, residual: torch.Tensor, weight: torch.Tensor, eps: float, *, dtype: torch.dtype | None = None,
                rows: torch.Tensor | None = None, out: torch.Tensor | None = None, new_residual: torch.Tensor | None = None) -> MicroscaledRows:
    """:func:`ops.add_rmsnorm` whose rows leave in 4 bits, bit for bit those that :func:`quantize_rows` makes of its output.

    ``dtype``: the type that the normed rows are rounded to before they are quantised (delta's; without a delta bfloat16).  ``rows``: indices of the rows to norm; the
    residual is then left as it is.  ``out``: takes the normed rows too, in ``dtype``.  ``new_residual``: takes residual + delta in place of ``residual``."""
    dtype, count = ops.quantized_norm_type(delta, dtype), residual.shape[0] if rows is None else rows.numel()
    made = MicroscaledRows(residual, count, residual.shape[-1], dtype)
    ops.quantized_norm(delta, residual, weight, eps, dtype, rows, out, new_residual, False, count, made.codes_at, made.scales_at, made.factors_at, 0)
    return made


# ------------------------------------------------------------------------------------------------ weights
class Tiles:
    """Matrices of one size as the kernels read them: ``codes`` [matrices, tiles of 128 rows, steps of 256 columns, 128, 128 bytes (pieces of 16 swizzled)], ``scales``
    [matrices, tiles, steps, 2048 bytes] and ``factors`` [matrices, N]; ``paired``: the matrices' rows are (gate i, up i); ``far``: a factor
    is outside ``ORDINARY`` (csrc/microscaled.cuh)."""
    __slots__ = ("codes", "scales", "factors", "count", "features", "columns", "paired", "far", "device_index", "numbers")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, factors: torch.Tensor, columns: int, paired: bool, far: bool) -> None:
        self.codes, self.scales, self.factors, self.count, self.features, self.columns, self.paired = codes, scales, factors, codes.shape[0], factors.shape[1], columns, paired
        self.far, self.device_index = far, codes.get_device()
        # (what a product is told of them)
        self.numbers = (codes.data_ptr(), scales.data_ptr(), factors.data_ptr(), int(paired) + 2 * far, self.features, columns, self.count)


def _laid_out(stacks: Sequence[Sequence[MicroscaledMatrix]], paired: bool) -> Tiles:
    """A stack of matrices over the same columns for each expert (or one): a stack's rows lie one behind the other, or (``paired``) alternate."""
    columns, device = stacks[0][0].columns, stacks[0][0].device
    heights = [m.shape[0] for m in stacks[0]]
    for stack in stacks:
        if [m.shape[0] for m in stack] != heights or any(m.columns != columns or m.device != device for m in stack):
            raise ValueError("matrices of one weight must be alike: " + ", ".join(f"{tuple(m.shape)} on {m.device}" for m in (*stacks[0], *stack)))
    if paired and (len(heights) != 2 or heights[0] != heights[1]):
        raise ValueError(f"a gate and an up matrix are needed, of one size, not {heights} rows")
    features, steps = sum(heights), _count(columns, STEP)
    tiles = _count(features, TILE)
    codes = torch.zeros((len(stacks), tiles * TILE, steps * (STEP // 2)), dtype=torch.uint8, device=device)
    scales = torch.zeros((len(stacks), tiles * TILE, steps * (STEP // RUN)), dtype=torch.uint8, device=device)
    factors = torch.empty((len(stacks), features), dtype=torch.float32, device=device)
    first, found = 0, []
    for j, height in enumerate(heights):      # (all stacks' j-th matrices at once)
        at = slice(j, features, 2) if paired else slice(first, first + height)
        part = [stack[j] for stack in stacks]
        codes[:, at, :part[0].codes.shape[1]] = torch.stack([m.codes for m in part]) if len(part) > 1 else part[0].codes
        scales[:, at, :part[0].scales.shape[1]] = torch.stack([m.scales.view(torch.uint8) for m in part]) if len(part) > 1 else part[0].scales.view(torch.uint8)
        factors[:, at] = of_part = torch.stack([m.factor.reshape(1) for m in part])
        found.append(of_part.view(-1))
        first += height
    if columns % 2:      # (the half byte behind the last column)
        codes[:, :, columns // 2] &= 15
    # (piece p of 16 bytes of a step of row i: to piece p ^ (i % 8))
    pieces = torch.arange(8, device=device) ^ (torch.arange(TILE, device=device) % 8)[:, None]
    codes = codes.view(len(stacks), tiles, TILE, steps, 8, 16).transpose(2, 3)[:, :, :, torch.arange(TILE, device=device)[:, None], pieces].contiguous()
    # (row 32 a + b of a tile, run 4 c + d of a step: to [c][b][a][d])
    scales = scales.view(len(stacks), tiles, 4, 32, steps, 4, 4).permute(0, 1, 4, 5, 3, 2, 6).contiguous()
    # (The products ask for their weights ahead of the kernels before them in the stream: this waits until all of the above is there.)
    *values, largest = torch.cat([*found, scales.max().to(torch.float32).view(1)]).tolist()
    if largest > 0x7e:
        raise ValueError("the scales of a 4-bit matrix must be numbers, and none of them negative")
    ordered = [stack[j] for j in range(len(heights)) for stack in stacks]      # (a factor is far where it matters: not that of a matrix of zeros)
    far = any(not ORDINARY[0] <= abs(f) <= ORDINARY[1] and f != 0 and math.isfinite(f) and bool(m.scales.view(torch.uint8).any()) for f, m in zip(values, ordered))
    if far and len(stacks) > FAR_EXPERTS:
        raise ValueError(f"factors of 4-bit matrices outside {ORDINARY[0]:g} .. {ORDINARY[1]:g} are not taken of more than {FAR_EXPERTS} experts")
    return Tiles(codes.view(len(stacks), tiles, steps, TILE, -1), scales.view(len(stacks), tiles, steps, -1), factors, columns, paired, far)


_NO_ROWS = (0, 0, 0)


def _product(x: "torch.Tensor | MicroscaledRows", tiles: Tiles, y: torch.Tensor, act: str, limit: float, alpha: float, offsets: int, order: int, top: int,
             x_by_pair: bool, row_scale: torch.Tensor | None, error_word: torch.Tensor | None, fresh: bool = False) -> None:
    # (fresh: y is memory that x is not)
    if isinstance(x, MicroscaledRows):
        x, rows = None, (x.codes_at, x.scales_at, x.factors_at)
    elif (fresh and not tiles.far and y.shape[0] <= GROUP and x.dtype is torch.bfloat16 and x.stride(0) % 8 == 0 and x.data_ptr() % 16 == 0 and
          _makes(y.shape[0], tiles.features, tiles.columns)):
        rows = _NO_ROWS
    else:
        scales, factors, size, _ = _sizes(y.shape[0], tiles.columns, tiles.count if offsets else 0)
        held = ops.new_bytes(x, size)
        at = held.data_ptr()
        rows = (at, at + scales, at + factors)
    ops.microscaled_product(tiles.numbers, x, rows, y, act, limit, alpha, offsets, order, top, x_by_pair, row_scale, error_word)


class MicroscaledWeight:
    """A projection of 4-bit codes, laid out for the kernels.  ``MicroscaledWeight(matrix)``; several matrices over the same columns
    (``MicroscaledWeight(q, k, v)``) give their outputs side by side; ``MicroscaledWeight(gate, up, epilogue="swiglu")`` is what
    :func:`gemm.linear_swiglu` takes."""

    def __init__(self, *matrices: MicroscaledMatrix, epilogue: str = "none") -> None:
        if epilogue not in ("none", "swiglu"):
            raise ValueError(f"unknown epilogue {epilogue!r}")
        if not matrices or any(not isinstance(m, MicroscaledMatrix) for m in matrices):
            raise ValueError("a microscaled weight is made of microscaled matrices")
        if epilogue == "swiglu" and len(matrices) != 2:
            raise ValueError("the swiglu epilogue takes a gate and an up matrix")
        self.epilogue, self.in_features = epilogue, matrices[0].columns
        self.tiles = _laid_out([matrices], epilogue == "swiglu")
        self.out_features = self.tiles.features

    @property
    def dtype(self) -> torch.dtype:
        return torch.uint8

    @property
    def device(self) -> torch.device:
        return self.tiles.codes.device

    def address(self) -> int:
        return self.tiles.numbers[0]

    def nbytes(self) -> int:
        return self.tiles.codes.numel() + self.tiles.scales.numel() + 4 * self.tiles.factors.numel()

    def rows(self, start: int, stop: int) -> "MicroscaledWeight":
        """The projection onto output features start .. stop-1 (a view; ``start`` a whole number of tiles of 128)."""
        if self.epilogue != "none" or not 0 <= start < stop <= self.out_features:
            raise ValueError(f"no features {start} .. {stop - 1} of {self.out_features} to take")
        if start % TILE:
            raise ValueError(f"feature {start} lies inside a tile of {TILE}")
        view = object.__new__(MicroscaledWeight)
        view.epilogue, view.in_features, view.out_features = "none", self.in_features, stop - start
        at = slice(start // TILE, _count(stop, TILE))
        view.tiles = Tiles(self.tiles.codes[:, at], self.tiles.scales[:, at], self.tiles.factors[:, start:stop], self.in_features, False, self.tiles.far)
        return view

    def _run(self, x: "torch.Tensor | MicroscaledRows", act: str, width: int, out_dtype: torch.dtype | None, out: torch.Tensor | None,
             error_word: torch.Tensor | None) -> torch.Tensor:
        if not isinstance(x, (torch.Tensor, MicroscaledRows)):
            raise ops.KernelError(f"linear: a 4-bit weight takes a tensor or MicroscaledRows, not {type(x).__name__}")
        rows = ops.need_rows(x, self.in_features, self.tiles.device_index, "linear")
        dtype = x.dtype if out_dtype is None else out_dtype
        if dtype not in _OUT_DTYPES:
            raise ops.KernelError(f"linear: unsupported output dtype {dtype}")
        fresh = out is None or out.dtype != dtype
        if fresh:
            out = ops.new_rows(x if isinstance(x, torch.Tensor) else x.buffer, rows, width, dtype)
        elif out.shape != (rows, width) or (out.stride(1) != 1 and width > 1) or out.get_device() != x.get_device():
            raise ops.KernelError(f"linear: out is {tuple(out.shape)} on {out.device}, wanted {(rows, width)} with unit inner stride on {x.device}")
        if rows:
            _product(x, self.tiles, out, act, 0.0, 0.0, 0, 0, 1, False, None, error_word, fresh)
        return out

    def product(self, x: "torch.Tensor | MicroscaledRows", *, out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
                error_word: torch.Tensor | None = None) -> torch.Tensor:
        """x [tokens, in] times the weight: [tokens, out] (a swiglu weight's gate and up sums side by side)."""
        return self._run(x, "none", self.out_features, out_dtype, out, error_word)

    def swiglu(self, x: "torch.Tensor | MicroscaledRows", *, out_dtype: torch.dtype | None = None, error_word: torch.Tensor | None = None) -> torch.Tensor:
        """silu(gate) * up of the 32-bit sums: [tokens, out / 2]."""
        if self.epilogue != "swiglu":
            raise ops.KernelError("linear_swiglu: the weight was not bound with epilogue='swiglu'")
        return self._run(x, "swiglu", self.out_features // 2, out_dtype, None, error_word)


class MicroscaledExperts:
    """The experts' matrices of one product of a routed feed-forward, all of one size: ``MicroscaledExperts(matrices)``, or
    ``MicroscaledExperts(gates, ups)`` for a gated unit.  :func:`ops.moe_expert_product` takes it in place of a tensor."""

    def __init__(self, matrices: Sequence[MicroscaledMatrix], ups: Sequence[MicroscaledMatrix] | None = None) -> None:
        if not matrices:
            raise ValueError("a product of experts needs at least one")
        if ups is not None and len(ups) != len(matrices):
            raise ValueError(f"{len(matrices)} gate and {len(ups)} up matrices")
        self.paired = ups is not None
        self.tiles = _laid_out([[m] for m in matrices] if ups is None else list(zip(matrices, ups)), self.paired)
        self.experts, self.in_features, self.out_features = len(matrices), self.tiles.columns, self.tiles.features

    @property
    def device(self) -> torch.device:
        return self.tiles.codes.device

    def address(self) -> int:
        return self.tiles.numbers[0]

    def nbytes(self) -> int:
        return self.tiles.codes.numel() + self.tiles.scales.numel() + 4 * self.tiles.factors.numel()

    def product(self, x: torch.Tensor, y: torch.Tensor, offsets: torch.Tensor, order: torch.Tensor, top: int, *, x_by_pair: bool,
                act: str = "none", limit: float = 0.0, alpha: float = 1.0, row_scale: torch.Tensor | None = None,
                error_word: torch.Tensor | None = None) -> torch.Tensor:
        """See :func:`ops.moe_expert_product`."""
        if not isinstance(x, torch.Tensor):
            raise ops.KernelError("moe_expert_product: rows by expert are quantised as they are sorted; they come as a tensor")
        pairs = ops.need_expert_product(x, y, offsets, order, top, x_by_pair, act, row_scale, self.experts, self.in_features, self.out_features, self.paired,
                                        self.tiles.device_index)
        if pairs:
            _product(x, self.tiles, y, act, limit, alpha, offsets.data_ptr(), order.data_ptr(), top, x_by_pair, row_scale, error_word)
        return y
