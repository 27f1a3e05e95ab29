"""8-bit weights with a scale for each block of 128 x 128, and the products of rows with them.

A matrix [N, K] is held as e4m3 codes with one fp32 scale S for each block of 128 x 128 (the last ones may be short): number (n, k)
stands for code(n, k) * S[n // 128, k // 128].  The rows x [M, K] of a product are quantised on the way: run b of 128
columns of a row, with the largest absolute value a, has the scale s = 2^p, p the smallest integer (at least -126) with
a * 2^-p <= 448 (1 where a is 0), and its codes are x / s rounded to e4m3, to nearest and ties to even.  Then

    y[m, n] = sum over b of s[m, b] * S[n // 128, b] * (sum over run b of code_x[m, k] * code_w[n, k])

with 32-bit sums and one rounding of y at the end, whatever the sizes of s and S (where no normal 32-bit number is their product, the
kernels take them one after the other).  A run that holds an infinity or a NaN makes its whole output row NaN.

A power of two as a run's scale divides without rounding, and its codes are the same on any machine.  Against a / 448, for which the
run's largest number is a code exactly, it costs some accuracy: relative rms error 0.0266 against 0.0257 on Gaussian rows, 0.0265
against 0.0226 on silu(g) * u of such, 0.0266 against 0.016 where one column in a hundred is 20 times as large.  Files in this format were
made with either; a file that says which (``scale_fmt``) and one that does not are read alike.

There is no backward pass: this is an inference engine's weight format.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Sequence

import torch

from torchinferno_b200.kernels import ops

BLOCK = 128
CODE_DTYPE = torch.float8_e4m3fn
_OUT_DTYPES = (torch.bfloat16, torch.float32)
# Up to so many rows (of an expert: on average) a product's kernel quantises its rows itself, in every tile of 128 features anew; more are quantised ahead
# of it.  One number for all sizes: what the first form saves is a kernel, what it costs grows with the tiles.  (us, itself / ahead: 8 rows 4,096 -> 4,096
# 7.9 / 10.1, 4,096 -> 6,144 8.9 / 11.7, 14,336 -> 4,096 13.7 / 16.7, 4,096 -> 28,672 21.2 / 23.9; 10 rows 8.7 / 10.1, 9.7 / 11.8, 15.0 / 16.7, 25.6 / 23.7; 16 rows
# 8.8 / 10.2, 10.0 / 11.8, 15.5 / 16.9, 27.1 / 23.0.  32 experts, gated 2,048 -> 2 x 1,024 and plain 1,024 -> 2,048: 2 rows an expert 24.3 / 24.6 and 14.5 / 14.8,
# 4 25.9 / 25.7 and 15.1 / 16.2, 6 29.0 / 26.9 and 16.3 / 16.4, 8 29.1 / 27.0 and 16.6 / 16.6, 12 29.1 / 27.3 and 17.0 / 16.7, 16 36.9 / 27.6 and 21.2 / 16.9.)
FEW_ROWS = 8
FEW_EXPERT_ROWS = 8


def blocks(count: int) -> int:
    return -(-count // BLOCK)


@dataclass(frozen=True)
class BlockScaledMatrix:
    """A matrix as a checkpoint stores it: ``codes`` [N, K] in e4m3 and ``scales`` [blocks of N, blocks of K] in fp32."""
    codes: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self) -> None:
        if self.codes.dtype != CODE_DTYPE or self.codes.dim() != 2 or 0 in self.codes.shape:
            raise ValueError(f"codes must be a non-empty 2-D tensor of {CODE_DTYPE}, got {self.codes.dtype} {tuple(self.codes.shape)}")
        wanted = tuple(blocks(d) for d in self.codes.shape)
        if self.scales.dtype != torch.float32 or tuple(self.scales.shape) != wanted:
            raise ValueError(f"scales of a {tuple(self.codes.shape)} matrix must be float32 {wanted}, got {self.scales.dtype} {tuple(self.scales.shape)}")
        if self.codes.device != self.scales.device:
            raise ValueError(f"codes are on {self.codes.device}, scales on {self.scales.device}")

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def to(self, device: torch.device | str) -> "BlockScaledMatrix":
        return BlockScaledMatrix(self.codes.to(device), self.scales.to(device))

    def widened(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The numbers the matrix stands for (on any device)."""
        n, k = self.codes.shape
        scales = self.scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
        return (self.codes.to(torch.float32) * scales).to(dtype)


def quantize_matrix(matrix: torch.Tensor) -> BlockScaledMatrix:
    """The e4m3 form of ``matrix`` [N, K]: a block's scale is its largest absolute value / 448 (1 for a block of zeros)."""
    if matrix.dim() != 2 or 0 in matrix.shape:
        raise ValueError(f"quantize_matrix takes a non-empty matrix, got {tuple(matrix.shape)}")
    n, k = matrix.shape
    tiles = torch.nn.functional.pad(matrix.to(torch.float32), (0, -k % BLOCK, 0, -n % BLOCK)).view(blocks(n), BLOCK, blocks(k), BLOCK)
    scales = tiles.abs().amax((1, 3)) / 448.0
    scales = torch.where(scales == 0, 1.0, scales).clamp(min=torch.finfo(torch.float32).tiny)
    codes = (tiles / scales[:, None, :, None]).clamp(-448.0, 448.0).view(blocks(n) * BLOCK, -1)[:n, :k]
    return BlockScaledMatrix(codes.to(CODE_DTYPE).contiguous(), scales.contiguous())


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes [M, K], scales [M, runs of 128]) of the rows ``x`` [M, K] (bfloat16 or float32, any row stride); see the module's text."""
    rows = ops.need_rows(x, None, None, "quantize_rows")
    columns = x.shape[1]
    runs, lds = blocks(columns), (rows + 3) & ~3
    codes = x.new_empty((rows, runs * BLOCK), dtype=CODE_DTYPE)
    scales = x.new_empty_strided((rows, runs), (1, lds), dtype=torch.float32)
    ops.quantize_rows(x, codes.data_ptr(), scales.data_ptr(), lds)
    return codes if columns == runs * BLOCK else codes[:, :columns], scales


def _code_buffer(x: torch.Tensor, rows: int, columns: int) -> torch.Tensor:
    """Room for the codes and scales of ``rows`` rows (see :func:`ops.block_scaled_product`)."""
    runs = -(-columns // BLOCK)
    return x.new_empty(runs * (rows * BLOCK + 4 * ((rows + 3) & ~3)), dtype=torch.uint8)


class BlockScaledRows:
    """Quantised rows [rows, columns] as the products read them, from :func:`add_rmsnorm`.  ``dtype``: the type that the rows were rounded to before."""
    __slots__ = ("buffer", "shape", "dtype", "codes_at", "scales_at", "lds")

    def __init__(self, like: torch.Tensor, rows: int, columns: int, dtype: torch.dtype) -> None:
        self.buffer = ops.new_bytes(like, blocks(columns) * (rows * BLOCK + 4 * ((rows + 3) & ~3)))
        self.shape, self.dtype, self.lds, self.codes_at = torch.Size((rows, columns)), dtype, (rows + 3) & ~3, self.buffer.data_ptr()
        self.scales_at = self.codes_at + blocks(columns) * BLOCK * rows

    @property
    def device(self) -> torch.device:
        return self.buffer.device

    def get_device(self) -> int:
        return self.buffer.get_device()

    def __len__(self) -> int:
        return self.shape[0]

    def parts(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(codes [rows, columns], scales [rows, runs of 128]), as :func:`quantize_rows` returns them (views)."""
        rows, runs = len(self), blocks(self.shape[1])
        codes, scales = self.buffer[:rows * runs * BLOCK], self.buffer[rows * runs * BLOCK:]
        return codes.view(CODE_DTYPE).view(rows, runs * BLOCK)[:, :self.shape[1]], scales.view(torch.float32).view(runs, self.lds).t()[:rows]

    def widened(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The numbers the rows stand for, in ``dtype`` (bfloat16 or float32; left out: the rows' own)."""
        dtype = self.dtype if dtype is None else dtype
        rows = ops.need_rows(self, None, None, "widened")
        if dtype not in _OUT_DTYPES:
            raise ops.KernelError(f"widened: unsupported dtype {dtype}")
        out = ops.new_rows(self.buffer, rows, self.shape[1], dtype)
        ops.widen_rows(self.codes_at, self.scales_at, self.lds, out)
        return out


def add_rmsnorm(delta: torch.Tensor | None, residual: torch.Tensor, weight: torch.Tensor, eps: float, *, dtype: torch.dtype | None = None,
                rows: torch.Tensor | None = None, out: torch.Tensor | None = None, new_residual: torch.Tensor | None = None) -> BlockScaledRows:
    """:func:`ops.add_rmsnorm` whose rows leave in 8 bits, bit for bit those that :func:`quantize_rows` makes of its output.

    ``dtype``: the type that the normed rows are rounded to before they are quantised (delta's; without a delta bfloat16).  ``rows``: indices of the rows to norm; the
    residual is then left as it is.  ``out``: takes the normed rows too, in ``dtype``.  ``new_residual``: takes residual + delta in place of ``residual``."""
    dtype, count = ops.quantized_norm_type(delta, dtype), residual.shape[0] if rows is None else rows.numel()
    made = BlockScaledRows(residual, count, residual.shape[-1], dtype)
    ops.quantized_norm(delta, residual, weight, eps, dtype, rows, out, new_residual, True, count, made.codes_at, 0, made.scales_at, made.lds)
    return made


def _normal_range(scales: torch.Tensor) -> tuple[float, float]:
    """The least and the largest of the powers of two whose product with every one of ``scales`` is a normal 32-bit number, or exact all the same
    (powers of at least 1: 1 always is one of them); the kernels look after other products one by one."""
    sizes = scales.abs()
    least, most = torch.stack(torch.aminmax(sizes)).tolist()
    if not (least > 0 and most < math.inf):      # (zeros are products already, infinities and NaNs remain ones)
        least = torch.where(sizes > 0, sizes, math.inf).amin().item()
        most = torch.where(torch.isfinite(sizes), sizes, 0.0).amax().item()
    low = -126 if math.isinf(least) else max(min(-125 - math.frexp(least)[1], 0), -126)      # (least is at least 2^(its exponent - 1))
    high = 120 if most == 0 else min(128 - math.frexp(most)[1], 120)                         # (most is less than 2^(its exponent))
    return 2.0 ** low, 2.0 ** high


class Blocks:
    """Matrices of one size as the kernels read them: ``codes`` [matrices, blocks of N, blocks of K, 128, 128], padded with zeros, and ``scales`` [matrices,
    blocks of N, blocks of K]; ``paired``: the matrices' rows are (gate i, up i), their scales' rows (gate block j, up block j)."""
    __slots__ = ("codes", "scales", "count", "features", "columns", "paired", "codes_at", "scales_at", "scale_rows", "device_index", "far_low", "far_high")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, features: int, columns: int, paired: bool, far: "tuple[float, float] | None" = None) -> None:
        if codes.shape[1] != blocks(features) or codes.shape[2] != blocks(columns) or scales.shape[1:] != (codes.shape[1] if not paired else 2 * blocks(features // 2), codes.shape[2]):
            raise ValueError(f"blocks {tuple(codes.shape)} and scales {tuple(scales.shape)} do not make matrices of {features} rows")
        if not codes.is_contiguous() or not scales.is_contiguous():
            raise ValueError("blocks and their scales must be contiguous")
        self.codes, self.scales, self.count, self.features, self.columns, self.paired = codes, scales, codes.shape[0], features, columns, paired
        self.codes_at, self.scales_at, self.scale_rows, self.device_index = codes.data_ptr(), scales.data_ptr(), scales.shape[1], codes.get_device()
        self.far_low, self.far_high = _normal_range(scales) if far is None else far      # (the scales are read: once a weight)


def _laid_out(matrices: Sequence[BlockScaledMatrix], ups: Sequence[BlockScaledMatrix] | None) -> Blocks:
    """Equally large matrices in blocks; with ``ups`` the rows of either alternate (gate i, up i; gate block j, up block j)."""
    shape, device = matrices[0].shape, matrices[0].device
    for m in [*matrices, *(ups or ())]:
        if m.shape != shape or m.device != device:
            raise ValueError(f"matrices of one weight must be alike: {tuple(m.shape)} on {m.device}, {tuple(shape)} on {device}")
    if ups is not None and len(ups) != len(matrices):
        raise ValueError(f"{len(matrices)} gate and {len(ups)} up matrices")
    n, k = shape
    parts, runs = 1 if ups is None else 2, blocks(k)
    tiles, each = blocks(n * parts), BLOCK // parts
    codes = torch.empty((len(matrices), tiles, runs, each, parts, BLOCK), dtype=torch.uint8, device=device)
    scales = torch.empty((len(matrices), blocks(n), parts, runs), dtype=torch.float32, device=device)
    pad = (0, runs * BLOCK - k, 0, tiles * each - n)
    for part, stack in enumerate((matrices,) if ups is None else (matrices, ups)):
        for i, m in enumerate(stack):
            stored = m.codes.view(torch.uint8)
            if any(pad):
                stored = torch.nn.functional.pad(stored, pad)
            codes[i, :, :, :, part].copy_(stored.reshape(tiles, each, runs, BLOCK).transpose(1, 2))
            scales[i, :, part].copy_(m.scales)
    return Blocks(codes.view(len(matrices), tiles, runs, BLOCK, BLOCK).view(CODE_DTYPE), scales.view(len(matrices), blocks(n) * parts, -1), n * parts, k,
                  ups is not None)


class BlockScaledWeight:
    """A projection of 8-bit blocks, laid out for the kernels.  ``BlockScaledWeight(matrix)``; several matrices over the same columns
    (``BlockScaledWeight(q, k, v)``) give their outputs side by side; ``BlockScaledWeight(gate, up, epilogue="swiglu")`` is what
    :func:`gemm.linear_swiglu` takes."""

    def __init__(self, *matrices: BlockScaledMatrix, epilogue: str = "none") -> None:
        if epilogue not in ("none", "swiglu"):
            raise ValueError(f"unknown epilogue {epilogue!r}")
        if not matrices or any(not isinstance(m, BlockScaledMatrix) for m in matrices):
            raise ValueError("a block-scaled weight is made of block-scaled matrices")
        if epilogue == "swiglu" and len(matrices) != 2:
            raise ValueError("the swiglu epilogue takes a gate and an up matrix")
        if any(m.shape[1] != matrices[0].shape[1] or m.device != matrices[0].device for m in matrices):
            raise ValueError("the matrices of a weight need the same columns and device")
        self.epilogue, self.in_features = epilogue, matrices[0].shape[1]
        self.out_features = sum(m.shape[0] for m in matrices)
        # (first output, blocks) of every product to run.  Matrices are put together while the ones before end with a whole block; where one
        # does not, its blocks' borders would not be the joint matrix's: it starts a product of its own.
        self.parts: list[tuple[int, Blocks]] = []
        if epilogue == "swiglu":
            self.parts.append((0, _laid_out(matrices[:1], matrices[1:])))
            return
        first, run = 0, []
        for i, m in enumerate(matrices):
            run.append(m)
            if m.shape[0] % BLOCK or i == len(matrices) - 1:
                joint = run[0] if len(run) == 1 else BlockScaledMatrix(
                    torch.cat([r.codes.view(torch.uint8) for r in run]).view(CODE_DTYPE), torch.cat([r.scales for r in run]))
                self.parts.append((first, _laid_out([joint], None)))
                first, run = first + joint.shape[0], []

    @property
    def dtype(self) -> torch.dtype:
        return CODE_DTYPE

    @property
    def device(self) -> torch.device:
        return self.parts[0][1].codes.device

    def address(self) -> int:
        return self.parts[0][1].codes_at

    def nbytes(self) -> int:
        return sum(part.codes.numel() + 4 * part.scales.numel() for _, part in self.parts)

    def rows(self, start: int, stop: int) -> "BlockScaledWeight":
        """The projection onto output features start .. stop-1 (views; ``start`` a whole number of blocks into its matrix)."""
        if self.epilogue != "none" or not 0 <= start < stop <= self.out_features:
            raise ValueError(f"no features {start} .. {stop - 1} of {self.out_features} to take")
        view = object.__new__(BlockScaledWeight)
        view.epilogue, view.in_features, view.out_features, view.parts = "none", self.in_features, stop - start, []
        for first, part in self.parts:
            lo, hi = max(start - first, 0), min(stop - first, part.features)
            if lo < hi:
                if lo % BLOCK:
                    raise ValueError(f"feature {start} lies inside a block")
                view.parts.append((first + lo - start, Blocks(part.codes[:, lo // BLOCK:blocks(hi)], part.scales[:, lo // BLOCK:blocks(hi)], hi - lo, self.in_features, False,
                                                          (part.far_low, part.far_high))))
        return view

    def _run(self, x: "torch.Tensor | BlockScaledRows", act: str, width: int, out_dtype: torch.dtype | None, out: torch.Tensor | None,
             error_word: torch.Tensor | None) -> torch.Tensor:
        ready = isinstance(x, BlockScaledRows)
        if not ready and not isinstance(x, torch.Tensor):
            raise ops.KernelError(f"linear: an 8-bit weight takes a tensor or BlockScaledRows, not {type(x).__name__}")
        rows = ops.need_rows(x, self.in_features, self.parts[0][1].device_index, "linear")
        like, dtype = x.buffer if ready else x, x.dtype if out_dtype is None else out_dtype
        if out is None or out.dtype != dtype:
            if dtype not in _OUT_DTYPES:
                raise ops.KernelError(f"linear: unsupported output dtype {dtype}")
            out = like.new_empty((rows, width)) if dtype == like.dtype else like.new_empty((rows, width), dtype=dtype)
        elif out.shape != (rows, width) or (out.stride(1) != 1 and width > 1) or out.get_device() != x.get_device():
            raise ops.KernelError(f"linear: out is {tuple(out.shape)} on {out.device}, wanted {(rows, width)} with unit inner stride on {x.device}")
        if rows == 0:
            return out
        # (codes that are there already: no kernel quantises them, at few rows neither)
        held = None if ready or rows <= FEW_ROWS else _code_buffer(x, rows, self.in_features)
        codes = x.codes_at if ready else 0 if held is None else held.data_ptr()
        source = None if ready else x
        if len(self.parts) == 1:
            ops.block_scaled_product(source, codes, not ready, self.parts[0][1], out, act, 0.0, 0.0, 0, 0, 1, False, None, error_word)
        else:
            for i, (first, part) in enumerate(self.parts):
                ops.block_scaled_product(source, codes, not ready and i == 0, part, out[:, first:first + part.features], act, 0.0, 0.0, 0, 0, 1, False, None, error_word)
        return out

    def product(self, x: "torch.Tensor | BlockScaledRows", *, out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
                error_word: torch.Tensor | None = None) -> torch.Tensor:
        """x [tokens, in] times the weight: [tokens, out] (a swiglu weight's gate and up sums side by side)."""
        return self._run(x, "none", self.out_features, out_dtype, out, error_word)

    def swiglu(self, x: "torch.Tensor | BlockScaledRows", *, out_dtype: torch.dtype | None = None, error_word: torch.Tensor | None = None) -> torch.Tensor:
        """silu(gate) * up of the 32-bit sums: [tokens, out / 2]."""
        if self.epilogue != "swiglu":
            raise ops.KernelError("linear_swiglu: the weight was not bound with epilogue='swiglu'")
        return self._run(x, "swiglu", self.out_features // 2, out_dtype, None, error_word)


class BlockScaledExperts:
    """The experts' matrices of one product of a routed feed-forward, all of one size: ``BlockScaledExperts(matrices)``, or
    ``BlockScaledExperts(gates, ups)`` for a gated unit.  :func:`ops.moe_expert_product` takes it in place of a tensor."""

    def __init__(self, matrices: Sequence[BlockScaledMatrix], ups: Sequence[BlockScaledMatrix] | None = None) -> None:
        if not matrices:
            raise ValueError("a product of experts needs at least one")
        self.paired = ups is not None
        self.blocks = _laid_out(matrices, ups)
        self.experts, self.in_features = len(matrices), matrices[0].shape[1]
        self.out_features = matrices[0].shape[0] * (2 if self.paired else 1)

    @property
    def device(self) -> torch.device:
        return self.blocks.codes.device

    def address(self) -> int:
        return self.blocks.codes_at

    def nbytes(self) -> int:
        return self.blocks.codes.numel() + 4 * self.blocks.scales.numel()

    def product(self, x: torch.Tensor, y: torch.Tensor, offsets: torch.Tensor, order: torch.Tensor, top: int, *, x_by_pair: bool,
                act: str = "none", limit: float = 0.0, alpha: float = 1.0, row_scale: torch.Tensor | None = None,
                error_word: torch.Tensor | None = None) -> torch.Tensor:
        """See :func:`ops.moe_expert_product`."""
        if not isinstance(x, torch.Tensor):
            raise ops.KernelError("moe_expert_product: rows by expert are quantised as they are sorted; they come as a tensor")
        pairs = ops.need_expert_product(x, y, offsets, order, top, x_by_pair, act, row_scale, self.experts, self.in_features, self.out_features, self.paired,
                                        self.blocks.device_index)
        if pairs == 0:
            return y
        held = None if pairs <= FEW_EXPERT_ROWS * self.experts else _code_buffer(x, pairs, self.in_features)
        ops.block_scaled_product(x, 0 if held is None else held.data_ptr(), True, self.blocks, y, act, limit, alpha, offsets.data_ptr(), order.data_ptr(), top,
                                 x_by_pair, row_scale, error_word)
        return y
