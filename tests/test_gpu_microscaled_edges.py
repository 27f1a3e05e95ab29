"""4-bit rows, norms that leave quantised rows and their products where 32-bit numbers end and where the kernels change, against the definition in 64 bits."""
import pytest
import torch

from gpu_common import need_gpu
from microscaled_oracle import matrix64, random_matrix, rows64
from test_gpu_microscaled import act64, check, rows, same, same_rows
from torchinferno_b200.kernels import block_scaled, gemm, microscaled, ops
from torchinferno_b200.kernels.microscaled import MicroscaledExperts, MicroscaledMatrix, MicroscaledWeight, quantize_rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


# ------------------------------------------------------------------------------------------------ subnormal numbers
def subnormal(m, k, power, seed):
    """Gaussian numbers of this size, most of them subnormal."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=g, dtype=torch.float64) * 2.0 ** power).to(F32).to(DEV)


@pytest.mark.parametrize("power", [-147, -140, -137, -134, -131, -128, -126, -124, -118])
@pytest.mark.parametrize("m, k", [(70, 400), (3, 1003), (1, 17000)])
def test_rows_of_subnormal_numbers(m, k, power):
    need_gpu()
    same_rows(subnormal(m, k, power, m - power))


def test_subnormal_numbers_beside_the_borders_of_codes():
    """Runs with each of the scales that are odd or even multiples of 2^-9, in rows whose factor is 2^-126: a code is a number of units of 2^-149."""
    need_gpu()
    runs = []
    for m in range(1, 16):
        unit = m << 14                                                       # m 2^-9 2^-126
        near = [int(b * unit) + off for b in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)
                for off in (-4097, -4096, -2049, -2048, -2047, -700, -1, 0, 1, 700, 2047, 2048, 4096)]
        near = [min(n, 6 * unit) for n in near] + [0] * (-len(near) % 15)
        for first in range(0, len(near), 15):
            runs.append([6 * unit] + near[first:first + 15])
    bits = torch.tensor(runs, dtype=torch.int32)
    sign = torch.where(torch.arange(16) % 3 == 1, -1.0, 1.0)
    x = bits.view(F32) * sign
    same_rows(x.to(DEV))
    same_rows(x.reshape(1, -1).to(DEV))                                      # (one row: the scales are of every size)
    one = torch.zeros(2, 16, dtype=torch.int32)
    one[:, 0], one[0, 1], one[1, 1] = 6 << 14, 0x1909, 0x262a
    assert quantize_rows(one.view(F32).to(DEV)).widened(F32)[:, 1].tolist() == [2.0 ** -136, 2.0 ** -136]


@pytest.mark.parametrize("m, k", [(4, 520), (3, 1003), (2, 9002), (2, 10240)])
def test_a_norm_of_subnormal_rows(m, k):
    need_gpu()
    residual, weight = rows(m, k, 3, F32, spread=0.3), subnormal(1, k, -131, k)[0]
    out = torch.empty(m, k, device=DEV)
    made = microscaled.add_rmsnorm(None, residual, weight, 1e-5, dtype=F32, out=out)
    assert (out.abs() < 2.0 ** -126).any() and same(made.widened(F32), rows64(out))


@pytest.mark.parametrize("m", [3, 40, 300])
def test_products_of_subnormal_rows(m):
    need_gpu()
    x, matrix = subnormal(m, 300, -130, m), random_matrix(260, 300, 6, DEV, 1e30)
    check(gemm.linear(x, MicroscaledWeight(matrix)), x, [matrix])


# ------------------------------------------------------------------------------------------------ norms whose row nearly fills, fills and overfills 48 KB of shared memory
WIDTHS = (8196, 12028, 12032, 12036, 12160, 12284, 12288, 12292, 16384)


def every_width():
    """Every kernel of norms of this width, the narrower rows first (what a wider row asks for would serve them too)."""
    for k in WIDTHS:
        for dtype in (BF16, F32):
            delta, residual, weight = rows(3, k, k, dtype), rows(3, k, k + 1, F32, spread=0.3), 1 + 0.1 * rows(1, k, k + 2, F32, spread=0.1)[0]
            want = torch.empty(3, k, dtype=dtype, device=DEV)
            ops.add_rmsnorm(delta, residual.clone(), weight, 1e-5, want)
            assert torch.equal(microscaled.add_rmsnorm(delta, residual.clone(), weight, 1e-5).widened(F32), quantize_rows(want).widened(F32)), (k, dtype)
            made, (codes, scales) = block_scaled.add_rmsnorm(delta, residual.clone(), weight, 1e-5), block_scaled.quantize_rows(want)
            assert torch.equal(made.parts()[0].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(made.parts()[1], scales), (k, dtype)


def test_norms_about_48_kb_of_shared_memory():
    """In a process of its own, whose kernels no wider row has met."""
    need_gpu()
    import subprocess
    import sys
    from pathlib import Path
    here = Path(__file__).resolve().parent
    code = f"import sys; sys.path[:0] = [{str(here)!r}, {str(here.parent)!r}]; import test_gpu_microscaled_edges as t; t.every_width(); print('every width')"
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "every width" in done.stdout, done.stdout[-2000:] + done.stderr[-3000:]


# ------------------------------------------------------------------------------------------------ factors at the ends of the range
def check_numbers(y, sums, slack):
    """y against sums in 64 bits that are off by ``slack`` at most, two multiplications and one rounding (check's text), and, of numbers at the lower end, by two steps
    of 2^-149: beyond the largest number y is infinite."""
    half, largest = torch.finfo(y.dtype).eps / 2, torch.finfo(y.dtype).max
    bound = slack + sums.abs() * (half + 2.0 ** -22) + 2.0 ** (-149 if y.dtype == F32 else -133) * 2
    beyond = sums.abs() - bound > largest * (1 + half)
    assert (y[beyond].double() == torch.copysign(torch.full_like(sums, float("inf")), sums)[beyond]).all()
    near = sums.abs() + bound < largest
    assert y[near].isfinite().all() and ((y.double() - sums).abs() <= bound)[near].all()
    return near


def sums_of(x, matrix):
    wide, w = rows64(x), matrix64(matrix)
    return wide @ w.t(), wide.abs() @ w.abs().t() * (x.shape[1] + 4) * 2.0 ** -24


# (the size of a row's largest numbers, the matrix's factor): products of factor and sum, or of row and sum, that are no 32-bit numbers, where the output is one
ENDS = [(2e-24, 1e33), (1e-30, 1e36), (3e-36, 3e38), (1e-38, 3e38), (1e-42, 3e38), (1e30, 1e-39), (1e36, 1e-43), (3e38, 2e-45), (3e38, 1e-38), (1.0, 3e38), (1.0, 1e-45), (3e38, 3e38),
        (1e-40, 1e-40)]


@pytest.mark.parametrize("size, factor", ENDS)
@pytest.mark.parametrize("m, k, n", [(1, 1000, 260), (8, 1000, 700), (3, 8320, 130), (40, 520, 260), (300, 300, 260), (700, 600, 4001)])
def test_products_at_the_ends_of_the_range(m, k, n, size, factor):
    """Rows that the product quantises, tiles of 32 and 128 rows, shared and not, and pairs of SMs."""
    need_gpu()
    matrix = random_matrix(n, k, n, DEV, factor)
    x = (rows(m, k, 5, F32, spread=0.1).clamp(-1, 1).double() * size).to(F32)
    weight = MicroscaledWeight(matrix)
    check_numbers(gemm.linear(x, weight), *sums_of(x, matrix))
    x = x.to(BF16)
    check_numbers(gemm.linear(x, weight, out_dtype=F32), *sums_of(x, matrix))


@pytest.mark.parametrize("m", [2, 40, 300])
def test_the_smallest_sums(m):
    """Two codes of 1/2 and two scales of 2^-9 make a sum of 2^-20: with the least normal factor no normal number, with the rows' it is one."""
    need_gpu()
    factor = 1.7 * 2.0 ** -126
    codes = torch.zeros(260, 16, dtype=torch.uint8)
    codes[:, 8] = torch.arange(260) % 16 << 4                                 # (column 17)
    scales = torch.zeros(260, 2)
    scales[:, 1] = torch.arange(1, 261) % 9 * 2.0 ** -9
    matrix = MicroscaledMatrix(codes.to(DEV), scales.to(torch.float8_e4m3fn).to(DEV), torch.tensor(factor, device=DEV))
    x = torch.zeros(m, 32, device=DEV)
    x[:, 0], x[:, 16], x[:, 17] = 2688.0, 4 * 2.0 ** -9, 0.5 * 2.0 ** -9
    x *= (2.0 ** (torch.arange(m, device=DEV) % 110))[:, None]
    for dtype in (F32, BF16):
        y = gemm.linear(x.to(dtype), MicroscaledWeight(matrix), out_dtype=F32)
        sums, slack = sums_of(x, matrix)
        assert (sums != 0).any() and check_numbers(y, sums, slack * 0).all()      # (one product each: no sum is rounded)


@pytest.mark.parametrize("m", [20, 300, 900])
@pytest.mark.parametrize("size, factor, scale", [(1e-30, 1e36, 1e-15), (3e36, 1e-30, 1e-15), (1e30, 1e12, 1e-10), (1e-30, 1e-22, 1e15), (1.0, 1e-3, 0.0), (1.0, 1e-3, -0.75), (3e38, 1e30, 1e-18),
                                                 (1e-38, 1e-15, 5e17)])
def test_factors_of_pairs_at_the_ends_of_the_range(m, size, factor, scale):
    need_gpu()
    matrix = random_matrix(300, 520, m, DEV, factor)
    x = (rows(m, 520, 5, F32, spread=0.1).clamp(-1, 1).double() * size).to(F32)
    row_scale = scale * (1 + 0.5 * torch.rand(m, generator=torch.Generator().manual_seed(m))).to(DEV)
    order = torch.randperm(m, generator=torch.Generator().manual_seed(m)).to(torch.int32).to(DEV)
    y = torch.empty(m, 300, device=DEV)
    ops.moe_expert_product(x, MicroscaledExperts([matrix]), y, torch.tensor([0, m], dtype=torch.int32, device=DEV), order, 1, x_by_pair=False, row_scale=row_scale)
    sums, slack = sums_of(x, matrix)
    each = row_scale.double()[order.long()][:, None]
    check_numbers(y, sums * each, slack * each.abs())


# ------------------------------------------------------------------------------------------------ blocks of several kernels on an SM
def test_short_products_of_every_kind_side_by_side():
    """4-bit, 8-bit and bf16 products with rings of one stage to full ones, tiles shared by clusters and not, behind one another in a stream and on three streams at once:
    the bits of each by itself."""
    need_gpu()
    g = torch.Generator().manual_seed(3)
    sizes = [(256, 512), (256, 2048), (512, 1024), (1024, 300 * 8), (2048, 1024), (768, 4096)]
    weights = []
    for i, (k, n) in enumerate(sizes):
        dense = torch.randn(n, k, generator=g).to(DEV) / k ** 0.5
        weights.append((k, MicroscaledWeight(random_matrix(n, k, i, DEV, 1e-5))))
        weights.append((k, gemm.LinearWeight(dense.to(BF16), few_rows_tcgen05=True)))
        weights.append((k, block_scaled.BlockScaledWeight(block_scaled.quantize_matrix(dense))))
    inputs = {(m, k): rows(m, k, m + k, spread=0.2) for m in (3, 40, 64, 100) for k in {k for k, _ in sizes}}
    calls = [(m, k, w) for m in (3, 40, 64, 100) for k, w in weights if m <= 64 or not isinstance(w, gemm.LinearWeight)]      # (bf16 above 64 rows: the library's)
    g = torch.Generator().manual_seed(4)
    want = {}
    for i, (m, k, w) in enumerate(calls):
        want[i] = gemm.linear(inputs[m, k], w)
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(6):
        order, outs = torch.randperm(len(calls), generator=g).tolist(), []
        for j, i in enumerate(order):
            m, k, w = calls[i]
            with torch.cuda.stream(streams[j % 3 if turn % 2 else 0]):
                outs.append((i, gemm.linear(inputs[m, k], w)))
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[i]) for i, y in outs)


@pytest.mark.parametrize("size", [1.0, 1e-30, 1e30])
def test_a_matrix_is_quantised_alike_on_the_host_and_on_the_device(size):
    need_gpu()
    w = torch.randn(5000, 3601, generator=torch.Generator().manual_seed(1)) * size
    for made in (w, w.to(BF16)):
        here, there = microscaled.quantize_matrix(made), microscaled.quantize_matrix(made.to(DEV)).to("cpu")
        assert torch.equal(here.codes, there.codes) and torch.equal(here.scales.view(torch.uint8), there.scales.view(torch.uint8)) and here.factor == there.factor


# ------------------------------------------------------------------------------------------------ pairs' factors and activations
def check_scaled(y, x, matrices, act, scale):
    """As check, of sums that are multiplied by a factor each row has ahead of the activation: one more product, 2^-24 of a sum."""
    half = torch.finfo(y.dtype).eps / 2
    wide, k, scale = rows64(x), x.shape[1], scale.double()[:, None]
    ws = [matrix64(m) for m in matrices]
    sums = [wide @ w.t() * scale for w in ws]
    slack = [wide.abs() @ w.abs().t() * scale.abs() * (k + 5) * 2.0 ** -24 for w in ws]
    want = act64(act, sums)
    bound = {"none": lambda: slack[0], "silu": lambda: 1.13 * slack[0], "gelu": lambda: 1.13 * slack[0], "relu2": lambda: 2 * sums[0].abs() * slack[0] + slack[0] ** 2,
             "swiglu": lambda: 1.13 * slack[0] * (sums[1].abs() + slack[1]) + sums[0].abs() * slack[1], "glu_clamp": lambda: 1.7 * slack[0] * 8.0 + 7.0 * slack[1]}[act]()
    bound = bound + want.abs() * (half + 2.0 ** -20) + (0 if act == "none" else 2.0 ** -20 * sums[0].abs().clamp(max=1.0))
    bad = (y.double() - want).abs() > bound
    assert not bad.any(), (int(bad.sum()), float(((y.double() - want).abs() / bound).max()))


@pytest.mark.parametrize("act", ["none", "relu2", "silu", "gelu", "swiglu", "glu_clamp"])
@pytest.mark.parametrize("counts, top", [([1, 0, 3, 0, 4], 2), ([30, 5, 0, 29, 28, 1, 27], 4), ([700, 0, 901, 3], 4), ([257, 0, 256, 1, 600, 130], 2)])
def test_pairs_factors_multiply_the_sums_ahead_of_every_activation(counts, top, act):
    """Factors of both signs and of sizes from 2^-8 to 2^3, the pair's and not the row's."""
    need_gpu()
    k, n, experts, pairs = 520, 260, len(counts), sum(counts)
    gates = [random_matrix(n, k, 7 * e, DEV, 1e-4 * (1 + e % 3)) for e in range(experts)]
    ups = [random_matrix(n, k, 7 * e + 1, DEV, 1e-4) for e in range(experts)] if act in ops.MOE_GATED else None
    weight = MicroscaledExperts(gates, ups)
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32).to(DEV)
    g = torch.Generator().manual_seed(pairs)
    order = torch.randperm(pairs, generator=g).to(torch.int32).to(DEV)
    scale = (torch.randn(pairs, generator=g).sign() * 2.0 ** (11 * torch.rand(pairs, generator=g) - 8)).to(DEV)
    for by_pair, out in ((True, F32), (False, BF16)):
        x = rows(pairs // top if by_pair else pairs, k, pairs, spread=0.5)
        y = torch.empty(pairs, n, dtype=out, device=DEV)
        ops.moe_expert_product(x, weight, y, offsets, order, top, x_by_pair=by_pair, act=act, limit=7.0, alpha=1.702, row_scale=scale)
        for e in range(experts):
            at = slice(int(offsets[e]), int(offsets[e + 1]))
            if at.start < at.stop:
                check_scaled(y[at], x[order[at].long() // top] if by_pair else x[at], [gates[e]] + ([ups[e]] if ups else []), act, scale[order[at].long()])


# ------------------------------------------------------------------------------------------------ operands of a norm that share memory
def test_operands_of_a_norm_that_overlap_are_refused():
    """Blocks write rows of what others still read: refused, and nothing is written.  Side by side in one piece of memory, or the same rows, is fine."""
    need_gpu()
    m, k = 40, 520
    weight = torch.ones(k, device=DEV)
    for dtype in (F32, BF16):
        size = m * k * (4 if dtype == F32 else 2)
        room = torch.zeros(8 * m * k, dtype=torch.float32, device=DEV)
        pieces = room.view(torch.uint8)
        at = lambda first, t, shape=(m, k): pieces[first:first + shape[0] * shape[1] * (2 if t == BF16 else 4)].view(t).view(shape)      # noqa: E731
        residual = at(0, F32)
        residual.copy_(rows(m, k, 1, F32, spread=0.2))
        delta = at(m * k * 4, dtype)
        delta.copy_(rows(m, k, 2, dtype, spread=0.2))
        kept = room.clone()
        end = m * k * 4 + size
        for form in (microscaled, block_scaled):
            for bad in (dict(out=at(m * k * 4 - 1024, dtype)), dict(out=at(end - 1024, dtype)), dict(out=at(512, dtype)), dict(out=at(0, dtype)), dict(out=at(m * k * 4, dtype)),
                        dict(new_residual=at(k * 4, F32)), dict(new_residual=at(end - 16, F32)), dict(new_residual=at(end, F32), out=at(end + 64, dtype)),
                        *([dict(new_residual=at(m * k * 4, F32))] if dtype == BF16 else [])):
                with pytest.raises(ops.KernelError, match="memory"):
                    form.add_rmsnorm(delta, residual, weight, 1e-5, **bad)
            torch.cuda.synchronize()
            assert torch.equal(room, kept)
            want, new = residual.clone(), residual.float() + delta.float()
            normed = torch.empty_like(delta)
            ops.add_rmsnorm(delta, want, weight, 1e-5, normed)
            made = form.add_rmsnorm(delta, residual, weight, 1e-5, new_residual=at(end, F32), out=at(end + m * k * 4, dtype))
            assert torch.equal(at(end, F32), new) and torch.equal(at(end + m * k * 4, dtype), normed) and torch.equal(residual, kept[:m * k].view(m, k))
            same_place = form.add_rmsnorm(delta, residual, weight, 1e-5, new_residual=residual)
            assert torch.equal(residual, new) and torch.equal(same_place.widened(F32), made.widened(F32))
            residual.copy_(kept[:m * k].view(m, k))
            if dtype == F32:      # (the sum takes the place of delta)
                form.add_rmsnorm(delta, residual, weight, 1e-5, new_residual=delta)
                assert torch.equal(delta, new)
            room.copy_(kept)


@pytest.mark.parametrize("m", [1, 8, 30, 200])
def test_far_factors_of_gated_weights_experts_and_views(m):
    """Matrices with far factors beside others: every output of each."""
    need_gpu()
    k, size = 520, 2.0 ** -60
    x = (rows(m, k, 5, F32, spread=0.1).clamp(-1, 1).double() * size).to(F32)
    matrices = [random_matrix(128, k, 1, DEV, 1e15), random_matrix(260, k, 2, DEV, 1e36), random_matrix(70, k, 3, DEV, 2e-20), random_matrix(130, k, 4, DEV, 1e-45)]
    weight = MicroscaledWeight(*matrices)
    y, first = gemm.linear(x, weight), 0
    for matrix in matrices:
        check_numbers(y[:, first:first + matrix.shape[0]], *sums_of(x, matrix))
        first += matrix.shape[0]
    assert torch.equal(gemm.linear(x, weight.rows(128, 458)), y[:, 128:458])
    word = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert torch.equal(weight.product(quantize_rows(x), error_word=word), y) and int(word) == 0
    gate, up = random_matrix(200, k, 7, DEV, 2.0 ** 55), random_matrix(200, k, 8, DEV, 2.0 ** 80)      # (sums about 1 and 2^25)
    x = x * 2.0 ** -18
    check(gemm.linear_swiglu(x, MicroscaledWeight(gate, up, epilogue="swiglu")), x, [gate, up], "swiglu")
    experts = MicroscaledExperts([matrices[1], random_matrix(260, k, 9, DEV, 1e18), random_matrix(260, k, 10, DEV, 1e-38)])
    offsets = torch.tensor([0, m // 3, m // 2, m], dtype=torch.int32, device=DEV)
    out, order = torch.empty(m, 260, device=DEV), torch.arange(m, dtype=torch.int32, device=DEV)
    ops.moe_expert_product(x, experts, out, offsets, order, 1, x_by_pair=False)
    for e, matrix in enumerate([matrices[1], random_matrix(260, k, 9, DEV, 1e18), random_matrix(260, k, 10, DEV, 1e-38)]):
        at = slice(int(offsets[e]), int(offsets[e + 1]))
        if at.start < at.stop:
            check_numbers(out[at], *sums_of(x[at], matrix))
