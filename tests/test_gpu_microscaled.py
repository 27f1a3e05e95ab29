"""4-bit microscaled rows and products, and norms that leave quantised rows, on the GPU against their definitions in 64 bits."""
import pytest
import torch

from gpu_common import need_gpu
from microscaled_oracle import matrix64, random_matrix, rows64
from torchinferno_b200.kernels import block_scaled, gemm, microscaled, ops
from torchinferno_b200.kernels.microscaled import MicroscaledExperts, MicroscaledMatrix, MicroscaledWeight, quantize_rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def rows(m, k, seed, dtype=BF16, spread=2.0):
    g = torch.Generator().manual_seed(1000 + seed)
    x = torch.randn(m, k, generator=g) * (spread * torch.randn(m, 1, generator=g)).exp() * (torch.randn(1, k, generator=g)).exp()
    return x.to(dtype).to(DEV)


def same(a, b):
    return torch.equal(a.double().nan_to_num(-1e30), b.double().nan_to_num(-1e30))


# ------------------------------------------------------------------------------------------------ rows to codes
def same_rows(x):
    made = quantize_rows(x)
    assert made.shape == x.shape and made.dtype == x.dtype and len(made) == len(x)
    wide = made.widened(F32)
    assert same(wide, rows64(x).float())
    return made


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m, k", [(1, 1), (1, 16), (3, 15), (8, 4096), (9, 257), (17, 127), (64, 520), (130, 1000), (5, 2055), (300, 33), (2, 17000), (3, 33000)])
def test_rows_become_codes(m, k, dtype):
    need_gpu()
    same_rows(rows(m, k, m + k, dtype))


def test_bf16_values_beside_every_border():
    """Runs of 16 over all finite bf16 numbers, so scales of all binades; rows of two runs whose scales differ by every ratio; numbers on
    the borders between codes, and next to them."""
    need_gpu()
    bits = torch.arange(0x7f80, dtype=torch.int32)
    x = (bits << 16).view(F32)[:0x7f80 // 16 * 16].view(-1, 16) * torch.where(torch.arange(16) % 3 == 0, -1.0, 1.0)
    same_rows(x.to(BF16).to(DEV))
    top = torch.full((1024, 1), 2688.0)
    second = (torch.arange(1024, dtype=torch.int32) + 0x3d80 - 512 << 16).view(F32)[:, None]         # (a scale on and beside every border, from its subnormal numbers up)
    scale_borders = torch.cat([top, torch.zeros(1024, 15), second, second.expand(1024, 15) * 0.5], 1)
    same_rows(scale_borders.to(BF16).to(DEV))
    same_rows(scale_borders.to(DEV))
    six = torch.cat([torch.tensor([2688.0] + [0.0] * 15), torch.tensor([6.0 * 15 / 16 * 2.0 ** -8] + [0.0] * 15)])
    same_rows(torch.stack([six, six * (1 + 2.0 ** -23), six * (1 - 2.0 ** -24)]).to(DEV))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_numbers_on_and_beside_the_borders_of_codes(dtype):
    need_gpu()
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    made = []
    for m in range(8, 16):                        # (scales of every mantissa)
        run = torch.cat([torch.tensor([6.0]), borders, -borders[:7]]) * m
        made.append(run)
        for step in (1, -1):
            near = (run.to(dtype).view(torch.int16 if dtype == BF16 else torch.int32) + step).view(dtype).float()
            near[0] = 6.0 * m
            near[8] = 5.5 * m
            made.append(near)
    x = torch.cat(made)[None]
    x = torch.cat([x * 2.0 ** p for p in range(-3, 4)], 1)
    same_rows(torch.cat([x * 2.0 ** p for p in (-120, -100, 0, 90)]).to(dtype).to(DEV))


def test_rows_of_any_stride_and_alignment():
    need_gpu()
    wide = rows(20, 1500, 3)
    same_rows(wide[:, 8:8 + 600])
    same_rows(wide[:, 3:3 + 601])
    same_rows(wide[::3, 1:130])
    same_rows(rows(40, 777, 4, F32)[1::2, 5:5 + 300])
    same_rows(rows(1, 300, 5).expand(6, 300))


def test_rows_that_are_empty_or_not_finite():
    need_gpu()
    x = rows(8, 400, 7, F32)
    x[0] = 0
    x[1, 130] = float("inf")
    x[2, 5] = float("nan")
    x[3, 399] = -float("inf")
    x[4] = 1e-42                    # subnormal numbers
    x[5, :128] = 3e38
    x[6] = -0.0
    same_rows(x)
    same_rows(x[:4].to(BF16))
    assert quantize_rows(x[:0]).widened(F32).shape == (0, 400)


def test_widened_rows_in_both_types():
    need_gpu()
    x = rows(140, 333, 11)
    made = quantize_rows(x)
    assert made.widened().dtype == BF16 and same(made.widened(), rows64(x).to(BF16)) and same(made.widened(F32), rows64(x))


# ------------------------------------------------------------------------------------------------ norms that leave quantised rows
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m, k", [(1, 1), (8, 4096), (3, 520), (130, 1000), (5, 2055), (2, 9000), (7, 8192), (1, 264)])
def test_a_norm_leaves_the_codes_of_its_rows(m, k, dtype):
    need_gpu()
    g = torch.Generator().manual_seed(m + k)
    delta, residual, weight = rows(m, k, m, dtype), 3.0 * torch.randn(m, k, generator=g).to(DEV), 1 + 0.3 * torch.randn(k, generator=g).to(DEV)
    want_residual, want = residual.clone(), torch.empty(m, k, dtype=dtype, device=DEV)
    ops.add_rmsnorm(delta, want_residual, weight, 1e-5, want)
    for form in (microscaled, block_scaled):
        kept, out, new = residual.clone(), torch.empty_like(want), torch.empty_like(residual)
        made = form.add_rmsnorm(delta, kept, weight, 1e-5)
        assert torch.equal(kept, want_residual) and made.dtype == dtype and made.shape == (m, k)
        wide = made.widened(F32)
        plain = quantize_rows(want).widened(F32) if form is microscaled else None
        if plain is None:
            codes, scales = block_scaled.quantize_rows(want)
            plain = codes.float() * scales.repeat_interleave(128, 1)[:, :k]
            assert torch.equal(made.parts()[0].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(made.parts()[1], scales)
        assert torch.equal(wide, plain)
        kept = residual.clone()
        again = form.add_rmsnorm(delta, kept, weight, 1e-5, out=out, new_residual=new)
        assert torch.equal(kept, residual) and torch.equal(new, want_residual) and torch.equal(out, want) and torch.equal(again.widened(F32), plain)
        alone = form.add_rmsnorm(None, want_residual, weight, 1e-5, dtype=dtype)
        assert torch.equal(alone.widened(F32), plain)
        index = torch.tensor([m - 1, 0, m // 2], dtype=torch.int32, device=DEV)
        picked = form.add_rmsnorm(delta, kept, weight, 1e-5, rows=index)
        assert torch.equal(kept, residual) and torch.equal(picked.widened(F32), plain[index.long()])


# ------------------------------------------------------------------------------------------------ products
def act64(name, sums, limit=7.0, alpha=1.702):
    if name == "swiglu":
        return sums[0] * torch.sigmoid(sums[0]) * sums[1]
    if name == "glu_clamp":
        g, u = sums[0].clamp(max=limit), sums[1].clamp(-limit, limit)
        return g * torch.sigmoid(alpha * g) * (u + 1)
    v = sums[0]
    return {"none": v, "relu2": v.clamp(min=0).square(), "silu": v * torch.sigmoid(v), "gelu": 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))}[name]


def check(y, x, matrices, act="none"):
    """y against the definition.  A sum of K products in 32 bits is off by at most K 2^-24 of the sum of the products' sizes in any order (products of codes, and of
    scales, are exact); two multiplications and the rounding of y add 2^-23 and eps / 2.  Activations pass an error on with a slope of at most 1.13 (gelu, silu), 2 |v|
    (relu2), and of products by their factors' sizes; the approximate exponential adds a few 2^-22 of the result."""
    wide, half = rows64(x), torch.finfo(y.dtype).eps / 2
    k = x.shape[1]
    ws = [matrix64(m) for m in matrices]
    sums = [wide @ w.t() for w in ws]
    slack = [wide.abs() @ w.abs().t() * (k + 4) * 2.0 ** -24 for w in ws]
    want = act64(act, sums)
    if act == "none":
        bound = slack[0]
    elif act in ("silu", "gelu"):
        bound = 1.13 * slack[0]
    elif act == "relu2":
        bound = 2 * sums[0].abs() * slack[0] + slack[0] ** 2
    elif act == "swiglu":
        bound = 1.13 * slack[0] * (sums[1].abs() + slack[1]) + sums[0].abs() * slack[1]
    else:
        bound = 1.7 * slack[0] * 8.0 + 7.0 * slack[1]
    bound = bound + want.abs() * (half + 2.0 ** -20) + (0 if act == "none" else 2.0 ** -20 * sums[0].abs().clamp(max=1.0))
    assert y.shape == want.shape
    bad = (y.double() - want).abs() > bound
    assert not bad.any(), (int(bad.sum()), float(((y.double() - want).abs() / bound).max()))


PLAIN = [(1, 4096, 4096), (1, 16, 8), (1, 1, 1), (2, 255, 129), (3, 257, 1), (8, 4096, 640), (8, 512, 28672), (16, 1000, 1302), (17, 2048, 300), (33, 300, 77), (64, 4096, 512),
         (128, 520, 1400), (129, 256, 130), (200, 1000, 257), (333, 1000, 1302), (600, 4096, 1024), (1000, 272, 2304), (2100, 600, 500),
         (2100, 600, 2500), (600, 4096, 4096), (129, 300, 9601), (1000, 272, 2561), (3000, 1100, 4000)]


@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("m, k, n", PLAIN)
def test_products(m, k, n, out):
    need_gpu()
    matrix = random_matrix(n, k, m + n, DEV)
    x = rows(m, k, m + k)
    weight = MicroscaledWeight(matrix)
    y = gemm.linear(x, weight, out_dtype=out)
    assert y.dtype == out
    check(y, x, [matrix])
    assert torch.equal(gemm.linear(quantize_rows(x), weight, out_dtype=out), y)


@pytest.mark.parametrize("m, k, n", [(1, 4096, 1024), (8, 512, 700), (20, 1000, 333), (130, 600, 129), (500, 1100, 1000), (2000, 512, 2304), (333, 1400, 4001)])
def test_gated_products(m, k, n):
    need_gpu()
    gate, up = random_matrix(n, k, m + n, DEV, 1e-4), random_matrix(n, k, m + n + 1, DEV, 2.3e-4)
    x = rows(m, k, m + k, spread=0.5)
    weight = MicroscaledWeight(gate, up, epilogue="swiglu")
    for out in (BF16, F32):
        check(gemm.linear_swiglu(x, weight, out_dtype=out), x, [gate, up], "swiglu")
    both = gemm.linear(x, weight, out_dtype=F32)
    check(both[:, 0::2], x, [gate])
    check(both[:, 1::2], x, [up])


@pytest.mark.parametrize("act", ["none", "relu2", "silu", "gelu", "swiglu", "glu_clamp"])
@pytest.mark.parametrize("counts, k, n, top", [([1, 0, 3, 0, 4], 520, 300, 2), ([0, 0, 1], 256, 40, 1), ([130, 5, 0, 129, 128, 1, 255], 300, 200, 3), ([16] * 60, 512, 96, 4),
                                               ([700, 0, 900, 3], 1000, 257, 1),
                                               ([257, 0, 256, 1, 600, 130], 1600, 520, 2)])
def test_products_of_experts(counts, k, n, top, act):
    need_gpu()
    experts, pairs = len(counts), sum(counts)
    pairs -= pairs % top
    counts = torch.tensor(counts)
    counts[counts.argmax()] -= int(counts.sum()) - pairs
    gated = act in ops.MOE_GATED
    gates = [random_matrix(n, k, 7 * e + n, DEV, 1e-4 * (1 + e % 3)) for e in range(experts)]
    ups = [random_matrix(n, k, 7 * e + n + 1, DEV, 1e-4) for e in range(experts)] if gated else None
    weight = MicroscaledExperts(gates, ups)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32).to(DEV)
    g = torch.Generator().manual_seed(pairs)
    order = torch.randperm(pairs, generator=g).to(torch.int32).to(DEV)
    row_scale = (0.5 + torch.rand(pairs, generator=g)).to(DEV)
    for by_pair, out, scale in ((True, BF16, None), (False, F32, None), (True, F32, row_scale)):
        x = rows(pairs // top if by_pair else pairs, k, pairs, spread=0.5)
        y = torch.full((pairs, n), 7.0, dtype=out, device=DEV)
        ops.moe_expert_product(x, weight, y, offsets, order, top, x_by_pair=by_pair, act=act, limit=7.0, alpha=1.702, row_scale=scale)
        for e in range(experts):
            at = slice(int(offsets[e]), int(offsets[e + 1]))
            if at.start == at.stop:
                continue
            taken = x[order[at].long() // top] if by_pair else x[at]
            if scale is None:
                check(y[at], taken, [gates[e]] + ([ups[e]] if gated else []), act)
            elif act == "none":      # (the factor multiplies the sums)
                check(y[at] / scale[order[at].long()][:, None], taken, [gates[e]])


def test_rows_behind_the_last_expert_are_left_alone():
    need_gpu()
    weight = MicroscaledExperts([random_matrix(70, 300, e, DEV) for e in range(3)])
    offsets, order = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device=DEV), torch.arange(8, dtype=torch.int32, device=DEV)
    x, y = rows(8, 300, 1), torch.full((8, 70), 3.0, device=DEV)
    ops.moe_expert_product(x, weight, y, offsets, order, 1, x_by_pair=False)
    assert (y[5:] == 3.0).all() and not (y[:5] == 3.0).any()
