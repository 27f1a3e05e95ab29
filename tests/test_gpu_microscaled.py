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
@pytest.mark.parametrize("m, k", [(1, 1), (8, 4096), (3, 520), (130, 1000), (5, 2055), (2, 9000), (7, 8192), (1, 264), (3, 1004), (9, 4100), (2, 8196), (300, 10240), (5, 16384), (2, 9002),
                                  (2, 16388)])
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


# ------------------------------------------------------------------------------------------------ every way through the kernels
def plan(rows, columns, features, experts=0):
    """The library's own account of how such a product runs."""
    import ctypes
    found = (ctypes.c_int * 4)()
    assert ops.lib().tib_microscaled_plan(rows, features, columns, experts, ctypes.addressof(found)) == 0
    return tuple(found)


def device_matrix(n, k, seed, factor=1e-3):
    """A large matrix, made on the device."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = (4.0 * torch.randn(n, -(-k // 16), generator=g, device=DEV).exp()).clamp(max=448.0)
    return MicroscaledMatrix(codes, scales.to(torch.float8_e4m3fn), torch.tensor(factor, device=DEV), k)


# Up to eight short rows (8,192 columns in all, of each row a multiple of eight) whose codes the product's kernel makes: rings that wrap, shared tiles, the last run and step in part.
MADE = [(1, 8, 1), (1, 8192, 1000), (1, 4096, 28672), (2, 4096, 640), (2, 3304, 36000), (3, 2048, 2048), (4, 1992, 130), (5, 1024, 30000), (7, 264, 300), (8, 1024, 1024), (8, 1000, 37000),
        (8, 16, 128)]


@pytest.mark.parametrize("m, k, n", MADE)
def test_rows_that_the_product_quantises(m, k, n):
    """One launch, and the bits of rows that were quantised before."""
    need_gpu()
    assert ops.microscaled_makes(m, n, k)
    matrix, x = device_matrix(n, k, m), rows(m, k, n)
    weight, strided = MicroscaledWeight(matrix), torch.zeros(m, k + 8, dtype=BF16, device=DEV)[:, :k]
    for out in (BF16, F32):
        word, before = torch.zeros(1, dtype=torch.int32, device=DEV), ops.launch_count()
        y = weight.product(x, out_dtype=out, error_word=word)
        assert ops.launch_count() == before + 1
        check(y, x, [matrix])
        assert torch.equal(y, weight.product(quantize_rows(x), out_dtype=out)) and int(word) == 0
        assert torch.equal(y, weight.product(strided.copy_(x), out_dtype=out))
    if n % 2 == 0:
        gated = MicroscaledWeight(*(MicroscaledMatrix(matrix.codes[i::2].contiguous(), matrix.scales[i::2].contiguous(), matrix.factor) for i in (0, 1)), epilogue="swiglu")
        assert torch.equal(gated.swiglu(x), gated.swiglu(quantize_rows(x)))


def test_rows_that_the_product_quantises_hold_anything():
    """Zeros, subnormal numbers, the largest, an infinity and a NaN, each a row of its own: as they are quantised before."""
    need_gpu()
    x = rows(8, 1000, 3)
    x[0], x[1], x[2], x[3, 7], x[4, 999], x[5, 0], x[6, 500] = 0, 1e-39, x[2] * 1e-30, float("inf"), float("nan"), 3e38, -float("inf")
    weight = MicroscaledWeight(device_matrix(700, 1000, 1))
    y, want = weight.product(x, out_dtype=F32), weight.product(quantize_rows(x), out_dtype=F32)
    assert torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(), want.nan_to_num())
    assert y[[3, 4, 6]].isnan().all() and not y[[0, 1, 2, 5, 7]].isnan().any() and not y[0].any()


def test_where_the_product_does_not_quantise():
    """More rows or columns than a round of loads takes, columns or strides that are no multiples of eight, more tiles than blocks; an output that lies over the rows."""
    need_gpu()
    assert not any(ops.microscaled_makes(*sizes) for sizes in ((9, 512, 512), (8, 512, 1032), (3, 512, 2056), (2, 512, 4104), (1, 512, 8200), (1, 512, 1001), (1, 300 * 128, 512)))
    weight, x = MicroscaledWeight(random_matrix(512, 512, 1, DEV)), rows(8, 512, 1)
    want = gemm.linear(x, weight)
    apart, shifted = torch.zeros(8, 513, dtype=BF16, device=DEV)[:, :512], torch.zeros(8 * 512 + 1, dtype=BF16, device=DEV)[1:].view(8, 512)
    for other in (apart, shifted):
        before = ops.launch_count()
        assert torch.equal(gemm.linear(other.copy_(x), weight), want) and ops.launch_count() == before + 2
    assert torch.equal(gemm.linear(apart.copy_(x), weight, out=apart), want)
    # (right behind the rows, or ahead of them, is not over them)
    gated = MicroscaledWeight(random_matrix(256, 512, 2, DEV), random_matrix(256, 512, 3, DEV), epilogue="swiglu")
    for made, act, width in ((weight, "none", 512), (gated, "swiglu", 256)):
        for first in (False, True):
            whole = torch.zeros(8 * (512 + width), dtype=BF16, device=DEV)
            at = 8 * width if first else 0
            near, y = whole[at:at + 8 * 512].view(8, 512), (whole[:at] if first else whole[8 * 512:]).view(8, width)
            ops.microscaled_product(made.tiles.numbers, near.copy_(x), (0, 0, 0), y, act, 0.0, 0.0, 0, 0, 1, False, None, None)
            assert torch.equal(near, x) and torch.equal(y, made.swiglu(x) if act == "swiglu" else want)
    over = x.clone()
    with pytest.raises(ops.KernelError):
        ops.microscaled_product(weight.tiles.numbers, over, (0, 0, 0), over, "none", 0.0, 0.0, 0, 0, 1, False, None, None)
    assert torch.equal(over, x) and torch.equal(gemm.linear(over, weight, out=over), want)


# (rows, columns, features, (rows of a tile, blocks that share it, steps of a block, stages of its ring)): rings that wrap and that do not, features that are no whole
# tiles, columns that are no whole steps, more tiles than blocks among them.
WAYS = [(8, 4096, 4096, (32, 4, 4, 3)), (8, 600, 38530, (32, 1, 6, 4)), (20, 2500, 19200, (32, 1, 10, 4)), (3, 8320, 4000, (32, 8, 5, 3)), (8, 900, 300, (32, 4, 1, 1)),
        (8, 2300, 16000, (32, 2, 5, 3)), (64, 1100, 500, (128, 4, 2, 2)), (50, 8320, 9001, (128, 2, 17, 4)), (100, 2500, 19200, (128, 1, 20, 6)), (300, 8192, 1024, (128, 4, 8, 4)),
        (333, 1000, 1302, (128, 1, 4, 4)), (1000, 300, 20000, (256, 1, 10, 5)), (700, 2600, 4001, (256, 1, 11, 5)), (2000, 128, 5000, (256, 1, 3, 5))]


@pytest.mark.parametrize("m, k, n, way", WAYS)
def test_every_way_of_a_product(m, k, n, way):
    """Within the bound, with no wait run out, and the same bits again."""
    need_gpu()
    assert plan(m, k, n) == way
    matrix, x = device_matrix(n, k, m), rows(m, k, n)
    weight = MicroscaledWeight(matrix)
    for out in (BF16, F32):
        word = torch.zeros(1, dtype=torch.int32, device=DEV)
        y = weight.product(x, out_dtype=out, error_word=word)
        check(y, x, [matrix])
        assert torch.equal(y, weight.product(x, out_dtype=out, error_word=word)) and int(word) == 0


@pytest.mark.parametrize("m, k, n", [(8, 4096, 2400), (5, 8320, 250), (20, 2500, 9603), (50, 8320, 4501), (100, 2500, 9601), (700, 2600, 2001)])
def test_every_way_of_a_gated_product(m, k, n):
    need_gpu()
    gate, up, x = device_matrix(n, k, m, 2e-5), device_matrix(n, k, m + 1, 3e-5), rows(m, k, n, spread=0.3)
    weight = MicroscaledWeight(gate, up, epilogue="swiglu")
    for out in (BF16, F32):
        word = torch.zeros(1, dtype=torch.int32, device=DEV)
        y = weight.swiglu(x, out_dtype=out, error_word=word)
        check(y, x, [gate, up], "swiglu")
        assert torch.equal(y, weight.swiglu(x, out_dtype=out)) and int(word) == 0


@pytest.mark.parametrize("pairs, experts, k, n, way", [(30, 32, 2100, 2050, (32, 1, 18, 4)), (250, 32, 2100, 2050, (128, 1, 36, 6)), (3000, 240, 1100, 200, (128, 1, 20, 6)),
                                                       (2400, 6, 1200, 2001, (256, 1, 10, 5)), (3600, 200, 300, 130, (256, 1, 6, 5)), (1500, 1024, 300, 70, (128, 1, 14, 5))])
def test_every_way_of_experts(pairs, experts, k, n, way):
    need_gpu()
    assert plan(pairs, k, n, experts) == way
    matrices = [device_matrix(n, k, e) for e in range(experts)]
    weight = MicroscaledExperts(matrices)
    g = torch.Generator().manual_seed(pairs)
    ids = (torch.rand(pairs, generator=g) ** 2 * experts).long()
    order = torch.sort(ids, stable=True).indices
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(ids, minlength=experts).cumsum(0)]).to(torch.int32).to(DEV)
    x, word = rows(pairs // 2, k, n, spread=0.5), torch.zeros(1, dtype=torch.int32, device=DEV)
    y = torch.empty(pairs, n, device=DEV)
    ops.moe_expert_product(x, weight, y, offsets, order.to(torch.int32).to(DEV), 2, x_by_pair=True, error_word=word)
    again = torch.empty_like(y)
    ops.moe_expert_product(x, weight, again, offsets, order.to(torch.int32).to(DEV), 2, x_by_pair=True, error_word=word)
    assert torch.equal(y, again) and int(word) == 0
    for e in range(experts):
        at = slice(int(offsets[e]), int(offsets[e + 1]))
        if at.start < at.stop and (experts < 100 or e % 17 == 0):
            check(y[at], x[order[at].to(DEV) // 2], [matrices[e]])


# ------------------------------------------------------------------------------------------------ what callers do
def test_32_bit_rows_and_several_matrices():
    need_gpu()
    q, k, v = random_matrix(256, 300, 1, DEV, 1e-3), random_matrix(64, 300, 2, DEV, 0.7), random_matrix(70, 300, 3, DEV, 3e-6)
    weight = MicroscaledWeight(q, k, v)
    for m in (1, 40, 700):
        x = rows(m, 300, m, F32)
        y = gemm.linear(x, weight)
        assert y.dtype == F32
        for at, matrix in ((slice(0, 256), q), (slice(256, 320), k), (slice(320, 390), v)):
            check(y[:, at], x, [matrix])
        assert torch.equal(gemm.linear(x, weight.rows(0, 256)), y[:, :256]) and torch.equal(gemm.linear(x, weight.rows(256, 390)), y[:, 256:])


@pytest.mark.parametrize("m", [3, 130, 300])
def test_strided_rows_and_outputs(m):
    need_gpu()
    matrix = random_matrix(390, 601, 1, DEV)
    weight, wide = MicroscaledWeight(matrix), rows(2 * m, 1500, 3)
    for x in (wide[:m, 8:609], wide[:m, 3:604], wide[::2, 1:602], wide[:1, :601].expand(m, 601)):
        want = gemm.linear(x.contiguous(), weight)
        check(want, x, [matrix])
        assert torch.equal(gemm.linear(x, weight), want)
        for room in (torch.full((m, 500), 9.0, dtype=BF16, device=DEV), torch.full((m + 1, 397), 9.0, dtype=BF16, device=DEV)[1:]):
            out = room[:, 3:393]
            assert gemm.linear(x, weight, out=out).data_ptr() == out.data_ptr() and torch.equal(out, want)
            assert (room[:, :3] == 9.0).all() and (room[:, 393:] == 9.0).all()


@pytest.mark.parametrize("m", [5, 100, 700])
def test_rows_that_are_not_finite_show(m):
    need_gpu()
    gate, up = random_matrix(200, 500, 1, DEV, 1e-4), random_matrix(200, 500, 2, DEV, 1e-4)
    x = rows(m, 500, 3, spread=0.3)
    x[1], x[2, 7], x[3, 499], x[m - 1, 250] = 0, float("nan"), float("inf"), -float("inf")
    fine = [i for i in range(m) if i not in (2, 3, m - 1)]
    for call, matrices, act in ((lambda: gemm.linear(x, MicroscaledWeight(gate)), [gate], "none"),
                                (lambda: gemm.linear_swiglu(x, MicroscaledWeight(gate, up, epilogue="swiglu")), [gate, up], "swiglu")):
        y = call()
        assert y[[2, 3, m - 1]].isnan().all() and not y[1].any()
        check(y[fine], x[fine], matrices, act)
    for act in ("relu2", "silu", "gelu"):
        y = torch.empty(m, 200, dtype=BF16, device=DEV)
        ops.moe_expert_product(x, MicroscaledExperts([gate]), y, torch.tensor([0, m], dtype=torch.int32, device=DEV), torch.arange(m, dtype=torch.int32, device=DEV), 1,
                               x_by_pair=False, act=act)
        assert y[[2, 3, m - 1]].isnan().all() and not y[fine].isnan().any()


def test_sizes_at_the_ends_of_the_range():
    """Rows of the least and of the largest numbers, factors of both kinds: sums are scaled in turn, so only outputs that are beyond 32 bits are lost."""
    need_gpu()
    for size, factor in ((1e-37, 1e25), (2e38, 1e-30), (1e-30, 1e30), (3e38, 1e-38)):
        for m in (2, 300):
            x = (rows(m, 300, 5, F32, spread=0.1).clamp(-1, 1) * size)
            matrix = random_matrix(260, 300, 6, DEV, factor)
            check(gemm.linear(x, MicroscaledWeight(matrix)), x, [matrix])


@pytest.mark.parametrize("m", [1, 8, 64, 100, 300])
def test_a_row_does_not_depend_on_the_others(m):
    need_gpu()
    weight, x = MicroscaledWeight(random_matrix(390, 1100, 3, DEV)), rows(m, 1100, 2)
    first = gemm.linear(x, weight)
    assert torch.equal(first, gemm.linear(x, weight))
    assert torch.equal(torch.roll(first, 1, 0), gemm.linear(torch.roll(x, 1, 0), weight))
    quiet = x.clone()
    quiet[1:] *= 1e-20
    assert torch.equal(first[0], gemm.linear(quiet, weight)[0])


def a_layer(seed):
    gate, up, down = random_matrix(260, 400, seed, DEV, 1e-4), random_matrix(260, 400, seed + 1, DEV, 1e-4), random_matrix(400, 260, seed + 2, DEV, 1e-3)
    norm = 1 + 0.1 * torch.randn(400, generator=torch.Generator().manual_seed(seed)).to(DEV)
    return norm, MicroscaledWeight(gate, up, epilogue="swiglu"), MicroscaledWeight(down), (gate, up, down)


@pytest.mark.parametrize("m", [1, 8, 40, 300, 700])
def test_a_feed_forward_from_its_norm_on(m):
    """residual + delta, the norm's rows in 4 bits, gate and up, down: each step against its definition on what the step before left."""
    need_gpu()
    norm, gated, down, matrices = a_layer(5)
    delta, residual = rows(m, 400, m, spread=0.3), 2.0 * rows(m, 400, m + 1, F32, spread=0.2)
    want, normed = residual.clone(), torch.empty(m, 400, dtype=BF16, device=DEV)
    ops.add_rmsnorm(delta, want, norm, 1e-5, normed)
    made = microscaled.add_rmsnorm(delta, residual, norm, 1e-5)
    assert torch.equal(residual, want) and same(made.widened(F32), rows64(normed))
    inner = gemm.linear_swiglu(made, gated)
    check(inner, normed, matrices[:2], "swiglu")
    assert torch.equal(inner, gemm.linear_swiglu(normed, gated))
    y = gemm.linear(inner, down)
    check(y, inner, matrices[2:])
    # the part that a model has, as a layer calls it
    from torchinferno_b200.parts.base import PartSpec, ResidualStream, build_part
    part = build_part("feed_forward", PartSpec("swiglu", {"hidden_size": 400, "intermediate_size": 260}), dtype=BF16, device=torch.device(DEV))
    part.bind(dict(zip(part.names, matrices)))
    rms = build_part("norm", PartSpec("rmsnorm", {"width": 400, "eps": 1e-5}), dtype=BF16, device=torch.device(DEV))
    rms.bind({"weight": norm})
    stream = ResidualStream(2.0 * rows(m, 400, m + 1, F32, spread=0.2), BF16)
    stream.add(delta)
    read = stream.normed(rms, form=part.rows_form(m))
    assert isinstance(read, microscaled.MicroscaledRows) and stream.pending is None and torch.equal(stream.residual, want)
    assert torch.equal(part.forward(read, None), y)


@pytest.mark.parametrize("m", [3, 8, 9, 100, 700])
def test_8_bit_products_take_the_rows_of_a_norm(m):
    """Codes made by the norm or by the product's own kernel are the same, so where the same kernel multiplies them (from nine rows on) the outputs are too."""
    need_gpu()
    g = torch.Generator().manual_seed(m)
    matrices = [block_scaled.quantize_matrix(torch.randn(n, 400, generator=g).to(DEV) / 20) for n in (256, 100, 36)]
    delta, residual, norm = rows(m, 400, m, spread=0.3), rows(m, 400, m + 1, F32), torch.ones(400, device=DEV)
    normed = torch.empty(m, 400, dtype=BF16, device=DEV)
    made = block_scaled.add_rmsnorm(delta, residual, norm, 1e-5, out=normed)
    for weight, product in ((block_scaled.BlockScaledWeight(*matrices), gemm.linear),
                            (block_scaled.BlockScaledWeight(matrices[0], matrices[0], epilogue="swiglu"), gemm.linear_swiglu)):
        y, plain = product(made, weight), product(normed, weight)
        assert y.dtype == BF16 and (torch.equal(y, plain) if m > block_scaled.FEW_ROWS else torch.allclose(y.float(), plain.float(), rtol=2.0 ** -7, atol=1e-4))
        assert torch.equal(product(made, weight, out_dtype=F32).to(BF16), y)


@pytest.mark.parametrize("m", [3, 100, 700])
def test_captured_and_on_two_streams(m):
    need_gpu()
    norm, gated, down, _ = a_layer(11)
    inputs = [rows(m, 400, i, spread=0.3) for i in range(4)]
    residual = rows(m, 400, 9, F32)

    def pass_of(x):
        new = torch.empty_like(residual)
        return gemm.linear(gemm.linear_swiglu(microscaled.add_rmsnorm(x, residual, norm, 1e-5, new_residual=new), gated), down), new
    want = [pass_of(x) for x in inputs]
    torch.cuda.synchronize()
    graphs, statics = [], []
    for i in range(2):                         # (two captured passes, replayed side by side: they share nothing but the weights)
        x = inputs[i].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = pass_of(x)
        graphs.append(graph), statics.append((x, y))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(8):
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                statics[i][0].copy_(inputs[(turn + i) % 4])
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(statics[i][1], want[(turn + i) % 4]))
    outs = []
    for turn in range(6):
        with torch.cuda.stream(streams[turn % 2]):
            outs.append(pass_of(inputs[turn % 4]))
    torch.cuda.synchronize()
    assert all(torch.equal(y[0], want[turn % 4][0]) for turn, y in enumerate(outs))


def test_refusals():
    need_gpu()
    weight, x = MicroscaledWeight(random_matrix(100, 200, 1, DEV)), rows(4, 200, 1)
    gated = MicroscaledWeight(random_matrix(100, 200, 1, DEV), random_matrix(100, 200, 2, DEV), epilogue="swiglu")
    residual, ones = torch.zeros(4, 200, device=DEV), torch.ones(200, device=DEV)
    for call in (lambda: gemm.linear(x[:, :199], weight), lambda: gemm.linear(x.half(), weight), lambda: gemm.linear(x, weight, out_dtype=torch.float16),
                 lambda: gemm.linear(x.t().contiguous().t(), weight), lambda: gemm.linear(x[0], weight), lambda: gemm.linear_swiglu(x, weight),
                 lambda: gemm.linear(x, weight, out=torch.empty(4, 99, dtype=BF16, device=DEV)), lambda: gemm.linear_swiglu(x.cpu(), gated),
                 lambda: gemm.linear(x, weight, out=torch.empty(100, 4, dtype=BF16, device=DEV).t()),
                 lambda: gemm.linear(x, MicroscaledWeight(random_matrix(100, 200, 1))), lambda: quantize_rows(x.half()), lambda: quantize_rows(x[0]),
                 lambda: quantize_rows(x).widened(torch.float16), lambda: quantize_rows(x[:, :0]),
                 lambda: gemm.linear(quantize_rows(x[:, :199]), weight), lambda: gemm.linear(quantize_rows(x), x),
                 lambda: microscaled.add_rmsnorm(x, residual[:3], ones, 1e-5), lambda: microscaled.add_rmsnorm(x, residual, ones[:199], 1e-5),
                 lambda: microscaled.add_rmsnorm(x, residual.to(BF16), ones, 1e-5), lambda: microscaled.add_rmsnorm(x, residual, ones, 1e-5, dtype=F32),
                 lambda: microscaled.add_rmsnorm(x, residual, ones, 1e-5, out=torch.empty(4, 200, device=DEV)),
                 lambda: microscaled.add_rmsnorm(x, residual, ones, 1e-5, new_residual=torch.empty(4, 199, device=DEV)),
                 lambda: microscaled.add_rmsnorm(x, residual, ones, 1e-5, rows=torch.zeros(2, dtype=torch.int64, device=DEV)),
                 lambda: microscaled.add_rmsnorm(x, residual, ones, 1e-5, rows=torch.zeros(2, dtype=torch.int32, device=DEV), new_residual=residual.clone()),
                 lambda: microscaled.add_rmsnorm(x, residual, ones, 1e-5, out=x), lambda: microscaled.add_rmsnorm(None, residual, ones, 1e-5, dtype=F32, out=residual),
                 lambda: block_scaled.add_rmsnorm(x.t().contiguous().t(), residual, ones, 1e-5)):
        with pytest.raises(ops.KernelError):
            call()
    assert not residual.any()
    assert gemm.linear(x[:0], weight).shape == (0, 100) and gemm.linear(quantize_rows(x[:0]), weight).shape == (0, 100)
    assert len(microscaled.add_rmsnorm(x[:0], residual[:0], ones, 1e-5)) == 0


def test_expert_refusals():
    need_gpu()
    weight = MicroscaledExperts([random_matrix(40, 100, e, DEV) for e in range(3)])
    offsets, order = torch.tensor([0, 2, 2, 4], dtype=torch.int32, device=DEV), torch.arange(4, dtype=torch.int32, device=DEV)
    x, y = rows(4, 100, 1), torch.empty(4, 40, device=DEV)

    def call(x=x, y=y, offsets=offsets, order=order, top=1, **options):
        return ops.moe_expert_product(x, weight, y, offsets, order, top, **{"x_by_pair": False, **options})
    call()
    for bad in (dict(x=rows(4, 99, 1)), dict(x=rows(3, 100, 1)), dict(y=y[:, :39]), dict(offsets=offsets[:3]), dict(offsets=offsets.long()), dict(order=order.long()), dict(top=0),
                dict(act="swiglu"), dict(act="tanh"), dict(row_scale=torch.ones(3, device=DEV)), dict(row_scale=torch.ones(4, dtype=BF16, device=DEV)),
                dict(x=quantize_rows(x)), dict(x=x.cpu()), dict(y=y.half()), dict(y=torch.empty(40, 4, device=DEV).t()), dict(x=rows(1, 100, 1), top=3, x_by_pair=True)):
        with pytest.raises(ops.KernelError):
            call(**bad)


# ------------------------------------------------------------------------------------------------ models
NVFP4 = {"quant_method": "modelopt", "quant_algo": "NVFP4"}


def _engine(folder, dtype, **options):
    from torchinferno_b200.config.engine_config import EngineConfig
    from torchinferno_b200.engine.engine import InferenceEngine
    return InferenceEngine.from_config(EngineConfig(model=str(folder), dtype=dtype, **options))


def _generate(engine, prompts, tokens):
    from torchinferno_b200.engine.types import GenerateRequest, SamplingConfig
    return [list(o.token_ids) for o in engine.generate_many([GenerateRequest(f"g{i}", prompt_token_ids=p, sampling=SamplingConfig(tokens))
                                                             for i, p in enumerate(prompts)])]


@pytest.mark.parametrize("name", ["B", "D"])
def test_a_model_in_codes(tmp_path, name):
    """In float32 the engine gives the tokens of the numbers the codes stand for; in bfloat16 every decode step is captured, gives the same tokens as
    uncaptured ones and run ahead or not, and its logits point where the float32 engine's do."""
    need_gpu()
    import numpy as np
    import plain_llama
    from conftest import TINY
    from gpu_common import requests_for
    from replay_util import InProcessReplayer, gather, trace_tail_decode
    from torchinferno_b200.weights.random_init import write_random_model
    config, seed = TINY[name]
    folder = write_random_model({**config, "quantization_config": NVFP4}, tmp_path, seed)
    cfg, stored = plain_llama.read_model_folder(folder)
    beside = {n + suffix for n in stored for suffix in ("_scale", "_scale_2") if n + "_scale_2" in stored}
    widened = {n: w if n + "_scale_2" not in stored else MicroscaledMatrix(w.to(torch.uint8), stored[n + "_scale"].to(torch.float8_e4m3fn),
                                                                           stored[n + "_scale_2"].float()).widened().double()
               for n, w in stored.items() if n not in beside}
    wanted = requests_for(config, seed, [9, 21, 3, 14])
    prompts = list(wanted.values())
    with _engine(folder, "float32", page_size=16, max_batch_size=4) as engine:
        assert _generate(engine, prompts, 8) == [plain_llama.generate_greedy(cfg, widened, p, 8) for p in prompts]
    outs = []
    for ahead in (True, False):
        with _engine(folder, "bfloat16", page_size=16, max_batch_size=4, async_scheduling=ahead) as engine:
            outs.append(_generate(engine, prompts, 12))
            assert engine.runner.counters["graph_steps"] > 0
    assert outs[0] == outs[1]
    rows_by_dtype = {}
    for dtype in ("float32", "bfloat16"):
        steps, index = trace_tail_decode(wanted, 3)
        rows_by_dtype[dtype] = gather(InProcessReplayer(folder, dtype, 512).run(steps), index)
    # A number of a row is off by at most half the distance of two codes, which is a quarter of the lower one or less from 1 on: by 0.25 / sqrt(3) / 1.5 = 0.1 of it in the mean
    # (the lower ends of the codes' intervals are off most), and so is a product.  A layer adds what four products behind one another make: gate, up and down
    # 0.1 sqrt(3) x 1.5 (the activation's slope) = 0.26, projections in and out of attention 0.14 twice over for the softmax = 0.28; three layers:
    # 0.38 sqrt(3) = 0.66 of the logits at the most, a cosine of 1 - 0.66^2 / 2 = 0.78.
    pairs = [tuple(np.asarray(rows_by_dtype[d][k][0], dtype=np.float64) for d in ("float32", "bfloat16")) for k in rows_by_dtype["float32"]]
    assert len(pairs) == 4 * 4 - 1      # (one prompt is shorter than its decoded tail)
    cosines = [float((a * b).sum() / np.sqrt((a * a).sum() * (b * b).sum())) for a, b in pairs]
    assert min(cosines) >= 0.78, min(cosines)


@pytest.mark.parametrize("module, name", [("giforax_configs", "GA"), ("vofidra_configs", "VA"), ("zipedra_configs", "ZA"), ("tadalorn_configs", "TB")])
def test_designs_with_experts_in_codes(tmp_path, module, name):
    """Their experts are bound in codes and a random model generates: prompts in portions beside decode steps, the same tokens twice."""
    need_gpu()
    import importlib
    from torchinferno_b200.weights.random_init import write_random_model
    config, seed = importlib.import_module(module).CONFIGS[name]
    folder = write_random_model({**config, "quantization_config": NVFP4}, tmp_path, seed)
    g = torch.Generator().manual_seed(seed)
    prompts = [torch.randint(0, config["vocab"], (n,), generator=g).tolist() for n in (11, 30, 2)]
    outs = []
    for _ in range(2):
        with _engine(folder, "bfloat16", page_size=16, max_batch_size=4, prefill_chunk_size=16) as engine:
            assert any(type(getattr(b.feed_forward, "up_weight", None)).__name__ == "MicroscaledExperts" for b in engine.runner.model.blocks
                       if getattr(b, "feed_forward", None) is not None)
            outs.append(_generate(engine, prompts, 6))
    assert outs[0] == outs[1] and all(len(o) == 6 for o in outs[0])


def test_a_layer_reads_its_norms_rows_in_8_bits_as_before(tmp_path, monkeypatch):
    """A model in 8-bit blocks: the same tokens whether its norms leave codes or its products make them."""
    need_gpu()
    from conftest import TINY
    from torchinferno_b200.parts import attention, mlp
    from torchinferno_b200.weights.random_init import write_random_model
    config, seed = TINY["B"]
    folder = write_random_model({**config, "quantization_config": {"quant_method": "fp8", "weight_block_size": [128, 128]}}, tmp_path, seed)
    g = torch.Generator().manual_seed(seed)
    prompts = [torch.randint(0, config["vocab_size"], (n,), generator=g).tolist() for n in (11, 30, 200)]
    outs = []
    for fused in (True, False):
        if not fused:
            for module in (attention, mlp):
                monkeypatch.setattr(module, "rows_form", lambda weight, count: None)
        with _engine(folder, "bfloat16", page_size=16, max_batch_size=4) as engine:
            outs.append(_generate(engine, prompts, 8))
    assert outs[0] == outs[1]


@pytest.mark.parametrize("form", [NVFP4, {"quant_method": "fp8", "weight_block_size": [128, 128]}])
def test_kernels_let_in_early_change_nothing(form):
    """Prompts in portions and captured decode steps give the same tokens whether a kernel is placed while the one ahead of it is at work or not."""
    need_gpu()
    from conftest import TINY_D
    from torchinferno_b200.engine.batch import StepEntry
    from torchinferno_b200.engine.factory import make_runner, random_model
    config = {**TINY_D, "quantization_config": form}
    outs = []
    with torch.inference_mode():
        model = random_model(config, seed=0, dtype="bfloat16")
        prompts = torch.randint(0, config["vocab_size"], (12, 90), generator=torch.Generator().manual_seed(1)).tolist()
        for early in (True, False):
            before = ops.set_dependent_launch(early)
            try:
                runner = make_runner(model, page_size=16, max_tokens=12 * 320, max_requests=12, max_request_tokens=300)
                ids = [f"r{i}" for i in range(12)]
                for at in (0, 40):
                    logits = runner.step([StepEntry(i, p[at:at + 50 if at else 40], [49] if at else []) for i, p in zip(ids, prompts)])
                first = logits.argmax(1).tolist()
                outs.append((first, runner.decode_loop(ids, first, 150, temperature=[0.0] * 12, seeds=list(range(12))).cpu().clone()))
                runner.end(ids)
            finally:
                ops.set_dependent_launch(before)
    assert outs[0][0] == outs[1][0] and torch.equal(outs[0][1], outs[1][1])
