"""Products of 8-bit block-scaled weights on the GPU against the definition in 64 bits (tests/block_scaled_oracle.py)."""
import pytest
import torch

from block_scaled_oracle import EXPERT_PATHS, GATED_PATHS, PLAIN_PATHS, act64, check, gated64, matrix64, product64, product_of_known64, random_matrix, requantised64, rows64, widened_rows64
from gpu_common import need_gpu
from torchinferno_b200.kernels import gemm, ops
from torchinferno_b200.kernels.block_scaled import BlockScaledExperts, BlockScaledMatrix, BlockScaledWeight, quantize_rows

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def rows(m, k, seed, dtype=BF16, spread=2.0):
    g = torch.Generator().manual_seed(1000 + seed)
    x = torch.randn(m, k, generator=g) * (spread * torch.randn(m, 1, generator=g)).exp() * (torch.randn(1, k, generator=g)).exp()
    return x.to(dtype).to(DEV)


def error_word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------------ rows to codes
def same_codes(x):
    codes, scales = quantize_rows(x)
    want_codes, want_scales = rows64(x)
    assert codes.shape == x.shape and scales.shape == want_scales.shape and codes.dtype == torch.float8_e4m3fn
    assert torch.equal(scales.double().nan_to_num(-1.0), want_scales.nan_to_num(-1.0))
    assert torch.equal(codes.double().nan_to_num(-1e9), want_codes.nan_to_num(-1e9))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m, k", [(1, 1), (1, 128), (3, 16), (8, 4096), (9, 129), (17, 127), (64, 520), (130, 1000), (5, 2055), (33, 15)])
def test_rows_become_codes(m, k, dtype):
    need_gpu()
    same_codes(rows(m, k, m + k, dtype))


def test_every_bf16_value_beside_every_border():
    """All finite bf16 numbers of a sign change pattern, run after run of one size: scales over the whole range of exponents, borders of
    448 * 2^p included."""
    need_gpu()
    bits = torch.arange(0x7f80, dtype=torch.int32)
    x = (bits << 16).view(F32)[:0x7f80 // 128 * 128].view(-1, 128)
    x = x * torch.where(torch.arange(128) % 3 == 0, -1.0, 1.0)
    same_codes(x.to(BF16).to(DEV))
    edges = torch.stack([torch.full((128,), 448.0 * 2.0 ** p) for p in range(-130, 119)])
    for factor in (1.0, 1 + 2.0 ** -7, 1 - 2.0 ** -8):
        same_codes((edges * factor).to(BF16).to(DEV))
    same_codes((edges * (1 + 2.0 ** -23)).to(DEV))


def test_rows_of_any_stride_and_alignment():
    need_gpu()
    wide = rows(20, 1500, 3)
    same_codes(wide[:, 8:8 + 600])
    same_codes(wide[:, 3:3 + 601])
    same_codes(wide[::3, 1:130])
    same_codes(rows(40, 777, 4, F32)[1::2, 5:5 + 300])
    one = rows(1, 300, 5).expand(6, 300)
    same_codes(one)


def test_runs_that_are_empty_or_not_finite():
    need_gpu()
    x = rows(6, 400, 7, F32)
    x[0] = 0
    x[1, 130] = float("inf")
    x[2, 5] = float("nan")
    x[3, 399] = -float("inf")
    x[4] = 1e-42                    # subnormal numbers
    x[5, :128] = 3e38
    same_codes(x)
    same_codes(x[:4].to(BF16))
    assert quantize_rows(x[:0])[0].shape == (0, 400)


# ------------------------------------------------------------------------------------------------ one matrix
SIZES = [(1, 1, 1), (1, 128, 128), (1, 4096, 512), (2, 129, 130), (7, 256, 127), (8, 1000, 1302), (15, 300, 257), (16, 2048, 384), (17, 640, 129),
         (32, 384, 2), (33, 127, 640), (47, 1152, 200), (63, 512, 1000), (64, 4096, 256), (65, 200, 129), (96, 1024, 512), (127, 400, 300), (128, 128, 128),
         (129, 2304, 136), (200, 512, 2560), (255, 1000, 258), (256, 256, 512), (257, 384, 770), (333, 1000, 1302), (520, 2048, 1280), (1030, 640, 390)]


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("m, k, n", SIZES)
def test_linear(m, k, n, out_dtype):
    need_gpu()
    matrix, x, word = random_matrix(n, k, m + n, DEV), rows(m, k, m), error_word()
    gemm.set_error_word(word)
    try:
        got = gemm.linear(x, BlockScaledWeight(matrix), out_dtype=out_dtype)
    finally:
        gemm.set_error_word(None)
    check(got, product64(x, matrix), out_dtype)
    assert int(word) == 0


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("m, k, n", [(1, 128, 1), (1, 4096, 1024), (3, 200, 130), (8, 1024, 257), (16, 2048, 640), (31, 500, 64), (64, 1024, 129), (65, 384, 130),
                                     (130, 1000, 300), (256, 512, 256), (300, 2048, 513), (700, 256, 1000)])
def test_linear_swiglu(m, k, n, out_dtype):
    need_gpu()
    gate, up = random_matrix(n, k, 1, DEV, (0.005, 0.2)), random_matrix(n, k, 2, DEV, (0.005, 0.2))
    x, weight = rows(m, k, m, spread=0.5), BlockScaledWeight(gate, up, epilogue="swiglu")
    check(gemm.linear_swiglu(x, weight, out_dtype=out_dtype), gated64(product64(x, gate), product64(x, up)), out_dtype)
    # (and without the activation: the two products side by side, row pairs)
    both = gemm.linear(x, weight, out_dtype=F32)
    for part, matrix in ((0, gate), (1, up)):
        check(both[:, part::2].contiguous(), product64(x, matrix), F32)


@pytest.mark.parametrize("m", [1, 20, 90, 300])
def test_32_bit_rows(m):
    need_gpu()
    matrix, x = random_matrix(260, 520, 5, DEV), rows(m, 520, m, F32)
    check(gemm.linear(x, BlockScaledWeight(matrix)), product64(x, matrix), F32)
    check(gemm.linear(x, BlockScaledWeight(matrix), out_dtype=BF16), product64(x, matrix), BF16)


@pytest.mark.parametrize("m", [1, 5, 64, 65, 140, 600])
def test_several_matrices_side_by_side(m):
    """Those whose rows end inside a block among them; into a slice of wider rows, whose other columns stay as they are."""
    need_gpu()
    parts = [random_matrix(n, 333, n, DEV) for n in (256, 130, 64, 1, 200)]
    weight, x = BlockScaledWeight(*parts), rows(m, 333, m)
    total = sum(p.shape[0] for p in parts)
    wide = torch.full((m, total + 7), 5.0, dtype=BF16, device=DEV)
    got = gemm.linear(x, weight, out=wide[:, 3:3 + total])
    assert got.data_ptr() == wide[:, 3:].data_ptr() and (wide[:, :3] == 5).all() and (wide[:, 3 + total:] == 5).all()
    want, bound = (torch.cat(t, 1) for t in zip(*(product64(x, p) for p in parts)))
    check(got, (want, bound), BF16)
    check(gemm.linear(x, weight.rows(128, 400)), (want[:, 128:400], bound[:, 128:400]), BF16)


@pytest.mark.parametrize("m", [4, 70, 300])
def test_strided_and_unaligned_rows(m):
    need_gpu()
    matrix, wide = random_matrix(200, 301, 5, DEV), rows(2 * m, 1000, m)
    for x in (wide[:m, 8:309], wide[:m, 3:304], wide[::2, 1:302], wide[:1, 16:317].expand(m, 301)):
        check(gemm.linear(x, BlockScaledWeight(matrix)), product64(x, matrix), BF16)


@pytest.mark.parametrize("m", [3, 64, 100, 400])
def test_rows_of_zeros_and_not_finite(m):
    """Rows of zeros give zeros; an infinity or a NaN makes its own row NaN and no other; NaN codes and scales their own features."""
    need_gpu()
    matrix, x = random_matrix(150, 300, 9, DEV), rows(m, 300, 1)
    x[0] = 0
    weight = BlockScaledWeight(matrix)
    clean = gemm.linear(x, weight)
    assert not clean[0].any()
    x[1, 290], x[2, 0] = float("inf"), float("nan")
    got = gemm.linear(x, weight)
    assert got[1:3].isnan().all() and torch.equal(got[3:], clean[3:]) and torch.equal(got[0], clean[0])
    codes, scales = matrix.codes.clone(), matrix.scales.clone()
    codes.view(torch.uint8)[7, 11] = 0x7f
    scales[1, 0] = float("nan")
    got = gemm.linear(x[3:] if m > 3 else x[:1], BlockScaledWeight(BlockScaledMatrix(codes, scales)))
    assert got[:, 7].isnan().all() and got[:, 128:].isnan().all() and not got[:, :7].isnan().any() and not got[:, 8:128].isnan().any()


@pytest.mark.parametrize("m", [2, 66, 260])
def test_sizes_at_the_ends_of_the_range(m):
    need_gpu()
    matrix = random_matrix(140, 256, 3, DEV, (1.0, 1.0))
    for size in (2.0 ** -100, 2.0 ** 90):
        x = (rows(m, 256, 1, F32, 0.1) * size).to(BF16)
        got, (want, bound) = gemm.linear(x, BlockScaledWeight(matrix), out_dtype=F32), product64(x, matrix)
        check(got / size, (want / size, bound / size), F32)


# ------------------------------------------------------------------------------------------------ scales whose product no 32-bit number holds
def far_rows(m, k, seed):
    """32-bit rows whose runs are of sizes from 2^-140 to 2^118, every run of a size of its own."""
    g = torch.Generator().manual_seed(seed)
    sizes = torch.tensor([-140.0, -118.0, -100.0, -60.0, 0.0, 60.0, 100.0, 118.0], dtype=torch.float64)
    power = sizes[torch.randint(0, len(sizes), (m, -(-k // 128)), generator=g)].repeat_interleave(128, 1)[:, :k]
    return (torch.randn(m, k, generator=g, dtype=torch.float64).clamp(-200, 200) * 2.0 ** power).to(F32).to(DEV)


def far_matrix(n, k, seed):
    """Scales over the whole range of 32-bit numbers, subnormal ones, zeros and either sign among them; some features are zeros."""
    matrix = random_matrix(n, k, seed)
    g = torch.Generator().manual_seed(seed)
    sizes = torch.tensor([0.0, 2.0 ** -149, 2.0 ** -130, 1.3 * 2.0 ** -100, -1.37 * 2.0 ** -10, 1.7, 1.1 * 2.0 ** 8, -2.0 ** 30, 1.9 * 2.0 ** 100, 2.0 ** 127], dtype=torch.float64)
    codes = matrix.codes.clone()
    codes.view(torch.uint8)[3::130] = 0
    return BlockScaledMatrix(codes, sizes[torch.randint(0, len(sizes), tuple(matrix.scales.shape), generator=g)].to(F32)).to(DEV)


def check_far(got, x, matrix):
    """Where no partial sum leaves the range.  A subnormal sum or share of one is a multiple of 2^-149: half of that more for every run, and for the last rounding."""
    want, bound = product64(x, matrix)
    size = widened_rows64(x).abs() @ matrix64(matrix).abs().t()
    kept = size < 2.0 ** 126
    assert kept.double().mean() > 0.3 and got.dtype == F32
    off = (got.double() - want).abs()
    bad = kept & ~(off <= bound + 2.0 ** -149 * (x.shape[1] / 128 + 2))
    assert not bad.any(), f"{int(bad.sum())} of {int(kept.sum())} off, {int((bad & got.isnan()).sum())} NaN, {int((bad & (got == 0)).sum())} zeros"


# (the kernel's own codes; tiles of 32, 64 and 128 rows; pairs of SMs)
FAR = [(5, 9600), (20, 9600), (60, 9600), (100, 9600), (200, 9600), (5, 300)]


@pytest.mark.parametrize("m, n", FAR)
def test_scales_whose_product_leaves_the_range(m, n):
    need_gpu()
    x, matrix = far_rows(m, 300, m), far_matrix(n, 300, 7)
    check_far(gemm.linear(x, BlockScaledWeight(matrix)), x, matrix)


@pytest.mark.parametrize("m, n", FAR)
def test_scales_of_gate_and_up_whose_product_leaves_the_range(m, n):
    need_gpu()
    x, gate, up = far_rows(m, 300, m), far_matrix(n // 2, 300, 8), far_matrix(n // 2, 300, 9)
    both = gemm.linear(x, BlockScaledWeight(gate, up, epilogue="swiglu"))
    check_far(both[:, 0::2].contiguous(), x, gate)
    check_far(both[:, 1::2].contiguous(), x, up)


@pytest.mark.parametrize("pairs", [6, 100, 500])
def test_scales_of_experts_whose_product_leaves_the_range(pairs):
    need_gpu()
    matrices, x = [far_matrix(300, 300, e) for e in range(4)], far_rows(pairs, 300, pairs)
    offsets, order, ids = routing(pairs, 1, 4, 1)
    y = torch.empty(pairs, 300, dtype=F32, device=DEV)
    ops.moe_expert_product(x, BlockScaledExperts(matrices), y, offsets, order, 1, x_by_pair=True)
    ends = offsets.tolist()
    for e in range(4):
        at = order[ends[e]:ends[e + 1]].long()
        if len(at):
            check_far(y[ends[e]:ends[e + 1]], x[at], matrices[e])


@pytest.mark.parametrize("m, n", FAR)
def test_small_gates_and_large_ups(m, n):
    """Gates of about 2^-120 whose scales' product is below the range, ups of about 2^30: the unit is far inside of it."""
    need_gpu()
    x = (rows(m, 300, m, F32, 0.1) * 2.0 ** -100).contiguous()
    gate, up = random_matrix(n // 2, 300, 1, DEV, (60 * 2.0 ** -31, 60 * 2.0 ** -30)), random_matrix(n // 2, 300, 2, DEV, (60 * 2.0 ** 119, 60 * 2.0 ** 120))
    got = gemm.linear_swiglu(x, BlockScaledWeight(gate, up, epilogue="swiglu"))
    # (a sum of subnormal size is a multiple of 2^-149 as well; its share in the bound: 2^-147 times the other factor)
    (g, eg), (u, eu) = product64(x, gate), product64(x, up)
    want, bound = gated64((g, eg + 2.0 ** -147), (u, eu))
    check(got, (want, bound), F32)
    assert want.abs().median() > 2.0 ** -105


@pytest.mark.parametrize("act", ["none", "relu2", "silu", "gelu", "swiglu", "glu_clamp"])
@pytest.mark.parametrize("pairs, out_dtype", [(6, F32), (100, F32), (500, F32), (6, BF16), (500, BF16)])
def test_activations_of_sums_with_far_scales(pairs, out_dtype, act):
    need_gpu()
    n = 130
    stacks = [[random_matrix(n, 300, e, DEV, (60 * 2.0 ** -31, 60 * 2.0 ** -30)) for e in range(3)]]
    if act in ops.MOE_GATED:
        stacks.append([random_matrix(n, 300, 10 + e, DEV, (60 * 2.0 ** 99, 60 * 2.0 ** 100)) for e in range(3)])
    x = (rows(pairs, 300, pairs, F32, 0.1) * 2.0 ** -100).contiguous()
    offsets, order, _ = routing(pairs, 1, 3, 1)
    scale = torch.rand(pairs, generator=torch.Generator().manual_seed(1)).to(DEV) + 0.5
    y = torch.empty(pairs, n, dtype=out_dtype, device=DEV)
    ops.moe_expert_product(x, BlockScaledExperts(*stacks), y, offsets, order, 1, x_by_pair=True, act=act, limit=2.0, alpha=1.702, row_scale=scale)
    ends = offsets.tolist()
    for e in range(3):
        at = order[ends[e]:ends[e + 1]].long()
        if len(at) == 0:
            continue
        s = scale[at].double()[:, None]
        sums = [product64(x[at], stack[e]) for stack in stacks]
        sums = [(v * s, b * s + 2.0 ** -23 * (v * s).abs() + 2.0 ** -147) for v, b in sums]
        want, bound = gated64(*sums, act=act, limit=2.0) if act in ops.MOE_GATED else act64(sums[0], act)
        check(y[ends[e]:ends[e + 1]], (want, bound + 2.0 ** -133), out_dtype)


@pytest.mark.parametrize("m, n", FAR)
def test_a_row_does_not_depend_on_others_of_far_sizes(m, n):
    """The same bits beside rows whose scales' product leaves the range."""
    need_gpu()
    weight, x = BlockScaledWeight(random_matrix(n, 300, 3, DEV, (1e-3, 1e-2))), rows(m, 300, 2, F32)
    before = gemm.linear(x, weight)
    x[1::3] = far_rows(m, 300, 5)[1::3]
    after = gemm.linear(x, weight)
    for at in (slice(0, None, 3), slice(2, None, 3)):
        assert torch.equal(before[at], after[at])


def test_no_rows():
    need_gpu()
    weight = BlockScaledWeight(random_matrix(100, 200, 1, DEV))
    assert gemm.linear(rows(0, 200, 1), weight).shape == (0, 100)


def test_refusals():
    need_gpu()
    weight, x = BlockScaledWeight(random_matrix(100, 200, 1, DEV)), rows(4, 200, 1)
    gated = BlockScaledWeight(random_matrix(100, 200, 1, DEV), random_matrix(100, 200, 2, DEV), epilogue="swiglu")
    for call in (lambda: gemm.linear(x[:, :199], weight), lambda: gemm.linear(x.half(), weight), lambda: gemm.linear(x, weight, out_dtype=torch.float16),
                 lambda: gemm.linear(x.t().contiguous().t(), weight), lambda: gemm.linear(x[0], weight), lambda: gemm.linear_swiglu(x, weight),
                 lambda: gemm.linear(x, weight, out=torch.empty(4, 99, dtype=BF16, device=DEV)), lambda: gemm.linear_swiglu(x.cpu(), gated),
                 lambda: gemm.linear(x, weight, out=torch.empty(100, 4, dtype=BF16, device=DEV).t()),
                 lambda: gemm.linear(x, BlockScaledWeight(random_matrix(100, 200, 1)))):
        with pytest.raises(ops.KernelError):
            call()


@pytest.mark.parametrize("m", [1, 8, 64, 100, 300])
def test_a_row_does_not_depend_on_the_others(m):
    """In a step of the same kernel: the same bits wherever a row stands, and from call to call."""
    need_gpu()
    weight, x = BlockScaledWeight(random_matrix(390, 1100, 3, DEV)), rows(m, 1100, 2)
    first = gemm.linear(x, weight)
    assert torch.equal(first, gemm.linear(x, weight))
    turned = torch.roll(x, 1, 0)
    assert torch.equal(torch.roll(first, 1, 0), gemm.linear(turned, weight))


@pytest.mark.parametrize("m", [3, 100, 300])
def test_captured_and_on_two_streams(m):
    need_gpu()
    gate, up, down = random_matrix(260, 400, 1, DEV, (0.01, 0.1)), random_matrix(260, 400, 2, DEV, (0.01, 0.1)), random_matrix(400, 260, 3, DEV)
    w1, w2 = BlockScaledWeight(gate, up, epilogue="swiglu"), BlockScaledWeight(down)
    inputs = [rows(m, 400, i) for i in range(4)]

    def pass_of(x):
        return gemm.linear(gemm.linear_swiglu(x, w1), w2)
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
            assert torch.equal(statics[i][1], want[(turn + i) % 4])
    outs = []
    for turn in range(6):
        with torch.cuda.stream(streams[turn % 2]):
            outs.append(pass_of(inputs[turn % 4]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[turn % 4]) for turn, y in enumerate(outs))


# ------------------------------------------------------------------------------------------------ every way through the kernels
def device_matrix(n, k, seed, size=1.0):
    """A large matrix, made on the device: codes of all sizes, scales up to ``size`` / 60."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = (torch.randn(n, k, generator=g, device=DEV) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    scales = (torch.rand(-(-n // 128), -(-k // 128), generator=g, device=DEV) + 0.02) * (size / 60)
    return BlockScaledMatrix(codes, scales)


def in_both_types(call, want):
    """``call(out type, error word)`` in 32 bits and in bf16, within the bound, with no wait run out, and the same bits again."""
    for dtype in (F32, BF16):
        word = error_word()
        got = call(dtype, word)
        check(got, want, dtype)
        assert torch.equal(got, call(dtype, word)) and int(word) == 0


@pytest.mark.parametrize("m, k, n", [sizes[:3] for sizes in PLAIN_PATHS])
def test_every_way_of_a_product(m, k, n):
    need_gpu()
    matrix, x = device_matrix(n, k, 1), rows(m, k, m)
    weight = BlockScaledWeight(matrix)
    in_both_types(lambda dtype, word: weight.product(x, out_dtype=dtype, error_word=word), product64(x, matrix))


@pytest.mark.parametrize("m, k, n", [sizes[:3] for sizes in GATED_PATHS])
def test_every_way_of_a_gated_product(m, k, n):
    need_gpu()
    gate, up = (device_matrix(n // 2, k, seed, (128 / k) ** 0.5 / 10) for seed in (1, 2))
    x, weight = rows(m, k, m, spread=0.5), BlockScaledWeight(gate, up, epilogue="swiglu")
    in_both_types(lambda dtype, word: weight.swiglu(x, out_dtype=dtype, error_word=word), gated64(product64(x, gate), product64(x, up)))


@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("pairs, count, k, n", [sizes[:4] for sizes in EXPERT_PATHS])
def test_every_way_of_experts(pairs, count, k, n, act):
    need_gpu()
    n = n // 2 if act == "swiglu" else n          # (features of either matrix)
    stacks = [[device_matrix(n, k, 100 * part + e, (128 / k) ** 0.5 / 10) for e in range(min(count, 4))] for part in range(2 if act == "swiglu" else 1)]
    offsets, order, ids = routing(pairs, 1, count, 3, empty=(1,))
    x, weight = rows(pairs, k, 5, spread=0.5), BlockScaledExperts(*([s[e % len(s)] for e in range(count)] for s in stacks))
    kind = ids.to(DEV)[order.long()] % len(stacks[0])
    want = [torch.empty(pairs, n, dtype=torch.float64, device=DEV) for _ in range(2)]
    for i in range(len(stacks[0])):
        at = (kind == i).nonzero()[:, 0]
        sums = [product64(x[order[at].long()], s[i]) for s in stacks]
        for to, part in zip(want, gated64(*sums) if act == "swiglu" else sums[0]):
            to[at] = part
    in_both_types(lambda dtype, word: ops.moe_expert_product(x, weight, torch.empty(pairs, n, dtype=dtype, device=DEV), offsets, order, 1, x_by_pair=True,
                                                             act=act, error_word=word), tuple(want))


# ------------------------------------------------------------------------------------------------ rows sorted by expert
def routing(tokens, top, experts, seed, empty=(), absent=0):
    """offsets, order, and ids of pairs sorted by expert; experts in ``empty`` get none; ``absent`` pairs at the end have no expert at all."""
    g = torch.Generator().manual_seed(seed)
    allowed = [e for e in range(experts) if e not in empty]
    ids = torch.tensor([allowed[i] for i in torch.randint(0, len(allowed), (tokens * top,), generator=g).tolist()])
    if absent:
        ids[torch.randperm(len(ids), generator=g)[:absent]] = experts
    order = torch.sort(ids, stable=True).indices.to(torch.int32)
    counts = torch.bincount(ids, minlength=experts + 1)[:experts]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    return offsets.to(DEV), order.to(DEV), ids


@pytest.mark.parametrize("act", ["none", "relu2", "silu", "gelu", "swiglu", "glu_clamp"])
@pytest.mark.parametrize("by_pair", [True, False])
@pytest.mark.parametrize("tokens, top, experts, k, n, out_dtype", [
    (1, 1, 1, 128, 128, F32), (1, 4, 8, 256, 96, BF16), (8, 4, 32, 1024, 256, BF16), (5, 3, 7, 200, 130, F32), (40, 2, 6, 640, 129, BF16),
    (100, 3, 5, 300, 200, F32), (150, 4, 4, 512, 256, BF16), (700, 2, 3, 200, 140, BF16), (64, 1, 300, 128, 64, F32)])
def test_expert_products(tokens, top, experts, k, n, out_dtype, by_pair, act):
    need_gpu()
    gated = act in ops.MOE_GATED
    sizes = (0.005, 0.2) if act != "none" else (0.02, 3.0)
    stacks = [[random_matrix(n, k, 100 * part + e, DEV, sizes) for e in range(min(experts, 6))] for part in range(2 if gated else 1)]
    stacks = [[stack[e % len(stack)] for e in range(experts)] for stack in stacks]
    empty = (0, experts - 1) if experts > 3 else ()
    pairs, absent = tokens * top, tokens if tokens * top > 8 else 0
    offsets, order, ids = routing(tokens, top, experts, tokens, empty, absent)
    x = rows(tokens if by_pair else pairs, k, tokens, spread=0.5)
    scale = torch.rand(pairs, generator=torch.Generator().manual_seed(1)).to(DEV) + 0.5 if act in ("glu_clamp", "none") else None
    y = torch.full((pairs, n), 9.0, dtype=out_dtype, device=DEV)
    word = error_word()
    assert ops.moe_expert_product(x, BlockScaledExperts(*stacks), y, offsets, order, top, x_by_pair=by_pair, act=act, limit=2.0, alpha=1.702,
                                  row_scale=scale, error_word=word) is y
    assert int(word) == 0
    ends = offsets.tolist()
    assert (y[ends[-1]:] == 9).all()                                 # (rows behind the last expert's: left as they were)
    for e in range(experts):
        at = torch.arange(ends[e], ends[e + 1], device=DEV)
        if len(at) == 0:
            continue
        source = order[at].long() // top if by_pair else at
        sums = [product64(x[source], stack[e]) for stack in stacks]
        if scale is not None:
            s = scale[order[at].long()].double()[:, None]
            sums = [(v * s, b * s + 2.0 ** -23 * (v * s).abs()) for v, b in sums]
        want = gated64(*sums, act=act, limit=2.0) if gated else act64(sums[0], act)
        check(y[at], want, out_dtype, f"expert {e}")


@pytest.mark.parametrize("experts, tokens, act", [(300, 40000, "none"), (300, 40000, "swiglu"), (200, 25000, "relu2"), (1024, 3000, "none")])
def test_many_experts(experts, tokens, act):
    """More than the pairs of SMs take, about as many, and the most; matrices repeat, so that the oracle is one product a matrix."""
    need_gpu()
    gated = act in ops.MOE_GATED
    stacks = [[random_matrix(60, 130, 100 * part + e, DEV, (0.005, 0.2)) for e in range(4)] for part in range(2 if gated else 1)]
    offsets, order, ids = routing(tokens, 1, experts, 3, empty=(1, experts - 1))
    x = rows(tokens, 130, 5, spread=0.5)
    y = torch.empty(tokens, 60, dtype=F32, device=DEV)
    word = error_word()
    ops.moe_expert_product(x, BlockScaledExperts(*([s[e % 4] for e in range(experts)] for s in stacks)), y, offsets, order, 1, x_by_pair=True, act=act,
                           error_word=word)
    assert int(word) == 0
    kind = ids.to(DEV)[order.long()] % 4
    for i in range(4):
        at = (kind == i).nonzero()[:, 0]
        sums = [product64(x[order[at].long()], s[i]) for s in stacks]
        check(y[at], gated64(*sums, act=act) if gated else act64(sums[0], act), F32)
    with pytest.raises(ops.KernelError):
        ops.moe_expert_product(x[:1], BlockScaledExperts([stacks[0][0]] * 1025), y[:1], torch.zeros(1026, dtype=torch.int32, device=DEV),
                               torch.zeros(1, dtype=torch.int32, device=DEV), 1, x_by_pair=True)


@pytest.mark.parametrize("act", ["none", "relu2", "silu", "gelu", "swiglu", "glu_clamp"])
@pytest.mark.parametrize("tokens", [4, 60, 400])
def test_rows_that_are_not_finite_show_through_every_activation(tokens, act):
    need_gpu()
    stacks = [[random_matrix(140, 200, 100 * part + e, DEV, (0.005, 0.2)) for e in range(2)] for part in range(2 if act in ops.MOE_GATED else 1)]
    offsets, order, _ = routing(tokens, 1, 2, tokens)
    x = rows(tokens, 200, tokens, spread=0.5)
    x[1, 7], x[2, 150] = float("nan"), float("inf")
    y = torch.empty(tokens, 140, dtype=BF16, device=DEV)
    ops.moe_expert_product(x, BlockScaledExperts(*stacks), y, offsets, order, 1, x_by_pair=True, act=act, limit=2.0, alpha=1.702)
    bad = ((order == 1) | (order == 2))
    assert y[bad].isnan().all() and not y[~bad].isnan().any()


def test_matrices_of_any_stride():
    need_gpu()
    wide = random_matrix(256, 512, 3, DEV)
    part = BlockScaledMatrix(wide.codes[:, 128:384], wide.scales[:, 1:3])
    turned = BlockScaledMatrix(wide.codes.view(torch.uint8)[:, :256].t().view(torch.float8_e4m3fn), wide.scales[:, :2].t())
    x = rows(5, 256, 1)
    for matrix in (part, turned):
        check(gemm.linear(x, BlockScaledWeight(matrix)), product64(x, matrix), BF16)


def test_expert_refusals():
    need_gpu()
    experts = BlockScaledExperts([random_matrix(64, 100, i, DEV) for i in range(4)])
    offsets, order, _ = routing(6, 2, 4, 0)
    x, y = rows(6, 100, 0), torch.empty(12, 64, dtype=BF16, device=DEV)
    good = dict(x_by_pair=True)
    ops.moe_expert_product(x, experts, y, offsets, order, 2, **good)
    for call in (lambda: ops.moe_expert_product(x, experts, y, offsets, order, 2, x_by_pair=False),               # rows by pair, not by token
                 lambda: ops.moe_expert_product(x, experts, y, offsets, order, 2, act="swiglu", **good),          # no gate rows
                 lambda: ops.moe_expert_product(x, experts, y, offsets, order, 2, act="tanh", **good),
                 lambda: ops.moe_expert_product(x, experts, y, offsets, order, 1, **good),                        # more sources than rows
                 lambda: ops.moe_expert_product(x, experts, y, offsets, order, 0, **good),
                 lambda: ops.moe_expert_product(x[:, :99], experts, y, offsets, order, 2, **good),
                 lambda: ops.moe_expert_product(x, experts, y[:11], offsets, order, 2, **good),
                 lambda: ops.moe_expert_product(x, experts, y, offsets[:4], order, 2, **good),
                 lambda: ops.moe_expert_product(x, experts, y, offsets, order.long(), 2, **good),
                 lambda: ops.moe_expert_product(x, experts, y, offsets.cpu(), order, 2, **good),
                 lambda: ops.moe_expert_product(x, experts, y, offsets, order, 2, row_scale=torch.ones(5, device=DEV), **good)):
        with pytest.raises(ops.KernelError):
            call()


def test_the_definition_by_itself():
    """The oracle's rows and matrices are what the tensors stand for (torch's own widening of e4m3)."""
    need_gpu()
    m, x = random_matrix(130, 200, 0, DEV), rows(9, 200, 1)
    assert torch.equal(m.widened(torch.float32).double(), matrix64(m).float().double())
    codes, scales = quantize_rows(x)
    assert torch.equal(widened_rows64(x), codes.double() * scales.double().repeat_interleave(128, 1)[:, :200])


# ------------------------------------------------------------------------------------------------ as the engine uses them
FP8 = {"quant_method": "fp8", "weight_block_size": [128, 128]}


@pytest.mark.parametrize("tokens", [1, 8, 40, 300])
def test_a_feed_forward_in_blocks(tokens):
    """Both products behind one another; the activation between them is known up to its own rounding, and so are its codes."""
    need_gpu()
    from torchinferno_b200.parts.base import PartSpec, build_part
    hidden, inter = 320, 450
    part = build_part("feed_forward", PartSpec("swiglu", {"hidden_size": hidden, "intermediate_size": inter}), dtype=BF16, device=torch.device(DEV))
    gate, up, down = random_matrix(inter, hidden, 1, DEV, (0.005, 0.1)), random_matrix(inter, hidden, 2, DEV, (0.005, 0.1)), random_matrix(hidden, inter, 3, DEV)
    part.bind(dict(zip(part.names, (gate, up, down))))
    x = rows(tokens, hidden, tokens, spread=0.5)
    act = gated64(product64(x, gate), product64(x, up))
    check(part.forward(x, None), product_of_known64(requantised64(act), down), BF16)


@pytest.mark.parametrize("activation, on_input", [("relu2", False), ("swiglu", False), ("glu_clamp", True), ("gelu", False)])
@pytest.mark.parametrize("tokens", [1, 7, 90, 400])
def test_routed_experts_in_blocks(tokens, activation, on_input):
    need_gpu()
    from torchinferno_b200.parts.base import PartSpec, build_part
    hidden, inter, experts, top, limit = 200, 140, 6, 2, 2.0
    part = build_part("feed_forward", PartSpec("routed_experts", {
        "hidden_size": hidden, "experts": experts, "top": top, "expert_size": inter, "activation": activation, "weight_on_input": on_input,
        "limit": limit}), dtype=BF16, device=torch.device(DEV))
    weights = {spec.name: random_matrix(*spec.shape, i, DEV, (0.005, 0.15) if spec.shape[0] == inter else (0.02, 3.0)) if spec.block_scaled else
               torch.randn(spec.shape, generator=torch.Generator().manual_seed(i)).to(DEV) * 0.1 for i, spec in enumerate(part.weight_specs())}
    part.bind(weights)
    x = rows(tokens, hidden, tokens, spread=0.5)
    logits = torch.empty(tokens, experts, device=DEV)
    ops.router_logits(x, part.router_weight, logits)
    ids, shares = torch.empty(tokens, top, dtype=torch.int32, device=DEV), torch.empty(tokens, top, device=DEV)
    ops.moe_route(logits, experts, top, ids, shares, normalize=True)
    want, bound = torch.zeros(tokens, hidden, dtype=torch.float64, device=DEV), torch.zeros(tokens, hidden, dtype=torch.float64, device=DEV)
    for e in range(experts):
        at, choice = (ids == e).nonzero(as_tuple=True)
        if len(at) == 0:
            continue
        share = shares[at, choice].double()[:, None]
        sums = [product64(x[at], weights[f"e{e}.{n}"]) for n in (("gate", "up") if part.glu else ("up",))]
        if on_input:
            sums = [(v * share, b * share + 2.0 ** -23 * (v * share).abs()) for v, b in sums]
        act = gated64(*sums, act=activation, limit=limit) if part.glu else act64(sums[0], activation)
        y, b = product_of_known64(requantised64(act), weights[f"e{e}.down"])
        share = torch.ones_like(share) if on_input else share
        want[at] += share * y
        # (the products with the shares and the sum over the choices: one rounding each)
        bound[at] += share * b + 2 * top * 2.0 ** -23 * (share * y).abs()
    check(part.forward(x, None), (want, bound), BF16)


def _blocks_folder(tmp_path, config, seed):
    from torchinferno_b200.weights.random_init import write_random_model
    return write_random_model({**config, "quantization_config": FP8}, tmp_path, seed)


def _engine(folder, dtype, **options):
    from torchinferno_b200.config.engine_config import EngineConfig
    from torchinferno_b200.engine.engine import InferenceEngine
    return InferenceEngine.from_config(EngineConfig(model=str(folder), dtype=dtype, **options))


def _generate(engine, prompts, tokens):
    from torchinferno_b200.engine.types import GenerateRequest, SamplingConfig
    return [list(o.token_ids) for o in engine.generate_many([GenerateRequest(f"g{i}", prompt_token_ids=p, sampling=SamplingConfig(tokens))
                                                             for i, p in enumerate(prompts)])]


@pytest.mark.parametrize("name", ["B", "D"])
def test_a_model_in_blocks(tmp_path, name):
    """In float32 the engine gives the tokens of the numbers the blocks stand for; in bfloat16 every decode step is captured, gives the same tokens as
    uncaptured ones and run ahead or not, and its logits point where the float32 engine's do."""
    need_gpu()
    import numpy as np
    import plain_llama
    from conftest import TINY
    from gpu_common import requests_for
    from replay_util import InProcessReplayer, gather, trace_tail_decode
    config, seed = TINY[name]
    folder = _blocks_folder(tmp_path, config, seed)
    cfg, stored = plain_llama.read_model_folder(folder)
    widened = {n: w if n + "_scale_inv" not in stored else
               w * stored[n + "_scale_inv"].repeat_interleave(128, 0)[:w.shape[0]].repeat_interleave(128, 1)[:, :w.shape[1]]
               for n, w in stored.items() if not n.endswith("_scale_inv")}
    # (the engine's float32 weights are the products of code and scale rounded to 24 bits)
    widened = {n: w.float().double() for n, w in widened.items()}
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
    # A product's terms are off by at most half a step of e4m3 (2^-4), by 2^-4 / sqrt(3) = 0.036 in the mean, and so is the product, its terms' errors
    # being independent.  A layer adds to the residual what four products behind one another make: gate, up and down 0.036 sqrt(3) x 1.5 (the
    # activation's slope) = 0.09, projections in and out of attention 0.05 twice over for the softmax = 0.1; three layers: 0.14 sqrt(3) = 0.24 of the
    # logits at the most, a cosine of 1 - 0.24^2 / 2 = 0.97.
    pairs = [tuple(np.asarray(rows_by_dtype[d][k][0], dtype=np.float64) for d in ("float32", "bfloat16")) for k in rows_by_dtype["float32"]]
    assert len(pairs) == 4 * 4 - 1      # (one prompt is shorter than its decoded tail)
    cosines = [float((a * b).sum() / np.sqrt((a * a).sum() * (b * b).sum())) for a, b in pairs]
    assert min(cosines) >= 0.97, min(cosines)


@pytest.mark.parametrize("module, name", [("giforax_configs", "GA"), ("vofidra_configs", "VA"), ("zipedra_configs", "ZA"), ("tadalorn_configs", "TB")])
def test_designs_with_experts_in_blocks(tmp_path, module, name):
    """Their experts are bound in blocks and a random model generates: prompts in portions beside decode steps, the same tokens twice."""
    need_gpu()
    import importlib
    config, seed = importlib.import_module(module).CONFIGS[name]
    folder = _blocks_folder(tmp_path, config, seed)
    vocab = config["vocab"]
    g = torch.Generator().manual_seed(seed)
    prompts = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (11, 30, 2)]
    outs = []
    for _ in range(2):
        with _engine(folder, "bfloat16", page_size=16, max_batch_size=4, prefill_chunk_size=16) as engine:
            assert any(type(getattr(b.feed_forward, "up_weight", None)).__name__ == "BlockScaledExperts" for b in engine.runner.model.blocks
                       if getattr(b, "feed_forward", None) is not None)
            outs.append(_generate(engine, prompts, 6))
    assert outs[0] == outs[1] and all(len(o) == 6 for o in outs[0])


def test_command_line_with_a_model_in_blocks(tmp_path):
    need_gpu()
    import json
    import subprocess
    import sys
    from pathlib import Path
    from conftest import TINY_D
    root = Path(__file__).resolve().parent.parent
    (tmp_path / "config.json").write_text(json.dumps({**TINY_D, "quantization_config": FP8}))
    run = [sys.executable, "-m", "torchinferno_b200"]
    subprocess.run([*run, "random-model", str(tmp_path / "config.json"), str(tmp_path / "model"), "--seed", "3"], check=True, cwd=root, timeout=300)
    out = subprocess.run([*run, "generate", str(tmp_path / "model"), "--input-ids", "1", "2", "3", "--new-tokens", "4"], check=True, cwd=root, timeout=300,
                         capture_output=True, text=True).stdout
    assert out.strip()
