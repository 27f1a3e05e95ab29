"""What can be checked on the host of 4-bit products and of how they share an SM."""
import ctypes
import random

import pytest
import torch

from microscaled_oracle import CODES, SCALES, random_matrix
from torchinferno_b200.kernels import ops
from torchinferno_b200.kernels.microscaled import MicroscaledExperts, MicroscaledMatrix, MicroscaledWeight, quantize_matrix


def room(rows, columns, features, experts=0, bits=4, codes=1):
    """{columns of tensor memory, bytes of shared memory} of a block of such a product."""
    found = (ctypes.c_int * 2)()
    at = ctypes.addressof(found)
    status = (ops.lib().tib_microscaled_room(rows, features, columns, experts, at) if bits == 4 else
              ops.lib().tib_block_scaled_tcgen05_room(codes, rows, features, columns, experts, at))
    assert status == 0, (rows, columns, features, experts, status)
    return tuple(found)


def shared(rows, columns, features, bits, codes):
    """How many blocks share a tile of such a product."""
    found = (ctypes.c_int * 4)()
    at = ctypes.addressof(found)
    status = (ops.lib().tib_microscaled_plan(rows, features, columns, 0, at) if bits == 4 else ops.lib().tib_block_scaled_plan(codes, rows, features, columns, 0, at))
    assert status == 0
    return found[1]


def test_blocks_that_fit_an_sm_together_find_their_columns():
    """512 columns and 228 KB an SM, 1 KB of that for each block itself.  A block of less shared memory than its columns' share can make another block wait that it
    waits for itself (csrc/tcgen05.cuh).  Of two blocks of 256 columns and more 56 columns' share may be left, 25 KB: less than the smallest block takes."""
    g = random.Random(5)
    seen = set()
    sizes = [(m, k, n, e) for m in (1, 8, 20, 33, 64, 128, 129, 300, 2000) for k in (16, 256, 300, 512, 768, 1000, 1300, 2048, 4096, 14336) for n in (64, 1024, 4096, 28672) for e in (0, 32)]
    sizes += [(int(2 ** g.uniform(0, 12)), int(2 ** g.uniform(0, 14)), int(2 ** g.uniform(0, 16)), g.choice([0, 0, 8, 200, 1024])) for _ in range(2000)]
    least = 228 * 1024
    for m, k, n, e in sizes:
        for bits, codes in ((4, 1), (8, 0), (8, 1)):
            columns, smem = room(m, k, n, e, bits, codes)
            seen.add((bits, columns))
            least = min(least, smem + 1024)
            assert columns in (32, 64, 128, 256, 512) and smem <= 227 * 1024, (m, k, n, e, bits)
            assert smem + 1024 >= (columns - (28 if columns >= 256 else 0)) * 228 * 1024 // 512, (m, k, n, e, bits, columns, smem)
            assert e or shared(m, k, n, bits, codes) == 1 or smem + 1024 > 30 * 1024      # (in clusters: beside 512 columns and 199 KB)
    assert {(4, 128), (4, 256), (4, 512), (8, 64), (8, 128), (8, 256), (8, 512)} <= seen and least > 56 * 228 * 1024 // 512


@pytest.mark.parametrize("sizes", [(0, 8, 8, 0), (8, 0, 8, 0), (8, 8, 0, 0), (8, 8, 8, -1)])
def test_no_room_for_no_product(sizes):
    m, n, k, e = sizes
    found = (ctypes.c_int * 2)()
    for status in (ops.lib().tib_microscaled_room(m, n, k, e, ctypes.addressof(found)), ops.lib().tib_block_scaled_tcgen05_room(1, m, n, k, e, ctypes.addressof(found)),
                   ops.lib().tib_microscaled_room(8, 8, 8, 0, 0), ops.lib().tib_block_scaled_tcgen05_room(1, 8, 8, 8, 0, 0)):
        assert status < 0


# ------------------------------------------------------------------------------------------------ checkpoints
def folder_of(tmp_path, said, **more):
    """A random model folder in 4-bit codes whose config.json says this, with these tensors beside its own."""
    import json
    from conftest import TINY_B
    from safetensors.torch import load_file, save_file
    from torchinferno_b200.weights.random_init import build_model, write_random_model
    write_random_model({**TINY_B, "quantization_config": {"quant_method": "modelopt", "quant_algo": "NVFP4"}}, tmp_path, seed=0)
    config = {**TINY_B} if said is None else {**TINY_B, "quantization_config": said}
    (tmp_path / "config.json").write_text(json.dumps(config))
    tensors = {k: v.clone() for k, v in load_file(str(tmp_path / "model.safetensors")).items()}
    save_file({**tensors, **more}, str(tmp_path / "model.safetensors"))
    return build_model(config, dtype=torch.bfloat16, device="cpu")


@pytest.mark.parametrize("said, form", [({"quant_method": "modelopt", "quant_algo": "FP8"}, "'FP8'"), ({"quant_method": "modelopt", "quant_algo": "W4A16_AWQ"}, "'W4A16_AWQ'"),
                                        ({"quant_algo": "MIXED_PRECISION"}, "'MIXED_PRECISION'"), ({"quant_method": "fp8", "weight_block_size": [128, 128]}, "'fp8'"),
                                        ({"quant_method": "awq", "bits": 4}, "'awq'")])
def test_codes_of_a_folder_that_names_another_form_are_refused(tmp_path, said, form):
    from torchinferno_b200.weights.loader import WeightError, load_weights
    with pytest.raises(WeightError, match=f"4-bit codes, but quantization_config names {form}"):
        load_weights(folder_of(tmp_path, said), tmp_path)


@pytest.mark.parametrize("said", [None, {}, {"quant_algo": "nvfp4"}, {"quant_method": "modelopt"}, {"quant_method": "modelopt_fp4"}, {"quant_method": "modelopt", "quant_algo": "NVFP4", "group_size": 16}])
def test_codes_of_a_folder_that_names_them_or_nothing_are_read(tmp_path, said):
    from torchinferno_b200.kernels.microscaled import MicroscaledWeight
    from torchinferno_b200.weights.loader import load_weights
    model = folder_of(tmp_path, said)
    load_weights(model, tmp_path)
    assert isinstance(model.blocks[0].feed_forward.down_weight, MicroscaledWeight)


CACHE_SCALES = {f"model.layers.{i}.self_attn.{p}_proj.{p}_scale": torch.tensor(0.05 * (i + 1)) for i in range(2) for p in "kv"}


def test_scales_of_an_8_bit_cache_are_left_aside(tmp_path):
    from torchinferno_b200.kernels.microscaled import MicroscaledWeight
    from torchinferno_b200.weights.loader import load_weights
    said = {"quant_method": "modelopt", "quant_algo": "NVFP4", "kv_cache_scheme": {"dynamic": False, "num_bits": 8, "type": "float"}}
    model = folder_of(tmp_path, said, **CACHE_SCALES, **{"model.layers.0.self_attn.k_proj.input_scale": torch.tensor(0.1)})
    report = load_weights(model, tmp_path)
    assert report["ignored"] == sorted([*CACHE_SCALES, "model.layers.0.self_attn.k_proj.input_scale"])
    plain = folder_of(tmp_path, said)
    load_weights(plain, tmp_path)
    assert isinstance(model.blocks[0].mixer.qkv_weight, MicroscaledWeight)
    assert torch.equal(model.blocks[0].mixer.qkv_weight.tiles.codes, plain.blocks[0].mixer.qkv_weight.tiles.codes)


def test_scales_of_a_cache_beside_other_tensors_are_not_known(tmp_path):
    from conftest import TINY_B
    from safetensors.torch import load_file, save_file
    from torchinferno_b200.weights.loader import WeightError, load_weights
    from torchinferno_b200.weights.random_init import build_model, write_random_model
    with pytest.raises(WeightError, match="unexpected"):
        load_weights(folder_of(tmp_path, None, **{"model.norm.k_scale": torch.ones(1)}), tmp_path)
    write_random_model(TINY_B, tmp_path, seed=0)      # (a folder without codes)
    save_file({**load_file(str(tmp_path / "model.safetensors")), **CACHE_SCALES}, str(tmp_path / "model.safetensors"))
    with pytest.raises(WeightError, match="unexpected"):
        load_weights(build_model(TINY_B, dtype=torch.bfloat16, device="cpu"), tmp_path)


# ------------------------------------------------------------------------------------------------ matrices
def check_nearest(matrix, made):
    """Every scale and every code is the nearest one, of two as near the even one: compared by products that are exact in 64 bits."""
    n, k = matrix.shape
    w, f = matrix.double(), made.factor.double()
    table = torch.tensor(SCALES, dtype=torch.float64)
    runs = torch.nn.functional.pad(w.abs(), (0, -k % 16)).view(n, -1, 16).amax(2)
    index = torch.searchsorted(table, made.scales.double())
    assert torch.equal(table[index], made.scales.double())
    even = index % 2 == 0
    below, above = (table[(index - 1).clamp(min=0)] + table[index]) / 2 * 6 * f, (table[(index + 1).clamp(max=len(SCALES) - 1)] + table[index]) / 2 * 6 * f
    assert ((index == 0) | (runs > below) | ((runs == below) & even)).all() and ((index == len(SCALES) - 1) | (runs < above) | ((runs == above) & even)).all()
    halves = torch.stack([made.codes % 16, made.codes // 16], 2).view(n, -1)[:, :k].long()
    code, codes = halves % 8, torch.tensor(CODES, dtype=torch.float64)
    unit = made.scales.double()[:, torch.arange(k) // 16] * f
    low, high = (codes[(code - 1).clamp(min=0)] + codes[code]) / 2 * unit, (codes[(code + 1).clamp(max=7)] + codes[code]) / 2 * unit
    size, even = torch.where(unit == 0, 0.0, w.abs()), code % 2 == 0
    assert ((code == 0) | (size > low) | ((size == low) & even)).all() and ((code == 7) | (size < high) | ((size == high) & even)).all()
    assert torch.equal(halves > 7, (w < 0) & (code > 0)) and not (code[unit == 0]).any()


@pytest.mark.parametrize("seed", range(6))
def test_a_matrix_gets_the_nearest_scales_and_codes(seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(1200, 1003, generator=g) * torch.randn(1200, 1, generator=g).exp()
    check_nearest(w, quantize_matrix(w))
    check_nearest(w.bfloat16(), quantize_matrix(w.bfloat16()))


@pytest.mark.parametrize("largest", [2688.0, 1.0, 0.1, 3.7e-3, 2688 * 1.2345678e-5, 3e38, 1e-30])
def test_numbers_of_a_matrix_beside_every_border(largest):
    """For the factor that this largest number gives: numbers on and next to each border of codes, under each scale, and runs' largest ones beside the borders of scales."""
    f = (torch.tensor(largest) / 2688.0).double()
    rows = []
    for s in SCALES[1::3] + [448.0]:
        top, near = (6 * s * f).float(), []
        for border in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
            b = (border * s * f).float()
            near += [torch.nextafter(b, torch.tensor(0.0)), b, torch.nextafter(b, torch.tensor(3e38))]
        rows += [torch.stack([top] + near[:15]), torch.stack([top] + near[6:])]
    for low, high in zip(SCALES[:-1], SCALES[1:]):
        b = ((low + high) / 2 * 6 * f).float()
        rows += [torch.cat([v[None], torch.zeros(15)]) for v in (torch.nextafter(b, torch.tensor(0.0)), b, torch.nextafter(b, torch.tensor(3e38)))]
    rows.append(torch.cat([torch.tensor([largest]), torch.zeros(15)]))
    w = torch.stack(rows).clamp(max=largest)
    made = quantize_matrix(w)
    assert made.factor == torch.tensor(largest) / 2688.0
    check_nearest(w, made)
    assert torch.equal(quantize_matrix(-w).scales.view(torch.uint8), made.scales.view(torch.uint8))


def test_operands_of_a_norm_that_overlap_are_refused():
    """By their addresses alone: 4 rows of 64 columns, 1,024 bytes in 32 bits and 512 in bf16."""
    lib, at = ops.lib(), 1 << 20      # (an address that nothing reads)
    norm = dict(delta=at + 4096, residual=at, sum=at + 8192, rows=0, weight=at + 12288, out=at + 16384, bytes=0, codes=at + 65536, scales=at + 131072, factors=at + 196608, lds=0, n_out=4,
                n_rows=4, hidden=64, eps=1e-5, dtype=1, stream=0)
    for wrong in (dict(sum=at + 16), dict(sum=at - 1008), dict(sum=at + 4096), dict(sum=at + 4096 - 1008, dtype=0), dict(sum=at + 12288 + 240), dict(out=at + 1008), dict(out=at - 496), dict(out=at),
                  dict(out=at + 4096 + 496), dict(out=at + 8192 + 512), dict(out=at + 12288 - 496), dict(sum=at, delta=at + 256, out=0)):
        assert lib.tib_quantized_norm(*{**norm, **wrong}.values()) == -8, wrong


def test_a_parameter_is_quantised_as_its_numbers():
    g = torch.Generator().manual_seed(1)
    w = torch.randn(40, 33, generator=g)
    for given in (torch.nn.Parameter(w.clone()), w.double(), w.t().contiguous().t()):
        made, want = quantize_matrix(given), quantize_matrix(w)
        assert torch.equal(made.codes, want.codes) and torch.equal(made.scales.view(torch.uint8), want.scales.view(torch.uint8)) and made.factor == want.factor
        assert not made.factor.requires_grad and not made.scales.requires_grad and MicroscaledWeight(made).tiles.numbers[3] == 0


# ------------------------------------------------------------------------------------------------ factors that are far from 1
def with_factor(n, factor, zeros=False):
    matrix = random_matrix(n, 32, n, factor=1.0)
    return MicroscaledMatrix(matrix.codes, torch.zeros_like(matrix.scales) if zeros else matrix.scales, torch.tensor(factor))


def test_which_weights_have_far_factors():
    """Those whose factor is outside 2^-100 .. 2^70 where it matters: not a matrix of zeros', whatever its factor."""
    tiny, least, most = 1e-38, 2.0 ** -100, 2.0 ** 70
    for factors, far in (((1e-3,), False), ((least,), False), ((most,), False), ((least * 0.999,), True), ((most * 1.001,), True), ((0.0,), False), ((-1e25,), True), ((1e-3, tiny), True),
                         ((tiny, 1e-3), True), ((3e38,), True)):
        weight = MicroscaledWeight(*(with_factor(140, f) for f in factors))
        assert weight.tiles.far is far and weight.tiles.numbers[3] == 2 * far and weight.rows(128, 140).tiles.numbers[3] == 2 * far
        gated = MicroscaledWeight(with_factor(6, 1e-3), with_factor(6, factors[-1]), epilogue="swiglu")
        assert gated.tiles.numbers[3] == 1 + 2 * (not least <= abs(factors[-1]) <= most and factors[-1] != 0)
    assert not MicroscaledWeight(with_factor(3, tiny, zeros=True), with_factor(5, 1.0)).tiles.far and not MicroscaledWeight(quantize_matrix(torch.zeros(4, 32))).tiles.far
    experts = [with_factor(4, 1e-3) for _ in range(300)]
    assert not MicroscaledExperts(experts).tiles.far
    experts[200] = with_factor(4, tiny)
    with pytest.raises(ValueError, match="more than 223 experts"):
        MicroscaledExperts(experts)
    assert MicroscaledExperts(experts[78:]).tiles.far and not MicroscaledExperts(experts[:200] + [with_factor(4, tiny, zeros=True)] + experts[201:]).tiles.far


def test_products_with_far_factors_are_told_so():
    """2 of `pairs`: no product that quantises its rows itself, and no more experts than pairs of SMs take."""
    lib, at = ops.lib(), 1 << 20
    product = dict(w=at, w_scales=at, w_factors=at, pairs=2, N=8, K=64, experts=1, x=at, x_dtype=1, ldx=64, x_rows=4, codes=0, scales=0, factors=0, make=1, y=at + 65536, y_dtype=1, ldy=8,
                   M=4, offsets=0, order=0, top=1, x_by_pair=0, act=0, limit=0.0, alpha=0.0, row_scale=0, error_word=0, stream=0)
    for wrong, status in ((dict(), -5), (dict(codes=at, scales=at, factors=at, make=0, act=4), -2), (dict(codes=at, scales=at, factors=at, make=0, pairs=3, N=7), -2),
                          (dict(codes=at, scales=at, factors=at, make=0, offsets=at, order=at, experts=224), -2)):
        assert lib.tib_microscaled_product(*{**product, **wrong}.values()) == status, wrong
