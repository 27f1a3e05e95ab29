"""4-bit microscaled matrices on the host: their types, how they are laid out, and what is refused before a kernel runs."""
import pytest
import torch

from microscaled_oracle import CODES, matrix64, nearest, random_matrix
from torchinferno_b200.kernels import block_scaled, gemm, microscaled, ops
from torchinferno_b200.kernels.microscaled import MicroscaledExperts, MicroscaledMatrix, MicroscaledWeight, quantize_matrix, quantize_rows


def test_a_matrix_stands_for_its_numbers():
    for n, k in ((1, 1), (3, 16), (5, 33), (130, 100)):
        matrix = random_matrix(n, k, n + k)
        assert matrix.shape == (n, k) and torch.equal(matrix.widened().double(), matrix64(matrix).float().double())
        assert matrix.widened(torch.bfloat16).dtype == torch.bfloat16


@pytest.mark.parametrize("n, k", [(1, 1), (7, 16), (40, 333), (3, 1000)])
def test_quantising_a_matrix(n, k):
    g = torch.Generator().manual_seed(n)
    w = torch.randn(n, k, generator=g) * torch.randn(n, 1, generator=g).exp()
    made = quantize_matrix(w)
    # a number lies between codes at most 2 apart, of a size up to 6 scales: it is off by at most one scale, and by what a scale rounded down (2^-4) cuts off above 6
    scale = made.scales.float().double()[:, torch.arange(k) // 16] * made.factor.double()
    assert ((made.widened().double() - w.double()).abs() <= scale * (1 + 2.0 ** -20)).all()
    # and no code is nearer than the one taken (but for the borders themselves)
    size = (w.double() / torch.where(scale == 0, 1.0, scale)).abs()
    best = torch.tensor(CODES, dtype=torch.float64)[nearest(size, CODES)]
    taken = (made.widened().double() / torch.where(scale == 0, 1.0, scale)).abs()
    assert ((taken - size).abs() <= (best - size).abs() + 1e-5).all()
    assert torch.equal(quantize_matrix(torch.zeros(2, 20)).widened(), torch.zeros(2, 20))


def number(tiles, i, n, k):
    """Number (n, k) of matrix i, read from where the kernels look for it."""
    tile, row, step, column = n // 128, n % 128, k // 256, k % 256
    byte = int(tiles.codes[i, tile, step, row, (column // 32 ^ row % 8) * 16 + column // 2 % 16])
    scales = tiles.scales[i, tile, step].view(torch.float8_e4m3fn)
    at = (column // 64) * 512 + (row % 32) * 16 + (row // 32) * 4 + (column % 64) // 16
    code = byte >> 4 if column % 2 else byte & 15
    return CODES[code & 7] * (-1 if code > 7 else 1) * float(scales[at]) * float(tiles.factors[i, n])


def test_where_the_kernels_find_a_matrix():
    a, b = random_matrix(150, 301, 1), random_matrix(20, 301, 2, factor=0.5)
    tiles = MicroscaledWeight(a, b).tiles
    assert tiles.codes.shape == (1, 2, 2, 128, 128) and tiles.scales.shape == (1, 2, 2, 2048) and tiles.features == 170
    wide = torch.cat([a.widened(), b.widened()])
    for n in (0, 1, 31, 32, 127, 128, 149, 150, 169):
        for k in (0, 1, 15, 16, 63, 64, 255, 256, 300):
            assert number(tiles, 0, n, k) == pytest.approx(float(wide[n, k]), rel=1e-6)
    assert not tiles.codes[0, 1, :, 42:].any() and int((tiles.codes[0, 0, 1] > 0).sum()) <= 128 * 23
    gates, ups = [random_matrix(70, 64, i) for i in (3, 4)], [random_matrix(70, 64, i, factor=0.3) for i in (5, 6)]
    tiles = MicroscaledExperts(gates, ups).tiles
    for i in range(2):
        for n in (0, 1, 64, 69):
            assert number(tiles, i, 2 * n, 20) == pytest.approx(float(gates[i].widened()[n, 20]), rel=1e-6)
            assert number(tiles, i, 2 * n + 1, 20) == pytest.approx(float(ups[i].widened()[n, 20]), rel=1e-6)


def test_views_of_a_weight():
    weight = MicroscaledWeight(random_matrix(300, 40, 1))
    view = weight.rows(128, 290)
    assert view.out_features == 162 and view.tiles.features == 162 and view.tiles.codes.shape[1] == 2
    tiles = weight.tiles
    assert view.tiles.numbers[:3] == (tiles.codes[:, 1].data_ptr(), tiles.scales[:, 1].data_ptr(), tiles.factors[:, 128:].data_ptr())
    with pytest.raises(ValueError, match="inside a tile"):
        weight.rows(64, 128)
    for start, stop in ((0, 301), (5, 5), (-1, 3)):
        with pytest.raises(ValueError, match="no features"):
            weight.rows(start, stop)
    assert weight.nbytes() == 3 * 128 * 128 + 3 * 2048 + 4 * 300 and weight.device.type == "cpu"


def test_matrices_that_are_refused():
    good = random_matrix(4, 32, 1)
    with pytest.raises(ValueError, match="uint8"):
        MicroscaledMatrix(good.codes.to(torch.int32), good.scales, good.factor)
    with pytest.raises(ValueError, match="bytes of codes"):
        MicroscaledMatrix(good.codes, good.scales, good.factor, columns=30)
    with pytest.raises(ValueError, match="scales of a"):
        MicroscaledMatrix(good.codes, good.scales[:, :1], good.factor)
    with pytest.raises(ValueError, match="scales of a"):
        MicroscaledMatrix(good.codes, good.scales.float(), good.factor)
    with pytest.raises(ValueError, match="one float32 number"):
        MicroscaledMatrix(good.codes, good.scales, good.factor.expand(2))
    for bad in (-1.0, float("nan")):
        scales = good.scales.float()
        scales[2, 1] = bad
        with pytest.raises(ValueError, match="none of them negative"):
            MicroscaledWeight(MicroscaledMatrix(good.codes, scales.to(torch.float8_e4m3fn), good.factor))
    with pytest.raises(ValueError, match="alike"):
        MicroscaledWeight(good, random_matrix(4, 48, 2))
    with pytest.raises(ValueError, match="gate and an up"):
        MicroscaledWeight(good, epilogue="swiglu")
    with pytest.raises(ValueError, match="of one size"):
        MicroscaledWeight(good, random_matrix(5, 32, 2), epilogue="swiglu")
    with pytest.raises(ValueError, match="unknown epilogue"):
        MicroscaledWeight(good, epilogue="gelu")
    with pytest.raises(ValueError, match="made of microscaled"):
        MicroscaledWeight(torch.zeros(3, 3))
    with pytest.raises(ValueError, match="at least one"):
        MicroscaledExperts([])
    with pytest.raises(ValueError, match="1 gate and 2 up"):
        MicroscaledExperts([good], [good, good])
    with pytest.raises(ValueError, match="non-empty matrix"):
        quantize_matrix(torch.zeros(0, 3))


def test_weights_from_matrices():
    four, eight = random_matrix(4, 32, 1), block_scaled.quantize_matrix(torch.ones(4, 32))
    assert isinstance(gemm.projection(four, four), MicroscaledWeight) and isinstance(gemm.gated_projection(four, four), MicroscaledWeight)
    assert isinstance(gemm.expert_matrices([four, four]), MicroscaledExperts)
    for other in (eight, torch.ones(4, 32)):
        with pytest.raises(ValueError, match="all be stored in 4-bit codes, or none"):
            gemm.projection(four, other)


def test_calls_that_are_refused_without_a_gpu():
    x, weight, residual = torch.zeros(2, 32), MicroscaledWeight(random_matrix(4, 32, 1)), torch.zeros(2, 32)
    for call in (lambda: quantize_rows(x), lambda: gemm.linear(x, weight), lambda: microscaled.add_rmsnorm(None, residual, torch.ones(32), 1e-5)):
        with pytest.raises(ops.KernelError, match="CUDA"):
            call()
    with pytest.raises(ops.KernelError, match="rows of 32"):
        gemm.linear(torch.zeros(2, 31), weight)
    with pytest.raises(ops.KernelError, match="epilogue='swiglu'"):
        gemm.linear_swiglu(x, weight)
    with pytest.raises(ops.KernelError, match="delta is"):
        microscaled.add_rmsnorm(x, residual, torch.ones(32), 1e-5, dtype=torch.bfloat16)
    eight_rows = block_scaled.BlockScaledRows(x, 2, 32, torch.bfloat16)
    with pytest.raises(ops.KernelError, match="not BlockScaledRows"):
        gemm.linear(eight_rows, weight)
    with pytest.raises(ops.KernelError, match="not MicroscaledRows"):
        gemm.linear(microscaled.MicroscaledRows(x, 2, 32, torch.bfloat16), block_scaled.BlockScaledWeight(block_scaled.quantize_matrix(torch.ones(4, 32))))
    for product in (gemm.linear, gemm.linear_swiglu):
        with pytest.raises(ops.KernelError, match="quantised rows are for quantised weights"):
            product(eight_rows, gemm.LinearWeight(torch.ones(4, 32), few_rows_tcgen05=False))


# ------------------------------------------------------------------------------------------------ checkpoints
NVFP4 = {"quant_method": "modelopt", "quant_algo": "NVFP4", "ignore": ["lm_head"],
         "config_groups": {"group_0": {"weights": {"num_bits": 4, "type": "float", "group_size": 16}, "targets": ["Linear"]}}}


def test_quantization_config():
    from torchinferno_b200.config.model_config import ConfigError
    from torchinferno_b200.config.quantization import BlockQuantization, MicroscaledQuantization, quantization_of
    assert quantization_of({}) is None and quantization_of({"quantization_config": None}) is None
    assert quantization_of({"quantization_config": {"quant_method": "modelopt", "quant_algo": "FP8"}}) is None
    assert isinstance(quantization_of({"quantization_config": {"quant_method": "fp8", "weight_block_size": [128, 128]}}), BlockQuantization)
    q = quantization_of({"quantization_config": {**NVFP4, "ignore": ["lm_head", "model.layers.1.mlp", "model.layers.2*", "o_proj"]}})
    assert isinstance(q, MicroscaledQuantization)
    assert [q.converts(n) for n in ("lm_head.weight", "model.layers.1.mlp.up_proj.weight", "model.layers.11.mlp.up_proj.weight", "model.layers.2.mlp.up_proj.weight",
                                    "model.layers.0.self_attn.o_proj.weight", "model.layers.0.self_attn.q_proj.weight")] == [False, False, True, False, False, True]
    for bad in ({**NVFP4, "config_groups": {"g": {"weights": {"group_size": 32}}}}, {**NVFP4, "group_size": 32}, {**NVFP4, "ignore": "lm_head"}, {**NVFP4, "ignore": [1]},
                {**NVFP4, "config_groups": [1]}):
        with pytest.raises(ConfigError):
            quantization_of({"quantization_config": bad})


def _folder(tmp_path, config, drop=(), **changes):
    """A random model folder with these tensors changed or left out, and its tensors as they were."""
    from safetensors.torch import load_file, save_file
    from torchinferno_b200.weights.random_init import write_random_model
    write_random_model(config, tmp_path, seed=0)
    tensors = {k: v.clone() for k, v in load_file(str(tmp_path / "model.safetensors")).items()}
    save_file({k: v for k, v in {**tensors, **changes}.items() if k not in drop}, str(tmp_path / "model.safetensors"))
    return tensors


def test_a_checkpoint_of_codes_is_bound_in_codes(tmp_path):
    from conftest import TINY_B
    from torchinferno_b200.kernels.gemm import LinearWeight
    from torchinferno_b200.kernels.microscaled import MicroscaledRows
    from torchinferno_b200.weights.loader import load_weights
    from torchinferno_b200.weights.random_init import build_model, init_random_weights
    config = {**TINY_B, "quantization_config": {**NVFP4, "ignore": ["model.layers.2.self_attn*"]}}
    name = "model.layers.0.mlp.down_proj.weight"
    tensors = _folder(tmp_path, config, **{"model.layers.0.mlp.down_proj.input_scale": torch.tensor(0.01)})
    model = build_model(config, dtype=torch.bfloat16, device="cpu")
    report = load_weights(model, tmp_path)
    assert report["stored_dtypes"] == ["bfloat16", "uint8"] and report["ignored"] == ["model.layers.0.mlp.down_proj.input_scale"]
    assert tensors[name].shape == (192, 256) and tensors[name + "_scale"].shape == (192, 32) and tensors[name + "_scale_2"].shape == ()
    block = model.blocks[0]
    down = block.feed_forward.down_weight
    assert isinstance(down, MicroscaledWeight) and down.in_features == 512 and down.out_features == 192
    want = MicroscaledWeight(MicroscaledMatrix(tensors[name], tensors[name + "_scale"], tensors[name + "_scale_2"])).tiles
    assert torch.equal(down.tiles.codes, want.codes) and torch.equal(down.tiles.scales, want.scales) and torch.equal(down.tiles.factors, want.factors)
    assert isinstance(block.mixer.qkv_weight, MicroscaledWeight) and block.feed_forward.gate_up_weight.tiles.paired
    assert isinstance(model.blocks[2].mixer.qkv_weight, LinearWeight) and isinstance(model.blocks[2].feed_forward.down_weight, MicroscaledWeight)
    # the norms ahead of 4-bit products leave rows of codes
    assert [b.mixer.rows_form(1) for b in model.blocks] == [MicroscaledRows, MicroscaledRows, None] and block.feed_forward.rows_form(4) is MicroscaledRows
    from torchinferno_b200.kernels import native_block
    assert native_block.block_weights(block) is None
    plain = build_model(TINY_B, dtype=torch.bfloat16, device="cpu")
    init_random_weights(plain, 0)
    assert model.weight_bytes() < plain.weight_bytes()
    same = build_model(config, dtype=torch.bfloat16, device="cpu")
    init_random_weights(same, 0, config=config)
    assert torch.equal(same.blocks[0].feed_forward.down_weight.tiles.codes, down.tiles.codes)
    # in 32 bits the numbers they stand for
    wide = build_model(config, dtype=torch.float32, device="cpu")
    load_weights(wide, tmp_path)
    assert torch.equal(wide.blocks[0].feed_forward.down_weight.tensor, MicroscaledMatrix(tensors[name], tensors[name + "_scale"], tensors[name + "_scale_2"]).widened())


UP = "model.layers.0.mlp.up_proj.weight"


@pytest.mark.parametrize("changes, drop, message", [
    ({UP + "_scale": torch.ones(512, 11).to(torch.float8_e4m3fn)}, (), r"_scale: file \[512, 11\] vs \[512, 12\]"),
    ({UP + "_scale": torch.ones(512, 12)}, (), "_scale: stored as F32"),
    ({UP + "_scale_2": torch.ones(2)}, (), r"_scale_2: file \[2\]"),
    ({UP + "_scale_2": torch.ones((), dtype=torch.bfloat16)}, (), "_scale_2: stored as BF16"),
    ({UP: torch.zeros(512, 95, dtype=torch.uint8)}, (), r"up_proj.weight: file \[512, 95\]"),
    ({UP: torch.zeros(512, 192, dtype=torch.bfloat16)}, (), "up_proj.weight: "),
    ({}, (UP + "_scale",), "_scale_2"),
    ({}, (UP + "_scale", UP + "_scale_2"), r"up_proj.weight: file \[512, 96\]"),
    ({"model.norm.weight_scale": torch.ones(1)}, (), "unexpected"),
    ({"model.norm.input_scale": torch.ones(1)}, (), "unexpected")])
def test_checkpoints_that_do_not_fit_are_refused(tmp_path, changes, drop, message):
    from conftest import TINY_B
    from torchinferno_b200.weights.loader import WeightError, load_weights
    from torchinferno_b200.weights.random_init import build_model
    config = {**TINY_B, "quantization_config": NVFP4}
    _folder(tmp_path, config, drop, **changes)
    for dtype in (torch.bfloat16, torch.float32):
        with pytest.raises(WeightError, match=message):
            load_weights(build_model(config, dtype=dtype, device="cpu"), tmp_path)


def test_codes_of_another_form_are_refused(tmp_path):
    """Scales that are no numbers, and a config.json that names another run of columns."""
    import json
    from conftest import TINY_B
    from torchinferno_b200.weights.loader import WeightError, load_weights
    from torchinferno_b200.weights.random_init import build_model, init_random_weights
    config = {**TINY_B, "quantization_config": NVFP4}
    _folder(tmp_path, config, **{UP + "_scale": torch.full((512, 12), -1.0).to(torch.float8_e4m3fn)})
    with pytest.raises(ValueError, match="none of them negative"):
        load_weights(build_model(config, dtype=torch.bfloat16, device="cpu"), tmp_path)
    _folder(tmp_path, config)
    other = {**config, "quantization_config": {**NVFP4, "group_size": 32}}
    (tmp_path / "config.json").write_text(json.dumps(other))
    with pytest.raises(WeightError, match="4-bit codes, but quantization_config"):
        load_weights(build_model(config, dtype=torch.bfloat16, device="cpu"), tmp_path)
    model = build_model(other, dtype=torch.bfloat16, device="cpu")
    init_random_weights(model, 0, config=other)      # (random weights are of the model's own type then)
    assert model.blocks[0].feed_forward.down_weight.dtype == torch.bfloat16


def test_fused_projections_are_stored_alike(tmp_path):
    from conftest import TINY_B
    from torchinferno_b200.weights.loader import load_weights
    from torchinferno_b200.weights.random_init import build_model
    config = {**TINY_B, "quantization_config": {**NVFP4, "ignore": ["k_proj"]}}
    _folder(tmp_path, config)
    with pytest.raises(ValueError, match="all be stored in 4-bit codes, or none"):
        load_weights(build_model(config, dtype=torch.bfloat16, device="cpu"), tmp_path)


def test_experts_are_bound_in_codes():
    from giforax_configs import GA
    from torchinferno_b200.weights.random_init import build_model, init_random_weights
    config = {**GA, "quantization_config": NVFP4}
    model = build_model(config, dtype=torch.bfloat16, device="cpu")
    init_random_weights(model, 1, config=config)
    moes = [b.feed_forward for b in model.blocks if type(b.feed_forward).__name__ == "RoutedExperts"]
    assert moes
    for moe in moes:
        assert isinstance(moe.up_weight, MicroscaledExperts) and moe.up_weight.paired == moe.glu and moe.up_weight.experts == moe.experts
        assert isinstance(moe.down_weight, MicroscaledExperts) and moe.router_weight.dtype == torch.float32 and moe.rows_form(3) is None


def test_what_the_library_refuses():
    """Refused by their arguments alone, before anything is launched: null pointers, sizes, types, alignment, and activations that do not fit."""
    lib = ops.lib()
    at = 1 << 20      # (an address that nothing reads)
    rows = dict(x=at, x_dtype=1, ldx=64, x_rows=4, codes=at, scales=at, factors=at, rows=4, K=64, offsets=0, order=0, experts=1, top=1, x_by_pair=0, stream=0)
    for wrong, status in ((dict(x=0), -5), (dict(codes=0), -5), (dict(K=0), -5), (dict(rows=-1), -5), (dict(x_rows=3), -5), (dict(x_dtype=2), -1), (dict(codes=at + 8), -3),
                          (dict(scales=at + 4), -3), (dict(offsets=at, x_by_pair=1), -5), (dict(top=0), -5), (dict(rows=0, x=0), 0)):
        assert lib.tib_microscaled_rows(*{**rows, **wrong}.values()) == status, wrong
    widen = dict(codes=at, scales=at, factors=at, out=at, out_dtype=1, ldo=64, rows=4, K=64, stream=0)
    for wrong, status in ((dict(out=0), -5), (dict(K=0), -5), (dict(out_dtype=7), -1), (dict(codes=at + 1), -3), (dict(rows=0), 0)):
        assert lib.tib_microscaled_widen(*{**widen, **wrong}.values()) == status, wrong
    product = dict(w=at, w_scales=at, w_factors=at, pairs=0, N=8, K=64, experts=1, x=0, x_dtype=1, ldx=0, x_rows=0, codes=at, scales=at, factors=at, make=0, y=at, y_dtype=1, ldy=8,
                   M=4, offsets=0, order=0, top=1, x_by_pair=0, act=0, limit=0.0, alpha=0.0, row_scale=0, error_word=0, stream=0)
    for wrong, status in ((dict(w=0), -5), (dict(y=0), -5), (dict(codes=0), -5), (dict(K=0), -5), (dict(M=-1), -5), (dict(experts=0), -5), (dict(make=1), -5), (dict(offsets=at), -5),
                          (dict(row_scale=at), -5), (dict(act=9), -2), (dict(act=4), -2), (dict(pairs=1, N=7), -2), (dict(y_dtype=2), -1), (dict(w=at + 8), -3),
                          (dict(offsets=at, order=at, experts=2000), -2), (dict(N=1 << 30, K=1 << 20), -2), (dict(M=0), 0), (dict(N=0), 0)):
        assert lib.tib_microscaled_product(*{**product, **wrong}.values()) == status, wrong
    norm = dict(delta=0, residual=at, sum=0, rows=0, weight=at, out=0, bytes=0, codes=at, scales=at, factors=at, lds=0, n_out=4, n_rows=4, hidden=64, eps=1e-5, dtype=1, stream=0)
    for wrong, status in ((dict(residual=0), -5), (dict(weight=0), -5), (dict(scales=0), -5), (dict(rows=at, sum=at), -5), (dict(n_out=5), -5), (dict(hidden=0), -5),
                          (dict(dtype=3), -1), (dict(bytes=1, lds=3), -2), (dict(codes=at + 4), -3), (dict(n_out=0), 0)):
        assert lib.tib_quantized_norm(*{**norm, **wrong}.values()) == status, wrong
