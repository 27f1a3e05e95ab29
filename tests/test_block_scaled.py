"""8-bit block-scaled weights on the host: their checks, their layout, their quantisation."""
import pytest
import torch

from block_scaled_oracle import EXPERT_PATHS, GATED_PATHS, PLAIN_PATHS, matrix64, plan, random_matrix, rows64
from torchinferno_b200.kernels import gemm, ops
from torchinferno_b200.kernels.block_scaled import BlockScaledExperts, BlockScaledMatrix, BlockScaledWeight, quantize_matrix, quantize_rows

CODES = torch.float8_e4m3fn


def codes(n, k):
    return torch.zeros(n, k, dtype=torch.uint8).view(CODES)


@pytest.mark.parametrize("c, s", [
    (torch.zeros(4, 4), torch.ones(1, 1)),                          # not codes
    (codes(4, 4).view(torch.uint8), torch.ones(1, 1)),              # bytes
    (codes(4, 4)[0], torch.ones(1)),                                # a vector
    (codes(0, 4), torch.ones(0, 1)),                                # empty
    (codes(129, 128), torch.ones(1, 1)),                            # a block of rows without a scale
    (codes(128, 129), torch.ones(1, 1)), (codes(128, 128), torch.ones(2, 1)),
    (codes(4, 4), torch.ones(1, 1, dtype=torch.bfloat16))])
def test_a_matrix_that_is_none_is_refused(c, s):
    with pytest.raises(ValueError):
        BlockScaledMatrix(c, s)


@pytest.mark.parametrize("make", [
    lambda a, b, w: BlockScaledWeight(), lambda a, b, w: BlockScaledWeight(torch.zeros(4, 4)), lambda a, b, w: BlockScaledWeight(a, epilogue="relu"),
    lambda a, b, w: BlockScaledWeight(a, epilogue="swiglu"), lambda a, b, w: BlockScaledWeight(a, b, epilogue="swiglu"),
    lambda a, b, w: BlockScaledWeight(a, w), lambda a, b, w: BlockScaledExperts([]), lambda a, b, w: BlockScaledExperts([a, b]),
    lambda a, b, w: BlockScaledExperts([a, a], [a])])
def test_weights_that_do_not_fit_are_refused(make):
    with pytest.raises(ValueError):
        make(random_matrix(130, 200, 0), random_matrix(64, 200, 1), random_matrix(130, 100, 2))


def flat(x, n):
    """The rows of codes in blocks [blocks, runs, 128, 128]."""
    return x.view(torch.uint8).transpose(1, 2).reshape(x.shape[0] * 128, -1)[:n]


def test_a_weight_keeps_its_matrices_in_whole_blocks():
    a, b, c = random_matrix(256, 200, 0), random_matrix(130, 200, 1), random_matrix(64, 200, 2)
    w = BlockScaledWeight(a, b, c)
    assert (w.out_features, w.in_features, w.dtype) == (450, 200, CODES)
    def shapes(weight):
        return [(first, p.features, tuple(p.codes.shape), tuple(p.scales.shape)) for first, p in weight.parts]
    assert shapes(w) == [(0, 386, (1, 4, 2, 128, 128), (1, 4, 2)), (386, 64, (1, 1, 2, 128, 128), (1, 1, 2))]
    x, s = w.parts[0][1].codes, w.parts[0][1].scales
    assert torch.equal(flat(x[0], 256)[:, :200], a.codes.view(torch.uint8)) and torch.equal(s[0, 2:], b.scales)
    assert torch.equal(flat(x[0], 386)[256:, :200], b.codes.view(torch.uint8))
    assert not flat(x[0], 512)[:, 200:].any() and not flat(x[0], 512)[386:].any()
    assert w.nbytes() == 5 * 2 * 128 * 128 + 4 * (8 + 2)
    view = w.rows(128, 400)
    assert view.out_features == 272 and shapes(view) == [(0, 258, (1, 3, 2, 128, 128), (1, 3, 2)), (258, 14, (1, 1, 2, 128, 128), (1, 1, 2))]
    assert torch.equal(view.parts[0][1].codes.view(torch.uint8), x[:, 1:].view(torch.uint8))
    for start, stop in ((64, 130), (0, 451), (5, 5), (-1, 4)):
        with pytest.raises(ValueError):
            w.rows(start, stop)


def test_gate_and_up_alternate():
    g, u = random_matrix(130, 300, 0), random_matrix(130, 300, 1)
    part = BlockScaledWeight(g, u, epilogue="swiglu").parts[0][1]
    x, s = flat(part.codes[0], 260), part.scales
    assert part.features == 260 and part.paired
    assert torch.equal(x[0::2, :300], g.codes.view(torch.uint8)) and torch.equal(x[1::2, :300], u.codes.view(torch.uint8))
    assert torch.equal(s[0, 0::2], g.scales) and torch.equal(s[0, 1::2], u.scales)
    e = BlockScaledExperts([g, u], [u, g])
    assert e.out_features == 260 and torch.equal(flat(e.blocks.codes[1], 260)[0::2, :300], u.codes.view(torch.uint8))


@pytest.mark.parametrize("scales, low, high", [
    ([1.0], -126, 120), ([0.0], -126, 120), ([2.0 ** -10], -116, 120), ([-2.0 ** -10, 1.9], -116, 120), ([1.99 * 2.0 ** -10], -116, 120), ([2.0 ** -126], 0, 120),
    ([2.0 ** -149], 0, 120), ([2.0 ** 8], -126, 119), ([1.9 * 2.0 ** 7], -126, 120), ([2.0 ** 127], -126, 0), ([2.0 ** -126, 2.0 ** 127], 0, 0),
    ([float("nan"), 2.0 ** -20, float("inf")], -106, 120)])
def test_rows_scales_that_a_matrix_keeps_normal(scales, low, high):
    """The range that the kernels compare with: all of it gives normal products (or powers of at least 1), a power outside of it does not."""
    import math
    codes_ = torch.zeros(128, 128 * len(scales), dtype=torch.uint8).view(CODES)
    part = BlockScaledWeight(BlockScaledMatrix(codes_, torch.tensor([scales]))).parts[0][1]
    assert (part.far_low, part.far_high) == (2.0 ** low, 2.0 ** high)

    def normal(p):
        return all(s == 0 or not math.isfinite(s) or (2.0 ** p * abs(s) < 2.0 ** 128 and (p >= 0 or 2.0 ** p * abs(s) >= 2.0 ** -126)) for s in scales)
    assert all(normal(p) for p in range(low, high + 1)) and (low == -126 or not normal(low - 1)) and (high == 120 or not normal(high + 1))


def test_products_need_a_gpu():
    w = BlockScaledWeight(random_matrix(64, 64, 0))
    for call in (lambda: gemm.linear(torch.zeros(2, 64), w), lambda: gemm.linear(torch.zeros(2, 63), w), lambda: quantize_rows(torch.zeros(2, 64)),
                 lambda: quantize_rows(torch.zeros(64)), lambda: quantize_rows(torch.zeros(4, 0)), lambda: gemm.linear_swiglu(torch.zeros(2, 64), w)):
        with pytest.raises(ops.KernelError):
            call()


@pytest.mark.parametrize("n, k", [(1, 1), (128, 128), (130, 200), (5, 300)])
def test_a_quantised_matrix_is_near_its_own(n, k):
    m = torch.randn(n, k, generator=torch.Generator().manual_seed(n)) * 3
    m[0, 0] = 0
    q = quantize_matrix(m)
    # half a step of e4m3 for normal codes; half of 2^-9 for the subnormal ones, in the block's scale; the scale itself rounds by 2^-24
    scale = q.scales.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k].double()
    assert ((matrix64(q) - m.double()).abs() <= (2.0 ** -4 + 2.0 ** -22) * m.double().abs() + 2.0 ** -10 * scale).all()
    assert torch.equal(q.widened().double(), (q.codes.float() * scale.float()).double())
    zeros = quantize_matrix(torch.zeros(n, k))
    assert not zeros.widened().any() and (zeros.scales == 1).all()


def test_the_oracle_rounds_as_e4m3_does():
    """Its codes against torch's own conversion, over every midpoint of neighbouring codes and beside them."""
    values = torch.arange(0, 127, dtype=torch.uint8).view(CODES).float()
    middles = (values[1:] + values[:-1]) / 2
    v = torch.cat([values, middles, middles * (1 + 2.0 ** -20), middles * (1 - 2.0 ** -20), -middles])
    v = torch.cat([v, torch.zeros(-len(v) % 127)]).view(-1, 127)
    v = torch.cat([v, torch.full((len(v), 1), 448.0)], 1)                      # (so that every run's scale is 1)
    c, s = rows64(v)
    assert (s == 1).all() and torch.equal(c.float(), v.to(CODES).float())


# ------------------------------------------------------------------------------------------------ which kernel runs, and how
def test_the_ways_through_the_kernels_are_those_that_the_gpu_tests_name():
    """Each of their sizes runs as it says, and between them they take every tile and split there is, with rings that wrap."""
    for rows, columns, features, want in (*PLAIN_PATHS, *GATED_PATHS):
        assert plan(rows, columns, features) == want, (rows, columns, features)
    for pairs, experts, columns, features, want in EXPERT_PATHS:
        assert plan(pairs, columns, features, experts) == want, (pairs, experts, columns, features)
    found = {plan(m, k, 128 * f)[:2] for m in (*range(1, 140, 3), *range(140, 2000, 117)) for f in range(1, 320) for k in (128, 1024, 4096, 8192)}
    assert found == {want[:2] for *_, want in PLAIN_PATHS}
    assert not {tiles for tiles in found if tiles[0] >= 128 and tiles[1] > 1}
    for paths in (PLAIN_PATHS, GATED_PATHS, EXPERT_PATHS):
        for rows in (16, 32, 64, 128, 256):
            deep = [want for *_, want in paths if want[0] == rows]
            assert any(steps > max(stages, 16 if rows <= 128 else 0) for _, _, steps, stages in deep) or (paths is EXPERT_PATHS and rows == 64)
    # more tiles than blocks, for each height of a tile
    blocks_of = {16: 296, 32: 296, 64: 148, 128: 148, 256: 74}
    for rows, blocks in blocks_of.items():
        edge = 256 if rows == 256 else 128
        assert any(want[0] == rows and want[1] == 1 and -(-m // rows) * -(-n // edge) > blocks for m, _, n, want in PLAIN_PATHS)


@pytest.mark.parametrize("codes, m, n, k, experts", [(0, 0, 8, 8, 0), (1, 8, 0, 8, 0), (1, 8, 8, 0, 0), (1, 8, 8, 8, -1), (0, 8, 8, 8, 1025)])
def test_no_plan_for_no_product(codes, m, n, k, experts):
    import ctypes
    found = (ctypes.c_int * 4)()
    assert ops.lib().tib_block_scaled_plan(codes, m, n, k, experts, ctypes.addressof(found)) < 0
    assert ops.lib().tib_block_scaled_plan(1, 8, 8, 8, 0, 0) < 0


# ------------------------------------------------------------------------------------------------ checkpoints
FP8 = {"quant_method": "fp8", "fmt": "e4m3", "weight_block_size": [128, 128], "activation_scheme": "dynamic"}


def test_quantization_config():
    from torchinferno_b200.config.model_config import ConfigError
    from torchinferno_b200.config.quantization import BlockQuantization
    assert BlockQuantization.from_config({}) is None and BlockQuantization.from_config({"quantization_config": None}) is None
    assert BlockQuantization.from_config({"quantization_config": {"quant_method": "other"}}) is None
    q = BlockQuantization.from_config({"quantization_config": {**FP8, "modules_to_not_convert": ["lm_head", "layers.1.mlp", "o_proj"]}})
    assert [q.converts(n) for n in ("lm_head.weight", "model.layers.1.mlp.up_proj.weight", "model.layers.11.mlp.up_proj.weight",
                                    "model.layers.0.self_attn.o_proj.weight", "model.layers.0.self_attn.q_proj.weight")] == [False, False, True, False, True]
    for bad in ("fp8", {"quant_method": "fp8"}, {**FP8, "weight_block_size": [64, 128]}, {**FP8, "fmt": "e5m2"}, {**FP8, "activation_scheme": "static"},
                {**FP8, "modules_to_not_convert": "lm_head"}):
        with pytest.raises(ConfigError):
            BlockQuantization.from_config({"quantization_config": bad})


@pytest.mark.parametrize("names", [5, True, {"lm_head": 1}, [1], ["lm_head", None]])
def test_modules_that_are_no_list_of_names_are_refused(names):
    from torchinferno_b200.config.model_config import ConfigError
    from torchinferno_b200.config.quantization import BlockQuantization
    with pytest.raises(ConfigError, match="list of names"):
        BlockQuantization.from_config({"quantization_config": {**FP8, "modules_to_not_convert": names}})


def _folder(tmp_path, config, **changes):
    """A random model folder with these tensors changed, and its tensors as they were."""
    from safetensors.torch import load_file, save_file
    from torchinferno_b200.weights.random_init import write_random_model
    write_random_model(config, tmp_path, seed=0)
    tensors = {k: v.clone() for k, v in load_file(str(tmp_path / "model.safetensors")).items()}      # (clones: the file is mapped)
    save_file({**tensors, **changes}, str(tmp_path / "model.safetensors"))
    return tensors


def test_a_checkpoint_of_blocks_is_bound_in_blocks(tmp_path):
    from conftest import TINY_B
    from torchinferno_b200.kernels.gemm import LinearWeight
    from torchinferno_b200.weights.loader import load_weights
    from torchinferno_b200.weights.random_init import build_model
    config = {**TINY_B, "quantization_config": {**FP8, "modules_to_not_convert": ["model.layers.2.self_attn"]}}
    tensors = _folder(tmp_path, config)
    model = build_model(config, dtype=torch.bfloat16, device="cpu")
    report = load_weights(model, tmp_path)
    assert report["stored_dtypes"] == ["bfloat16", "float8_e4m3fn"]
    name = "model.layers.0.mlp.down_proj.weight"
    assert tensors[name].dtype == CODES and tensors[name + "_scale_inv"].shape == (2, 4)
    block = model.blocks[0]
    down = block.feed_forward.down_weight
    assert isinstance(down, BlockScaledWeight) and torch.equal(flat(down.parts[0][1].codes[0], 192), tensors[name].view(torch.uint8))
    assert isinstance(block.mixer.qkv_weight, BlockScaledWeight) and isinstance(block.feed_forward.gate_up_weight, BlockScaledWeight)
    assert isinstance(model.blocks[2].mixer.qkv_weight, LinearWeight) and isinstance(model.blocks[2].feed_forward.down_weight, BlockScaledWeight)
    assert model.embedding.dtype == torch.bfloat16
    # the block is not one for the native call, and its bytes count once each
    from torchinferno_b200.kernels import native_block
    assert native_block.block_weights(block) is None
    plain = build_model(TINY_B, dtype=torch.bfloat16, device="cpu")
    from torchinferno_b200.weights.random_init import init_random_weights
    init_random_weights(plain, 0)
    assert model.weight_bytes() < plain.weight_bytes()
    # in 32 bits the numbers they stand for
    wide = build_model(config, dtype=torch.float32, device="cpu")
    load_weights(wide, tmp_path)
    want = BlockScaledMatrix(tensors[name], tensors[name + "_scale_inv"]).widened()
    assert torch.equal(wide.blocks[0].feed_forward.down_weight.tensor, want)


@pytest.mark.parametrize("name, tensor, message", [
    ("model.layers.0.mlp.up_proj.weight_scale_inv", torch.ones(3, 2), "a scale for each 128 x 128"),
    ("model.layers.0.mlp.up_proj.weight", torch.zeros(512, 192), "not stored as e4m3"),
    ("model.layers.0.mlp.up_proj.weight", torch.zeros(512, 191, dtype=torch.uint8).view(CODES), "up_proj.weight: file"),
    ("model.norm.weight_scale_inv", torch.ones(1, 1), "unexpected")])
def test_checkpoints_that_do_not_fit_are_refused(tmp_path, name, tensor, message):
    from conftest import TINY_B
    from torchinferno_b200.weights.loader import WeightError, load_weights
    from torchinferno_b200.weights.random_init import build_model
    config = {**TINY_B, "quantization_config": FP8}
    _folder(tmp_path, config, **{name: tensor})
    with pytest.raises(WeightError, match=message):
        load_weights(build_model(config, dtype=torch.bfloat16, device="cpu"), tmp_path)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("name", ["model.layers.0.self_attn.o_proj.weight", "model.layers.1.mlp.down_proj.weight", "model.layers.0.self_attn.k_proj.weight"])
def test_codes_without_their_scales_are_refused(tmp_path, name, dtype):
    """A lost tensor of scales is named, whether or not the matrix shares its product with others; unscaled codes are never bound as numbers."""
    from conftest import TINY_B
    from safetensors.torch import save_file
    from torchinferno_b200.weights.loader import WeightError, load_weights
    from torchinferno_b200.weights.random_init import build_model
    config = {**TINY_B, "quantization_config": FP8}
    tensors = _folder(tmp_path, config)
    del tensors[name + "_scale_inv"]
    save_file(tensors, str(tmp_path / "model.safetensors"))
    with pytest.raises(WeightError, match=name + ": stored as F8_E4M3 without " + name + "_scale_inv"):
        load_weights(build_model(config, dtype=dtype, device="cpu"), tmp_path)


@pytest.mark.parametrize("code", [CODES, torch.float8_e5m2])
def test_codes_of_what_is_never_in_blocks_are_refused(tmp_path, code):
    from conftest import TINY_B
    from torchinferno_b200.weights.loader import WeightError, load_weights
    from torchinferno_b200.weights.random_init import build_model
    shape = build_model(TINY_B, dtype=torch.bfloat16, device="cpu").expected_tensors()["model.norm.weight"].shape
    _folder(tmp_path, TINY_B, **{"model.norm.weight": torch.ones(shape).to(code)})
    with pytest.raises(WeightError, match="model.norm.weight: stored as F8_"):
        load_weights(build_model(TINY_B, dtype=torch.bfloat16, device="cpu"), tmp_path)


@pytest.mark.parametrize("change", [{"weight_block_size": [96, 128]}, {"weight_block_size": None}, {"activation_scheme": "static"}, {"fmt": "e5m2"}])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_blocks_of_another_form_are_refused(tmp_path, change, dtype):
    """Scales of blocks of 96 rows have the shape of those of 128 where the rows are 192: only config.json tells them apart.  The same folder without a
    tensor in 8 bits loads whatever its config.json says of them."""
    import json
    from conftest import TINY_B
    from torchinferno_b200.weights.loader import WeightError, load_weights
    from torchinferno_b200.weights.random_init import build_model, write_random_model
    _folder(tmp_path, {**TINY_B, "quantization_config": FP8})
    said = json.loads((tmp_path / "config.json").read_text())
    said["quantization_config"] = {**FP8, **change}
    (tmp_path / "config.json").write_text(json.dumps(said))
    with pytest.raises(WeightError, match="8-bit blocks, but quantization_config." + next(iter(change))):
        load_weights(build_model(TINY_B, dtype=dtype, device="cpu"), tmp_path)
    write_random_model(TINY_B, tmp_path, seed=0)
    (tmp_path / "config.json").write_text(json.dumps(said))
    load_weights(build_model(TINY_B, dtype=dtype, device="cpu"), tmp_path)


def test_scales_that_are_no_numbers_are_refused(tmp_path):
    """Bytes beside codes (exponents, say) are not read as numbers."""
    from conftest import TINY_B
    from torchinferno_b200.weights.loader import WeightError, load_weights
    from torchinferno_b200.weights.random_init import build_model
    config = {**TINY_B, "quantization_config": FP8}
    name = "model.layers.0.mlp.down_proj.weight_scale_inv"
    _folder(tmp_path, config, **{name: torch.full((2, 4), 120, dtype=torch.uint8)})
    with pytest.raises(WeightError, match="stored as U8"):
        load_weights(build_model(config, dtype=torch.bfloat16, device="cpu"), tmp_path)


@pytest.mark.parametrize("quantization", [{"quant_method": "fp8"}, {**FP8, "weight_block_size": [1, 128]}, {**FP8, "activation_scheme": "static"}, "fp8"])
def test_random_models_run_whatever_form_config_json_names(tmp_path, quantization):
    """A form of 8-bit weights that is not read is no reason against random ones: they are what they are without it."""
    from conftest import TINY_B
    from torchinferno_b200.weights.loader import load_weights
    from torchinferno_b200.weights.random_init import build_model, init_random_weights, write_random_model
    config = {**TINY_B, "quantization_config": quantization}
    models = [build_model(c, dtype=torch.bfloat16, device="cpu") for c in (TINY_B, config, config)]
    init_random_weights(models[0], 0, config=TINY_B)
    init_random_weights(models[1], 0, config=config)
    load_weights(models[2], write_random_model(config, tmp_path, 0))
    downs = [m.blocks[0].feed_forward.down_weight.tensor for m in models]
    assert torch.equal(downs[0], downs[1]) and torch.equal(downs[0], downs[2])


def test_fused_projections_are_stored_alike(tmp_path):
    from conftest import TINY_B
    from torchinferno_b200.weights.loader import load_weights
    from torchinferno_b200.weights.random_init import build_model
    config = {**TINY_B, "quantization_config": {**FP8, "modules_to_not_convert": ["k_proj"]}}
    _folder(tmp_path, config)
    with pytest.raises(ValueError, match="all be stored in 8-bit blocks, or none"):
        load_weights(build_model(config, dtype=torch.bfloat16, device="cpu"), tmp_path)


def test_experts_are_bound_in_blocks():
    """Every design with routed experts takes them in blocks; gated ones as row pairs, the router never."""
    from giforax_configs import GA
    from torchinferno_b200.kernels.block_scaled import BlockScaledExperts
    from torchinferno_b200.weights.random_init import build_model, init_random_weights
    config = {**GA, "quantization_config": FP8}
    model = build_model(config, dtype=torch.bfloat16, device="cpu")
    init_random_weights(model, 1, config=config)
    moes = [b.feed_forward for b in model.blocks if type(b.feed_forward).__name__ == "RoutedExperts"]
    assert moes
    for moe in moes:
        assert isinstance(moe.up_weight, BlockScaledExperts) and moe.up_weight.paired == moe.glu and moe.up_weight.experts == moe.experts
        assert isinstance(moe.down_weight, BlockScaledExperts) and moe.router_weight.dtype == torch.float32
