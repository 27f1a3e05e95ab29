"""8-bit block-scaled weights on the host: their checks, their layout, their quantisation."""
import pytest
import torch

from block_scaled_oracle import matrix64, random_matrix, rows64
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
