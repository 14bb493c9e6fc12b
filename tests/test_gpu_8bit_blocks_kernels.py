"""The kernels that the size rules of the product in 8 bits with scales by blocks choose between, each at sizes that reach it, with contractions that end with a step, inside
one, and before the first: against 64-bit evaluations, in place, between neighbours, and with scales whose product is no normal number."""
import pytest
import torch

import turbofno_amd as tf
from layer_norm_reference import Product, rounded, within
from operators_reference import EPS32, TYPES, act, randn
from test_gpu_8bit_blocks import SUMS_8BIT, product_operands

pytestmark = pytest.mark.gpu

# blocks of columns and rows decide: tiles of 128 rows (384 tiles or more), of 64 rows, waves that divide the steps (256 blocks of 64 x 16 or fewer), all of 64, fewer than 64 and
# fewer than four columns; complex: tiles of 64 and of 32 rows, and the same split
SHAPES = {
    "f32": [(256, 1030, 5637), (300, 1030, 5637), (100, 1030, 5637), (128, 256, 2049), (200, 70, 3000), (70, 513, 1030), (512, 200, 200), (1300, 40, 100), (900, 60, 63), (390, 300, 3), (65, 17, 1)],
    "c64": [(64, 500, 4100), (100, 500, 4100), (40, 500, 4100), (128, 200, 2049), (70, 30, 9000), (33, 200, 2049), (256, 100, 60), (300, 40, 32), (450, 60, 31), (100, 300, 2), (33, 9, 1)],
}
# whole steps and pieces of 16 columns: read into LDS directly, tiles of 128 rows from three steps on, tiles of 64 rows for one and two steps and for fewer columns
SHAPES["bf16"] = SHAPES["f32"] + [(384, 1030, 8208), (640, 520, 16400), (1024, 392, 16384), (512, 1030, 8064), (128, 1030, 8208), (256, 520, 16400), (384, 300, 1040), (640, 77, 3008),
                                  (896, 650, 528)]
# few tiles of 64 rows and many steps: two groups of waves with half of the steps each, an odd number of them too, the last one not whole
SHAPES["f32"] = SHAPES["f32"] + [(385, 300, 1001), (640, 100, 1001), (1100, 200, 700), (1024, 130, 2000)]
SHAPES["bf16"] = SHAPES["bf16"] + [(1024, 300, 1040), (1152, 130, 2000), (1200, 200, 1003), (1030, 500, 701), (1900, 260, 400), (2176, 300, 528)]
CASES = [(kind,) + shape for kind in TYPES for shape in SHAPES[kind]]


def check(kind, operands, activation, got, terms):
    """the sums' bound of 32 bits, with the fixed steps of numbers below 2^-126: 2^-149 in 32 bits, of which sums and scales round twice, and 2^-133 in bf16, whose rounding of a
    result z below 2^-134 to zero is right and off by all of z"""
    E = Product(*operands)
    bound = (terms + 12) * EPS32 * E.sizes + 4 * EPS32 * E.more + 2.0 ** -148
    if kind == "bf16":
        bound = bound + SUMS_8BIT * E.sizes
    bound = 1.13 * bound + (2.0 ** -20 * E.z.abs() if activation != "none" else 0)
    Y = act(activation, E.z)
    within(got, Y, rounded(Y, bound, TYPES[kind]) + (2.0 ** -134 if kind == "bf16" else 0), "y")


@pytest.mark.parametrize("kind,K,N,P", CASES)
def test_each_kernel(kind, K, N, P):
    operands = product_operands(kind, K, N, (P,), 3)
    terms = K * (2 if kind == "c64" else 1)
    y = tf.mix_8bit_blocks(*operands, activation="silu")
    check(kind, operands, "silu", y, terms)
    place = operands[5].clone()                         # the residual replaced: windows that share columns with their neighbours leave them alone
    tf.mix_8bit_blocks(*operands[:5], residual=place, activation="silu", y=place)
    assert torch.equal(place, y)
    xq, pair = operands[0], (2,) if kind == "c64" else ()
    if P % 16 == 0:                                     # channels a multiple of 16 bytes apart, as in the field itself
        apart = torch.full((K, P + 48) + pair, 448.0, device="cuda").to(torch.float8_e4m3fn)
        apart[:, 32:32 + P] = xq
        assert torch.equal(tf.mix_8bit_blocks(apart[:, 32:32 + P], *operands[1:], activation="silu"), y)
    apart = torch.full((K, P + 5) + pair, 448.0, device="cuda").to(torch.float8_e4m3fn)
    apart[:, 3:3 + P] = xq
    out = torch.full((N, P + 9), 7.0, dtype=y.dtype, device="cuda")
    tf.mix_8bit_blocks(apart[:, 3:3 + P], *operands[1:], activation="silu", y=out[:, 1:1 + P])
    assert torch.equal(out[:, 1:1 + P], y) and (out[:, :1] == 7).all() and (out[:, 1 + P:] == 7).all()


@pytest.mark.parametrize("kind,K,N,P", CASES)
def test_each_kernel_with_small_scales(kind, K, N, P):
    """one scale of x and one of W so small that their product is none, in a position and rows that the other sums have to be right beside"""
    xq, xscale, Wq, wscale, bias, _ = product_operands(kind, K, N, (P,), 9, residual=False)
    xscale, wscale = xscale.clone(), wscale.clone()
    xscale[:, P // 2] *= 2.0 ** -75
    wscale[-1] *= 2.0 ** -75
    operands = (xq, xscale, Wq, wscale, None, None)
    y = tf.mix_8bit_blocks(*operands, dtype=TYPES[kind])
    check(kind, operands, "none", y, K * (2 if kind == "c64" else 1))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("P", [1, 40, 200])
def test_channels_far_apart(kind, P):
    """48 channels of x, or twelve rows of the result, 2^32 bytes apart and more: views of one buffer"""
    K, N, dt, pair = 70, 20, TYPES[kind], (2,) if kind == "c64" else ()
    operands = product_operands(kind, K, N, (P,), 20)
    want = tf.mix_8bit_blocks(*operands, activation="relu")
    step = (1 << 32) // 48 + 17                         # bytes
    step -= step % 2
    xq = operands[0]
    far = torch.empty((K - 1) * step + 2 * P, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    x = far.as_strided((K, P) + pair, (step,) + ((2, 1) if pair else (1,)))
    x.copy_(xq)
    got = tf.mix_8bit_blocks(x, *operands[1:], activation="relu")
    check(kind, operands, "relu", got, K * (2 if pair else 1))
    del far, x
    step = ((1 << 32) // 12) // dt.itemsize + 5
    far = torch.empty((N - 1) * step + P, dtype=dt, device="cuda").as_strided((N, P), (step, 1))
    tf.mix_8bit_blocks(*operands, activation="relu", y=far)
    check(kind, operands, "relu", far, K * (2 if pair else 1))
    far.copy_(operands[5])
    tf.mix_8bit_blocks(*operands[:5], residual=far, activation="relu", y=far)
    check(kind, operands, "relu", far, K * (2 if pair else 1))
    assert (want - got).abs().max() <= 0.05 * want.abs().max()
    del far
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind", TYPES)
def test_one_block_of_channels_is_the_product_with_scales_per_position(kind):
    """up to 64 real values of the contraction: the same sums as mix_8bit with the scale of each block of rows"""
    for K, N, P in ((64, 300, 1000), (32, 17, 5), (3, 4, 2), (1, 1, 1)):
        if kind == "c64" and K > 32:
            continue
        xq, xscale, Wq, wscale, bias, residual = product_operands(kind, K, N, (P,), 40)
        y = tf.mix_8bit_blocks(xq, xscale, Wq, wscale, bias, residual, activation="gelu_tanh")
        same = tf.mix_8bit(xq, xscale[0], Wq, wscale[:, 0].repeat_interleave(128)[:N].contiguous(), bias, residual, activation="gelu_tanh")
        assert torch.equal(y, same)


@pytest.mark.parametrize("kind,K,N,P", CASES)
def test_scales_of_zero_and_none(kind, K, N, P):
    """a scale of zero takes its block out, infinite and NaN ones make their position or rows so, and nothing beside them"""
    xq, xscale, Wq, wscale, _, residual = product_operands(kind, K, N, (P,), 50, bias=False)
    xscale, wscale = xscale.clone(), wscale.clone()
    xscale[:, 0] = 0
    wscale[:, 0] = 0
    if P > 2:
        xscale[0, P // 2], xscale[0, P - 1] = float("nan"), float("inf")
    operands = (xq, xscale, Wq, wscale, None, residual)
    y = tf.mix_8bit_blocks(*operands)
    part = torch.view_as_real(y).sum(-1) if y.is_complex() else y
    if P > 2:
        assert not torch.isfinite(part[:, [P // 2, P - 1]]).any()
    kept = [p for p in range(P) if p not in ((P // 2, P - 1) if P > 2 else ())]
    assert torch.isfinite(part[:, kept]).all() and torch.equal(y[:, 0], residual[:, 0])
    if K <= 128:
        assert torch.equal(y[:128][:, kept], residual[:128][:, kept])
    few = (xq[:, kept], xscale[:, kept], Wq, wscale, None, residual[:, kept])
    check(kind, few, "none", y[:, kept], K * (2 if kind == "c64" else 1))


def test_on_two_streams_at_once():
    """calls of several kernels beside one another on two streams, each the result that it gives alone"""
    shapes = [("bf16", 256, 1030, 5637), ("f32", 512, 200, 200), ("c64", 100, 500, 4100), ("bf16", 900, 60, 63)]
    operands = [product_operands(kind, K, N, (P,), 60) for kind, K, N, P in shapes]
    want = [tf.mix_8bit_blocks(*o, activation="silu") for o in operands]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i, side in enumerate(sides):
        side.wait_stream(torch.cuda.current_stream())
    for turn in range(3):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                for n in range(len(operands)):
                    o = operands[(n + i) % len(operands)]
                    got.append(((n + i) % len(operands), tf.mix_8bit_blocks(*o, activation="silu")))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[n]) for n, y in got)


@pytest.mark.parametrize("kind,K,N,P", [("bf16", 384, 1030, 8208), ("bf16", 384, 300, 1040), ("bf16", 256, 1030, 5637), ("f32", 100, 1030, 5637), ("c64", 64, 500, 4100), ("bf16", 512, 200, 200)])
def test_each_kernel_in_a_graph(kind, K, N, P):
    """quantised and multiplied in a captured graph, replayed with other fields and eager calls in between: the eager result each time"""
    operands = product_operands(kind, K, N, (P,), 70)
    wide = torch.complex64 if kind == "c64" else torch.float32
    x, place = randn((K, P), wide, 71), operands[5].clone()
    q, scale = tf.quantise_8bit(x)
    y = torch.empty_like(operands[5])

    def run(q, scale, y):
        tf.quantise_8bit(x, q=q, scale=scale)
        tf.mix_8bit_blocks(q, scale, *operands[2:5], residual=place, activation="silu", y=y)
    run(q, scale, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(q, scale, y)
    for i in range(3):
        x.copy_(randn((K, P), wide, 80 + i))
        place.copy_(randn((N, P), place.dtype, 90 + i))
        want = torch.empty_like(y)
        run(torch.empty_like(q), torch.empty_like(scale), want)
        torch.cuda.synchronize()
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), i
