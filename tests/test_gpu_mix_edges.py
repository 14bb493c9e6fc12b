"""Channel product at the edges of its size rules: few weights, few and ragged positions, channels far apart, results in the residual's place."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import EPS32, TYPES, product_bound, randn, rounding, wide, within
from test_gpu_mix import check_backward, check_forward, operands, quantized

pytestmark = pytest.mark.gpu

# fewer than eight weights, eight and a few more, contractions that leave one to seven entries of a step, around 1024 tiles of 64 x 16
SIZES = [(1, 1, 64), (2, 3, 1000), (3, 1, 70), (1, 7, 65), (2, 2, 70001), (1, 8, 64), (3, 3, 66), (4, 2, 129), (33, 5, 91), (39, 9, 64), (5, 17, 127),
         (31, 40, 16383), (40, 33, 65600), (96, 20, 40003), (70, 260, 2050)]


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,N,P", SIZES)
def test_forward_and_backward(kind, K, N, P):
    x, W, bias, residual = operands(kind, K, N, (P,), 500)
    z = torch.empty_like(residual)
    y = tf.mix(x, W, bias, residual, "silu", z=z)
    check_forward(y, z, x, W, bias, residual, "silu")
    gy = randn((N, P), TYPES[kind], 504)
    check_backward(gy, x, W, z, "silu", tf.mix_backward(gy, x, W, z=z, activation="silu"))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,N,P", [(1, 3, 66), (2, 2, 131), (9, 4, 100), (70, 30, 20001)])
def test_8bit(kind, K, N, P):
    dt = TYPES[kind]
    pair = (2,) if dt.is_complex else ()
    xq, xs = quantized(randn((K, P) + pair, torch.float32, 510), (0, -1) if pair else 0)
    Wq, ws = quantized(randn((N, K) + pair, torch.float32, 511), (1, -1) if pair else 1)
    xs, ws = xs.reshape(P).contiguous(), ws.reshape(N).contiguous()
    got = tf.mix_8bit(xq, xs, Wq, ws, dtype=dt)
    X, V = xq.cpu().double(), Wq.cpu().double()
    if pair:
        X, V = torch.view_as_complex(X), torch.view_as_complex(V)
    X, V = X * wide(xs), V * wide(ws)[:, None]
    bound = product_bound(V, X, K * (2 if pair else 1), 3 * EPS32)
    within(got, V @ X, bound + rounding(dt) * ((V @ X).abs() + bound), "y")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("P", [1, 3, 15, 16, 17, 31, 33, 63, 255, 257, 1023])
def test_weight_gradients_of_few_positions(kind, P):
    for K, N in ((5, 3), (33, 70)):
        x, gz = randn((K, P), TYPES[kind], 520), randn((N, P), TYPES[kind], 521)
        gW, gbias = tf.mix_weight_grad(gz, x)
        G, X = wide(gz), wide(x)
        exact, terms = G @ X.mH, P * (2 if G.is_complex() else 1)
        bound = product_bound(G, X.mH, terms)
        within(gW, exact, bound + rounding(gz.dtype) * (exact.abs() + bound), "gW")
        bound = (terms + 4) * EPS32 * G.abs().sum(1)
        within(gbias, G.sum(1), bound + rounding(gz.dtype) * (G.sum(1).abs() + bound), "gbias")


@pytest.mark.parametrize("kind", TYPES)
def test_channels_far_apart(kind):
    """rows of x 2^31 values apart, of the others 2^24 and more: beyond 32 bits, from the first channel on"""
    K, N, P, dt = 5, 4, 83, TYPES[kind]
    parts = 2 if dt.is_complex else 1
    x, W, bias, residual = operands(kind, K, N, (P,), 530)

    def apart(t, ld):
        wide_rows = torch.empty(((t.shape[0] - 1) * ld + P,), dtype=dt, device="cuda").as_strided(t.shape, (ld, 1))
        return wide_rows.copy_(t)
    xf, rf = apart(x, (1 << 31) // parts), apart(residual, (1 << 24) // parts + 3)
    y, z = apart(torch.zeros_like(residual), (1 << 25) // parts + 1), apart(torch.zeros_like(residual), 1 << 24)
    tf.mix(xf, W, bias, rf, "gelu_tanh", y=y, z=z)
    check_forward(y, z, x, W, bias, residual, "gelu_tanh")
    gy = apart(randn((N, P), dt, 535), (1 << 24) + 7)
    gx = apart(torch.zeros_like(x), (1 << 31) // parts)
    check_backward(gy, xf, W, z, "gelu_tanh", tf.mix_backward(gy, xf, W, z=z, activation="gelu_tanh", gx=gx))
    del xf, rf, y, z, gy, gx
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind", TYPES)
def test_channels_almost_as_far_apart_as_32_bits_reach(kind):
    """24 rows of x, or 12 complex ones or rows of the results, just below 2^32 bytes apart, and sizes of the resident kernel"""
    K, N, P, dt = 40, 64, 20003, TYPES[kind]
    x, W, bias, residual = operands(kind, K, N, (P,), 550)
    size = 8 if dt.is_complex else 4 if dt == torch.float32 else 2
    ldx, ldy = ((1 << 32) - 8192) // (24 * size if not dt.is_complex else 12 * size), ((1 << 32) - 8192) // (12 * size)

    def apart(t, ld):
        return torch.empty(((t.shape[0] - 1) * ld + P,), dtype=dt, device="cuda").as_strided(t.shape, (ld, 1)).copy_(t)
    xf, y = apart(x, ldx), apart(torch.zeros_like(residual), ldy)
    z = torch.empty_like(residual)
    tf.mix(xf, W, bias, residual, "silu", y=y, z=z)
    check_forward(y, z, x, W, bias, residual, "silu")
    del y
    gy, gx = randn((N, P), dt, 555), apart(torch.zeros_like(x), ldx)
    check_backward(gy, x, W, z, "silu", tf.mix_backward(gy, xf, W, z=z, activation="silu", gx=gx))
    del xf, gx
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,N,P", [(8, 5, 33), (8, 5, 130), (40, 70, 20003)])
def test_residual_in_place_at_the_last_columns(kind, K, N, P):
    x, W, bias, residual = operands(kind, K, N, (P,), 540)
    y = residual.clone()
    tf.mix(x, W, bias, y, "silu", y=y)
    check_forward(y, None, x, W, bias, residual, "silu")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("activation", ["relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("K,N,P", [(200, 40, 6001), (520, 33, 4097), (140, 300, 20001)])
def test_gradients_of_many_channels(kind, activation, K, N, P):
    """sizes at which gz is formed by itself; rows that start anywhere and end inside a unit of 2048 columns, nothing written beside them"""
    dt = TYPES[kind]
    x, W = randn((K, P), dt, 560), randn((N, K), dt, 561, K ** -0.5)
    gy, z = randn((N, P + 5), dt, 562)[:, 2:2 + P], randn((N, P + 3), dt, 563)[:, 1:1 + P]
    gz, gx = torch.full((N, P + 7), 7.0, dtype=dt, device="cuda"), torch.full((K, P + 9), 7.0, dtype=dt, device="cuda")
    results = tf.mix_backward(gy, x, W, z=z, activation=activation, gz=gz[:, 3:3 + P], gx=gx[:, 5:5 + P])
    check_backward(gy, x, W, z, activation, results)
    for t, lo in ((gz, 3), (gx, 5)):
        assert (t[:, :lo] == 7).all() and (t[:, lo + P:] == 7).all()
