"""The kernels that the size rules choose between, each at sizes that reach it: contractions held in registers in 16 and 8 bits with every number of steps, more tiles
than there are waves; the direct kernel with 32 and 64 rows; wide strips of the norm. Against 64-bit evaluations on the GPU."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import EPS16, EPS32, TYPES, act, by_parts, product_bound, randn, rounding, slope

pytestmark = pytest.mark.gpu


def wide(t):
    return t.to(torch.complex128 if t.is_complex() else torch.float64)


def within(got, exact, bound, what):
    assert got.shape == exact.shape
    off = ((wide(got) - exact).abs() - bound).max().item()
    assert off <= 0, "%s: %g over its bound" % (what, off)


def check_forward(y, z, Z, bound, activation, dt):
    """Z: z in 64 bits, off by `bound` before its last rounding"""
    if z is not None:
        within(z, Z, bound + rounding(dt) * (Z.abs() + bound), "z")
    bound = 1.13 * bound + (2.0 ** -20 * Z.abs() if activation != "none" else 0)
    Y = act(activation, Z)
    within(y, Y, bound + 1.01 * rounding(dt) * (Y.abs() + bound), "y")


def check_input_gradient(gx, gz, gy, W, z, activation):
    dt, G, VH = gy.dtype, wide(gy), wide(W).mH.contiguous()
    GZ = by_parts(lambda g, s: g * s, G, slope(activation, wide(z))) if activation != "none" else G
    inside = 2.0 ** -19 * G.abs() if activation != "none" else 0 * G.abs()
    within(gz, GZ, inside + 1.01 * rounding(dt) * (GZ.abs() + inside), "gz")
    own = 1.01 * EPS16 if dt == torch.bfloat16 and activation != "none" else 0.0
    bound = product_bound(VH, GZ, W.shape[0] * (2 if dt.is_complex else 1), own) + VH.abs() @ inside
    E = VH @ GZ
    within(gx, E, bound + 1.01 * rounding(dt) * (E.abs() + bound), "gx")


def quantized(shape, pair, seed, dim):
    t = randn(shape + pair, torch.float32, seed)
    dims = (dim, -1) if pair else (dim,)
    scale = t.abs().amax(dim=dims, keepdim=True) / 448
    return (t / scale).to(torch.float8_e4m3fn), scale.flatten().contiguous()


def check_8bit(kind, xq, xs, Wq, ws, residual, P):
    dt = TYPES[kind]
    y = tf.mix_8bit(xq, xs, Wq, ws, residual=residual, activation="silu", dtype=dt)
    X, V = xq.double(), Wq.double()
    if dt.is_complex:
        X, V = torch.view_as_complex(X), torch.view_as_complex(V)
    X, V = X * xs.double(), V * ws.double()[:, None]
    Z = V @ X + wide(residual)
    bound = product_bound(V, X, X.shape[0] * (2 if dt.is_complex else 1)) + 5 * EPS32 * (Z.abs() + wide(residual).abs())
    check_forward(y, None, Z, bound, "silu", dt)


# real channels of the contraction: 1 to 8 steps of 32, the last one not whole, and where it is
STEPS = [20, 33, 72, 100, 129, 160, 190, 200, 224, 250, 256]


@pytest.mark.parametrize("K", STEPS)
@pytest.mark.parametrize("N,P", [(200, 140003), (72, 140064), (20, 140003)])
def test_held_steps_16_bits(K, N, P):
    x, W = randn((K, P), torch.bfloat16, 1), randn((N, K), torch.bfloat16, 2, K ** -0.5)
    bias, residual = randn((N,), torch.bfloat16, 3), randn((N, P), torch.bfloat16, 4)
    z = torch.empty_like(residual)
    y = tf.mix(x, W, bias, residual, "silu", z=z)
    Z = wide(W) @ wide(x) + wide(bias)[:, None] + wide(residual)
    bound = product_bound(wide(W), wide(x), K) + 3 * EPS32 * (Z.abs() + wide(bias).abs()[:, None])
    check_forward(y, z, Z, bound, "silu", torch.bfloat16)


@pytest.mark.parametrize("activation", ["none", "gelu_tanh"])
@pytest.mark.parametrize("N", STEPS)
@pytest.mark.parametrize("K,P", [(100, 140003), (72, 140064), (40, 140003), (20, 140003), (20, 50)])
def test_held_steps_of_the_gradient_16_bits(N, K, P, activation):
    gy, z, W = randn((N, P), torch.bfloat16, 5), randn((N, P), torch.bfloat16, 6), randn((N, K), torch.bfloat16, 7, N ** -0.5)
    gx, gz = tf.mix_input_grad(gy, W, z=z, activation=activation)
    check_input_gradient(gx, gz, gy, W, z, activation)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K", STEPS)
@pytest.mark.parametrize("N,P", [(200, 140004), (72, 140064), (20, 140004)])
def test_held_steps_8_bits(kind, K, N, P):
    dt, pair = TYPES[kind], (2,) if TYPES[kind].is_complex else ()
    if pair:
        K, P = (K + 1) // 2, P // 2
    xq, xs = quantized((K, P), pair, 8, 0)
    Wq, ws = quantized((N, K), pair, 9, 1)
    check_8bit(kind, xq, xs, Wq, ws, randn((N, P), dt, 10), P)


def apart(t, values):
    """rows of t that many real values apart: too far for 32 bits of a lane's offset, which the direct kernel takes"""
    ld = values // (2 if t.is_complex() else 1)
    buffer = torch.empty(((t.shape[0] - 1) * ld + t[0].numel(),), dtype=t.dtype, device="cuda")
    return buffer.as_strided(t.shape, (ld,) + t.stride()[1:]).copy_(t)


FAR = {"c64": (1 << 32) // 48, "f32": (1 << 32) // 96, "bf16": (1 << 32) // 48, "8bit": (1 << 32) // 24 * 2 + 2}


# 40 rows: three times 16; up to 2048 tiles of 64 x 16 in 32 rows, then in 64
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("columns", [25003, 45004])
@pytest.mark.parametrize("K", [20, 70])
def test_direct_kernel_of_many_rows(kind, columns, K):
    dt, N = TYPES[kind], 40
    parts = 2 if dt.is_complex else 1
    P = columns // parts
    x, W, residual = randn((K, P), dt, 11), randn((N, K), dt, 12, K ** -0.5), randn((N, P), dt, 13)
    far, z = apart(x, FAR[kind] + 64), torch.empty_like(residual)
    y = tf.mix(far, W, residual=residual, activation="gelu_tanh", z=z)
    Z = wide(W) @ wide(x) + wide(residual)
    check_forward(y, z, Z, product_bound(wide(W), wide(x), parts * K) + 3 * EPS32 * Z.abs(), "gelu_tanh", dt)
    print("gradient", flush=True)
    V = W.t().contiguous()                              # [K][N]: sums over the K far channels, 40 results
    pre = randn((K, P), dt, 14)
    for activation in ("none", "silu"):
        gx, gz = tf.mix_input_grad(far, V, z=pre, activation=activation)
        check_input_gradient(gx, gz, x, V, pre, activation)
    del far
    torch.cuda.empty_cache()
    print("8 bits", flush=True)
    pair = (2,) if parts == 2 else ()
    xq, xs = quantized((K, P), pair, 15, 0)
    Wq, ws = quantized((N, K), pair, 16, 1)
    far = torch.empty((K - 1) * FAR["8bit"] + 2 * P, dtype=torch.float8_e4m3fn, device="cuda").as_strided(xq.shape, (FAR["8bit"],) + xq.stride()[1:]).copy_(xq)
    check_8bit(kind, far, xs, Wq, ws, residual, P)
    del far
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K", [7, 32, 33, 64, 100, 128, 200, 256, 300, 512, 600])
def test_wide_strips_of_the_norm(kind, K):
    """from 2^17 real columns on; the last strip is not whole"""
    dt = TYPES[kind]
    P = 140003 // (2 if dt.is_complex else 1)
    x, r, gain = randn((K, P), dt, 17), randn((K, P), dt, 18), 1 + 0.2 * randn((K,), torch.float32, 19)
    relative = (K + 16) * EPS32
    y, s, rstd = tf.rms_norm(x, gain, r)
    S, g = wide(x) + wide(r), gain.double()[:, None]
    R = 1 / torch.sqrt((S.abs() ** 2).mean(0) + 1e-6)
    Y = S * R * g
    of_sum = 2 * EPS32 * (Y / S).abs().nan_to_num() * wide(x).abs()
    within(s, S, 1.01 * (rounding(dt) + EPS32) * S.abs(), "s")
    within(rstd, R, relative * R, "rstd")
    within(y, Y, (relative + 1.01 * rounding(dt)) * Y.abs() + of_sum, "y")
    q, scale, _ = tf.rms_norm_8bit(x, gain, r)
    parts = torch.view_as_real(Y) if dt.is_complex else Y[..., None]
    most = parts.abs().amax(dim=(0, 2)) / 448
    noise = relative + 8 * EPS32 * (wide(x).abs().amax() / S.abs().amax())
    within(scale, most, 4 * noise * most, "scale")
    exact = parts / most[None, :, None]
    got = q.double().reshape(exact.shape)
    assert ((got - exact).abs() <= exact.abs() * 2.0 ** -4 * (1 + 2.0 ** -10) + 2.0 ** -10).all() and got.abs().max() == 448
    G, R = wide(r), rstd.double()
    S = wide(s)                                         # what the gradient reads
    gx, ggain = tf.rms_norm_backward(r, s, gain, rstd, x)
    along, size = (S.conj() * G).real, S.abs() * G.abs()
    E = R * g * G - R ** 3 * (g * along).mean(0) * S + wide(x)
    mags = R * (g * G).abs() + R ** 3 * (g.abs() * size).mean(0) * S.abs() + wide(x).abs()
    within(gx, E, relative * mags + 1.01 * rounding(dt) * (E.abs() + relative * mags), "gx")
    # sums of at most 64 columns' products per lane and strip, over the strips of a block, lanes and blocks: fewer than 2048 roundings in a row
    within(ggain, (along * R).sum(1), (2048 + 16) * EPS32 * (size * R).sum(1), "ggain")
