"""Root-mean-square norm at the ends of the range: positions of zeros and of the smallest numbers between ordinary ones, gains of any size."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import EPS32, TYPES, randn, rounding, wide

pytestmark = pytest.mark.gpu

# channels held in narrow and wide strips, and channels that are read twice; strips that end inside
SIZES = [(3, 70), (40, 90), (200, 75), (600, 66), (30, 140003), (100, 140003), (300, 140003)]
GAINS = [1.0, 256.0, -256.0, 1e4, -1e4, 1e-3, 0.0, 1e9]


def check_8bit(x, gain, eps=1e-6, root=0.0):
    """q and scale against the definition in 64 bits: scale = max |y| / 448, or 1 where that is below the normal numbers. root: what
    the root of the mean is off by beside its roundings"""
    K = x.shape[0]
    q, scale, _ = tf.rms_norm_8bit(x, gain, eps=eps)
    S = wide(x)
    Y = S / torch.sqrt((S.abs() ** 2).mean(0) + eps) * wide(gain)[:, None]
    parts = torch.view_as_real(Y) if Y.is_complex() else Y[..., None]
    S = torch.view_as_real(S) if S.is_complex() else S[..., None]
    most = parts.abs().amax(dim=(0, 2))
    exact = torch.where(most / 448 < 2.0 ** -126, torch.ones_like(most), most / 448)
    assert not ((most / 448 / 2.0 ** -126 - 1).abs() < 0.01).any()          # which of the two it is does not hang on a rounding
    # the largest s gain is known to half of the smallest number, 2^-149, the rest is a sum of K squares and a few roundings
    largest = (S * wide(gain)[:, None, None]).abs().amax(dim=(0, 2))
    noise = (K + 24) * EPS32 + 2.0 ** -149 / largest.clamp_min(2.0 ** -149) + root
    assert ((wide(scale) - exact).abs() <= noise * exact).all(), ((wide(scale) - exact).abs() / exact).max()
    want = parts / exact[None, :, None]
    got = q.cpu().double().reshape(want.shape)
    assert ((got - want).abs() <= want.abs() * (2.0 ** -4 * (1 + 2.0 ** -10) + noise[None, :, None]) + 2.0 ** -10).all()
    assert (got[:, exact == 1] == 0).all() and (got.abs().amax(dim=(0, 2))[most / 448 >= 2.0 ** -126] == 448).all()
    return q, scale


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,P", SIZES)
def test_8bit_small_positions_and_large_gains(kind, K, P):
    dt = TYPES[kind]
    x, gain = randn((K, P), dt, 1), torch.tensor([GAINS[k % len(GAINS)] for k in range(K)], device="cuda")
    sizes = [0.0, 1e-20, 1e-29, 1e-30, 1e-33, 1e-34, 1e-36, 1e-37, 1e-38, 1e-43, 1.0, 1e10]
    for i, size in enumerate(sizes):                    # at the first columns, and at the last ones
        x[:, i] = x[:, i] * size
        x[:, P - 1 - 2 * i] = x[:, P - 1 - 2 * i] * size
    q, scale = check_8bit(x, gain)
    assert (q[:, 0].float() == 0).all() and scale[0] == 1 and scale[P - 1] == 1
    check_8bit(x, torch.ones_like(gain))
    # one channel alone, and the zeros of the others under the largest gain
    x[:, 20] = 0
    x[K - 1, 20] = 1e-29
    check_8bit(x, gain)


def test_8bit_position_of_zeros_through_the_product():
    """a masked position leaves bias and residual of the product that reads it"""
    K, N, P = 40, 24, 100
    x, gain = randn((K, P), torch.bfloat16, 1), torch.full((K,), 300.0, device="cuda")
    x[:, 17] = 0
    q, scale, _ = tf.rms_norm_8bit(x, gain)
    Wq, bias = randn((N, K), torch.float32, 2).to(torch.float8_e4m3fn), randn((N,), torch.bfloat16, 3)
    y = tf.mix_8bit(q, scale, Wq, torch.ones(N, device="cuda"), bias=bias)
    assert torch.equal(y[:, 17], bias) and torch.isfinite(y).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,P", [(3, 70), (40, 90), (600, 66), (100, 140003)])
def test_small_positions_without_eps(kind, K, P):
    """means of squares down to the smallest numbers: 2^-149 / mean of themselves is what they may be off by"""
    dt = TYPES[kind]
    x, gain = randn((K, P), dt, 4), 1 + 0.2 * randn((K,), torch.float32, 5)
    for i, size in enumerate((1e-10, 1e-17, 1e-18, 1e-19, 3e-20, 1e-20)):
        x[:, i] = x[:, i] * size
        x[:, P - 1 - 2 * i] = x[:, P - 1 - 2 * i] * size
    y, s, rstd = tf.rms_norm(x, gain, eps=0.0)
    S = wide(x)
    mean = (S.abs() ** 2).mean(0)
    R = 1 / torch.sqrt(mean)
    # of a mean of K squares, each of which and the mean itself may be rounded to a multiple of 2^-149 (real and imaginary parts: twice); half of it in the root
    noise = (K + 16) * EPS32 + 3 * 2.0 ** -149 / mean
    assert ((wide(rstd) - R).abs() <= noise * R).all(), ((wide(rstd) - R).abs() / R / noise).max()
    Y = S * R * wide(gain)[:, None]
    assert ((wide(y) - Y).abs() <= (noise + 1.01 * rounding(dt)) * Y.abs()).all()
    check_8bit(x, gain, eps=0.0, root=3 * 2.0 ** -149 / mean)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,P", [(3, 70), (40, 90), (300, 66), (100, 140003), (200, 70001)])
def test_gradient_of_small_positions_without_eps(kind, K, P):
    """rstd up to 1e19, whose cube is no float: the gradient is, wherever it is one"""
    dt = TYPES[kind]
    s, gy, gain = randn((K, P), dt, 6), randn((K, P), dt, 7), 1 + 0.2 * randn((K,), torch.float32, 8)
    for i, size in enumerate((1e-10, 1e-13, 1e-15, 1e-18, 1e-19)):
        s[:, i] = s[:, i] * size
        s[:, P - 1 - 2 * i] = s[:, P - 1 - 2 * i] * size
    rstd = (1 / torch.sqrt((s.to(torch.complex128 if dt.is_complex else torch.float64).abs() ** 2).mean(0))).float()
    gx, ggain = tf.rms_norm_backward(gy, s, gain, rstd)
    S, G, g, R = wide(s), wide(gy), wide(gain)[:, None], wide(rstd)
    along, size = (S.conj() * G).real, S.abs() * G.abs()
    E = R * g * G - R ** 3 * (g * along).mean(0) * S
    mags = R * (g * G).abs() + R ** 3 * (g.abs() * size).mean(0) * S.abs()
    assert ((wide(gx) - E).abs() <= (K + 16) * EPS32 * mags + 1.01 * rounding(dt) * (E.abs() + (K + 16) * EPS32 * mags)).all()
    assert ((wide(ggain) - (along * R).sum(1)).abs() <= (min(P, 2048) + 16) * EPS32 * (size * R).sum(1)).all()
