"""Root-mean-square norm over channels with the residual's addition, its 8-bit result and its gradient, against 64-bit evaluations."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import EPS32, TYPES, randn, rounding, wide, within

pytestmark = pytest.mark.gpu

# K, positions: one channel, sizes around what lanes, waves and registers hold (32, 64, 128, 256, 512 channels), strips that end inside
SIZES = [(1, (1,)), (4, (3,)), (31, (65,)), (32, (256,)), (33, (7, 19)), (64, (1000,)), (65, (129,)), (128, (31,)), (129, (515,)), (256, (70,)),
         (300, (100,)), (513, (67,)), (1000, (33,)), (20, (140001,))]


def square(t):
    return t.abs() ** 2


def expected(x, gain, residual, eps=1e-6):
    s = wide(x).flatten(1)
    if residual is not None:
        s = s + wide(residual).flatten(1)
    rstd = 1 / torch.sqrt(square(s).mean(0) + eps)
    return s, rstd, s * rstd * wide(gain)[:, None]


def operands(kind, K, places, seed=0, residual=True):
    dt = TYPES[kind]
    return randn((K,) + places, dt, seed), 1 + 0.2 * randn((K,), torch.float32, seed + 1), randn((K,) + places, dt, seed + 2) if residual else None


# a sum of squares of K terms in 32 bits is off by at most (K + 3) roundings of itself, its root by half of that
def relative(K):
    return (K + 16) * EPS32


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,places", SIZES)
@pytest.mark.parametrize("residual", [True, False])
def test_forward(kind, K, places, residual):
    x, gain, r = operands(kind, K, places, 0, residual)
    y, s, rstd = tf.rms_norm(x, gain, r)
    S, R, Y = expected(x, gain, r)
    assert rstd.shape == torch.Size(places) and (residual or s is x)
    within(s.flatten(1), S, 1.01 * (rounding(x.dtype) + EPS32) * S.abs(), "s")
    within(rstd.flatten(), R, relative(K) * R, "rstd")
    within(y.flatten(1), Y, (relative(K) + 1.01 * rounding(x.dtype)) * Y.abs() + 2 * EPS32 * (Y / S).abs().nan_to_num() * (wide(x).flatten(1).abs()), "y")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,places", SIZES)
def test_8bit(kind, K, places):
    x, gain, r = operands(kind, K, places, 3)
    q, scale, s = tf.rms_norm_8bit(x, gain, r)
    S, _, Y = expected(x, gain, r)
    y_parts = torch.view_as_real(Y) if Y.is_complex() else Y[..., None]
    most = y_parts.abs().amax(dim=(0, 2))
    noise = relative(K) + 8 * EPS32 * (wide(x).abs().flatten(1).amax() / S.abs().amax())
    within(scale.flatten(), most / 448, 4 * noise * most / 448, "scale")
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape + ((2,) if x.is_complex() else ())
    got = q.cpu().double().reshape(K, -1, 2 if x.is_complex() else 1)
    exact = y_parts / (most / 448)[None, :, None]
    # e4m3: half a step is 2^-4 of a number, 2^-10 below 2^-6
    bound = exact.abs() * 2.0 ** -4 * (1 + 2.0 ** -10) + 2.0 ** -10
    assert ((got - exact).abs() <= bound).all() and got.abs().max() == 448
    assert torch.equal(s, tf.rms_norm(x, gain, r)[1])
    # and the nearest of the type's numbers, except where rounding may tip a tie
    near = (exact.clamp(-448, 448)).to(torch.float32).to(torch.float8_e4m3fn).double()
    assert (near != got).double().mean() <= 1e-3 or got.numel() < 2000


@pytest.mark.parametrize("kind", TYPES)
def test_8bit_ends(kind):
    """positions of zeros, of one value, of values too small for a scale, and of values that are not finite"""
    dt = TYPES[kind]
    x = torch.zeros((40, 80), dtype=dt, device="cuda")
    x[7, 1] = -3.0
    x[:, 2] = 1e-38
    x[5, 3] = float("nan")
    x[6, 4] = float("inf")
    x[:, 66] = 2.0
    gain = torch.ones(40, device="cuda")
    q, scale, _ = tf.rms_norm_8bit(x, gain)
    v = q.float().reshape(40, 80, -1)
    assert (v[:, 0] == 0).all() and scale[0] == 1
    assert v[7, 1, 0] == -448 and (v.reshape(40, 80, -1)[:7, 1] == 0).all()
    assert torch.isfinite(v[:, 2]).all() and torch.isfinite(scale[2])
    assert torch.isnan(scale[3:5]).all() and torch.isnan(v[5, 3, 0]) and torch.isnan(v[6, 4, 0])
    assert (v[:, 66, 0] == 448).all()
    assert (v[:, 5:66] == 0).all() and (v[:, 67:] == 0).all()
    y, _, rstd = tf.rms_norm(x, gain)
    assert torch.isnan(rstd[3]) and rstd[4] == 0 and (y[:, 0] == 0).all()


@pytest.mark.parametrize("kind", TYPES)
def test_in_place_and_channels_apart(kind):
    dt = TYPES[kind]
    for K, P in ((50, 333), (600, 70)):
        x, gain, r = operands(kind, K, (P,), 9)
        y, s, rstd = tf.rms_norm(x, gain, r)
        stream = r.clone()
        y2, s2, _ = tf.rms_norm(x, gain, stream, s=stream)
        assert s2 is stream and torch.equal(stream, s) and torch.equal(y2, y)
        both, kept = x.clone(), r.clone()
        tf.rms_norm(both, gain, kept, y=both, s=kept)
        assert torch.equal(both, y) and torch.equal(kept, s)
        q, scale, _ = tf.rms_norm_8bit(x, gain, r)
        for shift in range(1, 5):
            wide_x = torch.full((K, P + 9), 7.0, dtype=dt, device="cuda")
            wide_x[:, shift:shift + P] = x
            out, sums = (torch.full((K, P + 5), 7.0, dtype=dt, device="cuda") for _ in range(2))
            tf.rms_norm(wide_x[:, shift:shift + P], gain, r, y=out[:, 2:2 + P], s=sums[:, shift:shift + P])
            assert torch.equal(out[:, 2:2 + P], y) and torch.equal(sums[:, shift:shift + P], s)
            assert (out[:, :2] == 7).all() and (out[:, 2 + P:] == 7).all() and (sums[:, :shift] == 7).all() and (sums[:, shift + P:] == 7).all()
            pair = (2,) if dt.is_complex else ()
            bytes_ = torch.zeros((K, P + 6) + pair, dtype=torch.float8_e4m3fn, device="cuda")
            tf.rms_norm_8bit(wide_x[:, shift:shift + P], gain, r, q=bytes_[:, shift:shift + P])
            raw = bytes_.view(torch.uint8)
            assert torch.equal(raw[:, shift:shift + P], q.view(torch.uint8)) and (raw[:, :shift] == 0).all() and (raw[:, shift + P:] == 0).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,places", SIZES)
@pytest.mark.parametrize("stream", [True, False])
def test_backward(kind, K, places, stream):
    dt = TYPES[kind]
    s, gy, gain = randn((K,) + places, dt, 1), randn((K,) + places, dt, 2), 1 + 0.2 * randn((K,), torch.float32, 3)
    gs = randn((K,) + places, dt, 4) if stream else None
    rstd = (1 / torch.sqrt(square(s.to(torch.complex64 if dt.is_complex else torch.float32)).mean(0) + 1e-6)).float()
    gx, ggain = tf.rms_norm_backward(gy, s, gain, rstd, gs)
    S, G, g, R = wide(s).flatten(1), wide(gy).flatten(1), wide(gain)[:, None], wide(rstd).flatten()
    along, size = (S.conj() * G).real, S.abs() * G.abs()
    E = R * g * G - R ** 3 * (g * along).mean(0) * S
    mags = R * (g * G).abs() + R ** 3 * (g.abs() * size).mean(0) * S.abs()
    if stream:
        E, mags = E + wide(gs).flatten(1), mags + wide(gs).flatten(1).abs()
    within(gx.flatten(1), E, relative(K) * mags + 1.01 * rounding(dt) * (E.abs() + relative(K) * mags), "gx")
    P = S.shape[1]
    # sums of at most 64 columns' products per lane and strip, added over lanes and blocks: fewer than 2048 roundings in a row
    within(ggain, (along * R).sum(1), (min(P, 2048) + 16) * EPS32 * (size * R).sum(1), "ggain")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K", [40, 700])
def test_backward_in_place(kind, K):
    dt, P = TYPES[kind], 203
    s, gy, gs, gain = (randn((K, P), dt, i) for i in (1, 2, 3)), None, None, randn((K,), torch.float32, 4)
    s, gy, gs = s
    rstd = torch.rand(P, device="cuda") + 0.5
    gx, ggain = tf.rms_norm_backward(gy, s, gain, rstd, gs)
    for which in range(3):
        ops = [gy.clone(), s.clone(), gs.clone()]
        got, ggain2 = tf.rms_norm_backward(ops[0], ops[1], gain, rstd, ops[2], gx=ops[which])
        assert got is ops[which] and torch.equal(got, gx) and torch.equal(ggain2, ggain)
    apart = torch.full((K, P + 5), 7.0, dtype=dt, device="cuda")
    tf.rms_norm_backward(gy, s, gain, rstd, gs, gx=apart[:, 3:3 + P])
    assert torch.equal(apart[:, 3:3 + P], gx) and (apart[:, :3] == 7).all() and (apart[:, 3 + P:] == 7).all()


@pytest.mark.parametrize("kind", ["c64", "f32"])
def test_gradient_against_differences(kind):
    dt, K, P, h = TYPES[kind], 24, 50, 2.0 ** -7
    x, gain, r = operands(kind, K, (P,), 7)
    c, cs = randn((K, P), dt, 8), randn((K, P), dt, 9)

    def loss(x, gain, r):
        y, s, _ = tf.rms_norm(x, gain, r)
        return ((wide(c).conj() * wide(y)).real.sum() + (wide(cs).conj() * wide(s)).real.sum()).item()
    _, s, rstd = tf.rms_norm(x, gain, r)
    gx, ggain = tf.rms_norm_backward(c, s, gain, rstd, cs)
    ops = [x, gain, r]
    for i, g in enumerate((gx, ggain, gx)):
        d = randn(ops[i].shape, ops[i].dtype, 20 + i)
        shifted = lambda t: loss(*[o + t * h * d if j == i else o for j, o in enumerate(ops)])  # noqa: E731
        along = (wide(g).conj() * wide(d)).real.sum().item()
        assert abs((shifted(1) - shifted(-1)) / (2 * h) - along) <= 5e-3 * wide(g).abs().norm().item() * wide(d).abs().norm().item(), i


def test_norm_feeds_the_8bit_product():
    """rms_norm_8bit -> mix_8bit against the product of the unrounded norm: e4m3 keeps 2^-4 of a number"""
    for kind, dt in TYPES.items():
        K, N, P = 48, 32, 500
        x, gain, r = operands(kind, K, (P,), 30)
        W = randn((N, K), dt, 31, K ** -0.5)
        parts = torch.view_as_real(W) if dt.is_complex else W.float()
        ws = (parts.flatten(1).abs().amax(1) / 448).contiguous()
        Wq = (parts / ws.reshape((N,) + (1,) * (parts.dim() - 1))).to(torch.float8_e4m3fn)
        q, scale, _ = tf.rms_norm_8bit(x, gain, r)
        y = tf.mix_8bit(q, scale, Wq, ws, dtype=dt)
        _, _, Y = expected(x, gain, r)
        exact = wide(W) @ Y
        assert (wide(y) - exact).abs().norm() <= 2.0 ** -4 * exact.abs().norm()


def test_no_positions():
    for dt in TYPES.values():
        x, gain = torch.empty((5, 0), dtype=dt, device="cuda"), torch.ones(5, device="cuda")
        y, s, rstd = tf.rms_norm(x, gain)
        assert y.shape == (5, 0) and rstd.shape == (0,)
        gx, ggain = tf.rms_norm_backward(x, x, gain, rstd, ggain=torch.ones(5, device="cuda"))
        assert (ggain == 0).all()


def test_refusals():
    x, gain = randn((6, 20), torch.float32, 1), torch.ones(6, device="cuda")
    with pytest.raises(ValueError, match="gain has shape"):
        tf.rms_norm(x, gain[:5])
    with pytest.raises(TypeError, match="gain must be"):
        tf.rms_norm(x, gain.double())
    with pytest.raises(TypeError, match="gain must be"):
        tf.rms_norm(x, None)
    with pytest.raises(tf.TurboFNOError, match="eps"):
        tf.rms_norm(x, gain, eps=-1.0)
    shared = randn((7, 20), torch.float32, 2)
    with pytest.raises(tf.TurboFNOError, match="without being it"):
        tf.rms_norm(shared[:6], gain, y=shared[1:])
    with pytest.raises(tf.TurboFNOError, match="the results overlap"):
        y = torch.empty_like(x)
        tf.rms_norm(x, gain, x.clone(), y=y, s=y)
    with pytest.raises(ValueError, match="rstd has shape"):
        tf.rms_norm_backward(x, x.clone(), gain, torch.ones(19, device="cuda"))
    with pytest.raises(TypeError, match="float64"):
        tf.rms_norm(x.double(), gain)


@pytest.mark.parametrize("K", [40, 130, 300])
def test_channels_further_apart_than_32_bits_of_an_offset(K):
    """2^28 values between channels: what lies between them is never touched"""
    P, ld = 100, (1 << 28) + 8
    x, gain, r = operands("bf16", K, (P,), 11)
    y, s, rstd = tf.rms_norm(x, gain, r)
    q, scale, _ = tf.rms_norm_8bit(x, gain, r)
    gx, ggain = tf.rms_norm_backward(x, s, gain, rstd, r)
    far = torch.empty((K, ld), dtype=torch.bfloat16, device="cuda")[:, 3:3 + P]
    far.copy_(x)
    y2, s2, _ = tf.rms_norm(far, gain, r)
    q2, scale2, _ = tf.rms_norm_8bit(far, gain, r)
    gx2, ggain2 = tf.rms_norm_backward(far, s, gain, rstd, r)
    # other kernels may run there, whose sums have another order: each is off by at most relative(K), and a rounding to bf16 may go the other way
    near = lambda a, b, what: within(a, wide(b), (2 * relative(K) + 2 * rounding(b.dtype)) * wide(b).abs().clamp_min(1e-3), what)  # noqa: E731
    assert torch.equal(s, s2)
    near(y2, y, "y")
    near(scale2, scale, "scale")
    near(gx2, gx, "gx")
    assert ((q2.float() - q.float()).abs() <= 2.0 ** -3 * q.float().abs() + 2.0 ** -9).all()
    within(ggain2, wide(ggain), 300 * EPS32 * ((wide(x) * wide(s)).abs() * wide(rstd)).sum(1), "ggain")
    near(tf.rms_norm(x, gain, r, y=far)[0], y, "y")
