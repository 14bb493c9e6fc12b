"""Layer norm over channels with residual and dropout, its 8-bit result and its gradient, against 64-bit evaluations."""
import pytest
import torch

import turbofno_amd as tf
from layer_norm_reference import Backward, Forward, check_eight, kept, rounded, wide, within
from operators_reference import EPS32, TYPES, randn

# K, positions: one channel, sizes around what lanes, waves and registers hold (32, 64, 128, 256, 512 channels), strips that end inside
SIZES = [(1, (1,)), (4, (3,)), (31, (65,)), (32, (256,)), (33, (7, 19)), (64, (1000,)), (65, (129,)), (128, (31,)), (129, (515,)), (256, (70,)),
         (300, (100,)), (513, (67,)), (1000, (33,)), (2100, (5,)), (20, (140001,)), (100, (131500,)), (200, (131100,))]
SEED = (77, 1 << 33)


def rng_of():
    return torch.tensor(SEED, dtype=torch.int64, device="cuda")


def operands(kind, K, places, seed=0, residual=True, offset=0.5):
    dt = TYPES[kind]
    wide_type = torch.complex64 if dt.is_complex else torch.float32
    x = (randn((K,) + places, wide_type, seed) + offset).to(dt)
    return x, 1 + 0.2 * randn((K,), torch.float32, seed + 1), 0.3 * randn((K,), wide_type, seed + 3), randn((K,) + places, dt, seed + 2) if residual else None


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,places", SIZES)
@pytest.mark.parametrize("residual,drop", [(True, 0.0), (False, 0.0), (True, 0.2)])
def test_forward(kind, K, places, residual, drop):
    x, gain, bias, r = operands(kind, K, places, 0, residual)
    y, s, mean, rstd = tf.layer_norm(x, gain, bias, r, drop=drop, rng=rng_of() if drop else None)
    E = Forward(x, gain, bias, r, drop=drop, rng=SEED)
    assert E.meaningful and rstd.shape == mean.shape == torch.Size(places) and (residual or s is x)
    within(s.flatten(1), E.s, rounded(E.s, E.s_off, x.dtype), "s")
    within(mean.flatten(), E.mean, E.mean_off, "mean")
    within(rstd.flatten(), E.rstd, E.rstd_off, "rstd")
    within(y.flatten(1), E.y, rounded(E.y, E.y_off, x.dtype), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,places", SIZES)
def test_8bit(kind, K, places):
    x, gain, bias, r = operands(kind, K, places, 3)
    q, scale, s = tf.layer_norm_8bit(x, gain, bias, r)
    E = Forward(x, gain, bias, r)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape + ((2,) if x.is_complex() else ()) and scale.shape == (-(-K // 128),) + places
    check_eight(q, scale, E.y, E.y_off, "layer_norm_8bit")
    assert torch.equal(s, tf.layer_norm(x, gain, bias, r)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,places", SIZES)
@pytest.mark.parametrize("stream,drop", [(True, 0.0), (False, 0.0), (True, 0.2)])
def test_gradient(kind, K, places, stream, drop):
    x, gain, bias, gs = operands(kind, K, places, 5, stream)
    gy = randn((K,) + places, x.dtype, 11)
    rng = rng_of() if drop else None
    _, s, mean, rstd = tf.layer_norm(x, gain, bias)
    gx, gr, ggain, gbias = tf.layer_norm_backward(gy, s, gain, mean, rstd, gs=gs, drop=drop, rng=rng)
    E = Backward(gy, s, gain, mean, rstd, gs, drop, SEED)
    within(gr.flatten(1), E.gr, rounded(E.gr, E.gr_off, x.dtype), "gr")
    within(gx.flatten(1), E.gx, rounded(E.gx, E.gx_off, x.dtype), "gx")
    within(ggain, E.ggain, E.ggain_off, "ggain")
    within(gbias, E.gbias, E.gbias_off, "gbias")
    assert (gr is gx) == (drop == 0.0)


@pytest.mark.parametrize("kind", ["c64", "f32"])
def test_formula_of_the_gradient_against_differences(kind):
    """Backward against central differences of Forward, both in 64 bits on the CPU: error of second order in the step"""
    dt, K, P, drop, gen = (torch.complex128 if kind == "c64" else torch.float64), 9, 6, 0.3, torch.Generator().manual_seed(3)
    new = lambda *shape, dtype=dt: torch.randn(shape, dtype=dtype, generator=gen)  # noqa: E731
    x, r, gain, bias, gy, gs = new(K, P), new(K, P), new(K, dtype=torch.float64), new(K), new(K, P), new(K, P)

    def loss(x, r, gain, bias):
        f = Forward(x, gain, bias, r, drop=drop, rng=SEED)
        return ((f.y.conj() * gy).real + (f.s.conj() * gs).real).sum() if dt.is_complex else (f.y * gy + f.s * gs).sum()
    f = Forward(x, gain, bias, r, drop=drop, rng=SEED)
    b = Backward(gy, f.s, gain, f.mean, f.rstd, gs, drop, SEED)
    args = [x, r, gain, bias]
    for i, got in enumerate((b.gx, b.gr, b.ggain, b.gbias)):
        for step in (1e-5, 1e-5j) if args[i].is_complex() else (1e-5,):
            direction = torch.randn(args[i].shape, dtype=torch.float64, generator=gen) * step
            ends = [loss(*[a + sign * direction if j == i else a for j, a in enumerate(args)]) for sign in (1, -1)]
            want = ((got.conj() * direction).real if got.is_complex() or direction.is_complex() else got * direction).sum()
            assert abs((ends[0] - ends[1]) / 2 - want) <= 1e-6 * abs(step) * K * P


@pytest.mark.gpu
def test_gradient_against_differences():
    """float32 on the GPU: the change of a loss formed in 64 bits from y, along a direction"""
    K, P = 24, 40
    x, gain, bias, r = operands("f32", K, (P,), 21)
    gy, rng = randn((K, P), torch.float32, 22), rng_of()
    run = lambda x, r, gain, bias: tf.layer_norm(x, gain, bias, r, drop=0.2, rng=rng)  # noqa: E731
    _, s, mean, rstd = run(x, r, gain, bias)
    got = tf.layer_norm_backward(gy, s, gain, mean, rstd, drop=0.2, rng=rng)
    args, names = [x, r, gain, bias], ("x", "residual", "gain", "bias")
    for i, g in enumerate(got):
        direction = 2.0 ** -6 * randn(args[i].shape, torch.float32, 30 + i)
        moved = [[a + sign * direction if j == i else a for j, a in enumerate(args)] for sign in (1, -1)]
        change = sum(sign * (run(*m)[0].double() * gy.double()).sum() for sign, m in zip((1, -1), moved)) / 2
        want = (g.double() * (moved[0][i].double() - moved[1][i].double()) / 2).sum()
        # rounding of 960 results of about 3, and the third order of the step: 2^-18 times derivatives of a few units each
        assert abs((change - want).item()) <= 960 * 3 * 3 * EPS32 + 960 * 2.0 ** -18 * 2, names[i]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["c64", "f32"])
@pytest.mark.parametrize("K", [64, 256, 700])
def test_a_mean_far_from_zero(kind, K):
    """means 3000 times the deviation: squares of deviations, not squares less the mean's, whose roundings would be as large as they"""
    x, gain, bias, _ = operands(kind, K, (300,), 40, False, 3000.0)
    y, _, mean, rstd = tf.layer_norm(x, gain, bias)
    X = wide(x)
    variance = ((X - X.mean(0)).abs() ** 2).mean(0)
    # the mean is off by a few roundings of itself; what that adds to the variance is the square of it
    off = 16 * EPS32 * 3000
    relative = (off / variance.sqrt()) ** 2 + (K + 8) * EPS32
    assert ((rstd.double() * torch.sqrt(variance + 1e-6) - 1).abs() <= relative).all()
    assert ((mean - X.mean(0)).abs() <= off).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_ends(kind):
    """positions of one value, of zeros, of values that are not finite, and their neighbours; no positions"""
    dt = TYPES[kind]
    x = randn((40, 80), dt, 50)
    x[:, 0] = 0
    x[:, 1] = 3.0
    x[5, 2], x[6, 66] = float("nan"), float("inf")
    gain, bias = torch.full((40,), 2.0, device="cuda"), randn((40,), torch.complex64 if dt.is_complex else torch.float32, 51)
    y, _, mean, rstd = tf.layer_norm(x, gain, bias)
    finite = lambda t: torch.isfinite(torch.view_as_real(t).sum(-1) if t.is_complex() else t)  # noqa: E731
    b = bias.to(dt)
    assert torch.equal(y[:, 0], b) and torch.equal(y[:, 1], b) and mean[1] == 3 and (rstd[:2] - 1000).abs().max() < 0.01
    for p in (2, 66):
        assert not finite(y[:, p]).any() and not torch.isfinite(rstd[p]) and not finite(mean[p:p + 1]).any()
    rest = [p for p in range(80) if p not in (2, 66)]
    assert finite(y[:, rest]).all()
    q, scale, _ = tf.layer_norm_8bit(x, gain, bias)
    assert torch.isnan(scale[0, [2, 66]]).all() and torch.isfinite(scale[0, rest]).all()
    assert torch.isnan(q.float().reshape(40, 80, -1)[:, [2, 66]]).all() and torch.isfinite(q.float().reshape(40, 80, -1)[:, rest]).all()
    q, scale, _ = tf.layer_norm_8bit(x[:, :1], gain)                        # nothing but zeros
    assert (scale == 1).all() and (q.float() == 0).all()
    y, s, mean, rstd = tf.layer_norm(x[:, :0], gain, bias, residual=x[:, :0])
    assert y.shape == s.shape == (40, 0) and mean.shape == rstd.shape == (0,)
    gx, _, ggain, gbias = tf.layer_norm_backward(x[:, :0], s, gain, mean, rstd, ggain=torch.full((40,), 7.0, device="cuda"), gbias=torch.full_like(bias, 7.0))
    assert gx.shape == (40, 0) and (ggain == 0).all() and (gbias == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,P", [(50, 333), (600, 70)])
def test_in_place_and_channels_apart(kind, K, P):
    dt = TYPES[kind]
    x, gain, bias, r = operands(kind, K, (P,), 60)
    rng = rng_of()
    run = lambda *a, **k: tf.layer_norm(*a, drop=0.25, rng=rng, **k)  # noqa: E731
    y, s, mean, rstd = run(x, gain, bias, r)
    stream = r.clone()
    y2, s2, _, _ = run(x, gain, bias, stream, s=stream)
    assert s2 is stream and torch.equal(stream, s) and torch.equal(y2, y)
    both, held = x.clone(), r.clone()
    run(both, gain, bias, held, y=both, s=held)
    assert torch.equal(both, y) and torch.equal(held, s)
    both, held = x.clone(), r.clone()
    run(both, gain, bias, held, y=held, s=both)
    assert torch.equal(held, y) and torch.equal(both, s)
    q, scale, _ = tf.layer_norm_8bit(x, gain, bias, r)
    gy, gs = randn((K, P), dt, 64), randn((K, P), dt, 65)
    back = lambda *a, **k: tf.layer_norm_backward(*a, drop=0.25, rng=rng, **k)  # noqa: E731
    want = back(gy, s, gain, mean, rstd, gs=gs)
    for names in (("gy", "s"), ("s", "gs"), ("gs", "gy")):
        own = dict(gy=gy.clone(), s=s.clone(), gs=gs.clone())
        got = back(own["gy"], own["s"], gain, mean, rstd, gs=own["gs"], gx=own[names[0]], gr=own[names[1]])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), names
    for shift in range(1, 5):
        apart = [torch.full((K, P + 9), 7.0, dtype=dt, device="cuda") for _ in range(6)]
        inside = [t[:, shift + i % 3:shift + i % 3 + P] for i, t in enumerate(apart)]
        untouched = lambda: all((t[:, :shift + i % 3] == 7).all() and (t[:, shift + i % 3 + P:] == 7).all() for i, t in enumerate(apart))  # noqa: E731
        inside[0].copy_(x)
        inside[1].copy_(r)
        run(inside[0], gain, bias, inside[1], y=inside[2], s=inside[3])
        assert torch.equal(inside[2], y) and torch.equal(inside[3], s) and untouched()
        pair = (2,) if dt.is_complex else ()
        bytes_ = torch.zeros((K, P + 6) + pair, dtype=torch.float8_e4m3fn, device="cuda")
        tf.layer_norm_8bit(inside[0], gain, bias, inside[1], q=bytes_[:, shift:shift + P])
        raw = bytes_.view(torch.uint8)
        assert torch.equal(raw[:, shift:shift + P], q.view(torch.uint8)) and (raw[:, :shift] == 0).all() and (raw[:, shift + P:] == 0).all()
        for i, t in enumerate((gy, s, gs)):
            inside[i].copy_(t)
        got = back(inside[0], inside[1], gain, mean, rstd, gs=inside[2], gx=inside[4], gr=inside[5])
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and untouched()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K", [5, 40, 130, 300])
def test_channels_far_apart(kind, K):
    """channels 2^28 values and more apart, where a lane's offset would pass 32 bits: views of one buffer whose rows overlap nothing that is compared"""
    dt, P = TYPES[kind], 70
    step = (1 << 28) // (2 if dt.is_complex else 1) + 11
    if K * step * dt.itemsize > 140 << 30:
        K = (140 << 30) // (step * dt.itemsize)
    x, gain, bias, _ = operands(kind, K, (P,), 70, False)
    far = torch.empty((K - 1) * step + P, dtype=dt, device="cuda").as_strided((K, P), (step, 1))
    far.copy_(x)
    want = tf.layer_norm(x, gain, bias)
    got = tf.layer_norm(far, gain, bias)
    E = Forward(x, gain, bias)
    within(got[0], E.y, rounded(E.y, E.y_off, dt), "y")
    q, scale, _ = tf.layer_norm_8bit(far, gain, bias)
    check_eight(q, scale, E.y, E.y_off, "8 bit")
    q, scale = tf.quantise_8bit(far)
    near = tf.quantise_8bit(x)
    assert torch.equal(q.view(torch.uint8), near[0].view(torch.uint8)) and torch.equal(scale, near[1])
    gy = randn((K, P), dt, 71)
    got = tf.layer_norm_backward(gy, far, gain, want[2], want[3])
    E = Backward(gy, x, gain, want[2], want[3])
    within(got[0], E.gr, rounded(E.gr, E.gr_off, dt), "gx")
    within(got[2], E.ggain, E.ggain_off, "ggain")
    rng = torch.tensor(SEED, dtype=torch.int64, device="cuda")
    assert torch.equal(tf.dropout(far, 0.5, rng), tf.dropout(x, 0.5, rng))
    del far
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_one_mask_everywhere():
    """layer_norm, its gradient and dropout keep the same elements, whatever kernel runs"""
    for kind in TYPES:
        for K, P in ((6, 50), (64, 131072), (200, 90), (600, 333)):
            x = torch.ones((K, P), dtype=TYPES[kind], device="cuda")
            gain, rng = torch.ones(K, device="cuda"), rng_of()
            alone = tf.dropout(x, 0.5, rng)
            _, s, mean, rstd = tf.layer_norm(x, gain, drop=0.5, rng=rng)
            gx, gr, _, _ = tf.layer_norm_backward(randn((K, P), x.dtype, 80), s, gain, mean, rstd, drop=0.5, rng=rng, gs=x)
            assert torch.equal(s, alone)
            assert torch.equal(gx, torch.where(alone != 0, 2 * gr, torch.zeros_like(gr)))
    assert torch.equal(kept(SEED, 600, 333, 0.5), alone != 0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_training_in_a_graph(kind):
    """forward and backward with dropout, captured with their random numbers and replayed: the eager result of each step"""
    dt, K, P = TYPES[kind], 96, 700
    x, gain, bias, r = operands(kind, K, (P,), 90)
    gy, rng = randn((K, P), dt, 94), rng_of()
    workspace = torch.empty(tf.layer_norm_backward_workspace_bytes(K, P, dt), dtype=torch.uint8, device="cuda")

    def step(x, rng, out):
        y, s, mean, rstd = tf.layer_norm(x, gain, bias, r, drop=0.1, rng=rng)
        grads = tf.layer_norm_backward(gy, s, gain, mean, rstd, gs=y, drop=0.1, rng=rng, workspace=workspace)
        for o, t in zip(out, (y, s) + grads):
            o.copy_(t)
    out = [torch.empty_like(x) for _ in range(4)] + [torch.empty_like(gain), torch.empty_like(bias)]
    eager = [torch.empty_like(t) for t in out]
    step(x, rng, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(x, rng, out)
        rng[1:] += 1
    rng.copy_(rng_of())
    for i in range(4):
        x.copy_(randn((K, P), dt, 95 + i))
        step(x, torch.tensor([SEED[0], SEED[1] + i], dtype=torch.int64, device="cuda"), eager)
        torch.cuda.synchronize()
        for o in out:
            o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), i


@pytest.mark.gpu
def test_on_another_stream():
    x, gain, bias, r = operands("bf16", 64, (5000,), 99)
    want = tf.layer_norm(x, gain, bias, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tf.layer_norm(x, gain, bias, r)
        grads = tf.layer_norm_backward(got[0], got[1], gain, got[2], got[3])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(grads, tf.layer_norm_backward(want[0], want[1], gain, want[2], want[3])))
