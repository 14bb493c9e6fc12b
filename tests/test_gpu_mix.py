"""Channel product with bias, residual and activation, its 8-bit form and its gradients, against 64-bit evaluations."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import (EPS16, EPS32, TYPES, act, by_parts, product_bound, randn, rounding, slope, wide, within)

pytestmark = pytest.mark.gpu

# K, N, positions: single elements, sizes around the tiles of 16 channels and 64 columns, steps that end inside, several row groups
SIZES = [(1, 1, (1,)), (3, 5, (7,)), (8, 64, (128,)), (17, 33, (65,)), (64, 64, (10, 100)), (72, 200, (3, 111)), (130, 131, (129,)), (300, 40, (70,)),
         (16, 300, (2, 5, 13)), (33, 16, (4099,)), (64, 128, (40001,)), (20, 1500, (6001,))]


def operands(kind, K, N, places, seed=0, bias=True, residual=True):
    dt = TYPES[kind]
    x, W = randn((K,) + places, dt, seed), randn((N, K), dt, seed + 1, K ** -0.5)
    return x, W, randn((N,), dt, seed + 2) if bias else None, randn((N,) + places, dt, seed + 3) if residual else None


def expected_z(x, W, bias, residual):
    """z and a bound of its error before its last rounding"""
    X, V = wide(x).flatten(1), wide(W)
    z, bound = V @ X, product_bound(V, X, V.shape[1] * (2 if X.is_complex() else 1))
    if bias is not None:
        z = z + wide(bias)[:, None]
    if residual is not None:
        z = z + wide(residual).flatten(1)
    return z, bound + 3 * EPS32 * (z.abs() + (0 if bias is None else wide(bias).abs()[:, None]))


def check_forward(y, z, x, W, bias, residual, activation):
    dt = x.dtype
    Z, bound = expected_z(x, W, bias, residual)
    if z is not None:
        within(z.flatten(1), Z, bound + rounding(dt) * (Z.abs() + bound), "z")
    Y = act(activation, Z)
    # slopes are at most 1.13; an activation adds at most 2^-20 of its argument (its exponential: |z| 2^-24 of itself, in a factor below 1)
    bound = 1.13 * bound + (2.0 ** -20 * Z.abs() if activation in ("silu", "gelu_tanh") else 0)
    within(y.flatten(1), Y, bound + 1.01 * rounding(dt) * (Y.abs() + bound), "y")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,N,places", SIZES)
def test_forward(kind, K, N, places):
    x, W, bias, residual = operands(kind, K, N, places)
    z = torch.empty_like(residual)
    y = tf.mix(x, W, bias, residual, "gelu_tanh", z=z)
    check_forward(y, z, x, W, bias, residual, "gelu_tanh")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("activation", ["none", "relu", "silu", "gelu_tanh"])
@pytest.mark.parametrize("bias,residual", [(False, False), (True, False), (False, True)])
def test_forward_parts(kind, activation, bias, residual):
    x, W, b, r = operands(kind, 20, 37, (203,), 10, bias, residual)
    check_forward(tf.mix(x, W, b, r, activation), None, x, W, b, r, activation)


@pytest.mark.parametrize("kind", TYPES)
def test_channels_apart_and_rows_that_start_anywhere(kind):
    """slices of larger fields: every offset of a row against 16 bytes, different distances for every operand"""
    dt = TYPES[kind]
    for shift in range(1, 8):
        K, N, P = 21, 35, 150 + shift
        x = randn((K, P + 9), dt, shift)[:, shift:shift + P]
        r = randn((N + 2, P + 5), dt, shift + 1)[1:-1, 3:3 + P]
        W, b = randn((N, K), dt, shift + 2, K ** -0.5), randn((N,), dt, shift + 3)
        y, z = (torch.full((N, P + 11 + i), 7.0, dtype=dt, device="cuda") for i in (0, 2))
        tf.mix(x, W, b, r, "silu", y=y[:, shift:shift + P], z=z[:, 2:2 + P])
        check_forward(y[:, shift:shift + P], z[:, 2:2 + P], x, W, b, r, "silu")
        for t, lo in ((y, shift), (z, 2)):              # nothing beside the rows is written
            assert (t[:, :lo] == 7).all() and (t[:, lo + P:] == 7).all()


@pytest.mark.parametrize("kind", TYPES)
def test_residual_in_place(kind):
    for N, P in ((64, 1000), (150, 77), (70, 60003)):
        x, W, b, r = operands(kind, 40, N, (P,), 5)
        want = tf.mix(x, W, b, r, "relu")
        stream = r.clone()
        assert tf.mix(x, W, b, stream, "relu", y=stream) is stream
        assert torch.equal(stream, want)
        saved, y = r.clone(), torch.empty_like(r)
        tf.mix(x, W, b, saved, "relu", y=y, z=saved)
        assert torch.equal(y, want) and torch.equal(by_parts(torch.relu, saved), want)


@pytest.mark.parametrize("kind", ["c64", "f32"])
def test_values_that_are_not_finite(kind):
    """infinities, NaN and the top of the range behave as in fp32, in their own columns only"""
    dt = TYPES[kind]
    K, N, P = 24, 20, 200
    x, W = randn((K, P), dt, 1), randn((N, K), dt, 2)
    top = torch.finfo(torch.float32).max
    clean = tf.mix(x, W)
    for c, v in ((3, float("inf")), (70, float("-inf")), (131, float("nan")), (199, top)):
        x[5, c] = v
        if v == top:
            x[:5, c], x[6:, c] = 0, 0
            W[:, 5] = W[:, 5] * 0.25
    clean = tf.mix(torch.where(torch.isfinite(x) & (x.abs() < 1e30), x, torch.zeros_like(x)), W)
    y = tf.mix(x, W)
    want = wide(W) @ wide(x)
    touched = [3, 70, 131, 199]
    rest = [c for c in range(P) if c not in touched]
    assert torch.equal(y[:, rest], clean[:, rest])
    parts = lambda t: torch.view_as_real(t) if t.is_complex() else t  # noqa: E731
    got = wide(y)
    for c in (3, 70):
        if kind == "f32":
            assert torch.equal(got[:, c], want[:, c])
        else:
            assert not torch.isfinite(parts(got[:, c])).any(dim=-1).all()
    assert torch.isnan(parts(got[:, 131])).any(dim=-1).all() if kind == "c64" else torch.isnan(got[:, 131]).all()
    inside = want[:, 199].abs() < top
    assert ((got[:, 199] - want[:, 199]).abs()[inside] <= 8 * EPS32 * want[:, 199].abs()[inside]).all() and inside.any()


def test_not_finite_in_16_bits():
    x, W = randn((24, 100), torch.bfloat16, 1), randn((20, 24), torch.bfloat16, 2)
    clean = tf.mix(x, W)
    x[3, 7], x[4, 50] = float("inf"), float("nan")
    y = tf.mix(x, W)
    rest = [c for c in range(100) if c not in (7, 50)]
    assert torch.equal(y[:, rest], clean[:, rest])
    assert torch.equal(y[:, 7].float(), torch.sign(W[:, 3].float()) * float("inf")) and torch.isnan(y[:, 50]).all()


def test_activations_at_their_ends():
    """large arguments of either sign, zeros and NaN: no overflow of the exponential shows"""
    v = torch.tensor([-1e30, -1e4, -100.0, -20.0, -0.0, 0.0, 20.0, 100.0, 1e4, 1e30, float("inf"), float("nan")], device="cuda")[None]
    W = torch.ones(1, 1, device="cuda")
    for name in ("relu", "silu", "gelu_tanh"):
        y = wide(tf.mix(v, W, activation=name))[0]
        z = wide(v)[0]
        assert torch.isnan(y[-1]) and y[-2] == float("inf")
        assert torch.equal(y[6:10], z[6:10]) and (y[:4].abs() <= 1e-6).all() and (y[4:6] == 0).all()
        gy = torch.ones_like(v)
        gx, gz = tf.mix_input_grad(gy, W, z=v, activation=name)
        g = wide(gz)[0]
        assert (g[:4].abs() <= 1e-6).all() and ((g[6:9] - 1).abs() <= 1e-6).all() and torch.isfinite(g[:9]).all()


def quantized(t, dim):
    scale = t.abs().amax(dim=dim, keepdim=True) / 448
    return (t / scale).to(torch.float8_e4m3fn), scale


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,N,places", SIZES)
def test_8bit(kind, K, N, places):
    dt = TYPES[kind]
    pair = (2,) if dt.is_complex else ()
    xq, xs = quantized(randn((K,) + places + pair, torch.float32, 1), (0, -1) if pair else 0)
    Wq, ws = quantized(randn((N, K) + pair, torch.float32, 2), (1, -1) if pair else 1)
    xs, ws = xs.reshape(places).contiguous(), ws.reshape(N).contiguous()
    b, r = randn((N,), dt, 3), randn((N,) + places, dt, 4)
    y = tf.mix_8bit(xq, xs, Wq, ws, b, r, "silu")
    assert y.dtype == dt and y.shape == r.shape
    X, V = xq.cpu().double(), Wq.cpu().double()
    if pair:
        X, V = torch.view_as_complex(X), torch.view_as_complex(V)
    X, V = X.flatten(1) * wide(xs).flatten(), V * wide(ws)[:, None]
    Z = V @ X + wide(b)[:, None] + wide(r).flatten(1)
    bound = product_bound(V, X, K * (2 if pair else 1)) + 5 * EPS32 * (Z.abs() + wide(b).abs()[:, None])
    Y = act("silu", Z)
    bound = 1.13 * bound + 2.0 ** -20 * Z.abs()
    within(y.flatten(1), Y, bound + 1.01 * rounding(dt) * (Y.abs() + bound), "y")


def test_8bit_strides_and_result_type():
    K, N, P = 19, 21, 75
    big, scale = quantized(randn((K, P + 6), torch.float32, 1), 0)
    Wq, ws = quantized(randn((N, K), torch.float32, 2), 1)
    xq, xs, ws = big[:, 3:3 + P], scale[0, 3:3 + P].contiguous(), ws[:, 0].contiguous()
    y = tf.mix_8bit(xq, xs, Wq, ws)
    assert y.dtype == torch.bfloat16
    assert torch.equal(y, tf.mix_8bit(xq.contiguous(), xs, Wq, ws))
    wide_y = tf.mix_8bit(xq, xs, Wq, ws, dtype=torch.float32)
    assert torch.equal(wide_y.to(torch.bfloat16), y)


def check_backward(gy, x, W, z, activation, results):
    gx, gW, gbias, gz = results
    dt = gy.dtype
    G, X, V = wide(gy).flatten(1), wide(x).flatten(1), wide(W)
    S = slope(activation, wide(z).flatten(1)) if activation != "none" else None
    GZ = by_parts(lambda g, s: g * s, G, S) if S is not None else G
    own = EPS16 if dt == torch.bfloat16 else 0.0        # the product takes gz as it was rounded
    inside = 2.0 ** -19 * G.abs() if activation in ("silu", "gelu_tanh") else 0 * G.abs()     # of the slope: z times a difference of rounded sigmoids
    within(gz.flatten(1), GZ, inside + 1.01 * rounding(dt) * (GZ.abs() + inside), "gz")
    parts = 2 if G.is_complex() else 1
    VH, XH = V.conj().T, X.conj().T
    bound = product_bound(VH, GZ, parts * V.shape[0], 1.01 * own) + VH.abs() @ inside
    E = VH @ GZ
    within(gx.flatten(1), E, bound + 1.01 * rounding(dt) * (E.abs() + bound), "gx")
    P = X.shape[1]
    # sums in parts: a wave's steps of 32, then the parts in turn
    bound = product_bound(GZ, XH, parts * min(P, 4096), 1.01 * own) + inside @ XH.abs()
    E = GZ @ XH
    within(gW, E, bound + 1.01 * rounding(dt) * (E.abs() + bound), "gW")
    bound = (min(P, 4096) * EPS32 + 1.01 * own) * GZ.abs().sum(1) + inside.sum(1)
    E = GZ.sum(1)
    within(gbias, E, bound + 1.01 * rounding(dt) * (E.abs() + bound), "gbias")


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,N,places", SIZES)
def test_backward(kind, K, N, places):
    dt = TYPES[kind]
    gy, z = randn((N,) + places, dt, 1), randn((N,) + places, dt, 2)
    x, W = randn((K,) + places, dt, 3), randn((N, K), dt, 4)
    check_backward(gy, x, W, z, "gelu_tanh", tf.mix_backward(gy, x, W, z, "gelu_tanh"))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("activation", ["none", "relu", "silu"])
def test_backward_activations(kind, activation):
    dt = TYPES[kind]
    gy, z = randn((37, 500), dt, 1), randn((37, 500), dt, 2)
    x, W = randn((20, 500), dt, 3), randn((37, 20), dt, 4)
    results = tf.mix_backward(gy, x, W, z, activation)
    check_backward(gy, x, W, z, activation, results)
    assert activation != "none" or results[3] is gy


@pytest.mark.parametrize("kind", TYPES)
def test_backward_channels_apart(kind):
    dt = TYPES[kind]
    for shift in range(1, 8):
        K, N, P = 18, 70, 301 + shift
        gy = randn((N, P + 9), dt, 1)[:, shift:shift + P]
        z = randn((N, P + 4), dt, 2)[:, 3:3 + P]
        x = randn((K + 1, P + 7), dt, 3)[1:, 5:5 + P]
        W = randn((N, K), dt, 4)
        gz, gx = torch.full((N, P + 5), 7.0, dtype=dt, device="cuda"), torch.full((K, P + 3), 7.0, dtype=dt, device="cuda")
        results = tf.mix_backward(gy, x, W, z, "silu", gz=gz[:, 2:2 + P], gx=gx[:, 1:1 + P])
        check_backward(gy, x, W, z, "silu", results)
        assert (gz[:, :2] == 7).all() and (gz[:, 2 + P:] == 7).all() and (gx[:, :1] == 7).all() and (gx[:, 1 + P:] == 7).all()


@pytest.mark.parametrize("kind", ["c64", "f32"])
def test_gradients_against_differences(kind):
    """(L(v + h d) - L(v - h d)) / 2 h of L = sum Re(conj(c) y) in the direction d of each operand, against Re(conj(g) d)"""
    dt, K, N, P, h = TYPES[kind], 12, 17, 90, 2.0 ** -7
    x, W, b, r = operands(kind, K, N, (P,), 20)
    c = randn((N, P), dt, 30)
    loss = lambda *v: (wide(c).conj() * wide(tf.mix(*v, "gelu_tanh"))).real.sum().item()  # noqa: E731
    z = torch.empty_like(c)
    tf.mix(x, W, b, r, "gelu_tanh", z=z)
    gx, gW, gbias, gz = tf.mix_backward(c, x, W, z, "gelu_tanh")
    ops = [x, W, b, r]
    for i, g in enumerate((gx, gW, gbias, gz)):
        d = randn(ops[i].shape, dt, 40 + i)
        shifted = lambda s: loss(*[o + s * h * d if j == i else o for j, o in enumerate(ops)])  # noqa: E731
        slope_along = (wide(g).conj() * wide(d)).real.sum().item()
        scale = wide(g).abs().norm().item() * wide(d).abs().norm().item()
        # third derivatives of gelu stay below 4: h^2 / 6 of them along d, cubed; a direction's size is of the order of one per element of z
        assert abs((shifted(1) - shifted(-1)) / (2 * h) - slope_along) <= 5e-3 * scale, i


def test_no_positions():
    for kind, dt in TYPES.items():
        x, W = torch.empty((5, 0), dtype=dt, device="cuda"), randn((3, 5), dt, 1)
        assert tf.mix(x, W).shape == (3, 0)
        gy = torch.empty((3, 0), dtype=dt, device="cuda")
        gx, gW, gbias, gz = tf.mix_backward(gy, x, W, gy, "silu", gW=torch.ones_like(W))
        assert gx.shape == (5, 0) and (gW == 0).all() and (gbias == 0).all()


def test_results_repeat_and_follow_their_stream():
    x, W, b, r = operands("c64", 64, 64, (70000,), 50)
    y = tf.mix(x, W, b, r, "gelu_tanh")
    gW, gbias = tf.mix_weight_grad(r, x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x2 = x * 1
        again = tf.mix(x2, W, b, r, "gelu_tanh")
        gW2, gbias2 = tf.mix_weight_grad(r, x2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, again) and torch.equal(gW, gW2) and torch.equal(gbias, gbias2)


def test_spectral_weight_gradient():
    """mix_weight_grad on truncated spectra: the gradient of layer_1d's weights, against the layer's own differences (it is linear in W)"""
    K, N, S, DY = 8, 64, 3, 128
    x, W = randn((K, S, DY), torch.complex64, 1), randn((N, K), torch.complex64, 2)
    g = randn((N, S, DY), torch.complex64, 3)
    spectra, product = torch.empty((K, S, 64), dtype=torch.complex64, device="cuda"), torch.empty((N, S, 64), dtype=torch.complex64, device="cuda")
    tf.fft_stride_DY(x, spectra, 8, K * S)
    tf.fft_stride_DY(g, product, 8, N * S)              # the adjoint of the padded backward transform
    gW, _ = tf.mix_weight_grad(product, spectra)
    d = randn((N, K), torch.complex64, 4)
    along = (wide(g).conj() * wide(tf.layer_1d(x, d))).real.sum().item()
    slope_along = (wide(gW).conj() * wide(d)).real.sum().item()
    assert abs(along - slope_along) <= 1e-5 * wide(gW).abs().norm().item() * wide(d).abs().norm().item()


def test_refusals():
    x, W = randn((4, 10), torch.float32, 1), randn((6, 4), torch.float32, 2)
    with pytest.raises(ValueError, match="one column per channel"):
        tf.mix(x, randn((6, 5), torch.float32, 2))
    with pytest.raises(TypeError, match="float16"):
        tf.mix(x.half(), W)
    with pytest.raises(TypeError, match="W must be"):
        tf.mix(x, W.to(torch.bfloat16))
    with pytest.raises(ValueError, match="side by side"):
        tf.mix(x.t().contiguous().t(), W)
    with pytest.raises(ValueError, match="activation"):
        tf.mix(x, W, activation="tanh")
    with pytest.raises(ValueError, match="residual has shape"):
        tf.mix(x, W, residual=x)
    with pytest.raises(tf.TurboFNOError, match="overlaps x"):
        tf.mix(x, randn((4, 4), torch.float32, 2), y=x)
    with pytest.raises(tf.TurboFNOError, match="channels"):
        tf.mix(x[:1].expand(4, 10), W)
    shared = randn((7, 10), torch.float32, 3)
    with pytest.raises(tf.TurboFNOError, match="without being it"):
        tf.mix(x, W, residual=shared[:6], y=shared[1:])
    with pytest.raises(ValueError, match="needs z"):
        tf.mix_backward(randn((6, 10), torch.float32, 1), x, W, activation="silu")
    with pytest.raises(tf.TurboFNOError, match="workspace"):
        tf.mix_weight_grad(randn((6, 10), torch.float32, 1), x, workspace=torch.empty(4, dtype=torch.uint8, device="cuda"))
    c = randn((4, 10), torch.complex64, 1)
    with pytest.raises(TypeError, match="conjugated"):
        tf.mix(c.conj(), randn((6, 4), torch.complex64, 1))
    with pytest.raises(TypeError, match="xq must be"):
        tf.mix_8bit(x, x[0], W, W[:, 0].contiguous())
