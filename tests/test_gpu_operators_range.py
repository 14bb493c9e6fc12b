"""Channel product and its gradients on 32-bit operands below the range of the split into bf16 parts (2^-110): fp32 precision down to the smallest normal
numbers, in columns and weights of any magnitude among others near one."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import EPS32, TYPES, product_bound, randn, rounding, slope, wide, within

pytestmark = pytest.mark.gpu
KINDS = ["f32", "c64"]
SCALES = [1e-33, 1e-35, 1e-37]

# real channels of the contraction, channels of the result, real columns (complex: half of the first and of the last): few weights and few columns, one
# to four tiles of 16 rows in the direct kernel, steps held and streamed with 64 and 32 rows in the resident one
SIZES = [(3, 2, 40), (2, 2, 200), (24, 40, 300), (70, 9, 130), (820, 40, 25000), (820, 40, 45000), (24, 40, 70000), (24, 20, 140001), (72, 40, 70002), (72, 20, 70001),
         (130, 200, 70000)]


def sized(kind, K, P):
    return (K, P) if kind == "f32" else (max(1, K // 2), max(1, P // 2))


def picked(P):
    """columns at both ends and in the middle; every third of 64 of them gets another magnitude"""
    idx = torch.tensor(sorted({p for a in (0, P // 2 - 64, P - 128) for p in range(max(0, a), min(P, a + 128))}), device="cuda")
    return idx, idx[idx % 64 % 3 == 1]


def tiny(terms, A):
    """what sums of `terms` products lose below the normal numbers"""
    return terms * 2.0 ** -149 * (1 + A.abs().amax())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("K,N,P", SIZES)
def test_forward(kind, K, N, P):
    dt, (K, P) = TYPES[kind], sized(kind, K, P)
    x, W = randn((K, P), dt, 1), randn((N, K), dt, 2, K ** -0.5)
    idx, small = picked(P)
    terms = K * (2 if dt.is_complex else 1)
    for scale in SCALES:
        xs = x.clone()
        xs[:, small] *= scale
        X, V = wide(xs[:, idx]), wide(W)
        within(tf.mix(xs, W)[:, idx], V @ X, product_bound(V, X, terms) + tiny(terms, V), "columns %g" % scale)
        Ws = W.clone()
        Ws[::3] *= scale
        X, V = wide(x[:, idx]), wide(Ws)
        within(tf.mix(x, Ws)[:, idx], V @ X, product_bound(V, X, terms) + tiny(terms, X), "weights %g" % scale)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("activation", ["none", "silu"])
@pytest.mark.parametrize("N,K,P", SIZES)
def test_input_gradient(kind, activation, N, K, P):
    """N: channels of gy, over which is summed"""
    dt, (N, P) = TYPES[kind], sized(kind, N, P)
    gy, z, W = randn((N, P), dt, 3), randn((N, P), dt, 4), randn((N, K), dt, 5, N ** -0.5)
    idx, small = picked(P)
    terms = N * (2 if dt.is_complex else 1)

    def check(gy, W, what):
        gx, gz = tf.mix_input_grad(gy, W, z=z, activation=activation)
        G, VH = wide(gy[:, idx]), wide(W).mH
        inside = 0 * G.abs()
        if activation != "none":
            S = slope(activation, wide(z[:, idx]))
            G, inside = (torch.complex(G.real * S.real, G.imag * S.imag) if dt.is_complex else G * S), 2.0 ** -19 * G.abs() + 2.0 ** -148
            within(gz[:, idx], G, inside + 1.01 * EPS32 * G.abs(), "gz " + what)
        within(gx[:, idx], VH @ G, product_bound(VH, G, terms) + VH.abs() @ inside + tiny(terms, VH) + tiny(terms, G), what)
    for scale in SCALES:
        gs = gy.clone()
        gs[:, small] *= scale
        check(gs, W, "columns %g" % scale)
        Ws = W.clone()
        Ws[:, ::3] *= scale
        check(gy, Ws, "weights %g" % scale)


def any_magnitude(shape, dt, seed):
    """values of either sign and of magnitudes from 1e-37 to 1e37, a tenth of them zeros"""
    gen = torch.Generator().manual_seed(seed)
    full = tuple(shape) + ((2,) if dt.is_complex else ())
    v = 10.0 ** (torch.rand(full, generator=gen, dtype=torch.float64) * 74 - 37) * torch.sign(torch.rand(full, generator=gen, dtype=torch.float64) - 0.5)
    v = torch.where(torch.rand(full, generator=gen) < 0.1, torch.zeros_like(v), v).float()
    return (torch.view_as_complex(v) if dt.is_complex else v).cuda()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("K,P", [(3, 40), (20, 200), (40, 300), (24, 70000), (72, 70000), (820, 25000)])
def test_a_permutation_returns_what_it_was_given(kind, K, P):
    """every value by itself, whatever stands beside it: products with ones and zeros are exact"""
    dt, (K, P) = TYPES[kind], sized(kind, K, P)
    x, order = any_magnitude((K, P), dt, 6), torch.randperm(K, generator=torch.Generator().manual_seed(7)).cuda()
    W = torch.eye(K, dtype=dt, device="cuda")[order].contiguous()
    assert torch.equal(tf.mix(x, W), x[order])
    assert torch.equal(tf.mix_input_grad(x[order], W)[0], x)


# channels of x and of gz, real columns (complex: half): fewer than a step, one tile of 32 x 32 and more, tiles of 64 x 64, and those with less than a step
WEIGHT_SIZES = [(5, 3, 20), (40, 70, 1001), (20, 30, 200), (64, 64, 140003), (70, 130, 140000), (4128, 4100, 20)]


def weight_gradient(gz, x):
    """gz x^H in 64 bits, real and imaginary parts apart: what is not finite is as the formula has it"""
    G, X = wide(gz), wide(x)
    if not G.is_complex():
        return G @ X.T
    return torch.complex(G.real @ X.real.T + G.imag @ X.imag.T, G.imag @ X.real.T - G.real @ X.imag.T)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("K,N,P", WEIGHT_SIZES)
def test_weight_gradient(kind, K, N, P):
    dt = TYPES[kind]
    parts = 2 if dt.is_complex else 1
    P //= parts
    gz, x = randn((N, P), dt, 8), randn((K, P), dt, 9)
    for scale in SCALES if N < 1000 else SCALES[1:2]:
        for which in (gz, x):
            kept = which.clone()
            which[::3] *= scale
            gW, gbias = tf.mix_weight_grad(gz, x)
            G, XH = wide(gz), wide(x).mH
            terms = parts * min(P, 4096)
            within(gW, weight_gradient(gz, x), product_bound(G, XH, terms) + P * parts * 2.0 ** -149 * 6, "gW %g" % scale)
            within(gbias, G.sum(1), (terms + 4) * EPS32 * G.abs().sum(1), "gbias %g" % scale)
            which.copy_(kept)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("K,N,P", WEIGHT_SIZES[:-1])
def test_weight_gradient_picks_single_values(kind, K, N, P):
    """x with one 1 per channel: every value of gz by itself, whatever stands beside it"""
    dt = TYPES[kind]
    P //= 2 if dt.is_complex else 1
    gz, where = any_magnitude((N, P), dt, 10), torch.randint(0, P, (K,), generator=torch.Generator().manual_seed(11)).cuda()
    where[0] = P - 1
    x = torch.zeros((K, P), dtype=dt, device="cuda")
    x[torch.arange(K, device="cuda"), where] = 1
    gW, _ = tf.mix_weight_grad(gz, x)
    assert torch.equal(gW, gz[:, where])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("K,N,P", WEIGHT_SIZES[:-1])
def test_weight_gradient_not_finite_and_at_the_top(kind, K, N, P):
    """infinities and NaN reach the sums that they take part in, the largest floats are numbers"""
    dt = TYPES[kind]
    P //= 2 if dt.is_complex else 1
    gz, x = randn((N, P), dt, 12), randn((K, P), dt, 13)
    top = torch.finfo(torch.float32).max
    real = lambda t: torch.view_as_real(t)[..., 0] if t.is_complex() else t  # noqa: E731
    real(gz)[0, P - 1] = float("inf")
    real(x)[1, 0] = float("-inf")
    real(x)[2, P // 2] = float("nan")
    x[:, P // 3] *= 0.125
    real(gz)[1, P // 3] = top
    gW, _ = tf.mix_weight_grad(gz, x)
    want, got = weight_gradient(gz, x), wide(gW)
    as_parts = lambda t: torch.view_as_real(t) if t.is_complex() else t  # noqa: E731
    want, got = as_parts(want), as_parts(got)
    beyond = want.abs() > top
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    finite = torch.isfinite(want) & ~beyond
    G, X = wide(gz).nan_to_num(0, 0, 0), wide(x).nan_to_num(0, 0, 0)
    bound = product_bound(G, X.mH, (2 if dt.is_complex else 1) * min(P, 4096))
    bound = bound[..., None] if dt.is_complex else bound
    assert ((got - want).abs() <= bound.expand_as(want))[finite].all() and finite.sum() > 0.5 * finite.numel() * (K - 2) / K * (N - 1) / N
    assert not beyond[torch.isfinite(want)].any()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,N,P", [(40, 20, 100), (100, 72, 140003)])
def test_8bit_scales_of_any_size(kind, K, N, P):
    """scales of positions down to the smallest normal number, as rms_norm_8bit gives them, and up to 1e30, with scales of weights around 1e-3"""
    dt = TYPES[kind]
    pair = (2,) if dt.is_complex else ()
    P //= 2 if pair else 1
    xq = (randn((K, P) + pair, torch.float32, 20) * 100).to(torch.float8_e4m3fn)
    Wq = (randn((N, K) + pair, torch.float32, 21) * 100).to(torch.float8_e4m3fn)
    ws = 1e-3 * (0.5 + torch.rand(N, generator=torch.Generator().manual_seed(22))).cuda()
    xs = torch.ones(P, device="cuda")
    idx, _ = picked(P)
    xs[idx] = (2.0 ** (torch.rand(len(idx), generator=torch.Generator().manual_seed(23)) * 226 - 126)).cuda()
    y = tf.mix_8bit(xq, xs, Wq, ws, dtype=dt)
    X, V = xq[:, idx].cpu().double(), Wq.cpu().double()
    if pair:
        X, V = torch.view_as_complex(X.contiguous()), torch.view_as_complex(V)
    X, V = X * wide(xs[idx]), V * wide(ws)[:, None]
    Z = V @ X
    bound = product_bound(V, X, K * (2 if pair else 1)) + 3 * EPS32 * Z.abs()
    smallest = 2.0 ** -133 if dt == torch.bfloat16 else 2.0 ** -149         # of the type, for results that are no normal numbers
    within(y[:, idx], Z, bound + 1.01 * rounding(dt) * (Z.abs() + bound) + 2 * smallest, "y")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("K,N,P", SIZES[2:])
def test_small_values_beside_a_nan(kind, K, N, P):
    """a column that is not a number, or infinite, beside one below the range of the split, which keeps fp32 precision, as the ordinary ones beside them do"""
    dt, (K, P) = TYPES[kind], sized(kind, K, P)
    x, W = randn((K, P), dt, 30), randn((N, K), dt, 31, K ** -0.5)
    idx, _ = picked(P)
    x[:, idx[0::4]] *= 1e-35
    x[:, idx[1::8]] = float("nan")
    x[:, idx[5::8]] = float("inf")
    rest = torch.tensor([i for i in range(len(idx)) if i % 4 != 1], device="cuda")
    terms = K * (2 if dt.is_complex else 1)
    for got in (tf.mix(x, W), tf.mix_input_grad(x, W.mH.contiguous())[0]):
        got = got[:, idx]
        X, V = wide(x[:, idx[rest]]), wide(W)
        within(got[:, rest], V @ X, product_bound(V, X, terms) + tiny(terms, V), "beside")
        touched = got[:, 1::8]
        assert torch.isnan(torch.view_as_real(touched.contiguous())).any(-1).all() if dt.is_complex else torch.isnan(touched).all()
