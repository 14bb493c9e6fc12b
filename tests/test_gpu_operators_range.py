"""Channel product and its gradients on 32-bit operands below the range of the split into bf16 parts (2^-110): fp32 precision down to the smallest normal
numbers, in columns and weights of any magnitude among others near one."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import EPS32, TYPES, product_bound, randn, slope, wide, within

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
