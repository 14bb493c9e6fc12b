"""Dropout from a counter-based generator, alone and with a residual, against the generator's definition and 64-bit evaluations."""
import pytest
import torch

import turbofno_amd as tf
from layer_norm_reference import dropped, kept, philox, rounded, wide, within
from operators_reference import EPS32, TYPES, randn

SEED = (0x0123456789ABCDEF, -5)         # both words of both numbers in use


def rng_of(seed=SEED[0], offset=SEED[1]):
    return torch.tensor([seed, offset], dtype=torch.int64, device="cuda")


def test_generator_against_its_published_vectors():
    """the three known answers that its authors publish for philox4x32 with ten rounds"""
    words = lambda text: [torch.tensor(int(w, 16)) for w in text.split()]  # noqa: E731
    for counter, key, answer in (("0 0 0 0", "0 0", "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
                                 ("ffffffff ffffffff ffffffff ffffffff", "ffffffff ffffffff", "408f276d 41c83b0e a20bc7c6 6d5451fd"),
                                 ("243f6a88 85a308d3 13198a2e 03707344", "a4093822 299f31d0", "d16cfe09 94fdcceb 5001e420 24126ea1")):
        assert philox(words(counter), words(key)) == words(answer)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,places", [(1, (1,)), (3, (5,)), (1, (1030,)), (2, (2, 2)), (70, (3,)), (33, (7, 19)), (5, (1000,)), (9, (4097,)), (300, (130,)), (1025, (2,))])
@pytest.mark.parametrize("residual", [True, False])
def test_against_the_definition(kind, K, places, residual):
    dt = TYPES[kind]
    x, r = randn((K,) + places, dt, 1), randn((K,) + places, dt, 2) if residual else None
    for drop in (0.1, 0.5, 0.973):
        y = tf.dropout(x, drop, rng_of(), residual=r)
        X = dropped(wide(x).flatten(1), SEED, drop)
        R = wide(r).flatten(1) if residual else torch.zeros_like(X)
        within(y.flatten(1), X + R, rounded(X + R, 3 * EPS32 * (X.abs() + R.abs()), dt), "y")
        if not residual:
            assert torch.equal(y.flatten(1) == 0, ~kept(SEED, K, y[0].numel(), drop))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_numbers_depend_on_seed_and_offset_alone(kind):
    """strides, alignment and a residual change nothing; other seeds and offsets, in either of their words, do"""
    dt, K, P = TYPES[kind], 37, 515
    x = torch.ones((K, P), dtype=dt, device="cuda")
    y = tf.dropout(x, 0.5, rng_of())
    wide_x, wide_y = torch.ones((K, P + 9), dtype=dt, device="cuda"), torch.full((K, P + 11), 7.0, dtype=dt, device="cuda")
    for shift in range(5):
        tf.dropout(wide_x[:, shift:shift + P], 0.5, rng_of(), y=wide_y[:, 3 + shift:3 + shift + P])
        assert torch.equal(wide_y[:, 3 + shift:3 + shift + P], y)
        assert (wide_y[:, :3 + shift] == 7).all() and (wide_y[:, 3 + shift + P:] == 7).all()
        wide_y.fill_(7.0)
    assert torch.equal(tf.dropout(x, 0.5, rng_of(), residual=x), y + 1)
    for other in (rng_of(SEED[0] + 1), rng_of(SEED[0] + (1 << 40)), rng_of(SEED[0], 3), rng_of(SEED[0], SEED[1] - (1 << 35))):
        different = (tf.dropout(x, 0.5, other) != y).float().mean().item()
        assert 0.45 < different < 0.55              # 19055 elements: five deviations are 0.018
    assert torch.equal(tf.dropout(x.view(K, 5, 103), 0.5, rng_of()).view(K, P), y)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_in_place_and_ends(kind):
    dt = TYPES[kind]
    x, r = randn((40, 333), dt, 3), randn((40, 333), dt, 4)
    y = tf.dropout(x, 0.3, rng_of(), residual=r)
    a, b = x.clone(), r.clone()
    assert tf.dropout(a, 0.3, rng_of(), residual=r, y=a) is a and torch.equal(a, y)
    tf.dropout(x, 0.3, rng_of(), residual=b, y=b)
    assert torch.equal(b, y)
    assert torch.equal(tf.dropout(x, 0.0, rng_of()), x)
    keep = kept(SEED, 40, 333, 0.3)
    x[:] = float("nan")                                 # what is dropped is 0 whatever was there
    y = tf.dropout(x, 0.3, rng_of())
    assert (y[~keep] == 0).all() and torch.isnan(y)[keep].all()
    assert tf.dropout(x[:, :0], 0.3, rng_of()).shape == (40, 0)


@pytest.mark.gpu
def test_gradient_is_the_same_call():
    """against differences of the forward pass: it is linear, so differences are exact to rounding"""
    x, g = randn((12, 50), torch.float32, 5), randn((12, 50), torch.float32, 6)
    gx = tf.dropout(g, 0.4, rng_of())
    y0 = tf.dropout(x, 0.4, rng_of()).double()
    step = randn((12, 50), torch.float32, 7)
    y1 = tf.dropout(x + step, 0.4, rng_of()).double()
    moved = (x + step).double() - x.double()
    left, right = (g.double() * (y1 - y0)).sum(), (gx.double() * moved).sum()
    assert abs((left - right).item()) <= 600 * 8 * EPS32 * 10


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_positions_beyond_32_bits_of_bytes(kind):
    """one long channel: the last positions of more than 2^32 bytes, and of more than 2^31 elements in 16 bits"""
    dt = TYPES[kind]
    P = {"c64": (1 << 29) + 333, "f32": (1 << 30) + 333, "bf16": (1 << 31) + 333}[kind]
    x = torch.ones((1, P), dtype=dt, device="cuda")
    tf.dropout(x, 0.5, rng_of(), y=x)
    for first in (0, P // 2 // 4 * 4, (P - 4001) // 4 * 4):
        assert torch.equal(x[0, first:first + 4001] != 0, kept(SEED, 1, 4001, 0.5, first=first)[0])
    del x
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_in_a_graph():
    """each replay draws what rng holds then"""
    x, rng = randn((20, 700), torch.bfloat16, 8), rng_of()
    y = torch.empty_like(x)
    tf.dropout(x, 0.2, rng, y=y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tf.dropout(x, 0.2, rng, y=y)
        rng[1:] += 1
    rng.copy_(rng_of())
    for i in range(4):
        want = tf.dropout(x, 0.2, rng_of(SEED[0], SEED[1] + i))
        torch.cuda.synchronize()
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), i
