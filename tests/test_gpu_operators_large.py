"""Sizes at which a launch has more threads than a dimension of a grid holds, 2^32: one channel of billions of positions, a billion weights."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import EPS32

pytestmark = pytest.mark.gpu
PART = 1 << 27                          # positions compared at once


def filled(shape, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.empty(shape, dtype=dtype, device="cuda")
    for part in t.view(-1).split(PART):
        part.copy_(torch.randn(part.shape, device="cuda", generator=gen))
    return t


@pytest.fixture(autouse=True)
def memory_given_back():
    yield
    torch.cuda.empty_cache()


def test_norm_of_billions_of_positions():
    P = (1 << 31) + 333
    x, gain = filled((1, P), torch.bfloat16, 1), torch.full((1,), 1.5, device="cuda")
    y, _, rstd = tf.rms_norm(x, gain)
    for a, b, r in zip(x[0].split(PART), y[0].split(PART), rstd.split(PART)):
        want = 1 / torch.sqrt(a.double() ** 2 + 1e-6)
        assert ((r.double() - want).abs() <= 16 * EPS32 * want).all()
        want = 1.5 * want * a.double()
        assert ((b.double() - want).abs() <= (2.0 ** -8 + 32 * EPS32) * want.abs()).all()
    del y, rstd
    print("norm", flush=True)
    q, scale, _ = tf.rms_norm_8bit(x, gain)
    for a, b, r in zip(x[0].split(PART), q[0].split(PART), scale.split(PART)):
        want = 1.5 * a.double().abs() / torch.sqrt(a.double() ** 2 + 1e-6) / 448
        want = torch.where(want > 0, want, torch.ones_like(want))
        assert ((r.double() - want).abs() <= 32 * EPS32 * want).all()
        assert torch.equal(b.float(), 448 * torch.sign(a.float()))


def test_product_of_billions_of_positions():
    P = (1 << 32) + 77
    x, W, bias = filled((1, P), torch.float32, 2), torch.full((1, 1), 0.75, device="cuda"), torch.full((1,), 0.5, device="cuda")
    y = tf.mix(x, W, bias)
    for a, b in zip(x[0].split(PART), y[0].split(PART)):
        want = 0.75 * a.double() + 0.5
        assert ((b.double() - want).abs() <= 4 * EPS32 * (want.abs() + 1)).all()


def test_gradient_of_a_billion_weights():
    """gz x^H of one position: each product is exact in fp32"""
    N = K = 32768
    gz, x = filled((N, 1), torch.bfloat16, 3), filled((K, 1), torch.bfloat16, 4)
    gW, gbias = tf.mix_weight_grad(gz, x)
    assert torch.equal(gbias, gz[:, 0])
    for rows, g in zip(gW.split(2048), gz.split(2048)):
        assert torch.equal(rows, (g.float() * x.float().t()).to(torch.bfloat16))
