"""Norms whose result replaces x: the s that the gradient takes is what x was."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import TYPES, randn

pytestmark = pytest.mark.gpu


def operands(kind, K, P):
    dt = TYPES[kind]
    return randn((K, P), dt, 1), 1 + 0.2 * randn((K,), torch.float32, 2), randn((K,), torch.complex64 if dt.is_complex else torch.float32, 3), randn((K, P), dt, 4)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,P", [(20, 300), (600, 70)])
@pytest.mark.parametrize("drop", [0.0, 0.3])
def test_layer_norm(kind, K, P, drop):
    x, gain, bias, gy = operands(kind, K, P)
    rng = torch.tensor([5, 6], device="cuda") if drop else None
    want = tf.layer_norm(x, gain, bias, drop=drop, rng=rng)
    grads = tf.layer_norm_backward(gy, want[1], gain, want[2], want[3], drop=drop, rng=rng)
    for y in (x.clone(), torch.zeros((K, P + 8), dtype=x.dtype, device="cuda")[:, 3:3 + P]):
        y.copy_(x)
        got = tf.layer_norm(y[:], gain, bias, drop=drop, rng=rng, y=y)
        assert got[0] is y and all(torch.equal(a, b) for a, b in zip(got, want))
        again = tf.layer_norm_backward(gy, got[1], gain, got[2], got[3], drop=drop, rng=rng)
        assert all(torch.equal(a, b) for a, b in zip(again, grads))
    place, s = x.clone(), torch.empty_like(x)
    got = tf.layer_norm(place, gain, bias, drop=drop, rng=rng, y=place, s=s)
    assert got[1] is s and all(torch.equal(a, b) for a, b in zip(got, want))
    empty = x[:, :0].contiguous()
    assert tf.layer_norm(empty, gain, bias, y=empty)[1].shape == (K, 0)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,P", [(20, 300), (600, 70)])
@pytest.mark.parametrize("passed", [True, False])
def test_rms_norm(kind, K, P, passed):
    x, gain, _, gy = operands(kind, K, P)
    want = tf.rms_norm(x, gain)
    grads = tf.rms_norm_backward(gy, want[1], gain, want[2])
    place, rstd = x.clone(), torch.empty(P, device="cuda") if passed else None
    got = tf.rms_norm(place, gain, y=place, rstd=rstd)
    assert got[0] is place and all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(tf.rms_norm_backward(gy, got[1], gain, got[2]), grads))
    place, s = x.clone(), torch.empty_like(x)
    got = tf.rms_norm(place, gain, y=place, s=s, rstd=rstd)
    assert got[1] is s and all(torch.equal(a, b) for a, b in zip(got, want))
