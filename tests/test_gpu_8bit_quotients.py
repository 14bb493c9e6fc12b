"""The values of 8-bit fields are the quotients by their scale, rounded as a division and a conversion round them: ties between two numbers of e4m3 go to the even one."""
import pytest
import torch

import turbofno_amd as tf
from layer_norm_reference import BLOCK, per_channel
from operators_reference import TYPES, randn

pytestmark = pytest.mark.gpu


def parts_of(t):
    """[K][P][1 or 2] in float32 on the CPU"""
    t = t.detach().cpu().flatten(1)
    return torch.view_as_real(t) if t.is_complex() else t.float()[..., None]


def check(v, q, scale):
    """every value of v [K][P][1 or 2]: the CPU's division and conversion round to nearest, ties to even"""
    K = v.shape[0]
    want = torch.stack([b.abs().amax((0, 2)) for b in v.split(BLOCK)]) / 448
    assert torch.equal(scale.cpu().flatten(1), want)
    quotients = (v / per_channel(want, K)[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    got = q.cpu().reshape(v.shape)
    off = (got.float() != quotients.float()).sum().item()
    assert off == 0, "%d of %d values" % (off, got.numel())


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,P", [(128, 4001), (300, 70), (20, 70001), (260, 66000)])
@pytest.mark.parametrize("size", [0, -110, 100])
def test_quantise(kind, K, P, size):
    """bf16 values, of which one in a thousand has a quotient half way between two numbers; scales near both ends of the normal numbers too"""
    dt = TYPES[kind]
    wide = torch.complex64 if dt.is_complex else torch.float32
    x = randn((K, P), wide, 1)
    x = (torch.view_as_complex(torch.view_as_real(x).bfloat16().float()) if dt.is_complex else x.bfloat16()).to(dt) * 2.0 ** size
    q, scale = tf.quantise_8bit(x)
    check(parts_of(x), q, scale)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K,P", [(64, 131073), (200, 1001), (128, 40004), (512, 333), (512, 9000), (1000, 33), (2000, 130), (2500, 900), (2500, 9001)])
def test_layer_norm(kind, K, P):
    """half of a position's values 1 and half -1: mean 0, deviation 1, so that y is the gain or its negative whatever the roundings"""
    dt = TYPES[kind]
    x = torch.ones((K, P), dtype=dt, device="cuda")
    x[::2] = -1
    x[:, P // 2:] *= -1
    gain = randn((K,), torch.float32, 2).bfloat16().float()
    y, _, mean, rstd = tf.layer_norm(x, gain, eps=0.0)
    assert (mean == 0).all() and (rstd == 1).all()
    q, scale, _ = tf.layer_norm_8bit(x, gain, eps=0.0)
    check(parts_of(x) * gain.cpu()[:, None, None], q, scale)
