"""Sums over many positions do not drift: the error of the weights' gradient grows like that of random roundings, not with the number of positions."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import EPS32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,P,C", [(torch.float32, (1 << 24) + 5, 16), (torch.complex64, (1 << 23) + 5, 16), (torch.float32, 1 << 27, 16),
                                    (torch.float32, (1 << 24) + 5, 40), (torch.complex64, (1 << 23) + 5, 40)])
def test_weight_gradient_of_many_positions(dt, P, C):
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, gz = (torch.randn((C, P), dtype=dt, device="cuda", generator=gen) for _ in range(2))
    gW, gbias = tf.mix_weight_grad(gz, x)
    wide = torch.complex128 if dt.is_complex else torch.float64
    exact, bias = torch.zeros((C, C), dtype=wide, device="cuda"), torch.zeros(C, dtype=wide, device="cuda")
    for g, v in zip(gz.split(1 << 21, 1), x.split(1 << 21, 1)):
        exact += g.to(wide) @ v.to(wide).mH.contiguous()
        bias += g.to(wide).sum(1)
    # roundings in a row: six products of each of a run's 16 steps, the runs of a wave (2048 waves, steps of 32 values), four waves, 128 parts
    runs = P * (2 if dt.is_complex else 1) / (2048 * 16 * 32)
    bound = 2 * (96 + runs + 4 + 128) ** 0.5 * EPS32
    off = ((gW.to(wide) - exact).norm() / exact.norm()).item()
    print("error %.2e, bound %.2e" % (off, bound), flush=True)
    assert off <= bound
    # a lane adds eight values of each of a wave's steps, one after the other's sum
    steps = P * (2 if dt.is_complex else 1) / (2048 * 32)
    assert ((gbias.to(wide) - bias).norm() / bias.norm()).item() <= 2 * (steps + 3 + 20 + 128) ** 0.5 * EPS32
