"""The product in 8 bits with scales by blocks with so many rows that tiles are plenty at few positions: around the columns that the widest tiles take."""
import pytest
import torch

import turbofno_amd as tf
from test_gpu_8bit_blocks import product_operands
from test_gpu_8bit_blocks_kernels import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,K,N,P", [(kind,) + shape for kind in ("f32", "bf16") for shape in ((65, 24600, 129), (200, 32000, 200), (65, 49200, 128), (130, 24600, 255), (256, 24600, 256),
                                                                                           (512, 24460, 257), (384, 49200, 144))] + [("c64", 40, 24600, 64), ("c64", 65, 24600, 100)])
def test_many_rows(kind, K, N, P):
    """x and its scales start their memory: nothing ahead of them is read, whose scales would have sent waves another way"""
    operands = product_operands(kind, K, N, (P,), 3)
    y = tf.mix_8bit_blocks(*operands, activation="silu")
    check(kind, operands, "silu", y, K * (2 if kind == "c64" else 1))
    xq, xscale = operands[:2]
    whole = torch.full((256 + xscale.numel(),), float("nan"), device="cuda")          # scales ahead of the first that are none
    whole[256:] = xscale.flatten()
    place = operands[5].clone()
    tf.mix_8bit_blocks(xq, whole[256:].view(xscale.shape), *operands[2:5], residual=place, activation="silu", y=place)
    assert torch.equal(place, y)
