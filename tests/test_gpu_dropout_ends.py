"""Dropout at the ends of its range: almost everything and almost nothing dropped."""
import pytest
import torch

import turbofno_amd as tf
from layer_norm_reference import kept

pytestmark = pytest.mark.gpu
SEED = (11, 12)


@pytest.mark.parametrize("drop", [1 - 2.0 ** -53, 1 - 2.0 ** -33, 1 - 2.0 ** -20, 2.0 ** -33, 2.0 ** -34, 2.0 ** -60, 5e-324])
def test_threshold(drop):
    """the whole number nearest to drop 2^32, at most 2^32 - 1: a word of all ones is kept whatever is dropped"""
    x, rng = torch.ones((64, 100003), device="cuda"), torch.tensor(SEED, device="cuda")
    y = tf.dropout(x, drop, rng)
    keep = kept(SEED, 64, 100003, drop)
    assert torch.equal(y != 0, keep) and (y[keep] == torch.tensor(1 / (1 - drop), dtype=torch.float32)).all()
    if drop <= 2.0 ** -33:                              # half, and less: to 0, the even number
        assert keep.all()
