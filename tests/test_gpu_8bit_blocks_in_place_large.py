"""The product in 8 bits with scales by blocks over the residual, where a launch has several rows of blocks and tiles side by side go to one XCD: added and activated once each."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import TYPES, randn
from test_gpu_8bit_blocks import quantised_weights
from test_gpu_8bit_blocks_kernels import check

pytestmark = pytest.mark.gpu


# more than 2^22 tiles of 128 columns (complex64: 256 real ones): staged, direct, and the complex tiles; float32, whose tiles go to the XCDs in turns, has none to spare
@pytest.mark.parametrize("kind,K,N,P", [("bf16", 65, 4, (1 << 29) + 77), ("bf16", 128, 4, (1 << 29) + 48), ("c64", 33, 2, (1 << 29) + 5), ("f32", 65, 2, (1 << 29) + 77)])
def test_once_each(kind, K, N, P):
    dt, pair = TYPES[kind], (2,) if kind == "c64" else ()
    xq = torch.empty((K, P) + pair, dtype=torch.uint8, device="cuda").random_(0, 0x60).view(torch.float8_e4m3fn)
    xscale = torch.rand((-(-K // 128), P), device="cuda") + 0.5
    Wq, wscale = quantised_weights(randn((N, K) + pair, torch.float32, 2, K ** -0.5))
    bias, place = randn((N,), dt, 3), randn((N, P), dt, 4)
    parts = [slice(p, p + 3000) for p in (0, (1 << 28) - 77, P // 8 - 1000, P // 2 - 999, 5 * P // 8, P - 3000)]
    before = [place[:, p].clone() for p in parts]
    want = tf.mix_8bit_blocks(xq, xscale, Wq, wscale, bias=bias, residual=place, activation="silu")
    got = tf.mix_8bit_blocks(xq, xscale, Wq, wscale, bias=bias, residual=place, activation="silu", y=place)
    assert got is place and torch.equal(got, want)
    for p, r in zip(parts, before):
        check(kind, (xq[:, p], xscale[:, p], Wq, wscale, bias, r), "silu", got[:, p], K * (2 if pair else 1))
    del xq, place, want, got
    torch.cuda.empty_cache()
