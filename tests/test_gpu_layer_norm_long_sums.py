"""Gradient of the layer norm over more strips than one launch takes: sums over positions that do not drift, and every strip's results."""
import pytest
import torch

import turbofno_amd as tf
from layer_norm_reference import along, wide
from operators_reference import EPS32, TYPES, randn
from test_gpu_layer_norm import rng_of

pytestmark = pytest.mark.gpu


def chain(columns, lanes):
    """additions in a row: four columns of each of a block's strips, at most 64 of a launch, the lanes, and the blocks of all launches, 64 at a time, and those sums"""
    strips = -(-columns // (4 * lanes))
    return 4 * min(65, -(-strips // 512)) + 6 + -(-strips // (64 * 512)) * 512 // 64 + 2 + 16


@pytest.mark.parametrize("K,P", [(2, 1 << 28), (70, 1 << 25)])
def test_sums_do_not_drift(K, P):
    """the same gradient everywhere: every rounding of a sum that grows is off in the same direction"""
    gy, s = torch.full((K, P), 0.1, device="cuda"), torch.ones((K, P), device="cuda")
    mean, rstd, gain = torch.zeros(P, device="cuda"), torch.ones(P, device="cuda"), torch.ones(K, device="cuda")
    _, _, ggain, gbias = tf.layer_norm_backward(gy, s, gain, mean, rstd, gx=gy)
    want = torch.tensor(0.1).double().item() * P
    bound = chain(P, 64 if K <= 64 else 16) * EPS32
    off = max((t.double() / want - 1).abs().max().item() for t in (ggain, gbias))
    print("off %.2e, bound %.2e" % (off, bound), flush=True)
    assert off <= bound
    del gy, s
    torch.cuda.empty_cache()


# strips of 256 columns, of 64, of 32 (32-bit fields of 257 to 512 channels) and of 64 read twice: one launch and a little more, and several
@pytest.mark.parametrize("kind,K,P", [("f32", 3, (1 << 23) + 77), ("bf16", 70, (1 << 21) + 35), ("c64", 66, (3 << 20) + 5), ("f32", 300, (1 << 20) + 64), ("f32", 300, (1 << 20) + 3), ("bf16", 530, (1 << 21) + 1)])
def test_several_launches(kind, K, P):
    dt, drop, rng = TYPES[kind], 0.2, rng_of()
    wide_type = torch.complex64 if dt.is_complex else torch.float32
    gy, s, gs = (randn((K, P), dt, seed) for seed in (1, 2, 3))
    mean, rstd, gain = 0.1 * randn((P,), wide_type, 4), 0.5 + torch.rand(P, device="cuda"), 1 + 0.2 * randn((K,), torch.float32, 5)
    room = tf.layer_norm_backward_workspace_bytes(K, P, dt)
    workspace = torch.full((room + 4096,), 77, dtype=torch.uint8, device="cuda")
    gx, gr, ggain, gbias = tf.layer_norm_backward(gy, s, gain, mean, rstd, gs=gs, drop=drop, rng=rng, workspace=workspace[:room])
    assert (workspace[room:] == 77).all()
    gains, biases = torch.zeros(K, dtype=torch.float64, device="cuda"), torch.zeros(K, dtype=torch.complex128 if dt.is_complex else torch.float64, device="cuda")
    sizes, bias_sizes = torch.zeros_like(gains), torch.zeros_like(gains)
    step = 1 << 18
    for a in range(0, P, step):
        p = slice(a, min(P, a + step))
        h, g = (wide(s[:, p]) - wide(mean[p])) * wide(rstd[p]), wide(gy[:, p])
        gains += along(h, g).sum(1)
        biases += g.sum(1)
        sizes += (h.abs() * g.abs()).sum(1)
        bias_sizes += g.abs().sum(1)
        # the gradients of these positions by themselves; gx is dropout of gr as it stands in 32 bits
        alone = tf.layer_norm_backward(gy[:, p], s[:, p], gain, mean[p].contiguous(), rstd[p].contiguous(), gs=gs[:, p])[0]
        off = (wide(alone) - wide(gr[:, p])).abs()
        assert (off <= 64 * EPS32 * (wide(gr[:, p]).abs() + 4) + (2.0 ** -7 * wide(gr[:, p]).abs() if kind == "bf16" else 0)).all(), a
        del h, g, alone, off
    if kind != "bf16":
        assert torch.equal(gx, tf.dropout(gr, drop, rng))
    else:
        assert torch.equal(gx == 0, tf.dropout(gr, drop, rng) == 0)
    bound = (chain(P * (2 if dt.is_complex else 1), 64 if K <= 64 else 8 if K == 300 else 16) + 4) * EPS32 * (2 if dt.is_complex else 1)
    assert ((ggain.double() - gains).abs() <= bound * sizes).all()
    assert ((gbias.to(biases.dtype) - biases).abs() <= bound * bias_sizes).all()
    del gy, s, gs, gx, gr
    torch.cuda.empty_cache()
