"""Which operands of the operators around the layer may share memory: every result is apart from what the call reads or writes, except in the places
that the header names. Refusals are checked without a GPU, on addresses that are never looked at."""
import random

import pytest
import torch

import turbofno_amd as tf
from operators_reference import TYPES, randn
from turbofno_amd import operators

BASE = 1 << 32                          # an address, for calls that are refused
INVALID, WORKSPACE = 1, 3               # TURBOFNO_ERR_INVALID_ARG, _WORKSPACE


def _meet(a, b, width):
    """the bytes of rows (address, rows, pitch) one by one"""
    def covered(place):
        at, rows, pitch = place
        return {at + i * pitch + j for i in range(rows) for j in range(width)}
    return bool(covered(a) & covered(b))


def test_rows_that_meet_and_rows_that_do_not():
    """gx against gy and s of the norm's gradient: refused for their memory, or, one check further, for the missing workspace"""
    L, rng = operators._lib(), random.Random(5)
    outcomes = []
    for _ in range(4000):
        K, P = rng.randint(1, 6), rng.randint(1, 5)
        ld = lambda: rng.randint(P, 4 * P + 3)  # noqa: E731
        lx, lg = ld(), ld()
        if rng.random() < 0.5:
            lg = lx                     # column ranges of one buffer
        gx, gy = BASE + 4 * rng.randint(0, 60), BASE + 4 * rng.randint(0, 60)
        rc = L.turbofno_rms_norm_backward(1, P, K, gy, lg, BASE << 1, P, 1, 1, None, 0, gx, lx, 1, None, 0, None)
        same = gx == gy and (lx == lg or K == 1)
        expected = INVALID if _meet((gx, K, 4 * lx), (gy, K, 4 * lg), 4 * P) and not same else WORKSPACE
        assert rc == expected, (K, P, lx, lg, (gx - BASE) // 4, (gy - BASE) // 4, L.turbofno_last_error_string())
        outcomes.append(rc)
    assert 500 < outcomes.count(INVALID) < 3500


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_column_ranges_of_one_buffer(kind):
    """x, residual and results side by side in the rows of one buffer"""
    K, N, P, dt = 24, 24, 70, TYPES[kind]
    x, r, W = randn((K, P), dt, 1), randn((N, P), dt, 2), randn((N, K), dt, 3, K ** -0.5)
    rows = torch.zeros((N, 4 * P), dtype=dt, device="cuda")
    bx, br, by, bz = (rows[:, i * P:(i + 1) * P] for i in range(4))
    bx.copy_(x)
    br.copy_(r)
    z = torch.empty_like(r)
    y = tf.mix(x, W, residual=r, activation="silu", z=z)
    tf.mix(bx, W, residual=br, activation="silu", y=by, z=bz)
    assert torch.equal(by, y) and torch.equal(bz, z) and torch.equal(bx, x) and torch.equal(br, r)
    gain = randn((K,), torch.float32, 4)
    want = tf.rms_norm(x, gain, r)
    tf.rms_norm(bx, gain, br, y=by, s=bz)
    assert torch.equal(by, want[0]) and torch.equal(bz, want[1]) and torch.equal(bx, x) and torch.equal(br, r)
    gx, ggain = tf.rms_norm_backward(x, want[1], gain, want[2])
    tf.rms_norm_backward(bx, bz, gain, want[2], gx=by)
    assert torch.equal(by, gx) and torch.equal(bx, x)
