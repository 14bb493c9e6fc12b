"""Which operands of the operators around the layer may share memory: every result is apart from what the call reads or writes, except in the places
that the header names. Refusals are checked without a GPU, on addresses that are never looked at."""
import ctypes
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


def test_weight_gradient_apart_from_its_operands():
    """gW, gbias and the workspace against gz, x and one another, in fields of 6 and 4 channels of 10 float32 values"""
    L = operators._lib()
    need = L.turbofno_mix_weight_grad_workspace_bytes(1, 10, 6, 4)
    gz, x, gW, gbias, ws = (BASE + (i << 20) for i in range(5))

    def refused(**k):
        o = {**dict(gz=gz, ldgz=10, x=x, ldx=10, gW=gW, gbias=gbias, ws=ws, bytes=need), **k}
        rc = L.turbofno_mix_weight_grad(1, 10, 6, 4, o["gz"], o["ldgz"], o["x"], o["ldx"], o["gW"], o["gbias"], o["ws"], o["bytes"], None)
        return rc == INVALID and b"overlap" in L.turbofno_last_error_string()
    assert refused(gW=x) and refused(gW=gz + 4 * 59) and refused(gW=x - 4 * 23) and refused(gbias=gz) and refused(gbias=x + 4 * 39)
    assert refused(ws=x) and refused(ws=gz + 4 * 59) and refused(gW=ws) and refused(gbias=gW + 4 * 23) and refused(gbias=ws + need - 4)
    # beside them, one check further: for a workspace that is too small
    for k in (dict(gW=x + 160), dict(gW=gz + 240), dict(gbias=gW + 96), dict(gbias=None), dict(x=gz), dict(ldx=40, gbias=x + 40), dict(gW=ws + need)):
        assert not refused(**k, bytes=4) and b"workspace of 4 bytes" in L.turbofno_last_error_string(), k


@pytest.mark.gpu
@pytest.mark.parametrize("kind", TYPES)
def test_weight_gradient_refusals(kind):
    dt = TYPES[kind]
    gz, x = randn((6, 40), dt, 1), randn((4, 40), dt, 2)
    with pytest.raises(tf.TurboFNOError, match="overlaps gz or x"):
        tf.mix_weight_grad(gz, x, gW=x.flatten()[:24].view(6, 4))
    with pytest.raises(tf.TurboFNOError, match="overlaps gz or x"):
        tf.mix_weight_grad(gz, x, gbias=gz[0, :6])
    want, _ = tf.mix_weight_grad(gz, x)
    between = torch.cat([x, x], 1)      # gbias in the columns that x leaves free
    got, gbias = tf.mix_weight_grad(gz, between[:, :40], gbias=between[0, 40:46])
    assert torch.equal(got, want) and torch.equal(between[0, :40], x[0])


def test_results_apart_from_weights_scales_and_the_workspace():
    """fields of 6 and 4 channels of 10 float32 values; the overlap is looked for last of what is checked before the launch, or before the workspace"""
    L = operators._lib()
    x, W, bias, r, y, z, xs, ws = (BASE + (i << 20) for i in range(8))

    def says(rc, text):
        return rc == INVALID and text in L.turbofno_last_error_string()

    def mix(**k):
        o = {**dict(x=x, W=W, bias=bias, r=r, y=y, z=z), **k}
        return L.turbofno_mix(1, 10, 6, 4, o["x"], 10, o["W"], o["bias"], o["r"], 10, 0, o["z"], 10, o["y"], 10, None)
    assert says(mix(W=y + 4 * 59), b"W or bias") and says(mix(bias=z - 4 * 5), b"W or bias") and says(mix(bias=y), b"W or bias") and says(mix(W=z), b"W or bias")

    def mix8(**k):
        o = {**dict(x=x, W=W, bias=bias, r=r, y=y, xs=xs, ws=ws), **k}
        return L.turbofno_mix_8bit(1, 10, 6, 4, o["x"], 10, o["xs"], o["W"], o["ws"], o["bias"], o["r"], 10, 0, o["y"], 10, None)
    assert all(says(mix8(**{name: y + 8}), b"a scale") for name in ("W", "bias", "xs", "ws")) and says(mix8(W=y - 23), b"a scale")

    def input_grad(**k):
        o = {**dict(gy=r, z=z, W=W, gz=y, gx=x), **k}
        return L.turbofno_mix_input_grad(1, 10, 6, 4, o["gy"], 10, o["z"], 10, o["W"], 1, o["gz"], 10, o["gx"], 10, None)
    assert says(input_grad(W=x), b"overlaps W") and says(input_grad(W=y + 4 * 59), b"overlaps W")

    def norm(call, **k):
        o = {**dict(x=x, r=r, gain=W, s=z, y=y, rstd=xs), **k}
        return getattr(L, call)(1, 10, 4, o["x"], 10, o["r"], 10, o["gain"], 1e-6, o["s"], 10, o["y"], 10, o["rstd"], None)
    for call in ("turbofno_rms_norm", "turbofno_rms_norm_8bit"):
        assert says(norm(call, gain=y + 8), b"gain") and says(norm(call, gain=z), b"gain")
        assert all(says(norm(call, rstd=p + 8), b"another operand") for p in (x, r, z, y, W))

    def norm_grad(need=0, **k):
        o = {**dict(gy=y, s=z, gain=W, rstd=xs, gs=r, gx=x, ggain=bias, ws=ws), **k}
        return L.turbofno_rms_norm_backward(1, 10, 4, o["gy"], 10, o["s"], 10, o["gain"], o["rstd"], o["gs"], 10, o["gx"], 10, o["ggain"], o["ws"], need, None)
    assert all(says(norm_grad(**{name: x + 8}), b"gx overlaps gain") for name in ("gain", "rstd", "ggain"))
    assert all(says(norm_grad(ws=p + 8), b"the workspace overlaps") for p in (y, z, r, x, W, xs, bias))
    assert norm_grad() == WORKSPACE and norm_grad(ggain=W) == WORKSPACE      # gain is read before ggain is written


def test_places_of_tensors():
    """the rule of the binding against single elements"""
    rng = random.Random(9)
    outcomes = []
    for _ in range(3000):
        base = torch.arange(90)

        def part():
            rows, width = rng.randint(1, 5), rng.randint(1, 5)
            pitch = rng.choice([10, rng.randint(width, 16)])
            return base.as_strided((rows, width), (pitch, 1), rng.randint(0, 90 - (rows - 1) * pitch - width))
        a, b = part(), part()
        expected = bool(set(a.flatten().tolist()) & set(b.flatten().tolist()))
        assert operators._meet(a, b) == expected and operators._meet(b, a) == expected, (a, b)
        outcomes.append(expected)
    assert 300 < sum(outcomes) < 2700
    assert not operators._meet(None, base) and not operators._meet(base, "x") and not operators._meet(base[:0], base)


@pytest.mark.gpu
@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("kind", TYPES)
def test_backward_results_apart_from_x(kind, compiled, monkeypatch):
    """what the second of the two products reads is not written by the first, nor what the first wrote by the second"""
    if not compiled:
        monkeypatch.setattr(operators.api, "_operands", None)
    dt, C, P = TYPES[kind], 12, 50
    gy, x, z, W = randn((C, P), dt, 1), randn((C, P), dt, 2), randn((C, P), dt, 3), randn((C, C), dt, 4)
    gx, gW, gbias, gz = tf.mix_backward(gy, x, W, z, "silu")
    kept = x.clone()
    rows = torch.cat([x, x], 1)
    for activation in ("silu", "none"):
        with pytest.raises(ValueError, match="gx overlaps x"):
            tf.mix_backward(gy, x, W, z, activation, gx=x)
        with pytest.raises(ValueError, match="gx overlaps x"):
            tf.mix_backward(gy, rows[:, :P], W, z, activation, gx=rows[:, 1:1 + P])
        with pytest.raises(ValueError, match="gW overlaps gx"):
            tf.mix_backward(gy, x, W, z, activation, gx=gx, gW=gx.flatten()[:C * C].view(C, C))
        with pytest.raises(ValueError, match="gbias overlaps gx"):
            tf.mix_backward(gy, x, W, z, activation, gx=gx, gbias=gx[3, :C])
        with pytest.raises(ValueError, match="workspace overlaps gx"):
            tf.mix_backward(gy, x, W, z, activation, gx=gx, workspace=torch.view_as_real(gx).view(torch.uint8) if dt.is_complex else gx.view(torch.uint8))
    with pytest.raises(ValueError, match="gz overlaps x"):
        tf.mix_backward(gy, x, W, z, "silu", gz=x)
    assert torch.equal(x, kept)
    with pytest.raises(tf.TurboFNOError, match="0 elements between channels"):
        tf.mix_backward(gy, x[:1].expand(C, P), W, z, "silu", gx=rows[:, :P])
    with pytest.raises(tf.TurboFNOError, match="0 elements between channels"):
        tf.mix_backward(gy, kept[:1].expand(C, P), W, z, "silu", gx=kept)
    # beside x in the same rows, and over operands that both products have read by then
    rows = torch.cat([x, x], 1)
    results = tf.mix_backward(gy, rows[:, :P], W, z, "silu", gx=rows[:, P:])
    assert torch.equal(rows[:, P:], gx) and torch.equal(rows[:, :P], x) and torch.equal(results[1], gW)
    own = W.clone()
    results = tf.mix_backward(gy, x, own, z, "silu", gW=own)
    assert torch.equal(own, gW) and torch.equal(results[0], gx) and torch.equal(results[2], gbias) and torch.equal(results[3], gz)


def test_clipped_tensors_that_meet():
    """lists of one to five tensors against single bytes: refused for their memory, or, one check further, for the missing workspace"""
    L, rng = operators._lib(), random.Random(11)
    bytes_of = {0: 8, 1: 4, 2: 2}
    outcomes = []
    for round_ in range(6000):
        n = rng.randint(1, 5)
        kinds, sizes = [rng.randint(0, 2) for _ in range(n)], [rng.choice([0, 1, 2, 3, 5]) for _ in range(n)]
        where = lambda: BASE + 2 * rng.randint(0, 200)  # noqa: E731
        grads = [where() for _ in range(n)]
        out = [g if rng.random() < 0.7 else where() for g in grads]
        norm = BASE + 1000 if rng.random() < 0.9 else where()
        rc = L.turbofno_clip_grad_norm(n, (ctypes.c_void_p * n)(*grads), (ctypes.c_void_p * n)(*out), (ctypes.c_long * n)(*sizes), (ctypes.c_int * n)(*kinds),
                                       1.0, norm, None, 0, None)
        covered = lambda at, i: set(range(at, at + sizes[i] * bytes_of[kinds[i]]))  # noqa: E731
        at_norm = set(range(norm, norm + 4))
        meet = any(covered(out[i], i) & covered(out[j], j) for i in range(n) for j in range(i))
        meet |= any(covered(out[i], i) & covered(grads[j], j) for i in range(n) for j in range(n) if i != j or out[i] != grads[j])
        meet |= any((covered(out[i], i) | covered(grads[i], i)) & at_norm for i in range(n))
        assert rc == (INVALID if meet else WORKSPACE), (grads, out, sizes, kinds, norm, L.turbofno_last_error_string())
        outcomes.append(rc)
    assert 1000 < outcomes.count(INVALID) < 5000


@pytest.mark.gpu
@pytest.mark.parametrize("count", [3, 150])
def test_clip_refuses_shared_memory(count):
    flat = randn((count * 100,), torch.float32, 1)
    grads = [flat[i * 100:(i + 1) * 100] for i in range(count)]
    kept = flat.clone()
    for again in (grads[1], flat[250:260], flat[:7], flat[99:101]):
        with pytest.raises(tf.TurboFNOError, match="overlap"):
            tf.clip_grad_norm(grads + [again], 0.1)
        with pytest.raises(tf.TurboFNOError, match="overlap"):
            tf.clip_grad_norm(grads + [again], 0.1, out=grads + [torch.empty_like(again)])
    with pytest.raises(tf.TurboFNOError, match="overlaps the norm"):
        tf.clip_grad_norm(grads, 0.1, norm=flat[5])
    assert torch.equal(flat, kept)
    # parts of one buffer, and a gradient that is read twice, are taken
    out = torch.empty_like(flat)
    norm = tf.clip_grad_norm(grads + [grads[0]], 0.1, out=[out[i * 100:(i + 1) * 100] for i in range(count)] + [torch.empty(100, device="cuda")])
    exact = (flat.double().square().sum() + grads[0].double().square().sum()).sqrt()
    assert abs(norm.item() - exact.item()) <= 2.0 ** -22 * exact.item()
    tf.clip_grad_norm(list(reversed(grads)), 0.1)
    assert not torch.equal(flat, kept)
