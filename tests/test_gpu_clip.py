"""Global gradient norm and clipping over lists of tensors, against 64-bit evaluations."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import EPS32, TYPES, randn, rounding, wide, within

pytestmark = pytest.mark.gpu


def tensors(count, largest, seed=0):
    """all types in turn, sizes from one value to `largest`, odd ones and multiples of the kernels' units among them"""
    sizes = [max(1, largest // (i * i + 1) - i) for i in range(count)]
    return [randn((n,), list(TYPES.values())[i % 3], seed + i, 0.1) for i, n in enumerate(sizes)]


def exact_norm(grads):
    return sum(float((wide(g).abs() ** 2).sum()) for g in grads) ** 0.5


def check(norm, out, grads, max_norm):
    want = exact_norm(grads)
    assert norm.dim() == 0 and norm.dtype == torch.float32 and abs(norm.item() - want) <= 4 * EPS32 * want
    factor = min(1.0, max_norm / (want + 1e-6))
    for g, o in zip(grads, out):
        E = wide(g) * factor
        within(o, E, (8 * EPS32 + 1.01 * rounding(g.dtype)) * E.abs(), "clipped")


@pytest.mark.parametrize("count,largest", [(1, 1), (1, 4096), (3, 8193), (60, 100003), (97, 5000), (200, 3001), (2, 9_000_001)])
@pytest.mark.parametrize("max_norm", [0.25, 1e6])
def test_clip(count, largest, max_norm):
    grads = tensors(count, largest)
    out = [torch.full_like(g, 7.0) for g in grads]
    kept = [g.clone() for g in grads]
    check(tf.clip_grad_norm(grads, max_norm, out=out), out, kept, max_norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, kept))
    norm = tf.clip_grad_norm(grads, max_norm)
    check(norm, grads, kept, max_norm)
    assert all(torch.equal(a, b) for a, b in zip(grads, out))


def test_rows_that_start_anywhere_and_empty_tensors():
    for dt in TYPES.values():
        for shift in range(1, 8):
            base = randn((9000,), dt, shift)
            g = [base[shift:shift + 4500 + shift], base[:0], base[5001:8999].reshape(2, 1999)]
            out = [torch.full((5000,), 7.0, dtype=dt, device="cuda"), torch.empty(0, dtype=dt, device="cuda"), torch.empty(2, 1999, dtype=dt, device="cuda")]
            view = out[0][1:1 + 4500 + shift]
            check(tf.clip_grad_norm(g, 2.0, out=[view] + out[1:]), [view, out[2]], [g[0], g[2]], 2.0)
            assert out[0][0] == 7 and (out[0][1 + 4500 + shift:] == 7).all()


def test_values_that_are_not_finite_and_ends_of_the_range():
    g = [torch.ones(5000, device="cuda"), torch.ones(10, dtype=torch.bfloat16, device="cuda")]
    g[0][4321] = float("nan")
    out = [torch.empty_like(t) for t in g]
    assert torch.isnan(tf.clip_grad_norm(g, 1.0, out=out)) and all(torch.isnan(t).all() for t in out)
    g[0][4321] = float("inf")
    assert tf.clip_grad_norm(g, 1.0, out=out) == float("inf")
    assert torch.isnan(out[0][4321]) and (out[0][:4321] == 0).all() and (out[1] == 0).all()
    big = [torch.full((100,), 1e30, device="cuda")]
    check(tf.clip_grad_norm(big, 3.0, out=[out_big := torch.empty_like(big[0])]), [out_big], big, 3.0)
    zero = [torch.zeros(100, device="cuda")]
    assert tf.clip_grad_norm(zero, 1.0) == 0 and (zero[0] == 0).all()
    some = [torch.ones(100, device="cuda")]
    tf.clip_grad_norm(some, 0.0)
    assert (some[0] == 0).all()
    assert tf.clip_grad_norm([], 1.0) == 0


def test_results_repeat_and_follow_their_stream():
    grads = tensors(20, 300001)
    out = [torch.empty_like(g) for g in grads]
    norm = tf.clip_grad_norm(grads, 0.5, out=out)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        copies = [g * 1 for g in grads]
        again = tf.clip_grad_norm(copies, 0.5)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(norm, again) and all(torch.equal(a, b) for a, b in zip(out, copies))


def test_refusals():
    g = [torch.ones(5, device="cuda")]
    with pytest.raises(TypeError, match="float64"):
        tf.clip_grad_norm([g[0].double()], 1.0)
    with pytest.raises(ValueError, match="contiguous"):
        tf.clip_grad_norm([torch.ones(4, 4, device="cuda").t()[1:]], 1.0)
    with pytest.raises(ValueError, match="out has"):
        tf.clip_grad_norm(g, 1.0, out=[])
    with pytest.raises(ValueError, match=r"out\[0\] has shape"):
        tf.clip_grad_norm(g, 1.0, out=[torch.ones(6, device="cuda")])
    with pytest.raises(tf.TurboFNOError, match="max_norm"):
        tf.clip_grad_norm(g, -1.0)
