"""The Fourier block of examples/fourier_block.py: its gradients against the derivatives of a 64-bit evaluation, its steps, its 8-bit form, and the whole
of it in a HIP graph."""
import importlib.util
import os

import pytest
import torch

from operators_reference import act, wide

pytestmark = pytest.mark.gpu

_path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "fourier_block.py")
_spec = importlib.util.spec_from_file_location("fourier_block", _path)
fourier_block = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(fourier_block)

CHANNELS, HIDDEN, SIGNALS, SAMPLES = 64, 96, 3, 128


def fields(seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(CHANNELS, SIGNALS, SAMPLES, dtype=torch.complex64, generator=g).cuda()


def plain(p, x):
    def norm(v, gain):
        return gain[:, None, None] * v / torch.sqrt(v.abs().square().mean(0) + 1e-6)

    def product(W, v):
        return (W @ v.flatten(1)).unflatten(1, v.shape[1:])
    h = norm(x, p["gain1"])
    kept = product(p["R"], torch.fft.fft(h)[..., :64])
    u = torch.fft.ifft(torch.nn.functional.pad(kept, (0, SAMPLES - 64)))
    t = act("gelu_tanh", u + product(p["W"], h) + p["b"][:, None, None]) + x
    v = act("gelu_tanh", product(p["W1"], norm(t, p["gain2"])) + p["b1"][:, None, None])
    return t + product(p["W2"], v) + p["b2"][:, None, None]


def off(a, b):
    return ((wide(a) - b).norm() / b.norm()).item()


def test_gradients():
    block = fourier_block.FourierBlock(CHANNELS, HIDDEN)
    x, gy = fields(1), fields(2)
    y, saved = block.forward(x)
    gx, g = block.backward(gy, saved)
    p = {name: wide(v).requires_grad_() for name, v in block.parameters.items()}
    x64 = wide(x).requires_grad_()
    y64 = plain(p, x64)
    y64.backward(wide(gy))
    # a dozen products, transforms and norms after one another, each off by less than 10^-6 of its result
    assert off(y, y64.detach()) < 2e-5
    assert off(gx, x64.grad) < 2e-5
    for name in p:
        assert off(g[name], p[name].grad) < 2e-5, name


def loss_of(block, x, target):
    y = block.forward(x)[0]
    return 0.5 * ((wide(y) - wide(target)).abs().square().sum() / y.numel()).item()


def test_steps():
    block = fourier_block.FourierBlock(CHANNELS, HIDDEN)
    x = fields(3)
    target = fourier_block.FourierBlock(CHANNELS, HIDDEN, seed=2).forward(x)[0]
    before = {name: v.clone() for name, v in block.parameters.items()}
    start = loss_of(block, x, target)
    loss, norm = block.train_step(x, target, rate=0.0, max_norm=1e9)
    assert abs(loss.item() - start) < 1e-5 * start
    # along the gradient the loss changes at the rate of its squared norm: steps of a thousandth of the loss, forward and back; losses are off by some 10^-6
    # of themselves, their difference by 10^-3 of itself, and its third order by a like part
    rate, ends = 1e-3 * start / norm.item() ** 2, []
    for sign in (1, -1):
        for name, v in block.parameters.items():
            v.copy_(before[name])
        block.train_step(x, target, rate=sign * rate, max_norm=1e9)
        ends.append(loss_of(block, x, target))
    assert abs((ends[1] - ends[0]) / (2e-3 * start) - 1) < 0.01, (start, ends)
    # clipped to a tenth of their norm, the gradients go a tenth as far
    moved = {}
    for part in (1.0, 0.1):
        for name, v in block.parameters.items():
            v.copy_(before[name])
        block.train_step(x, target, rate=1.0, max_norm=part * norm.item())
        moved[part] = {name: wide(v) - wide(before[name]) for name, v in block.parameters.items()}
    # differences of parameters of size 1, each rounded to 2^-24 of it
    for name in before:
        bound = 2 * 2.0 ** -24 * (wide(before[name]).abs().max() + moved[1.0][name].abs().max()) + 1e-5 * moved[1.0][name].abs().max()
        assert ((moved[0.1][name] - 0.1 * moved[1.0][name]).abs() <= bound).all(), name


def test_8_bits():
    block, x = fourier_block.FourierBlock(CHANNELS, HIDDEN), fields(3)
    block.quantise()
    # e4m3 keeps four significant bits: operands off by at most 2^-4 each, at random, so their product by less than 2^-4 of itself, and it is one of three terms
    assert off(block.serve(x), wide(block.forward(x)[0])) < 2.0 ** -4


def test_in_a_graph():
    block = fourier_block.FourierBlock(CHANNELS, HIDDEN)
    import turbofno_amd as tf

    def step(x, gy):
        y, saved = block.forward(x)
        gx, g = block.backward(gy, saved)
        grads = list(g.values())
        norm = tf.clip_grad_norm(grads, 0.5)
        return [y, gx, norm, block.serve(x)] + grads
    block.quantise()
    inputs = [(fields(10 + i), fields(20 + i)) for i in range(3)]
    x, gy = inputs[0][0].clone(), inputs[0][1].clone()
    step(x, gy)                             # first launches outside the capture (kernel attributes)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = step(x, gy)
    for i in (1, 2, 0, 1):
        x.copy_(inputs[i][0])
        gy.copy_(inputs[i][1])
        expect = step(*inputs[i])
        torch.cuda.synchronize()
        for t in results:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(results, expect):
            assert torch.equal(got, want), i
