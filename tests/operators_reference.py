"""Plain 64-bit forms of the operators around the spectral layer, on the CPU, and bounds of their error."""
import math

import torch

EPS32 = 2.0 ** -24                      # one rounding to 32 bits
EPS16 = 2.0 ** -8                       # one rounding to bf16, which holds 8 significant bits
TYPES = {"c64": torch.complex64, "f32": torch.float32, "bf16": torch.bfloat16}


def wide(t):
    return t.detach().cpu().to(torch.complex128 if t.is_complex() else torch.float64)


def rounding(dtype):
    return EPS16 if dtype == torch.bfloat16 else EPS32


def randn(shape, dtype, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    t = torch.randn(shape, dtype=torch.float32 if dtype == torch.bfloat16 else dtype, generator=gen) * scale
    return t.to(dtype).cuda()


def by_parts(f, *ts):
    if not ts[0].is_complex():
        return f(*ts)
    return torch.complex(f(*[t.real for t in ts]), f(*[t.imag for t in ts]))


def act(name, z):
    def f(v):
        if name == "none":
            return v
        if name == "relu":
            return torch.where(v <= 0, torch.zeros_like(v), v)
        if name == "silu":
            return v / (1 + torch.exp(-v))
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    return by_parts(f, z)


def slope(name, z):
    def f(v):
        if name == "none":
            return torch.ones_like(v)
        if name == "relu":
            return (v > 0).to(v.dtype)
        if name == "silu":
            s = 1 / (1 + torch.exp(-v))
            return s + v * s * (1 - s)
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (v + 0.044715 * v ** 3))
        return 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * c * (1 + 3 * 0.044715 * v * v)
    return by_parts(f, z)


def largest_part(t):
    """elementwise: the larger magnitude of the parts' errors is at most that of the complex number"""
    return t.abs()


def within(got, exact, bound, what=""):
    """|got - exact| <= bound for every element"""
    got = wide(got)
    off = (got - exact).abs()
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert got.shape == exact.shape and worst <= 0, "%s: %g over its bound (largest error %g)" % (what, worst, off.max().item())


def product_bound(A, B, terms, inputs=0.0):
    """error of a product A B summed over `terms` real values in 32 bits, its operands off by `inputs` of themselves: every rounding of a sum, and
    of a product, is at most EPS32 of the sum of magnitudes"""
    return ((terms + 4) * EPS32 + inputs) * (A.abs() @ B.abs())
