"""Cases of the operators around the spectral layer: channel product with epilogue, root-mean-square norm, gradient clipping.

A case names an operator (`op`) and its form:

  mix   forward   z = W x + bias + residual, y = activation(z); x[K][positions] -> y[N][positions]
        backward  gradients of x, W, bias and residual from that of y and the saved z
        8bit      forward with x and W in e4m3, a scale per position and a scale per output channel
  norm  forward   s = x + residual, y = s / sqrt(mean over channels of |s|^2 + eps) * gain
        8bit      the same with y in e4m3 and a scale per position
        backward  gradients of s and gain
  clip  forward   norm over all values of a list of gradients, and the gradients scaled to at most that norm

Where `own` is false, `run` computes them in elementary operations of torch, in 32 bits; where it is true, through `turbofno_amd`.
Fields are channel-outermost, as everywhere in the framework. `type` is c64, f32 or bf16; activations act on real and imaginary parts.
"""
import math

import torch

own = False

_TYPES = {"c64": torch.complex64, "f32": torch.float32, "bf16": torch.bfloat16}
_E4M3_MAX = 448.0
_EPS = 1e-6
_FIELDS = 16 * 256 * 256                # positions of the training batch of bench.py: 16 fields of 256 x 256


def listed():
    return [
        # one signal of 128 samples through a narrow block: the latency of a call
        dict(name="mix_single", op="mix", form="forward", type="c64", K=8, N=64, P=128, act="gelu_tanh", residual=True, save=False),
        # the pointwise half of a block in training, at the sizes of bench.py: residual = the spectral layer's output, z saved
        dict(name="mix_fields", op="mix", form="forward", type="c64", K=64, N=64, P=_FIELDS, act="gelu_tanh", residual=True, save=True),
        # a widening product on real fields in 16 bits, channels and positions that fit no tile, no residual
        dict(name="mix_ragged_bf16", op="mix", form="forward", type="bf16", K=72, N=200, P=100003, act="silu", residual=False, save=False),
        # the backward pass of mix_fields
        dict(name="mix_backward_fields", op="mix", form="backward", type="c64", K=64, N=64, P=_FIELDS, act="gelu_tanh", residual=True, save=True),
        # a backward pass of odd sizes on real fields
        dict(name="mix_backward_ragged", op="mix", form="backward", type="f32", K=40, N=100, P=50021, act="silu", residual=False, save=True),
        # serving in 8 bits: four fields of 256 x 256, 256 channels, the residual stream in 16 bits
        dict(name="mix_8bit", op="mix", form="8bit", type="bf16", K=256, N=256, P=4 * 65536, act="none", residual=True, save=False),
        # the norm of a residual stream in training
        dict(name="norm_fields", op="norm", form="forward", type="c64", K=64, P=_FIELDS, residual=True),
        # what mix_8bit reads
        dict(name="norm_8bit", op="norm", form="8bit", type="bf16", K=256, P=4 * 65536, residual=True),
        # the backward pass of norm_fields
        dict(name="norm_backward_fields", op="norm", form="backward", type="c64", K=64, P=_FIELDS, residual=True),
        # a short batch of odd sizes, no gradient into the residual stream
        dict(name="norm_backward_ragged", op="norm", form="backward", type="bf16", K=100, P=6001, residual=False),
        # the gradients of a few narrow blocks: many small tensors of three types
        dict(name="clip_many_small", op="clip", form="forward", count=60, values=250_000, mixed=True),
        # the gradients of a large model, most of them in a few tensors
        dict(name="clip_large", op="clip", form="forward", count=24, values=100_000_000, mixed=False),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """One more case: any sizes in the range (over their logarithm), any type, form and activation."""
    most = max(work(c)["bytes"] for c in listed())
    most_flops = max(work(c)["flops"] for c in listed())
    while True:
        op = rng.choice(["mix", "mix", "mix", "norm", "norm", "clip"])
        if op == "clip":
            case = dict(op=op, form="forward", count=rng.randint(1, 60), values=_log_uniform(rng, 2_000, 100_000_000), mixed=rng.random() < 0.5)
        else:
            case = dict(op=op, form=rng.choice(["forward", "backward", "8bit"]), type=rng.choice(["c64", "f32", "bf16"]))
            wide = 128 if case["type"] == "c64" else 256
            case.update(K=_log_uniform(rng, 4, wide), P=_log_uniform(rng, 64, _FIELDS))
            if op == "mix":
                case.update(N=_log_uniform(rng, 4, wide), act=rng.choice(["none", "relu", "silu", "gelu_tanh"]))
                case.update(residual=rng.random() < 0.6, save=case["form"] == "backward" or (case["form"] == "forward" and rng.random() < 0.5))
            else:
                case.update(residual=rng.random() < 0.6)
        w = work(case)
        if w["bytes"] <= most and w["flops"] <= most_flops:
            return case


# ---- inputs ----

def _normal(gen, shape, dtype, scale=1.0):
    real = torch.float32 if dtype == torch.bfloat16 else dtype
    return (torch.randn(shape, dtype=real, device="cuda", generator=gen) * scale).to(dtype)


def _quantized(v, dim):
    """v in e4m3 and its scales: the largest magnitude along `dim` (a dimension or several) becomes 448"""
    scale = v.abs().amax(dim=dim, keepdim=True).clamp_min(1e-30) / _E4M3_MAX
    return (v / scale).to(torch.float8_e4m3fn), scale


def _clip_sizes(case):
    """Sizes of the tensors: the i-th holds a share of 1 / (i + 1), at least one value each. complex64 where i % 3 == 0 of a mixed list,
    float32 where it is 1, bfloat16 where it is 2; a list that is not mixed is float32."""
    share = sum(1.0 / (i + 1) for i in range(case["count"]))
    sizes = [max(1, int(case["values"] / share / (i + 1))) for i in range(case["count"])]
    types = [("c64", "f32", "bf16")[i % 3] if case["mixed"] else "f32" for i in range(case["count"])]
    return sizes, types


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = dict(case=case)
    if case["op"] == "clip":
        sizes, types = _clip_sizes(case)
        st["grads"] = [_normal(gen, (n,), _TYPES[t], 0.01) for n, t in zip(sizes, types)]
        st["out"] = [torch.empty_like(g) for g in st["grads"]]
        st["max_norm"] = 1.0
        return st
    dt, K, P = _TYPES[case["type"]], case["K"], case["P"]
    form, part = case["form"], (2,) if dt.is_complex else ()
    real = torch.float32
    new = lambda *shape, dtype=dt: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    if case["op"] == "norm":
        st["gain"] = 1.0 + 0.1 * torch.randn(K, dtype=real, device="cuda", generator=gen)
        if form == "backward":
            st["gy"], st["s"] = _normal(gen, (K, P), dt), _normal(gen, (K, P), dt)
            s = st["s"] if dt.is_complex else st["s"].to(real)
            st["rstd"] = torch.rsqrt((s.abs() ** 2).mean(dim=0) + _EPS)
            st["gs"] = _normal(gen, (K, P), dt) if case["residual"] else None
            st["gx"], st["ggain"] = new(K, P), new(K, dtype=real)
            return st
        st["x"] = _normal(gen, (K, P), dt)
        st["residual"] = _normal(gen, (K, P), dt) if case["residual"] else None
        st["s"] = new(K, P) if case["residual"] else None
        if form == "8bit":
            st["q"], st["scale"] = new(K, P, *part, dtype=torch.float8_e4m3fn), new(P, dtype=real)
        else:
            st["y"], st["rstd"] = new(K, P), new(P, dtype=real)
        return st
    N = case["N"]
    st["bias"] = _normal(gen, (N,), dt, 0.1)
    if form == "8bit":
        st["xq"], xs = _quantized(torch.randn((K, P) + part, device="cuda", generator=gen), (0, 2) if part else 0)
        st["Wq"], ws = _quantized(torch.randn((N, K) + part, device="cuda", generator=gen) / math.sqrt(K), (1, 2) if part else 1)
        st["xscale"], st["wscale"] = xs.reshape(P).contiguous(), ws.reshape(N).contiguous()
        st["residual"], st["y"] = _normal(gen, (N, P), dt) if case["residual"] else None, new(N, P)
        return st
    st["x"], st["W"] = _normal(gen, (K, P), dt), _normal(gen, (N, K), dt, 1.0 / math.sqrt(K))
    if form == "forward":
        st["residual"] = _normal(gen, (N, P), dt) if case["residual"] else None
        st["y"], st["z"] = new(N, P), new(N, P) if case["save"] else None
        return st
    st["gy"], st["z"] = _normal(gen, (N, P), dt), _normal(gen, (N, P), dt)
    st["gx"], st["gW"], st["gbias"], st["gz"] = new(K, P), new(N, K), new(N), new(N, P)
    return st


# ---- plain forms: 32 bits, rounded once at the end ----

def _wide(t):
    return t if t.is_complex() else t.to(torch.float32)


def _by_parts(f, *tensors):
    """f on real tensors; on complex ones, on real and imaginary parts"""
    if not tensors[0].is_complex():
        return f(*tensors)
    return torch.view_as_complex(f(*[torch.view_as_real(t.resolve_conj()) for t in tensors]))


def _sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


_G0, _G1 = 2.0 * math.sqrt(2.0 / math.pi), 0.044715     # gelu_tanh(z) = z sigmoid(_G0 (z + _G1 z^3))


def _activate(act, z):
    if act == "none":
        return z
    if act == "relu":
        return _by_parts(lambda v: torch.where(v > 0, v, torch.zeros_like(v)), z)
    if act == "silu":
        return _by_parts(lambda v: v * _sigmoid(v), z)
    return _by_parts(lambda v: v * _sigmoid(_G0 * (v + _G1 * v * v * v)), z)


def _slope(act, z):
    """the activation's derivative at real z"""
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = _sigmoid(z)
        return s + z * s * (1.0 - s)
    s = _sigmoid(_G0 * (z + _G1 * z * z * z))
    return s + z * s * (1.0 - s) * (_G0 * (1.0 + 3.0 * _G1 * z * z))


_BLOCK = 4096                           # positions whose products are summed at once: one sum over a million loses three digits


def _over_positions(g, x):
    """g x^H, the sum over positions in blocks"""
    whole = x.shape[1] // _BLOCK * _BLOCK
    out = g[:, whole:] @ x[:, whole:].mH
    if whole:
        a = g[:, :whole].reshape(g.shape[0], -1, _BLOCK).permute(1, 0, 2).contiguous()
        b = x[:, :whole].reshape(x.shape[0], -1, _BLOCK).permute(1, 2, 0).conj().resolve_conj().contiguous()
        out = out + (a @ b).sum(dim=0)
    return out


def _plain_mix(st, case):
    dt = _TYPES[case["type"]]
    if case["form"] == "backward":
        gy, x, W, z = _wide(st["gy"]), _wide(st["x"]), _wide(st["W"]), _wide(st["z"])
        gz = gy if case["act"] == "none" else _by_parts(lambda g, v: g * _slope(case["act"], v), gy, z)
        gx, gW, gbias = W.mH @ gz, _over_positions(gz, x), gz.sum(dim=1)
        return dict(gx=gx.to(dt), gW=gW.to(dt), gbias=gbias.to(dt), gz=gz.to(dt))
    if case["form"] == "8bit":
        x, W = st["xq"].to(torch.float32), st["Wq"].to(torch.float32)
        if dt.is_complex:
            x, W = torch.view_as_complex(x), torch.view_as_complex(W)
        z = (W * st["wscale"][:, None]) @ (x * st["xscale"])
    else:
        z = _wide(st["W"]) @ _wide(st["x"])
    z = z + _wide(st["bias"])[:, None]
    if st["residual"] is not None:
        z = z + _wide(st["residual"])
    y = _activate(case["act"], z).to(dt)
    return dict(y=y, z=z.to(dt)) if case["save"] else dict(y=y)


def _square(t):
    return t.real ** 2 + t.imag ** 2 if t.is_complex() else t * t


def _plain_norm(st, case):
    dt, gain = _TYPES[case["type"]], st["gain"][:, None]
    if case["form"] == "backward":
        gy, s, rstd = _wide(st["gy"]), _wide(st["s"]), st["rstd"]
        along = (gy * s.conj()).real if dt.is_complex else gy * s
        gx = rstd * (gain * gy) - s * (rstd ** 3 * (gain * along).mean(dim=0))
        if st["gs"] is not None:
            gx = gx + _wide(st["gs"])
        return dict(gx=gx.to(dt), ggain=(along * rstd).sum(dim=1))
    s = _wide(st["x"])
    if st["residual"] is not None:
        s = s + _wide(st["residual"])
    rstd = torch.rsqrt(_square(s).mean(dim=0) + _EPS)
    y = s * rstd * gain
    out = dict(s=s.to(dt)) if st["residual"] is not None else {}
    if case["form"] == "forward":
        return dict(out, y=y.to(dt), rstd=rstd)
    parts = torch.view_as_real(y) if dt.is_complex else y[..., None]
    amax = parts.abs().amax(dim=(0, 2))
    scale = torch.where(amax > 0, amax / _E4M3_MAX, torch.ones_like(amax))
    q = (parts / scale[:, None]).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)
    return dict(out, q=q if dt.is_complex else q[..., 0], scale=scale)


def _plain_clip(st, case):
    norm = torch.sqrt(torch.stack([_square(_wide(g)).sum() for g in st["grads"]]).sum())
    factor = torch.clamp(st["max_norm"] / (norm + 1e-6), max=1.0)
    return dict(norm=norm, grads=[(_wide(g) * factor).to(g.dtype) for g in st["grads"]])


# ---- the framework's operators ----

def _own_mix(st, case):
    import turbofno_amd as tf
    if case["form"] == "forward":
        y = tf.mix(st["x"], st["W"], bias=st["bias"], residual=st["residual"], activation=case["act"], y=st["y"], z=st["z"])
        return dict(y=y, z=st["z"]) if case["save"] else dict(y=y)
    if case["form"] == "8bit":
        return dict(y=tf.mix_8bit(st["xq"], st["xscale"], st["Wq"], st["wscale"], bias=st["bias"], residual=st["residual"],
                                  activation=case["act"], y=st["y"]))
    gx, gW, gbias, gz = tf.mix_backward(st["gy"], st["x"], st["W"], z=st["z"], activation=case["act"], gz=st["gz"], gx=st["gx"],
                                        gW=st["gW"], gbias=st["gbias"])
    return dict(gx=gx, gW=gW, gbias=gbias, gz=gz)


def _own_norm(st, case):
    import turbofno_amd as tf
    if case["form"] == "backward":
        gx, ggain = tf.rms_norm_backward(st["gy"], st["s"], st["gain"], st["rstd"], gs=st["gs"], gx=st["gx"], ggain=st["ggain"])
        return dict(gx=gx, ggain=ggain)
    out = dict(s=st["s"]) if st["residual"] is not None else {}
    if case["form"] == "forward":
        tf.rms_norm(st["x"], st["gain"], residual=st["residual"], eps=_EPS, y=st["y"], s=st["s"], rstd=st["rstd"])
        return dict(out, y=st["y"], rstd=st["rstd"])
    tf.rms_norm_8bit(st["x"], st["gain"], residual=st["residual"], eps=_EPS, q=st["q"], scale=st["scale"], s=st["s"])
    return dict(out, q=st["q"], scale=st["scale"])


def _own_clip(st, case):
    import turbofno_amd as tf
    norm = tf.clip_grad_norm(st["grads"], st["max_norm"], out=st["out"])
    return dict(norm=norm, grads=st["out"])


def run(state):
    case = state["case"]
    forms = {"mix": _own_mix, "norm": _own_norm, "clip": _own_clip} if own else {"mix": _plain_mix, "norm": _plain_norm, "clip": _plain_clip}
    return forms[case["op"]](state, case)


# ---- from the definitions, in 64 bits, on real and imaginary parts ----

def _parts64(t):
    """(real, imaginary) in 64 bits; the imaginary part of a real tensor is None"""
    return (t.real.to(torch.float64), t.imag.to(torch.float64)) if t.is_complex() else (t.to(torch.float64), None)


def _joined(re, im):
    return re if im is None else torch.complex(re, im)


def _product64(a, b, conj_a=False, conj_b=False):
    """a b of two pairs of parts; with a flag, of the conjugate of that operand"""
    (ar, ai), (br, bi) = a, b
    if ai is None:
        return torch.matmul(ar, br), None
    sa, sb = -1.0 if conj_a else 1.0, -1.0 if conj_b else 1.0
    return torch.matmul(ar, br) - sa * sb * torch.matmul(ai, bi), sb * torch.matmul(ar, bi) + sa * torch.matmul(ai, br)


def _transposed(p):
    return p[0].t(), None if p[1] is None else p[1].t()


def _act64(act, v):
    if v is None or act == "none":
        return v
    if act == "relu":
        return torch.clamp(v, min=0.0)
    if act == "silu":
        return 0.5 * v * (1.0 + torch.tanh(0.5 * v))
    return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v.pow(3))))


def _slope64(act, v):
    if act == "none":
        return torch.ones_like(v)
    if act == "relu":
        return torch.heaviside(v, torch.zeros_like(v))
    if act == "silu":
        t = torch.tanh(0.5 * v)
        return 0.5 * (1.0 + t) + 0.25 * v * (1.0 - t * t)
    c = math.sqrt(2.0 / math.pi)
    t = torch.tanh(c * (v + 0.044715 * v.pow(3)))
    return 0.5 * (1.0 + t) + 0.5 * v * (1.0 - t * t) * c * (1.0 + 0.134145 * v.pow(2))


def _plus(p, q):
    return tuple(None if u is None else u + v for u, v in zip(p, q))


def _exact_mix(st, case):
    act = case["act"]
    if case["form"] == "backward":
        gy, z = _parts64(st["gy"]), _parts64(st["z"])
        gz = tuple(None if g is None else g * _slope64(act, v) for g, v in zip(gy, z))
        gx = _product64(_transposed(_parts64(st["W"])), gz, conj_a=True)
        gW = _product64(gz, _transposed(_parts64(st["x"])), conj_b=True)
        return dict(gx=_joined(*gx), gW=_joined(*gW), gbias=_joined(*(None if g is None else g.sum(dim=1) for g in gz)), gz=_joined(*gz))
    if case["form"] == "8bit":
        x, W = st["xq"].to(torch.float64), st["Wq"].to(torch.float64)
        pair = lambda t: (t[..., 0], t[..., 1]) if case["type"] == "c64" else (t, None)  # noqa: E731
        both = st["wscale"].to(torch.float64)[:, None] * st["xscale"].to(torch.float64)
        z = tuple(None if v is None else v * both for v in _product64(pair(W), pair(x)))
    else:
        z = _product64(_parts64(st["W"]), _parts64(st["x"]))
    z = _plus(z, tuple(None if v is None else v[:, None] for v in _parts64(st["bias"])))
    if st["residual"] is not None:
        z = _plus(z, _parts64(st["residual"]))
    y = _joined(*(_act64(act, v) for v in z))
    return dict(y=y, z=_joined(*z)) if case["save"] else dict(y=y)


def _exact_norm(st, case):
    gain = st["gain"].to(torch.float64).reshape(-1, 1)
    some = lambda p: [v for v in p if v is not None]  # noqa: E731
    if case["form"] == "backward":
        gy, s, rstd = _parts64(st["gy"]), _parts64(st["s"]), st["rstd"].to(torch.float64)
        dot = sum(g * v for g, v in zip(some(gy), some(s)))
        shrink = rstd.pow(3) * (gain * dot).sum(dim=0) / case["K"]
        gx = tuple(None if g is None else gain * g * rstd - v * shrink for g, v in zip(gy, s))
        if st["gs"] is not None:
            gx = _plus(gx, _parts64(st["gs"]))
        return dict(gx=_joined(*gx), ggain=torch.matmul(dot, rstd))
    s = _parts64(st["x"])
    if st["residual"] is not None:
        s = _plus(s, _parts64(st["residual"]))
    rstd = 1.0 / torch.sqrt(sum(v.pow(2).sum(dim=0) for v in some(s)) / case["K"] + _EPS)
    y = tuple(None if v is None else v * rstd * gain for v in s)
    out = dict(s=_joined(*s)) if st["residual"] is not None else {}
    if case["form"] == "forward":
        return dict(out, y=_joined(*y), rstd=rstd)
    scale = torch.stack([v.abs().amax(dim=0) for v in some(y)]).amax(dim=0) / _E4M3_MAX
    q = torch.stack([v / scale for v in some(y)], dim=-1)           # before its rounding to 8 bits
    return dict(out, q=q if case["type"] == "c64" else q[..., 0], scale=scale)


def _exact_clip(st, case):
    parts = [[v for v in _parts64(g) if v is not None] for g in st["grads"]]
    norm = math.sqrt(sum(float(torch.dot(v, v)) for p in parts for v in p))
    factor = min(1.0, st["max_norm"] / (norm + 1e-6))
    return dict(norm=norm, grads=[_joined(*(factor * v for v in p), *([None] if len(p) == 1 else [])) for p in parts])


def exact(case, seed):
    forms = {"mix": _exact_mix, "norm": _exact_norm, "clip": _exact_clip}
    return forms[case["op"]](prepare(case, seed), case)


# ---- what a pass cannot do without ----

def work(case):
    if case["op"] == "clip":
        sizes, types = _clip_sizes(case)
        size = sum(n * _TYPES[t].itemsize for n, t in zip(sizes, types))
        values = sum(n * (2 if t == "c64" else 1) for n, t in zip(sizes, types))
        return dict(bytes=2 * size + 4, flops=3.0 * values)
    e, K, P, parts = _TYPES[case["type"]].itemsize, case["K"], case["P"], 2 if case["type"] == "c64" else 1
    if case["op"] == "norm":
        more = 1 if case["residual"] else 0
        if case["form"] == "backward":
            return dict(bytes=e * K * P * (3 + more) + 4 * (P + 2 * K), flops=(8.0 + more) * parts * K * P)
        y = parts if case["form"] == "8bit" else e
        return dict(bytes=K * P * (e * (1 + 2 * more) + y) + 4 * (P + K), flops=(4.0 + more) * parts * K * P)
    N = case["N"]
    product = (8.0 if parts == 2 else 2.0) * N * K * P
    if case["form"] == "backward":
        known = 0 if case["act"] == "none" else 1                   # z is read, gz differs from gy
        return dict(bytes=e * P * (2 * K + N * (1 + 2 * known)) + e * (2 * N * K + N), flops=2.0 * product)
    outs = N * (1 + (1 if case["residual"] else 0) + (1 if case["save"] else 0))
    if case["form"] == "8bit":
        return dict(bytes=parts * K * (P + N) + 4 * (P + N) + e * (P * outs + N), flops=product)
    return dict(bytes=e * P * (K + outs) + e * (N * K + N), flops=product)
