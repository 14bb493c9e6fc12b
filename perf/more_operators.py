"""Cases of the further operators around the spectral layer: layer norm, dropout, and products in 8 bits with a scale for each block of 128 channels.

A case names an operator (`op`) and its form:

  norm     forward   s = residual + dropout(x), m = mean over channels of s, y = gain (s - m) / sqrt(mean over channels of |s - m|^2 + eps) + bias
           backward  gradients of x, residual, gain and bias from that of y and from gs, what reaches s by the residual stream
           8bit      forward without dropout, y in e4m3 with a scale per position and block of 128 channels
  dropout  plain     y = residual + dropout(x)
  quantise plain     x in e4m3 with a scale per position and block of 128 channels
  product  blocks    y = activation(W x + bias + residual), x as quantise gives it, W in e4m3 with a scale per block of 128 x 128

dropout(x) = x / (1 - drop) where a word of a counter-based generator is at least drop 2^32, and 0 elsewhere. The generator is Philox 4x32 with ten
rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; 2011): key = seed, counter = (low word of q, channel + 2^16 high word of
q, offset), q = position / 4, and word position % 4 of the four that it gives.

Where `own` is false, `run` computes them in elementary operations of torch, in 32 bits; where it is true, through `turbofno_amd`.
Fields are channel-outermost, as everywhere in the framework. `type` is c64, f32 or bf16; a complex element is kept or dropped as a whole.
"""
import math

import torch

own = False

_TYPES = {"c64": torch.complex64, "f32": torch.float32, "bf16": torch.bfloat16}
_E4M3_MAX = 448.0
_EPS = 1e-6
_BLOCK = 128
_FIELDS = 16 * 256 * 256                # positions of the training batch of bench.py: 16 fields of 256 x 256


def listed():
    return [
        # the residual stream of a block in training, at the sizes of bench.py: dropout, addition and norm in one pass
        dict(name="norm_fields", op="norm", form="forward", type="c64", K=64, P=_FIELDS, residual=True, drop=0.1),
        # one signal of 128 samples: the latency of a call
        dict(name="norm_single", op="norm", form="forward", type="f32", K=64, P=128, residual=False, drop=0.0),
        # the backward pass of norm_fields
        dict(name="norm_backward_fields", op="norm", form="backward", type="c64", K=64, P=_FIELDS, residual=True, drop=0.1),
        # a short batch of odd sizes in 16 bits, without dropout, no gradient into the residual stream
        dict(name="norm_backward_ragged", op="norm", form="backward", type="bf16", K=200, P=30011, residual=False, drop=0.0),
        # serving: the norm that feeds a product in 8 bits, four blocks of channels
        dict(name="norm_8bit", op="norm", form="8bit", type="bf16", K=512, P=65536, residual=True, drop=0.0),
        # regularisation of a wide real field in 16 bits, added to the residual stream
        dict(name="dropout_fields_bf16", op="dropout", form="plain", type="bf16", K=256, P=4 * 65536, residual=True, drop=0.1),
        # a short batch of complex fields of odd sizes
        dict(name="dropout_ragged", op="dropout", form="plain", type="c64", K=100, P=50021, residual=False, drop=0.3),
        # the result of a wide activation, on its way into the second product
        dict(name="quantise_fields", op="quantise", form="plain", type="bf16", K=1024, P=65536),
        # channels that fill no block, positions that fill no tile
        dict(name="quantise_ragged", op="quantise", form="plain", type="f32", K=200, P=10007),
        # a wide product of a served batch: one field of 256 x 256
        dict(name="product_fields", op="product", form="blocks", type="bf16", K=1024, N=1024, P=65536, act="gelu_tanh", residual=False),
        # few positions through wide layers: the weights are what is read
        dict(name="product_few", op="product", form="blocks", type="bf16", K=2048, N=2048, P=16, act="none", residual=True),
        # complex fields with a complex64 result, channels and positions that fit nothing
        dict(name="product_ragged", op="product", form="blocks", type="c64", K=200, N=136, P=30011, act="silu", residual=True),
    ]


def _log_uniform(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    """One more case: any sizes in the range (over their logarithm), any type, form and activation."""
    most = max(work(c)["bytes"] for c in listed())
    most_flops = max(work(c)["flops"] for c in listed())
    while True:
        op = rng.choice(["norm", "norm", "dropout", "quantise", "product", "product"])
        kind = rng.choice(["c64", "f32", "bf16"])
        wide = 512 if kind == "c64" else 2048
        case = dict(op=op, type=kind, K=_log_uniform(rng, 4, wide), P=_log_uniform(rng, 1, _FIELDS))
        if op == "product":
            case.update(form="blocks", N=_log_uniform(rng, 4, wide), act=rng.choice(["none", "relu", "silu", "gelu_tanh"]), residual=rng.random() < 0.6)
        else:
            case.update(form=rng.choice(["forward", "backward", "8bit"]) if op == "norm" else "plain")
            if op != "quantise":
                case.update(residual=rng.random() < 0.6)
                case.update(drop=0.0 if case["form"] == "8bit" or (op == "norm" and rng.random() < 0.4) else rng.choice([0.05, 0.1, 0.2, 0.5]))
        w = work(case)
        if 4096 <= w["bytes"] <= most and w["flops"] <= most_flops:
            return case


# ---- inputs ----

def _normal(gen, shape, dtype, scale=1.0):
    real = torch.float32 if dtype == torch.bfloat16 else dtype
    return (torch.randn(shape, dtype=real, device="cuda", generator=gen) * scale).to(dtype)


def _activations(gen, K, P, part):
    """values whose spread differs from channel to channel, as those of a trained network do"""
    spread = torch.exp(0.5 * torch.randn((K, 1) + (1,) * len(part), device="cuda", generator=gen))
    return torch.randn((K, P) + part, device="cuda", generator=gen) * spread


def _quantised_fields(v):
    """[K][P](2) in e4m3, and scales [K / 128][P]"""
    blocks = list(torch.split(v, _BLOCK, dim=0))
    scale = torch.stack([b.abs().amax(dim=0) if b.dim() == 2 else b.abs().amax(dim=(0, 2)) for b in blocks]).clamp_min(1e-30) / _E4M3_MAX
    per_channel = scale.repeat_interleave(_BLOCK, dim=0)[:v.shape[0]]
    return (v / (per_channel if v.dim() == 2 else per_channel[..., None])).to(torch.float8_e4m3fn), scale


def _quantised_weights(v):
    """[N][K](2) in e4m3, and scales [N / 128][K / 128]"""
    tiles = [[t.abs().amax() for t in torch.split(rows, _BLOCK, dim=1)] for rows in torch.split(v, _BLOCK, dim=0)]
    scale = torch.stack([torch.stack(t) for t in tiles]).clamp_min(1e-30) / _E4M3_MAX
    per_entry = scale.repeat_interleave(_BLOCK, dim=0)[:v.shape[0]].repeat_interleave(_BLOCK, dim=1)[:, :v.shape[1]]
    return (v / (per_entry if v.dim() == 2 else per_entry[..., None])).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = dict(case=case)
    dt, K, P = _TYPES[case["type"]], case["K"], case["P"]
    part = (2,) if dt.is_complex else ()
    wide = torch.complex64 if dt.is_complex else torch.float32
    new = lambda *shape, dtype=dt: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    blocks = -(-K // _BLOCK)
    if case["op"] == "product":
        N = case["N"]
        st["xq"], st["xscale"] = _quantised_fields(_activations(gen, K, P, part))
        st["Wq"], st["wscale"] = _quantised_weights(torch.randn((N, K) + part, device="cuda", generator=gen) / math.sqrt(K))
        st["bias"] = _normal(gen, (N,), dt, 0.1)
        st["residual"], st["y"] = _normal(gen, (N, P), dt) if case["residual"] else None, new(N, P)
        return st
    if case["op"] == "quantise":
        x = _activations(gen, K, P, part)
        st["x"] = torch.view_as_complex(x) if part else x.to(dt)
        st["q"], st["scale"] = new(K, P, *part, dtype=torch.float8_e4m3fn), new(blocks, P, dtype=torch.float32)
        return st
    if case["drop"]:
        st["rng"] = torch.tensor([0x243F6A8885A308D3 ^ seed, 1000 + seed % 17], dtype=torch.int64, device="cuda")      # seed and offset
    else:
        st["rng"] = None
    if case["op"] == "dropout":
        st["x"], st["residual"], st["y"] = _normal(gen, (K, P), dt), _normal(gen, (K, P), dt) if case["residual"] else None, new(K, P)
        return st
    st["gain"] = 1.0 + 0.1 * torch.randn(K, dtype=torch.float32, device="cuda", generator=gen)
    st["bias"] = 0.1 * torch.randn(K, dtype=wide, device="cuda", generator=gen)
    if case["form"] == "backward":
        s = torch.randn((K, P), dtype=wide, device="cuda", generator=gen) + 0.5
        st["s"], st["gy"] = s.to(dt), _normal(gen, (K, P), dt)
        s = st["s"].to(wide)
        st["mean"] = s.mean(dim=0)
        st["rstd"] = torch.rsqrt(((s - st["mean"]).abs() ** 2).mean(dim=0) + _EPS)
        st["gs"] = _normal(gen, (K, P), dt) if case["residual"] else None
        st["gx"], st["gr"] = new(K, P), new(K, P) if case["drop"] else None
        st["ggain"], st["gbias"] = new(K, dtype=torch.float32), new(K, dtype=wide)
        return st
    st["x"] = (torch.randn((K, P), dtype=wide, device="cuda", generator=gen) + 0.5).to(dt)
    st["residual"] = _normal(gen, (K, P), dt) if case["residual"] else None
    st["s"] = new(K, P) if case["residual"] or case["drop"] else None
    if case["form"] == "8bit":
        st["q"], st["scale"] = new(K, P, *part, dtype=torch.float8_e4m3fn), new(blocks, P, dtype=torch.float32)
    else:
        st["y"], st["mean"], st["rstd"] = new(K, P), new(P, dtype=wide), new(P, dtype=torch.float32)
    return st


# ---- plain forms: 32 bits, rounded once at the end ----

_LOW = 0xFFFFFFFF


def _keep(rng, K, P, drop):
    """[K][P], true where an element is kept. Products of two words fill 64 bits, which wrap around without losing any."""
    quad = torch.arange(-(-P // 4), dtype=torch.int64, device=rng.device)
    c0 = (quad & _LOW).expand(K, -1)
    c1 = torch.arange(K, dtype=torch.int64, device=rng.device)[:, None] + ((quad >> 32) << 16)
    c2, c3 = (rng[1] & _LOW).expand_as(c0), ((rng[1] >> 32) & _LOW).expand_as(c0)
    k0, k1 = rng[0] & _LOW, (rng[0] >> 32) & _LOW
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack([c0, c1, c2, c3], dim=-1).reshape(K, -1)[:, :P]
    return words >= round(drop * 2.0 ** 32)


def _wide(t):
    return t if t.is_complex() else t.to(torch.float32)


def _by_parts(f, t):
    """f on a real tensor; on a complex one, on real and imaginary parts"""
    return torch.view_as_complex(f(torch.view_as_real(t))) if t.is_complex() else f(t)


def _square(t):
    return t.real ** 2 + t.imag ** 2 if t.is_complex() else t * t


def _dropped(t, st, case):
    if not case["drop"]:
        return t
    keep = _keep(st["rng"], case["K"], case["P"], case["drop"])
    return torch.where(keep, t * (1.0 / (1.0 - case["drop"])), torch.zeros_like(t))


def _plain_dropout(st, case):
    y = _dropped(_wide(st["x"]), st, case)
    if st["residual"] is not None:
        y = y + _wide(st["residual"])
    return dict(y=y.to(_TYPES[case["type"]]))


def _blocks_of(parts):
    """[K][P](2) -> [blocks][128][P](2), zeros in channels that there are not"""
    blocks = -(-parts.shape[0] // _BLOCK)
    padded = torch.zeros((blocks * _BLOCK,) + parts.shape[1:], dtype=parts.dtype, device=parts.device)
    padded[:parts.shape[0]] = parts
    return padded.reshape((blocks, _BLOCK) + parts.shape[1:])


def _eight_bits(v):
    parts = torch.view_as_real(v) if v.is_complex() else v[..., None]
    amax = _blocks_of(parts).abs().amax(dim=(1, 3))
    scale = torch.where(amax > 0, amax / _E4M3_MAX, torch.ones_like(amax))
    per_channel = scale.repeat_interleave(_BLOCK, dim=0)[:v.shape[0], :, None]
    q = (parts / per_channel).clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)
    return dict(q=q if v.is_complex() else q[..., 0], scale=scale)


def _plain_quantise(st, case):
    return _eight_bits(_wide(st["x"]))


def _plain_norm(st, case):
    dt, gain = _TYPES[case["type"]], st["gain"][:, None]
    if case["form"] == "backward":
        gy, rstd = _wide(st["gy"]), st["rstd"]
        h = (_wide(st["s"]) - st["mean"]) * rstd
        g = gain * gy
        along = (gy * h.conj()).real if dt.is_complex else gy * h
        gr = rstd * (g - g.mean(dim=0) - h * (gain * along).mean(dim=0))
        if st["gs"] is not None:
            gr = gr + _wide(st["gs"])
        gx = _dropped(gr, st, case)
        out = dict(gr=gr.to(dt)) if case["drop"] else {}
        return dict(out, gx=gx.to(dt), ggain=along.sum(dim=1), gbias=gy.sum(dim=1))
    s = _dropped(_wide(st["x"]), st, case)
    if st["residual"] is not None:
        s = s + _wide(st["residual"])
    mean = s.mean(dim=0)
    rstd = torch.rsqrt(_square(s - mean).mean(dim=0) + _EPS)
    y = (s - mean) * rstd * gain + st["bias"][:, None]
    out = dict(s=s.to(dt)) if st["s"] is not None else {}
    if case["form"] == "8bit":
        return dict(out, **_eight_bits(y))
    return dict(out, y=y.to(dt), mean=mean, rstd=rstd)


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


def _plain_product(st, case):
    K, N = case["K"], case["N"]
    x, W = st["xq"].to(torch.float32), st["Wq"].to(torch.float32)
    xs = st["xscale"].repeat_interleave(_BLOCK, dim=0)[:K]
    ws = st["wscale"].repeat_interleave(_BLOCK, dim=0)[:N].repeat_interleave(_BLOCK, dim=1)[:, :K]
    if case["type"] == "c64":
        x, W = torch.view_as_complex(x * xs[..., None]), torch.view_as_complex(W * ws[..., None])
    else:
        x, W = x * xs, W * ws
    z = W @ x + _wide(st["bias"])[:, None]
    if st["residual"] is not None:
        z = z + _wide(st["residual"])
    return dict(y=_activate(case["act"], z).to(_TYPES[case["type"]]))


# ---- the framework's operators ----

def _own_dropout(st, case):
    import turbofno_amd as tf
    return dict(y=tf.dropout(st["x"], case["drop"], st["rng"], residual=st["residual"], y=st["y"]))


def _own_quantise(st, case):
    import turbofno_amd as tf
    q, scale = tf.quantise_8bit(st["x"], q=st["q"], scale=st["scale"])
    return dict(q=q, scale=scale)


def _own_norm(st, case):
    import turbofno_amd as tf
    if case["form"] == "backward":
        gx, gr, ggain, gbias = tf.layer_norm_backward(st["gy"], st["s"], st["gain"], st["mean"], st["rstd"], gs=st["gs"], drop=case["drop"], rng=st["rng"],
                                                      gx=st["gx"], gr=st["gr"], ggain=st["ggain"], gbias=st["gbias"])
        out = dict(gr=gr) if case["drop"] else {}
        return dict(out, gx=gx, ggain=ggain, gbias=gbias)
    out = dict(s=st["s"]) if st["s"] is not None else {}
    if case["form"] == "8bit":
        q, scale, _ = tf.layer_norm_8bit(st["x"], st["gain"], bias=st["bias"], residual=st["residual"], eps=_EPS, q=st["q"], scale=st["scale"], s=st["s"])
        return dict(out, q=q, scale=scale)
    y, _, mean, rstd = tf.layer_norm(st["x"], st["gain"], bias=st["bias"], residual=st["residual"], eps=_EPS, drop=case["drop"], rng=st["rng"], y=st["y"],
                                     s=st["s"], mean=st["mean"], rstd=st["rstd"])
    return dict(out, y=y, mean=mean, rstd=rstd)


def _own_product(st, case):
    import turbofno_amd as tf
    return dict(y=tf.mix_8bit_blocks(st["xq"], st["xscale"], st["Wq"], st["wscale"], bias=st["bias"], residual=st["residual"], activation=case["act"], y=st["y"]))


def run(state):
    case = state["case"]
    forms = ({"norm": _own_norm, "dropout": _own_dropout, "quantise": _own_quantise, "product": _own_product} if own else
             {"norm": _plain_norm, "dropout": _plain_dropout, "quantise": _plain_quantise, "product": _plain_product})
    return forms[case["op"]](state, case)


# ---- from the definitions, in 64 bits, on real and imaginary parts ----

def _words_times(a, m):
    """(high word, low word) of the product of the words `a` by the word `m`, by halves of 16 bits"""
    a1, a0, m1, m0 = a >> 16, a & 0xFFFF, m >> 16, m & 0xFFFF
    low = a0 * m0
    middle = a1 * m0 + (low >> 16)
    other = a0 * m1 + (middle & 0xFFFF)
    return a1 * m1 + (middle >> 16) + (other >> 16), ((other & 0xFFFF) << 16) | (low & 0xFFFF)


def _factors64(st, case):
    """what an element is multiplied with, channel by channel: 0 or 1 / (1 - drop)"""
    K, P, least = case["K"], case["P"], int(case["drop"] * 2 ** 32 + 0.5)
    seed, offset = (int(v) % 2 ** 64 for v in st["rng"].tolist())
    position = torch.arange(P, dtype=torch.int64, device="cuda")
    q = torch.arange(-(-P // 4), dtype=torch.int64, device="cuda")
    rows = []
    for k in range(K):
        counter = [q % 2 ** 32, k + 2 ** 16 * (q // 2 ** 32), torch.full_like(q, offset % 2 ** 32), torch.full_like(q, offset // 2 ** 32)]
        for r in range(10):
            key = [(seed + r * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32]
            (h0, l0), (h1, l1) = _words_times(counter[0], 0xD2511F53), _words_times(counter[2], 0xCD9E8D57)
            counter = [h1 ^ counter[1] ^ key[0], l1, h0 ^ counter[3] ^ key[1], l0]
        word = torch.stack(counter)[position % 4, position // 4]
        rows.append((word >= least).to(torch.float64) / (1.0 - case["drop"]))
    return torch.stack(rows)


def _parts64(t):
    """[real] or [real, imaginary] in 64 bits"""
    return [t.real.to(torch.float64), t.imag.to(torch.float64)] if t.is_complex() else [t.to(torch.float64)]


def _joined(parts):
    return parts[0] if len(parts) == 1 else torch.complex(parts[0], parts[1])


def _through_dropout64(parts, st, case):
    if not case["drop"]:
        return parts
    factor = _factors64(st, case)
    return [v * factor for v in parts]


def _exact_dropout(st, case):
    parts = _through_dropout64(_parts64(st["x"]), st, case)
    if st["residual"] is not None:
        parts = [u + v for u, v in zip(parts, _parts64(st["residual"]))]
    return dict(y=_joined(parts))


def _quantised64(parts):
    """values over their scale, before their rounding to 8 bits, and the scales"""
    scales, rows = [], []
    for first in range(0, parts[0].shape[0], _BLOCK):
        block = torch.stack([v[first:first + _BLOCK] for v in parts], dim=-1)
        scales.append(block.abs().flatten(2).amax(dim=(0, 2)) / _E4M3_MAX)
        rows.append(block / scales[-1][:, None])
    q = torch.cat(rows)
    return dict(q=q if len(parts) == 2 else q[..., 0], scale=torch.stack(scales))


def _exact_quantise(st, case):
    return _quantised64(_parts64(st["x"]))


def _exact_norm(st, case):
    gain, K = st["gain"].to(torch.float64).reshape(-1, 1), case["K"]
    if case["form"] == "backward":
        rstd = st["rstd"].to(torch.float64)
        h = [(v - m) * rstd for v, m in zip(_parts64(st["s"]), _parts64(st["mean"]))]
        gy = _parts64(st["gy"])
        dot = sum(u * v for u, v in zip(gy, h))
        slope = (gain * dot).sum(dim=0) / K
        gr = [rstd * (gain * g - (gain * g).sum(dim=0) / K - v * slope) for g, v in zip(gy, h)]
        if st["gs"] is not None:
            gr = [u + v for u, v in zip(gr, _parts64(st["gs"]))]
        out = dict(gr=_joined(gr)) if case["drop"] else {}
        return dict(out, gx=_joined(_through_dropout64(gr, st, case)), ggain=dot.sum(dim=1), gbias=_joined([g.sum(dim=1) for g in gy]))
    s = _through_dropout64(_parts64(st["x"]), st, case)
    if st["residual"] is not None:
        s = [u + v for u, v in zip(s, _parts64(st["residual"]))]
    mean = [v.sum(dim=0) / K for v in s]
    centred = [v - m for v, m in zip(s, mean)]
    rstd = 1.0 / torch.sqrt(sum(v.pow(2).sum(dim=0) for v in centred) / K + _EPS)
    y = [v * rstd * gain + b[:, None] for v, b in zip(centred, _parts64(st["bias"]))]
    out = dict(s=_joined(s)) if st["s"] is not None else {}
    if case["form"] == "8bit":
        return dict(out, **_quantised64(y))
    return dict(out, y=_joined(y), mean=_joined(mean), rstd=rstd)


def _act64(act, v):
    if act == "none":
        return v
    if act == "relu":
        return torch.clamp(v, min=0.0)
    if act == "silu":
        return 0.5 * v * (1.0 + torch.tanh(0.5 * v))
    return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v.pow(3))))


def _exact_product(st, case):
    K, N = case["K"], case["N"]
    split = lambda t: [t[..., 0], t[..., 1]] if case["type"] == "c64" else [t]  # noqa: E731
    z = [0.0] * len(split(st["xq"]))
    row_block = torch.arange(N, device="cuda") // _BLOCK
    for b in range(-(-K // _BLOCK)):                    # the definition: block by block
        lo, hi = b * _BLOCK, min(K, (b + 1) * _BLOCK)
        x = split(st["xq"][lo:hi].to(torch.float64))
        W = split(st["Wq"][:, lo:hi].to(torch.float64))
        scale = st["wscale"].to(torch.float64)[row_block, b][:, None] * st["xscale"][b].to(torch.float64)
        if len(z) == 1:
            sums = [W[0] @ x[0]]
        else:
            sums = [W[0] @ x[0] - W[1] @ x[1], W[0] @ x[1] + W[1] @ x[0]]
        z = [u + scale * v for u, v in zip(z, sums)]
    z = [u + v[:, None] for u, v in zip(z, _parts64(st["bias"]))]
    if st["residual"] is not None:
        z = [u + v for u, v in zip(z, _parts64(st["residual"]))]
    return dict(y=_joined([_act64(case["act"], v) for v in z]))


def exact(case, seed):
    forms = {"norm": _exact_norm, "dropout": _exact_dropout, "quantise": _exact_quantise, "product": _exact_product}
    return forms[case["op"]](prepare(case, seed), case)


# ---- what a pass cannot do without ----

def work(case):
    e, K, P, parts = _TYPES[case["type"]].itemsize, case["K"], case["P"], 2 if case["type"] == "c64" else 1
    values, blocks = parts * K * P, -(-K // _BLOCK)
    if case["op"] == "product":
        N = case["N"]
        flops = (8.0 if parts == 2 else 2.0) * N * K * P
        outs = 2 if case["residual"] else 1
        return dict(bytes=values + 4 * blocks * P + parts * N * K + 4 * blocks * -(-N // _BLOCK) + e * N * (P * outs + 1), flops=flops)
    if case["op"] == "quantise":
        return dict(bytes=e * K * P + values + 4 * blocks * P, flops=3.0 * values)
    more, dropped = 1 if case["residual"] else 0, 1 if case["drop"] else 0
    if case["op"] == "dropout":
        return dict(bytes=e * K * P * (2 + more) + 16, flops=(2.0 + more) * values)
    ends = 4 * (parts + 1)                              # mean and rstd of a position; gain and bias of a channel
    if case["form"] == "backward":
        return dict(bytes=e * K * P * (3 + more + dropped) + ends * (P + 2 * K) + 16 * dropped, flops=(13.0 + more + dropped) * values)
    sums = 1 if more or dropped else 0
    if case["form"] == "8bit":
        return dict(bytes=e * K * P * (1 + more + sums) + values + 4 * blocks * P + ends * K, flops=(10.0 + more) * values)
    return dict(bytes=e * K * P * (2 + more + sums) + ends * (P + K) + 16 * dropped, flops=(7.0 + more + dropped) * values)
