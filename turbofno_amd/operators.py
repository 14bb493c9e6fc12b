"""Binding of the operators around the spectral layer (include/turbofno.h): channel product with epilogue, root-mean-square norm and layer norm, dropout, fields
in 8 bits, gradient clipping.

Fields are channel outermost like the layer's, x[K][positions...]: any trailing dimensions, contiguous among themselves, with any distance
between channels (a slice of a larger batch of channels is taken as it is). Types: complex64, float32, bfloat16. Results are
allocated where they are not passed. Every call is asynchronous on torch's current stream.

Nothing is recorded for autograd, as with the layer: a result is cut off from the graph, also where an operand requires a gradient. The gradients are calls
of their own (mix_backward, rms_norm_backward, layer_norm_backward, mix_weight_grad; dropout is its own), to be made by a training step like examples/fourier_block.py or by the backward of an
autograd function.
"""
import ctypes

import torch

from . import api
from .api import _check, _need, _stream

_TYPES = {torch.complex64: 0, torch.float32: 1, torch.bfloat16: 2}
_ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu_tanh": 3}
_LIB = None
_AT = {}                                # addresses of the entry points, for the compiled checks (csrc/operands.cpp)


def _lib():
    global _LIB
    if _LIB is None:
        L = api.lib()
        vp, i, l, f, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_long, ctypes.c_float, ctypes.c_size_t
        L.turbofno_mix.argtypes = [i, l, i, i, vp, l, vp, vp, vp, l, i, vp, l, vp, l, vp]
        L.turbofno_mix_8bit.argtypes = [i, l, i, i, vp, l, vp, vp, vp, vp, vp, l, i, vp, l, vp]
        L.turbofno_mix_input_grad.argtypes = [i, l, i, i, vp, l, vp, l, vp, i, vp, l, vp, l, vp]
        L.turbofno_mix_weight_grad_workspace_bytes.argtypes = [i, l, i, i]
        L.turbofno_mix_weight_grad.argtypes = [i, l, i, i, vp, l, vp, l, vp, vp, vp, sz, vp]
        L.turbofno_rms_norm.argtypes = [i, l, i, vp, l, vp, l, vp, f, vp, l, vp, l, vp, vp]
        L.turbofno_rms_norm_8bit.argtypes = [i, l, i, vp, l, vp, l, vp, f, vp, l, vp, l, vp, vp]
        L.turbofno_rms_norm_backward_workspace_bytes.argtypes = [i, l, i]
        L.turbofno_rms_norm_backward.argtypes = [i, l, i, vp, l, vp, l, vp, vp, vp, l, vp, l, vp, vp, sz, vp]
        L.turbofno_clip_grad_norm_workspace_bytes.argtypes = [i]
        d = ctypes.c_double
        L.turbofno_dropout.argtypes = [i, l, i, vp, l, vp, l, d, vp, vp, l, vp]
        L.turbofno_layer_norm.argtypes = [i, l, i, vp, l, vp, l, vp, vp, f, d, vp, vp, l, vp, l, vp, vp, vp]
        L.turbofno_layer_norm_8bit.argtypes = [i, l, i, vp, l, vp, l, vp, vp, f, vp, l, vp, l, vp, vp]
        L.turbofno_layer_norm_backward_workspace_bytes.argtypes = [i, l, i]
        L.turbofno_layer_norm_backward.argtypes = [i, l, i, vp, l, vp, l, vp, vp, vp, vp, l, d, vp, vp, l, vp, l, vp, vp, vp, sz, vp]
        L.turbofno_quantise_8bit.argtypes = [i, l, i, vp, l, vp, l, vp, vp]
        L.turbofno_mix_8bit_blocks.argtypes = [i, l, i, i, vp, l, vp, vp, vp, vp, vp, l, i, vp, l, vp]
        L.turbofno_clip_grad_norm.argtypes = [i, vp, vp, vp, vp, f, vp, vp, sz, vp]
        for name in ("turbofno_mix", "turbofno_mix_8bit", "turbofno_mix_input_grad", "turbofno_mix_weight_grad", "turbofno_rms_norm",
                     "turbofno_rms_norm_8bit", "turbofno_rms_norm_backward", "turbofno_clip_grad_norm", "turbofno_dropout", "turbofno_layer_norm",
                     "turbofno_layer_norm_8bit", "turbofno_layer_norm_backward", "turbofno_quantise_8bit", "turbofno_mix_8bit_blocks"):
            getattr(L, name).restype = i
        for name in ("mix_weight_grad", "rms_norm_backward", "layer_norm_backward", "clip_grad_norm"):
            getattr(L, "turbofno_%s_workspace_bytes" % name).restype = sz
        for name in ("mix", "mix_8bit", "mix_input_grad", "mix_weight_grad", "mix_weight_grad_workspace_bytes", "rms_norm", "rms_norm_8bit",
                     "rms_norm_backward", "rms_norm_backward_workspace_bytes", "clip_grad_norm", "clip_grad_norm_workspace_bytes", "dropout", "layer_norm",
                     "layer_norm_8bit", "layer_norm_backward", "layer_norm_backward_workspace_bytes", "quantise_8bit", "mix_8bit_blocks"):
            _AT[name] = ctypes.cast(getattr(L, "turbofno_" + name), vp).value
        _LIB = L
    return _LIB


def _compiled(call, functions, *args):
    """The call through the compiled checks: True, or False where an operand is for the checks here to judge. They do the same, without a trip
    through Python for every attribute of a tensor."""
    if api._operands is None:
        return False
    if _LIB is None:
        _lib()
    device = torch.cuda.current_device()
    rc = getattr(api._operands, call)(*[_AT[f] for f in functions], *args, device, api._raw_stream(device) if api._raw_stream is not None else _stream())
    if rc > 0:
        _check(rc)
    return rc == 0


def _type(dtype, name):
    if dtype not in _TYPES:
        raise TypeError("%s is %s: complex64, float32 and bfloat16 are taken" % (name, dtype))
    return _TYPES[dtype]


def _activation(name):
    _need(name in _ACTIVATIONS, "activation %r is none of %s", name, ", ".join(_ACTIVATIONS))
    return _ACTIVATIONS[name]


def _on_gpu(t, name, dtype, device):
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == dtype):
        raise TypeError("%s must be a %s tensor on the GPU" % (name, dtype))
    if t.is_conj() or t.is_neg():                       # such views keep other values in memory than they stand for
        raise TypeError("%s is a conjugated or negated view: resolve it first" % name)
    _need(t.device == device, "%s is on %s, expected %s: all operands must live on one GPU", name, t.device, device)


def _spread(t, name, parts=1):
    """distance between channels of a field, in elements of `parts` values; the other dimensions have to lie side by side"""
    step = 1
    for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        _need(size == 1 or stride == step, "%s: the positions of a channel must lie side by side (strides %s)", name, t.stride())
        step *= size
    ld = t.stride(0) if t.shape[0] > 1 else step
    _need(ld % parts == 0, "%s: complex values are pairs, but channels are %d values apart", name, ld)
    return ld // parts


def _field(t, name, shape, dtype, device):
    """address and distance between channels of a field of that shape; (None, 0) for None"""
    if t is None:
        return None, 0
    _need(isinstance(t, torch.Tensor) and tuple(t.shape) == tuple(shape), "%s has shape %s, expected %s", name, tuple(getattr(t, "shape", ())), tuple(shape))
    _on_gpu(t, name, dtype, device)
    return t.data_ptr(), _spread(t, name)


def _packed(t, name, shape, dtype, device):
    """address of a contiguous tensor of that shape; None for None"""
    if t is None:
        return None
    _need(isinstance(t, torch.Tensor) and tuple(t.shape) == tuple(shape), "%s has shape %s, expected %s", name, tuple(getattr(t, "shape", ())), tuple(shape))
    _on_gpu(t, name, dtype, device)
    _need(t.is_contiguous(), "%s must be contiguous", name)
    return t.data_ptr()


def _place(t):
    """memory of a tensor whose rows lie side by side each: address, rows, bytes from row to row, bytes of a row; None for what is no such tensor"""
    if not isinstance(t, torch.Tensor) or not t.numel():
        return None
    if t.is_contiguous():
        return t.data_ptr(), 1, 0, t.numel() * t.element_size()
    if t.dim() < 2 or t.stride(0) <= 0 or not t[0].is_contiguous():
        return None
    return t.data_ptr(), t.shape[0], t.stride(0) * t.element_size(), t[0].numel() * t.element_size()


def _meet(a, b):
    """do two tensors share a byte"""
    a, b = _place(a), _place(b)
    if a is None or b is None or a[0] >= b[0] + (b[1] - 1) * b[2] + b[3] or b[0] >= a[0] + (a[1] - 1) * a[2] + a[3]:
        return False
    (at, rows, pitch, width), (other, others, other_pitch, other_width) = (a, b) if a[1] <= b[1] else (b, a)
    for start in range(at, at + rows * pitch if rows > 1 else at + 1, pitch or 1):
        before = start - other - other_width            # the first of the other's rows that ends behind `start`
        row = 0 if before < 0 or others == 1 else before // other_pitch + 1
        if row < others and other + row * other_pitch < start + width and start < other + row * other_pitch + other_width:
            return True
    return False


def _over(y, x):
    """is the result to take the place of x"""
    return isinstance(y, torch.Tensor) and isinstance(x, torch.Tensor) and y.numel() > 0 and y.data_ptr() == x.data_ptr()


def _input(x, name):
    """type, device, channels and positions of the field a call starts from"""
    if not isinstance(x, torch.Tensor):
        raise TypeError("%s must be a tensor" % name)
    _need(x.dim() >= 2 and x.shape[0] > 0, "%s must be [channels][positions...]", name)
    return _type(x.dtype, name), x.device, x.shape[0], x.numel() // x.shape[0]


def _current(device):
    _need(device.index == torch.cuda.current_device(), "the operands are on %s, the current device is cuda:%d", device, torch.cuda.current_device())


def _result(t, shape, dtype, device):
    return torch.empty(shape, dtype=dtype, device=device) if t is None else t


def _workspace(t, need, device):
    if t is None:
        t = torch.empty(need, dtype=torch.uint8, device=device)
    if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype == torch.uint8 and t.is_contiguous()):
        raise TypeError("workspace must be a contiguous uint8 tensor on the GPU")
    _need(t.device == device, "workspace is on %s, expected %s", t.device, device)
    return t


def mix(x, W, bias=None, residual=None, activation="none", y=None, z=None):
    """z = W x + bias + residual, y = activation(z): x[K][...], W[N][K] -> y[N][...]. `z`, where passed, receives the pre-activation that
    mix_backward takes. `residual` may be `y` or `z` itself. Activations: none, relu, silu, gelu_tanh; on real and imaginary parts. Not recorded for
    autograd: the gradients are mix_backward's."""
    if y is None and isinstance(x, torch.Tensor) and isinstance(W, torch.Tensor) and x.is_cuda and x.dim() and W.dim():
        y = torch.empty(W.shape[:1] + x.shape[1:], dtype=x.dtype, device=x.device)
    if getattr(y, "is_cuda", False) and _compiled("mix", ("mix",), x, W, bias, residual, _ACTIVATIONS.get(activation, -1), y, z):
        return y
    kind, device, K, P = _input(x, "x")
    act = _activation(activation)
    _need(isinstance(W, torch.Tensor) and W.dim() == 2 and W.shape[1] == K and W.shape[0] > 0, "W must be [N][%d], one column per channel of x", K)
    N, dtype = W.shape[0], x.dtype
    shape = (N,) + tuple(x.shape[1:])
    px, ldx = _field(x, "x", x.shape, dtype, device)
    y = _result(y, shape, dtype, device)
    pr, ldr = _field(residual, "residual", shape, dtype, device)
    pz, ldz = _field(z, "z", shape, dtype, device)
    py, ldy = _field(y, "y", shape, dtype, device)
    pW, pb = _packed(W, "W", (N, K), dtype, device), _packed(bias, "bias", (N,), dtype, device)
    _current(device)
    _check(_lib().turbofno_mix(kind, P, N, K, px, ldx, pW, pb, pr, ldr, act, pz, ldz, py, ldy, _stream()))
    return y


def mix_8bit(xq, xscale, Wq, wscale, bias=None, residual=None, activation="none", y=None, dtype=None):
    """mix from 8-bit operands: x = xscale[position] xq, W = wscale[n] Wq, all of float8_e4m3fn with float32 scales; xq and xscale as
    rms_norm_8bit gives them. The result has the type of `y`, `residual` or `dtype`, whichever is there (bfloat16 if none is). Complex
    operands are (re, im) pairs along a last dimension of two: xq[K][...][2], Wq[N][K][2]."""
    if getattr(y, "is_cuda", False) and dtype in (None, y.dtype) and _compiled("mix_8bit", ("mix_8bit",), xq, xscale, Wq, wscale, bias, residual, _ACTIVATIONS.get(activation, -1), y):
        return y
    if dtype is None:
        dtype = next((t.dtype for t in (y, residual) if isinstance(t, torch.Tensor)), torch.bfloat16)
    kind = _type(dtype, "the result")
    act = _activation(activation)
    tail = (2,) if dtype == torch.complex64 else ()
    if not isinstance(xq, torch.Tensor) or not isinstance(Wq, torch.Tensor):
        raise TypeError("xq and Wq must be tensors")
    _need(xq.dim() >= 2 + len(tail) and xq.shape[0] > 0 and (not tail or xq.shape[-1] == 2), "xq must be [K][positions...]%s", "[2]" if tail else "")
    K, device = xq.shape[0], xq.device
    _need(Wq.dim() == 2 + len(tail) and Wq.shape[0] > 0 and tuple(Wq.shape[1:]) == (K,) + tail, "Wq must be [N][%d]%s", K, "[2]" if tail else "")
    N, places = Wq.shape[0], tuple(xq.shape[1:-1] if tail else xq.shape[1:])
    P = xq.numel() // (K * (2 if tail else 1))
    f8 = torch.float8_e4m3fn
    _on_gpu(xq, "xq", f8, device)
    ldx = _spread(xq, "xq", 2 if tail else 1)
    y = _result(y, (N,) + places, dtype, device)
    pr, ldr = _field(residual, "residual", (N,) + places, dtype, device)
    py, ldy = _field(y, "y", (N,) + places, dtype, device)
    pxs, pW = _packed(xscale, "xscale", places, torch.float32, device), _packed(Wq, "Wq", Wq.shape, f8, device)
    pws, pb = _packed(wscale, "wscale", (N,), torch.float32, device), _packed(bias, "bias", (N,), dtype, device)
    _current(device)
    _check(_lib().turbofno_mix_8bit(kind, P, N, K, xq.data_ptr(), ldx, pxs, pW, pws, pb, pr, ldr, act, py, ldy, _stream()))
    return y


def mix_input_grad(gy, W, z=None, activation="none", gz=None, gx=None):
    """(gx, gz): gz = gy activation'(z), the gradient of the residual, and gx = W^H gz. Without an activation gz is gy itself. In bfloat16 gx is formed from
    gz as it is returned, rounded to bfloat16."""
    kind, device, N, P = _input(gy, "gy")
    act = _activation(activation)
    _need(isinstance(W, torch.Tensor) and W.dim() == 2 and W.shape[0] == N and W.shape[1] > 0, "W must be [%d][K], one row per channel of gy", N)
    K, dtype = W.shape[1], gy.dtype
    pg, ldg = _field(gy, "gy", gy.shape, dtype, device)
    if act:
        _need(z is not None, "the gradient of %s needs z", activation)
        gz = _result(gz, gy.shape, dtype, device)
    else:
        gz = gy
    gx = _result(gx, (K,) + tuple(gy.shape[1:]), dtype, device)
    pz, ldz = _field(z if act else None, "z", gy.shape, dtype, device)
    po, ldo = _field(gz, "gz", gy.shape, dtype, device)
    px, ldx = _field(gx, "gx", (K,) + tuple(gy.shape[1:]), dtype, device)
    pW = _packed(W, "W", (N, K), dtype, device)
    _current(device)
    _check(_lib().turbofno_mix_input_grad(kind, P, N, K, pg, ldg, pz, ldz, pW, act, po if act else None, ldo, px, ldx, _stream()))
    return gx, gz


def mix_weight_grad_workspace_bytes(N, K, P, dtype):
    return int(_lib().turbofno_mix_weight_grad_workspace_bytes(_type(dtype, "the operand"), P, N, K))


def mix_weight_grad(gz, x, gW=None, gbias=None, workspace=None):
    """(gW, gbias): gW[n][k] = sum over positions of gz[n] conj(x[k]), gbias[n] = sum over positions of gz[n]. On truncated spectra, gW is also the
    gradient of the spectral layer's weights. `workspace`: uint8 GPU tensor (allocated here when omitted)."""
    kind, device, N, P = _input(gz, "gz")
    _need(isinstance(x, torch.Tensor) and x.dim() >= 2 and x.shape[0] > 0 and x.shape[1:] == gz.shape[1:], "x must be [K]%s like gz", list(gz.shape[1:]))
    K, dtype = x.shape[0], gz.dtype
    pg, ldg = _field(gz, "gz", gz.shape, dtype, device)
    px, ldx = _field(x, "x", x.shape, dtype, device)
    gW, gbias = _result(gW, (N, K), dtype, device), _result(gbias, (N,), dtype, device)
    pW, pb = _packed(gW, "gW", (N, K), dtype, device), _packed(gbias, "gbias", (N,), dtype, device)
    workspace = _workspace(workspace, _lib().turbofno_mix_weight_grad_workspace_bytes(kind, P, N, K), device)
    _current(device)
    _check(_lib().turbofno_mix_weight_grad(kind, P, N, K, pg, ldg, px, ldx, pW, pb, workspace.data_ptr(), workspace.numel(), _stream()))
    return gW, gbias


def mix_backward(gy, x, W, z=None, activation="none", gz=None, gx=None, gW=None, gbias=None, workspace=None):
    """(gx, gW, gbias, gz) from the gradient of y, and the x, W and z of mix; gz is the gradient of its residual. x is read after gx and gz are written:
    they share no memory with it. In bfloat16 gx, gW and gbias are formed from gz as it is returned, rounded to bfloat16."""
    act = _ACTIVATIONS.get(activation, -1)
    if isinstance(gy, torch.Tensor) and isinstance(x, torch.Tensor) and isinstance(W, torch.Tensor) and gy.is_cuda:
        gz = gy if act == 0 else _result(gz, gy.shape, gy.dtype, gy.device)
        gx, gW, gbias = _result(gx, x.shape, x.dtype, x.device), _result(gW, W.shape, W.dtype, W.device), _result(gbias, gy.shape[:1], gy.dtype, gy.device)
        if _compiled("mix_backward", ("mix_input_grad", "mix_weight_grad", "mix_weight_grad_workspace_bytes"), gy, x, W, z, act, gz, gx, gW, gbias, workspace):
            return gx, gW, gbias, gz
    for name, t in (("gx", gx), ("gz", None if act == 0 else gz)):
        _need(not _meet(t, x), "%s overlaps x, which the gradient of W is formed from afterwards", name)
    for name, t in (("gW", gW), ("gbias", gbias), ("workspace", workspace)):
        _need(not _meet(t, gx), "%s overlaps gx", name)
    gx, gz = mix_input_grad(gy, W, z=z, activation=activation, gz=gz, gx=gx)
    gW, gbias = mix_weight_grad(gz, x, gW=gW, gbias=gbias, workspace=workspace)
    return gx, gW, gbias, gz


def _norm(x, gain, residual, eps, y, scale, s, rstd, eight):
    row = scale if eight else rstd
    if residual is None and s is None and _over(y, x):
        s = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if row is not None and (residual is None or s is not None) and getattr(y, "is_cuda", False):
        if _compiled("rms_norm", ("rms_norm_8bit" if eight else "rms_norm",), int(eight), x, gain, residual, eps, s, y, row):
            return y, row, x if s is None else s
    kind, device, K, P = _input(x, "x")
    dtype = x.dtype
    places = tuple(x.shape[1:])
    px, ldx = _field(x, "x", x.shape, dtype, device)
    pr, ldr = _field(residual, "residual", x.shape, dtype, device)
    pg = _packed(gain, "gain", (K,), torch.float32, device)
    if residual is not None:
        s = _result(s, x.shape, dtype, device)
    ps, lds = _field(s, "s", x.shape, dtype, device)
    if eight:
        parts = 2 if dtype == torch.complex64 else 1
        shape = tuple(x.shape) + ((2,) if parts == 2 else ())
        y, scale = _result(y, shape, torch.float8_e4m3fn, device), _result(scale, places, torch.float32, device)
        py, ldy = _field(y, "q", shape, torch.float8_e4m3fn, device)
        ldy = _spread(y, "q", parts)
        pc = _packed(scale, "scale", places, torch.float32, device)
    else:
        y, rstd = _result(y, x.shape, dtype, device), _result(rstd, places, torch.float32, device)
        py, ldy = _field(y, "y", x.shape, dtype, device)
        pc = _packed(rstd, "rstd", places, torch.float32, device)
    if pg is None:
        raise TypeError("gain must be a float32 tensor on the GPU")
    _current(device)
    call = _lib().turbofno_rms_norm_8bit if eight else _lib().turbofno_rms_norm
    _check(call(kind, P, K, px, ldx, pr, ldr, pg, float(eps), ps, lds, py, ldy, pc, _stream()))
    return y, scale if eight else rstd, x if s is None else s


def rms_norm(x, gain, residual=None, eps=1e-6, y=None, s=None, rstd=None):
    """s = x + residual, rstd = 1 / sqrt(mean over channels of |s|^2 + eps), y = gain rstd s: x[K][...], gain[K] in float32 -> (y, s, rstd).
    Without a residual s is x itself, or what x was where y replaces it. `s` and `y` may be `x` or `residual` themselves; rstd has the shape of the positions.
    Not recorded for autograd: the gradients are rms_norm_backward's."""
    y, rstd, s = _norm(x, gain, residual, eps, y, None, s, rstd, False)
    return y, s, rstd


def rms_norm_8bit(x, gain, residual=None, eps=1e-6, q=None, scale=None, s=None):
    """rms_norm with its result in float8_e4m3fn and a float32 scale per position, the largest magnitude of its channels over 448: (q, scale, s). q has a
    last dimension of two, (re, im), for complex fields."""
    return _norm(x, gain, residual, eps, q, scale, s, None, True)


def rms_norm_backward_workspace_bytes(K, P, dtype):
    return int(_lib().turbofno_rms_norm_backward_workspace_bytes(_type(dtype, "the operand"), P, K))


def rms_norm_backward(gy, s, gain, rstd, gs=None, gx=None, ggain=None, workspace=None):
    """(gx, ggain) from the gradient of y, the s and rstd of rms_norm, and gs, what reaches s by the residual stream. gx is the gradient of x and of
    residual; it may be gy, s or gs itself."""
    if ggain is not None and getattr(gx, "is_cuda", False):
        if _compiled("rms_norm_backward", ("rms_norm_backward", "rms_norm_backward_workspace_bytes"), gy, s, gain, rstd, gs, gx, ggain, workspace):
            return gx, ggain
    kind, device, K, P = _input(gy, "gy")
    dtype, places = gy.dtype, tuple(gy.shape[1:])
    if not all(isinstance(t, torch.Tensor) for t in (s, gain, rstd)):
        raise TypeError("s, gain and rstd must be tensors")
    py, ldy = _field(gy, "gy", gy.shape, dtype, device)
    ps, lds = _field(s, "s", gy.shape, dtype, device)
    pgs, ldgs = _field(gs, "gs", gy.shape, dtype, device)
    gx, ggain = _result(gx, gy.shape, dtype, device), _result(ggain, (K,), torch.float32, device)
    px, ldx = _field(gx, "gx", gy.shape, dtype, device)
    pg, pr = _packed(gain, "gain", (K,), torch.float32, device), _packed(rstd, "rstd", places, torch.float32, device)
    po = _packed(ggain, "ggain", (K,), torch.float32, device)
    workspace = _workspace(workspace, _lib().turbofno_rms_norm_backward_workspace_bytes(kind, P, K), device)
    _current(device)
    _check(_lib().turbofno_rms_norm_backward(kind, P, K, py, ldy, ps, lds, pg, pr, pgs, ldgs, px, ldx, po, workspace.data_ptr(),
                                             workspace.numel(), _stream()))
    return gx, ggain


_BLOCK = 128                            # channels of a scale


def _blocks(channels):
    return -(-channels // _BLOCK)


def _wide(dtype):
    """the 32-bit type of values that accompany a field"""
    return torch.complex64 if dtype.is_complex else torch.float32


def _rng(rng, device):
    return _packed(rng, "rng", (2,), torch.int64, device)


def dropout(x, drop, rng, residual=None, y=None):
    """y = residual + dropout(x): x / (1 - drop) where the element is kept, 0 elsewhere. `rng`: int64 GPU tensor (seed, offset), read when the kernel runs (in a
    captured graph, at each replay); no mask is stored, the same rng gives the same one. Every use in a model and every step takes an offset of its own. The
    gradient of x is dropout(gy, drop, rng), that of residual is gy. `y` may be `x` or `residual` itself. The elements that are kept depend on rng, drop, the
    channel and the position, on nothing else: include/turbofno.h has the generator."""
    if y is None and isinstance(x, torch.Tensor) and x.is_cuda:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if getattr(y, "is_cuda", False) and _compiled("dropout", ("dropout",), x, residual, drop, rng, y):
        return y
    kind, device, K, P = _input(x, "x")
    px, ldx = _field(x, "x", x.shape, x.dtype, device)
    pr, ldr = _field(residual, "residual", x.shape, x.dtype, device)
    y = _result(y, x.shape, x.dtype, device)
    py, ldy = _field(y, "y", x.shape, x.dtype, device)
    pd = _rng(rng, device)
    _current(device)
    _check(_lib().turbofno_dropout(kind, P, K, px, ldx, pr, ldr, float(drop), pd, py, ldy, _stream()))
    return y


def layer_norm(x, gain, bias=None, residual=None, eps=1e-6, drop=0.0, rng=None, y=None, s=None, mean=None, rstd=None):
    """s = residual + dropout(x), mean over channels of s, rstd = 1 / sqrt(mean over channels of |s - mean|^2 + eps), y = gain rstd (s - mean) + bias: x[K][...],
    gain[K] in float32, bias[K] in float32, complex64 for complex fields -> (y, s, mean, rstd). Without residual and dropout s is x itself, or what x was where y replaces it. `s` and `y`
    may be `x` or `residual` themselves; mean (of the type of bias) and rstd have the shape of the positions. drop, rng: as dropout takes them. Not recorded for autograd:
    the gradients are layer_norm_backward's."""
    summed = residual is not None or drop or _over(y, x)
    if isinstance(x, torch.Tensor) and x.is_cuda and x.dim() >= 2:
        y, mean = _result(y, x.shape, x.dtype, x.device), _result(mean, x.shape[1:], _wide(x.dtype), x.device)
        rstd = _result(rstd, x.shape[1:], torch.float32, x.device)
        if summed:
            s = _result(s, x.shape, x.dtype, x.device)
        if _compiled("layer_norm", ("layer_norm",), x, gain, bias, residual, eps, drop, rng, s, y, mean, rstd):
            return y, x if s is None else s, mean, rstd
    kind, device, K, P = _input(x, "x")
    dtype, places = x.dtype, tuple(x.shape[1:])
    px, ldx = _field(x, "x", x.shape, dtype, device)
    pr, ldr = _field(residual, "residual", x.shape, dtype, device)
    if not isinstance(gain, torch.Tensor):
        raise TypeError("gain must be a float32 tensor on the GPU")
    pg, pb = _packed(gain, "gain", (K,), torch.float32, device), _packed(bias, "bias", (K,), _wide(dtype), device)
    pd = _rng(rng, device)
    if summed:
        s = _result(s, x.shape, dtype, device)
    y, mean, rstd = _result(y, x.shape, dtype, device), _result(mean, places, _wide(dtype), device), _result(rstd, places, torch.float32, device)
    ps, lds = _field(s, "s", x.shape, dtype, device)
    py, ldy = _field(y, "y", x.shape, dtype, device)
    pm, pt = _packed(mean, "mean", places, _wide(dtype), device), _packed(rstd, "rstd", places, torch.float32, device)
    _current(device)
    _check(_lib().turbofno_layer_norm(kind, P, K, px, ldx, pr, ldr, pg, pb, float(eps), float(drop), pd, ps, lds, py, ldy, pm, pt, _stream()))
    return y, x if s is None else s, mean, rstd


def _eight_results(x, q, scale):
    """the 8-bit field and scales of a field, where they are not passed"""
    q = _result(q, tuple(x.shape) + ((2,) if x.dtype.is_complex else ()), torch.float8_e4m3fn, x.device)
    return q, _result(scale, (_blocks(x.shape[0]),) + tuple(x.shape[1:]), torch.float32, x.device)


def _eight_fields(x, q, scale, device):
    pair = (2,) if x.dtype.is_complex else ()
    pq, _ = _field(q, "q", tuple(x.shape) + pair, torch.float8_e4m3fn, device)
    return pq, _spread(q, "q", 2 if pair else 1), _packed(scale, "scale", (_blocks(x.shape[0]),) + tuple(x.shape[1:]), torch.float32, device)


def layer_norm_8bit(x, gain, bias=None, residual=None, eps=1e-6, q=None, scale=None, s=None):
    """layer_norm without dropout and with its result as quantise_8bit gives it: (q, scale, s)."""
    if isinstance(x, torch.Tensor) and x.is_cuda and x.dim() >= 2:
        q, scale = _eight_results(x, q, scale)
        if residual is not None:
            s = _result(s, x.shape, x.dtype, x.device)
        if _compiled("layer_norm_8bit", ("layer_norm_8bit",), x, gain, bias, residual, eps, s, q, scale):
            return q, scale, x if s is None else s
    kind, device, K, P = _input(x, "x")
    dtype = x.dtype
    px, ldx = _field(x, "x", x.shape, dtype, device)
    pr, ldr = _field(residual, "residual", x.shape, dtype, device)
    if not isinstance(gain, torch.Tensor):
        raise TypeError("gain must be a float32 tensor on the GPU")
    pg, pb = _packed(gain, "gain", (K,), torch.float32, device), _packed(bias, "bias", (K,), _wide(dtype), device)
    if residual is not None:
        s = _result(s, x.shape, dtype, device)
    ps, lds = _field(s, "s", x.shape, dtype, device)
    q, scale = _eight_results(x, q, scale)
    pq, ldq, pc = _eight_fields(x, q, scale, device)
    _current(device)
    _check(_lib().turbofno_layer_norm_8bit(kind, P, K, px, ldx, pr, ldr, pg, pb, float(eps), ps, lds, pq, ldq, pc, _stream()))
    return q, scale, x if s is None else s


def layer_norm_backward_workspace_bytes(K, P, dtype):
    return int(_lib().turbofno_layer_norm_backward_workspace_bytes(_type(dtype, "the operand"), P, K))


def layer_norm_backward(gy, s, gain, mean, rstd, gs=None, drop=0.0, rng=None, gx=None, gr=None, ggain=None, gbias=None, workspace=None):
    """(gx, gr, ggain, gbias) from the gradient of y, the s, mean and rstd of layer_norm, and gs, what reaches s by the residual stream. gr is the gradient of s and of
    residual, gx = dropout(gr) that of x, with the drop and rng of layer_norm; without dropout gr is gx itself, and what is passed for it is not used. gx
    and gr may be gy, s or gs themselves. gbias has the type of bias."""
    if isinstance(gy, torch.Tensor) and gy.is_cuda and gy.dim() >= 2:
        gx, gr = _result(gx, gy.shape, gy.dtype, gy.device), _result(gr, gy.shape, gy.dtype, gy.device) if drop else None
        ggain, gbias = _result(ggain, gy.shape[:1], torch.float32, gy.device), _result(gbias, gy.shape[:1], _wide(gy.dtype), gy.device)
        if _compiled("layer_norm_backward", ("layer_norm_backward", "layer_norm_backward_workspace_bytes"), gy, s, gain, mean, rstd, gs, drop, rng, gx, gr, ggain,
                     gbias, workspace):
            return gx, gr if drop else gx, ggain, gbias
    kind, device, K, P = _input(gy, "gy")
    dtype, places = gy.dtype, tuple(gy.shape[1:])
    if not all(isinstance(t, torch.Tensor) for t in (s, gain, mean, rstd)):
        raise TypeError("s, gain, mean and rstd must be tensors")
    py, ldy = _field(gy, "gy", gy.shape, dtype, device)
    ps, lds = _field(s, "s", gy.shape, dtype, device)
    pgs, ldgs = _field(gs, "gs", gy.shape, dtype, device)
    gx, gr = _result(gx, gy.shape, dtype, device), _result(gr, gy.shape, dtype, device) if drop else None
    px, ldx = _field(gx, "gx", gy.shape, dtype, device)
    pr, ldr = _field(gr, "gr", gy.shape, dtype, device)
    pg, pm, pt = _packed(gain, "gain", (K,), torch.float32, device), _packed(mean, "mean", places, _wide(dtype), device), _packed(rstd, "rstd", places, torch.float32, device)
    pd = _rng(rng, device)
    ggain, gbias = _result(ggain, (K,), torch.float32, device), _result(gbias, (K,), _wide(dtype), device)
    po, pb = _packed(ggain, "ggain", (K,), torch.float32, device), _packed(gbias, "gbias", (K,), _wide(dtype), device)
    workspace = _workspace(workspace, _lib().turbofno_layer_norm_backward_workspace_bytes(kind, P, K), device)
    _current(device)
    _check(_lib().turbofno_layer_norm_backward(kind, P, K, py, ldy, ps, lds, pg, pm, pt, pgs, ldgs, float(drop), pd, pr, ldr, px, ldx, po, pb, workspace.data_ptr(),
                                               workspace.numel(), _stream()))
    return gx, gr if drop else gx, ggain, gbias


def quantise_8bit(x, q=None, scale=None):
    """x in float8_e4m3fn with a float32 scale for each position and block of 128 channels, its largest magnitude over 448: (q, scale), what mix_8bit_blocks takes.
    scale has the shape [ceil(K / 128)][positions...]; q has a last dimension of two, (re, im), for complex fields."""
    if isinstance(x, torch.Tensor) and x.is_cuda and x.dim() >= 2:
        q, scale = _eight_results(x, q, scale)
        if _compiled("quantise_8bit", ("quantise_8bit",), x, q, scale):
            return q, scale
    kind, device, K, P = _input(x, "x")
    px, ldx = _field(x, "x", x.shape, x.dtype, device)
    q, scale = _eight_results(x, q, scale)
    pq, ldq, pc = _eight_fields(x, q, scale, device)
    _current(device)
    _check(_lib().turbofno_quantise_8bit(kind, P, K, px, ldx, pq, ldq, pc, _stream()))
    return q, scale


def mix_8bit_blocks(xq, xscale, Wq, wscale, bias=None, residual=None, activation="none", y=None, dtype=None):
    """mix from 8-bit operands with a scale for each block of 128 channels: x = xscale[k / 128][position] xq, W = wscale[n / 128][k / 128] Wq, all of float8_e4m3fn
    with float32 scales; xq and xscale as quantise_8bit and layer_norm_8bit give them. For the rest like mix_8bit."""
    if getattr(y, "is_cuda", False) and dtype in (None, y.dtype) and _compiled("mix_8bit_blocks", ("mix_8bit_blocks",), xq, xscale, Wq, wscale, bias, residual,
                                                                               _ACTIVATIONS.get(activation, -1), y):
        return y
    if dtype is None:
        dtype = next((t.dtype for t in (y, residual) if isinstance(t, torch.Tensor)), torch.bfloat16)
    kind = _type(dtype, "the result")
    act = _activation(activation)
    tail = (2,) if dtype == torch.complex64 else ()
    if not isinstance(xq, torch.Tensor) or not isinstance(Wq, torch.Tensor):
        raise TypeError("xq and Wq must be tensors")
    _need(xq.dim() >= 2 + len(tail) and xq.shape[0] > 0 and (not tail or xq.shape[-1] == 2), "xq must be [K][positions...]%s", "[2]" if tail else "")
    K, device = xq.shape[0], xq.device
    _need(Wq.dim() == 2 + len(tail) and Wq.shape[0] > 0 and tuple(Wq.shape[1:]) == (K,) + tail, "Wq must be [N][%d]%s", K, "[2]" if tail else "")
    N, places = Wq.shape[0], tuple(xq.shape[1:-1] if tail else xq.shape[1:])
    P = xq.numel() // (K * (2 if tail else 1))
    f8 = torch.float8_e4m3fn
    _on_gpu(xq, "xq", f8, device)
    ldx = _spread(xq, "xq", 2 if tail else 1)
    y = _result(y, (N,) + places, dtype, device)
    pr, ldr = _field(residual, "residual", (N,) + places, dtype, device)
    py, ldy = _field(y, "y", (N,) + places, dtype, device)
    pxs, pW = _packed(xscale, "xscale", (_blocks(K),) + places, torch.float32, device), _packed(Wq, "Wq", Wq.shape, f8, device)
    pws, pb = _packed(wscale, "wscale", (_blocks(N), _blocks(K)), torch.float32, device), _packed(bias, "bias", (N,), dtype, device)
    _current(device)
    _check(_lib().turbofno_mix_8bit_blocks(kind, P, N, K, xq.data_ptr(), ldx, pxs, pW, pws, pb, pr, ldr, act, py, ldy, _stream()))
    return y

def clip_grad_norm(grads, max_norm, out=None, norm=None, workspace=None):
    """The norm over all values of the tensors in `grads` (complex64, float32 and bfloat16, contiguous, in any mixture), as a float32 tensor of no
    dimensions on the GPU; each is scaled by min(1, max_norm / (norm + 1e-6)), into the tensor of the same place in `out`, or in place. A gradient that
    several parameters share is given once: results that overlap are refused."""
    grads = list(grads)
    out = grads if out is None else list(out)
    _need(len(out) == len(grads), "out has %d tensors, grads %d", len(out), len(grads))
    if grads and isinstance(grads[0], torch.Tensor) and grads[0].is_cuda:
        norm = _result(norm, (), torch.float32, grads[0].device)
        if _compiled("clip_grad_norm", ("clip_grad_norm", "clip_grad_norm_workspace_bytes"), grads, out, max_norm, norm, workspace):
            return norm
    device = grads[0].device if grads and isinstance(grads[0], torch.Tensor) else torch.device("cuda", torch.cuda.current_device())
    count = len(grads)
    kinds, sizes = (ctypes.c_int * count)(), (ctypes.c_long * count)()
    sources, results = (ctypes.c_void_p * count)(), (ctypes.c_void_p * count)()
    for i, (g, o) in enumerate(zip(grads, out)):
        if not isinstance(g, torch.Tensor):
            raise TypeError("grads[%d] must be a tensor" % i)
        kinds[i], sizes[i] = _type(g.dtype, "grads[%d]" % i), g.numel()
        sources[i] = _packed(g, "grads[%d]" % i, g.shape, g.dtype, device)
        results[i] = sources[i] if o is g else _packed(o, "out[%d]" % i, g.shape, g.dtype, device)
    norm = _result(norm, (), torch.float32, device)
    pn = _packed(norm, "norm", (), torch.float32, device)
    workspace = _workspace(workspace, _lib().turbofno_clip_grad_norm_workspace_bytes(count), device)
    _current(device)
    _check(_lib().turbofno_clip_grad_norm(count, sources, results, sizes, kinds, float(max_norm), pn, workspace.data_ptr(), workspace.numel(), _stream()))
    return norm
