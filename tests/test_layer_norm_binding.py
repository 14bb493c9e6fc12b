"""The binding of layer norm, dropout and the 8-bit operators with scales by blocks: the compiled checks (csrc/operands.cpp) against those in Python, refusals without a GPU,
and which operands may share memory."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import TYPES
from turbofno_amd import api, operators

needs_module = pytest.mark.skipif(api._operands is None, reason="extension not built")
K, N, P = 140, 20, (3, 50)
BASE = 1 << 32                          # an address, for calls that are refused
INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3


def _operands(dt, device):
    gen = torch.Generator().manual_seed(3)
    wide_type = torch.complex64 if dt.is_complex else torch.float32
    new = lambda *s, t=dt: torch.randn(s, dtype=torch.float32 if t == torch.bfloat16 else t, generator=gen).to(t).to(device)  # noqa: E731
    real = lambda *s: torch.rand(s, generator=gen).to(device)  # noqa: E731
    pair = (2,) if dt.is_complex else ()
    eight = lambda *s: torch.randn(s + pair, generator=gen).to(torch.float8_e4m3fn).to(device)  # noqa: E731
    return dict(x=new(K, *P), r=new(K, *P), s=new(K, *P), y=new(K, *P), gy=new(K, *P), gx=new(K, *P), gr=new(K, *P), gain=real(K), bias=new(K, t=wide_type),
                mean=new(*P, t=wide_type), rstd=real(*P), rng=torch.tensor([3, 4]).to(device), q=eight(K, *P), scale=real(2, *P), ggain=real(K),
                gbias=new(K, t=wide_type), Wq=eight(N, K), wscale=real(1, 2), b=new(N), nr=new(N, *P), ny=new(N, *P))


def _forms(dt, device):
    """(name, call): every entry point, with operands right and wrong in one respect each"""
    o = _operands(dt, device)
    wide = torch.zeros((2 * K, 3, 100), dtype=dt, device=device)
    views = dict(gap=wide[:K, :, :50], short=o["x"][:, :, :49], flat=o["x"].reshape(K, -1), host=o["x"].cpu(), apart=torch.zeros((K + 4,) + P, dtype=dt, device=device)[2:-2],
                 other=o["x"].to(torch.float16 if not dt.is_complex else torch.complex128), none=None, text="x", parameter=torch.nn.Parameter(o["x"]),
                 channel_last=o["x"].permute(1, 2, 0).contiguous().permute(2, 0, 1))
    if dt.is_complex:
        views["conjugated"] = o["x"].conj()
    call = lambda f, **base: lambda **k: f(**{**base, **k})  # noqa: E731
    drop = call(tf.dropout, x=o["x"], drop=0.5, rng=o["rng"], residual=o["r"], y=o["y"])
    norm = call(tf.layer_norm, x=o["x"], gain=o["gain"], bias=o["bias"], residual=o["r"], drop=0.5, rng=o["rng"], y=o["y"], s=o["s"], mean=o["mean"], rstd=o["rstd"])
    norm8 = call(tf.layer_norm_8bit, x=o["x"], gain=o["gain"], bias=o["bias"], residual=o["r"], q=o["q"], scale=o["scale"], s=o["s"])
    back = call(tf.layer_norm_backward, gy=o["gy"], s=o["s"], gain=o["gain"], mean=o["mean"], rstd=o["rstd"], gs=o["r"], drop=0.5, rng=o["rng"], gx=o["gx"], gr=o["gr"],
                ggain=o["ggain"], gbias=o["gbias"])
    quantise = call(tf.quantise_8bit, x=o["x"], q=o["q"], scale=o["scale"])
    mix = call(tf.mix_8bit_blocks, xq=o["q"], xscale=o["scale"], Wq=o["Wq"], wscale=o["wscale"], bias=o["b"], residual=o["nr"], activation="silu", y=o["ny"])
    out = [("dropout", drop), ("layer_norm", norm), ("layer_norm_8bit", norm8), ("layer_norm_backward", back), ("quantise", quantise), ("mix", mix)]
    for name, v in views.items():
        for form, args in ((("dropout", drop), ("x", "residual", "y")), (("layer_norm", norm), ("x", "residual", "s", "y")), (("layer_norm_8bit", norm8), ("x", "s")),
                           (("layer_norm_backward", back), ("gy", "s", "gs", "gx", "gr")), (("quantise", quantise), ("x",))):
            out += [("%s %s %s" % (form[0], a, name), lambda f=form[1], a=a, v=v: f(**{a: v})) for a in args]
    small = torch.zeros(4, dtype=torch.uint8, device=device)
    for value in (0.0, 1.0, -0.1, float("nan"), "a", None, 1 - 2.0 ** -40):
        out += [("dropout drop %s" % value, lambda v=value: drop(drop=v)), ("layer_norm drop %s" % value, lambda v=value: norm(drop=v)), ("back drop %s" % value, lambda v=value: back(drop=v))]
    for value in (None, o["rng"].int(), o["rng"][:1], torch.stack([o["rng"], o["rng"]]).t()[0], o["rng"].cpu(), 7):
        label = type(value).__name__ + str(len(out))
        out += [("dropout rng " + label, lambda v=value: drop(rng=v)), ("norm rng " + label, lambda v=value: norm(rng=v)), ("norm rng, no drop " + label, lambda v=value: norm(rng=v, drop=0.0)),
                ("back rng " + label, lambda v=value: back(rng=v))]
    for name, values in (("gain", (None, o["gain"][:-1], o["gain"].double(), "g")), ("bias", (None, o["bias"][:-1], o["bias"].double() if not dt.is_complex else o["gain"])),
                         ("mean", (None, o["mean"].t(), o["mean"][:, :-1])), ("rstd", (None, o["rstd"].t(), o["rstd"].double()))):
        for i, v in enumerate(values):
            out += [("norm %s %d" % (name, i), lambda n=name, v=v: norm(**{n: v}))]
            if name != "bias":
                out += [("back %s %d" % (name, i), lambda n=name, v=v: back(**{n: v}))]
            if name in ("gain", "bias"):
                out += [("norm8 %s %d" % (name, i), lambda n=name, v=v: norm8(**{n: v}))]
    out += [("norm eps", lambda: norm(eps=-1)), ("norm eps text", lambda: norm(eps="a")), ("norm no results", lambda: norm(y=None, s=None, mean=None, rstd=None)),
            ("norm plain", lambda: norm(residual=None, drop=0.0, s=None, rng=None, bias=None)), ("norm in place", lambda: norm(s=o["r"], y=o["x"])),
            ("norm results one", lambda: norm(s=o["y"])), ("norm8 no results", lambda: norm8(q=None, scale=None, s=None)), ("norm8 scale", lambda: norm8(scale=o["scale"][:1])),
            ("norm8 q", lambda: norm8(q=o["y"])), ("quantise no results", lambda: quantise(q=None, scale=None)), ("quantise scale", lambda: quantise(scale=o["scale"][:, :, :-1])),
            ("back no results", lambda: back(gx=None, gr=None, ggain=None, gbias=None)), ("back plain", lambda: back(drop=0.0, rng=None, gs=None)), ("back workspace", lambda: back(workspace=small)),
            ("back float workspace", lambda: back(workspace=o["rstd"])), ("back ggain", lambda: back(ggain=o["ggain"][:-1])), ("back gbias", lambda: back(gbias=o["gbias"][:-1])),
            ("back one result", lambda: back(gr=o["gx"])), ("mix no y", lambda: mix(y=None)), ("mix y type", lambda: mix(y=o["ny"].to(torch.complex128 if dt.is_complex else torch.float64))),
            ("mix wscale", lambda: mix(wscale=o["wscale"].t())), ("mix xscale", lambda: mix(xscale=o["scale"][:1])), ("mix float x", lambda: mix(xq=o["x"])),
            ("mix W columns", lambda: mix(Wq=o["Wq"][:, :-1])), ("mix bias", lambda: mix(bias=o["b"][:-1])), ("mix residual is y", lambda: mix(residual=o["ny"])),
            ("mix activation", lambda: mix(activation="tanh")), ("mix nothing", lambda: mix(bias=None, residual=None, dtype=dt, y=None)), ("mix W none", lambda: mix(Wq=None)),
            ("mix dtype", lambda: mix(dtype=torch.float64)), ("mix W vector", lambda: mix(Wq=o["Wq"].flatten()))]
    assert len(dict(out)) == len(out)
    return out


def _outcome(call):
    try:
        got = call()
        got = got if isinstance(got, tuple) else (got,)
        return "returned", tuple(t.float().cpu() if t.dtype == torch.float8_e4m3fn else t.detach().cpu().clone() for t in got)
    except Exception as e:
        return type(e), str(e)


def _same(a, b):
    if a.is_complex():
        a, b = torch.view_as_real(a), torch.view_as_real(b)
    return torch.equal(a.nan_to_num(), b.nan_to_num()) and torch.equal(torch.isnan(a), torch.isnan(b))


def _compare(dt, device, monkeypatch):
    for name, call in _forms(dt, device):
        print("form", dt, name, flush=True)
        fresh = dict(_forms(dt, device))                # results of one form are operands of others
        with_module = _outcome(fresh[name])
        fresh = dict(_forms(dt, device))
        with monkeypatch.context() as m:
            m.setattr(api, "_operands", None)
            without = _outcome(fresh[name])
        assert with_module[0] == without[0], (name, with_module, without)
        if with_module[0] == "returned":
            # what is allocated and not written does not stand in any result
            assert all(_same(a, b) for a, b in zip(with_module[1], without[1])), name
        else:
            assert with_module[1] == without[1], name


@needs_module
@pytest.mark.parametrize("dt", TYPES.values())
def test_same_refusals_without_a_gpu(dt, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)        # asked for before an operand is looked at
    _compare(dt, "cpu", monkeypatch)


@needs_module
@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES.values())
def test_same_forms_taken_and_refused(dt, monkeypatch):
    _compare(dt, "cuda", monkeypatch)


@needs_module
@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES.values())
def test_module_takes_the_plain_calls(dt, monkeypatch):
    """the short way is the one that runs, with results passed and without, with and without what is optional"""
    taken = []
    compiled = operators._compiled
    monkeypatch.setattr(operators, "_compiled", lambda call, *a: taken.append((call, compiled(call, *a))) or taken[-1][1])
    forms = dict(_forms(dt, "cuda"))
    names = ["dropout", "layer_norm", "layer_norm_8bit", "layer_norm_backward", "quantise", "mix", "norm no results", "norm plain", "back no results", "back plain", "norm8 no results",
             "quantise no results"]
    for name in names:
        forms[name]()
    assert len(taken) == len(names) and all(ok for _, ok in taken), taken


def test_refusals_of_the_library():
    """before any GPU call; the pointers are never looked at"""
    L = operators._lib()
    says = lambda rc, code, text: rc == code and text in L.turbofno_last_error_string()  # noqa: E731
    x, r, s, y, gain, bias, rng, mean, rstd, gy, gs, gx, gr, og, ob, ws = (BASE + (i << 20) for i in range(16))

    def norm(type=1, P=10, K=4, **k):
        o = {**dict(x=x, ldx=10, r=r, gain=gain, bias=bias, eps=1e-6, drop=0.5, rng=rng, s=s, y=y, ldy=10, mean=mean, rstd=rstd), **k}
        return L.turbofno_layer_norm(type, P, K, o["x"], o["ldx"], o["r"], 10, o["gain"], o["bias"], o["eps"], o["drop"], o["rng"], o["s"], 10, o["y"], o["ldy"], o["mean"], o["rstd"], None)
    assert says(norm(type=7), INVALID, b"type") and says(norm(P=-1), INVALID, b"positions") and says(norm(K=70000), UNSUPPORTED, b"70000") and says(norm(K=0), INVALID, b"positive")
    assert says(norm(x=None), INVALID, b"x is null") and says(norm(gain=None), INVALID, b"gain is null") and says(norm(ldx=9), INVALID, b"between channels") and says(norm(y=None), INVALID, b"y is null")
    for drop in (1.0, -0.5, float("nan"), float("inf")):
        assert says(norm(drop=drop), INVALID, b"drop")
    assert says(norm(rng=None), INVALID, b"rng is null") and says(norm(eps=-1.0), INVALID, b"eps") and says(norm(eps=float("nan")), INVALID, b"eps")
    assert says(norm(s=y), INVALID, b"results overlap") and says(norm(s=x + 4), INVALID, b"without being it") and says(norm(y=r, ldy=11), INVALID, b"without being it")
    for name in ("gain", "bias", "rng"):
        assert says(norm(**{name: y + 156}), INVALID, b"gain, bias or rng") and says(norm(**{name: s}), INVALID, b"gain, bias or rng")
    for name in ("mean", "rstd"):
        for place in (x + 156, r, s + 4, y, gain + 12, bias, rng, mean if name == "rstd" else rstd + 36):
            assert says(norm(**{name: place}), INVALID, b"mean or rstd overlaps"), (name, place)

    def norm8(**k):
        o = {**dict(q=y, scale=rstd, s=s, gain=gain, bias=bias), **k}
        return L.turbofno_layer_norm_8bit(1, 10, 130, x, 10, r, 10, o["gain"], o["bias"], 1e-6, o["s"], 10, o["q"], 10, o["scale"], None)
    assert says(norm8(q=x + 5199), INVALID, b"without being it") and says(norm8(q=x), INVALID, b"without being it") and says(norm8(scale=None), INVALID, b"scale is null")
    assert says(norm8(scale=gain - 76), INVALID, b"scale overlaps") and says(norm8(scale=y + 1299), INVALID, b"scale overlaps") and says(norm8(q=s + 4), INVALID, b"results overlap")

    need = L.turbofno_layer_norm_backward_workspace_bytes(1, 10, 4)

    def back(**k):
        o = {**dict(gy=gy, s=s, gain=gain, mean=mean, rstd=rstd, gs=gs, drop=0.5, rng=rng, gr=gr, gx=gx, og=og, ob=ob, ws=ws, bytes=need), **k}
        return L.turbofno_layer_norm_backward(1, 10, 4, o["gy"], 10, o["s"], 10, o["gain"], o["mean"], o["rstd"], o["gs"], 10, o["drop"], o["rng"], o["gr"], 10, o["gx"], 10, o["og"], o["ob"],
                                              o["ws"], o["bytes"], None)
    for name, text in (("gy", b"gy is null"), ("s", b"s is null"), ("gain", b"gain is null"), ("mean", b"mean is null"), ("rstd", b"rstd is null"), ("gr", b"gr is null"), ("gx", b"gx is null"),
                       ("og", b"ggain is null"), ("rng", b"rng is null"), ("ws", b"workspace")):
        assert says(back(**{name: None}), WORKSPACE if name == "ws" else INVALID, text), name
    assert says(back(bytes=need - 1), WORKSPACE, b"are needed") and says(back(bytes=4, gr=None, drop=0.0), WORKSPACE, b"are needed")
    assert says(back(gx=gr + 156), INVALID, b"gx and gr overlap") and says(back(gx=gy + 4), INVALID, b"without being it") and says(back(gr=s - 4), INVALID, b"without being it")
    assert says(back(gx=gy, gr=gs, bytes=0), WORKSPACE, b"are needed")
    for name in ("gain", "mean", "rstd", "rng", "og", "ob"):
        for place in (gx + 152, gr):
            assert says(back(**{name: place}), INVALID, b"gx or gr overlaps"), name
    assert says(back(ob=og + 12), INVALID, b"ggain and gbias")
    for place in (gy, s, gs, gx, gr, gain, mean, rstd, rng, og, ob):
        assert says(back(ws=place), INVALID, b"workspace overlaps"), place

    def dropout(**k):
        o = {**dict(x=x, r=r, drop=0.5, rng=rng, y=y, ldy=10), **k}
        return L.turbofno_dropout(1, 10, 4, o["x"], 10, o["r"], 10, o["drop"], o["rng"], o["y"], o["ldy"], None)
    assert says(dropout(drop=1.0), INVALID, b"drop") and says(dropout(rng=None, drop=0.0), INVALID, b"rng is null") and says(dropout(y=x, ldy=12), INVALID, b"without being it")
    assert says(dropout(y=r + 4), INVALID, b"without being it") and says(dropout(rng=y + 144), INVALID, b"overlaps rng")

    def quantise(**k):
        o = {**dict(x=x, q=y, scale=rstd), **k}
        return L.turbofno_quantise_8bit(0, 10, 130, o["x"], 10, o["q"], 10, o["scale"], None)
    assert says(quantise(q=x + 8), INVALID, b"overlap") and says(quantise(scale=x), INVALID, b"overlap") and says(quantise(scale=y + 2599), INVALID, b"overlap") and says(quantise(scale=None), INVALID, b"null")
    assert says(quantise(scale=y - 76), INVALID, b"overlap")

    def mix(**k):
        o = {**dict(x=x, xs=mean, W=gain, ws=rstd, bias=bias, r=r, act=0, y=y, ldy=10), **k}
        return L.turbofno_mix_8bit_blocks(1, 10, 6, 130, o["x"], 10, o["xs"], o["W"], o["ws"], o["bias"], o["r"], 10, o["act"], o["y"], o["ldy"], None)
    assert says(mix(act=9), INVALID, b"activation") and says(mix(xs=None), INVALID, b"xscale is null") and says(mix(ws=None), INVALID, b"wscale is null") and says(mix(W=None), INVALID, b"Wq is null")
    assert says(mix(y=x + 1299), INVALID, b"overlaps xq") and says(mix(y=r, ldy=11), INVALID, b"without being it")
    assert all(says(mix(**{name: y + 236}), INVALID, b"a scale") for name in ("W", "bias", "xs", "ws")) and says(mix(xs=y - 76), INVALID, b"a scale") and says(mix(W=y - 779), INVALID, b"a scale")


def test_refusals_in_python():
    x, rng = torch.zeros(4, 10), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(TypeError, match="on the GPU"):
        tf.dropout(x, 0.5, rng)
    with pytest.raises(TypeError, match="float64"):
        tf.layer_norm(x.double(), torch.ones(4))
    with pytest.raises(ValueError, match="channels"):
        tf.quantise_8bit(x[0])
    with pytest.raises(TypeError, match="tensors"):
        tf.mix_8bit_blocks(None, None, None, None)
    assert tf.layer_norm_backward_workspace_bytes(64, 1 << 20, torch.bfloat16) > 0
