"""The binding of the operators around the layer: the compiled checks (csrc/operands.cpp) against those in Python, and refusals without a GPU."""
import pytest
import torch

import turbofno_amd as tf
from turbofno_amd import api, operators

needs_module = pytest.mark.skipif(api._operands is None, reason="extension not built")
K, N, P = 12, 20, (3, 50)


def _operands(dt, device):
    gen = torch.Generator().manual_seed(3)
    new = lambda *s: torch.randn(s, dtype=torch.float32 if dt == torch.bfloat16 else dt, generator=gen).to(dt).to(device)  # noqa: E731
    real = lambda *s: torch.rand(s, generator=gen).to(device)  # noqa: E731
    pair = (2,) if dt.is_complex else ()
    eight = lambda *s: torch.randn(s + pair, generator=gen).to(torch.float8_e4m3fn).to(device)  # noqa: E731
    return dict(x=new(K, *P), W=new(N, K), bias=new(N), r=new(N, *P), y=new(N, *P), z=new(N, *P), xq=eight(K, *P), xs=real(*P), Wq=eight(N, K), ws=real(N),
                gy=new(N, *P), gz=new(N, *P), gx=new(K, *P), gW=new(N, K), gb=new(N), gain=real(K), s=new(K, *P), xr=new(K, *P), xy=new(K, *P),
                rstd=real(*P), q=eight(K, *P), ggain=real(K), norm=real())


def _forms(dt, device):
    """(name, call, results): every entry point, with operands right and wrong in one respect each"""
    o = _operands(dt, device)
    wide = torch.zeros((2 * K, 3, 100), dtype=dt, device=device)
    views = dict(every_other_channel=wide[::2, :, :50].contiguous()[:, :, :], apart=torch.zeros((K + 4,) + P, dtype=dt, device=device)[2:-2],
                 gap=wide[:K, :, :50], short=o["x"][:, :, :49], flat=o["x"].reshape(K, -1), host=o["x"].cpu(), other=o["x"].to(torch.float16 if not dt.is_complex else torch.complex128), none=None, text="x",
                 parameter=torch.nn.Parameter(o["x"]), channel_last=o["x"].permute(1, 2, 0).contiguous().permute(2, 0, 1))
    if dt.is_complex:
        views["conjugated"] = o["x"].conj()
    mix = lambda **k: tf.mix(**{**dict(x=o["x"], W=o["W"], bias=o["bias"], residual=o["r"], activation="silu", y=o["y"], z=o["z"]), **k})  # noqa: E731
    mix8 = lambda **k: tf.mix_8bit(**{**dict(xq=o["xq"], xscale=o["xs"], Wq=o["Wq"], wscale=o["ws"], bias=o["bias"], residual=o["r"], activation="relu", y=o["y"]), **k})  # noqa: E731
    back = lambda **k: tf.mix_backward(**{**dict(gy=o["gy"], x=o["x"], W=o["W"], z=o["z"], activation="gelu_tanh", gz=o["gz"], gx=o["gx"], gW=o["gW"], gbias=o["gb"]), **k})  # noqa: E731
    norm = lambda **k: tf.rms_norm(**{**dict(x=o["x"], gain=o["gain"], residual=o["xr"], y=o["xy"], s=o["s"], rstd=o["rstd"]), **k})  # noqa: E731
    norm8 = lambda **k: tf.rms_norm_8bit(**{**dict(x=o["x"], gain=o["gain"], residual=o["xr"], q=o["q"], scale=o["rstd"], s=o["s"]), **k})  # noqa: E731
    nback = lambda **k: tf.rms_norm_backward(**{**dict(gy=o["x"], s=o["s"], gain=o["gain"], rstd=o["rstd"], gs=o["xr"], gx=o["gx"], ggain=o["ggain"]), **k})  # noqa: E731
    clip = lambda **k: tf.clip_grad_norm(**{**dict(grads=[o["x"], o["W"], o["gain"]], max_norm=1.0, out=[o["gx"], o["gW"], o["ggain"]], norm=o["norm"]), **k})  # noqa: E731
    small = torch.zeros(4, dtype=torch.uint8, device=device)
    forms = [("mix", mix), ("mix_8bit", mix8), ("mix_backward", back), ("rms_norm", norm), ("rms_norm_8bit", norm8), ("rms_norm_backward", nback), ("clip", clip)]
    out = [(n, c) for n, c in forms]
    for name, v in views.items():
        out += [("mix x " + name, lambda v=v: mix(x=v)), ("mix_backward x " + name, lambda v=v: back(x=v)), ("rms_norm x " + name, lambda v=v: norm(x=v)),
                ("rms_norm_8bit residual " + name, lambda v=v: norm8(residual=v)), ("rms_norm_backward s " + name, lambda v=v: nback(s=v)),
                ("clip " + name, lambda v=v: clip(grads=[v, o["W"], o["gain"]]))]
    out += [("no bias", lambda: mix(bias=None)), ("no residual", lambda: mix(residual=None)), ("no z", lambda: mix(z=None)), ("no y", lambda: mix(y=None)),
            ("activation", lambda: mix(activation="tanh")), ("activation none", lambda: mix(activation=None)), ("W columns", lambda: mix(W=o["W"][:, :-1])),
            ("W rows apart", lambda: mix(W=torch.cat([o["W"], o["W"]], 1)[:, :K])), ("bias long", lambda: mix(bias=o["r"][0, 0])), ("y over x", lambda: mix(x=o["y"][:K])),
            ("residual is y", lambda: mix(residual=o["y"])), ("y text", lambda: mix(y="y")),
            ("8bit wscale", lambda: mix8(wscale=o["ws"][:-1])), ("8bit xscale", lambda: mix8(xscale=o["xs"][:, :-1])), ("8bit no y", lambda: mix8(y=None)),
            ("8bit float x", lambda: mix8(xq=o["x"])), ("8bit y type", lambda: mix8(y=o["y"].to(torch.complex128 if dt.is_complex else torch.float64))),
            ("backward without", lambda: back(activation="none")), ("backward no z", lambda: back(z=None)), ("backward no results", lambda: back(gz=None, gx=None, gW=None, gbias=None)),
            ("backward workspace", lambda: back(workspace=small)), ("backward float workspace", lambda: back(workspace=o["ws"])), ("backward gW", lambda: back(gW=o["gW"].t())),
            ("norm gain", lambda: norm(gain=o["gain"][:-1])), ("norm no gain", lambda: norm(gain=None)), ("norm eps", lambda: norm(eps=-1)), ("norm eps text", lambda: norm(eps="a")),
            ("norm no residual", lambda: norm(residual=None)), ("norm no results", lambda: norm(y=None, s=None, rstd=None)), ("norm in place", lambda: norm(s=o["xr"])),
            ("norm rstd", lambda: norm(rstd=o["rstd"].t())), ("norm 8bit q", lambda: norm8(q=o["xy"])), ("norm 8bit no residual", lambda: norm8(residual=None, s=None)),
            ("norm backward no gs", lambda: nback(gs=None)), ("norm backward workspace", lambda: nback(workspace=small)), ("norm backward no results", lambda: nback(gx=None, ggain=None)),
            ("clip in place", lambda: clip(out=None)), ("clip out", lambda: clip(out=[o["gx"]])), ("clip negative", lambda: clip(max_norm=-1.0)), ("clip norm text", lambda: clip(max_norm="a")),
            ("clip tuple", lambda: clip(grads=(o["x"], o["W"], o["gain"]))), ("clip nothing", lambda: clip(grads=[], out=[])), ("clip workspace", lambda: clip(workspace=small)),
            ("clip strided", lambda: clip(grads=[o["x"], o["W"].t().contiguous().t(), o["gain"]]))]
    assert len(dict(out)) == len(out)
    return out


def _outcome(call):
    try:
        got = call()
        got = got if isinstance(got, tuple) else (got,)
        return "returned", tuple(t.float().cpu() if t.dtype == torch.float8_e4m3fn else t.detach().cpu().clone() for t in got)
    except Exception as e:
        return type(e), str(e)


def _compare(dt, device, monkeypatch):
    fresh = lambda name: dict(_forms(dt, device))[name]  # noqa: E731   (results of one form are operands of others)
    for name, _ in _forms(dt, device):
        print("form", dt, name, flush=True)
        with_module = _outcome(fresh(name))
        with monkeypatch.context() as m:
            m.setattr(api, "_operands", None)
            without = _outcome(fresh(name))
        assert with_module[0] == without[0], (name, with_module, without)
        if with_module[0] == "returned":
            assert all(torch.equal(a.nan_to_num() if a.is_floating_point() else a, b.nan_to_num() if b.is_floating_point() else b)
                       for a, b in zip(with_module[1], without[1])), name
        else:
            assert with_module[1] == without[1], name


@needs_module
@pytest.mark.parametrize("dt", [torch.complex64, torch.float32, torch.bfloat16])
def test_same_refusals_without_a_gpu(dt, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)        # asked for before an operand is looked at
    _compare(dt, "cpu", monkeypatch)


@needs_module
@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.complex64, torch.float32, torch.bfloat16])
def test_same_forms_taken_and_refused(dt, monkeypatch):
    _compare(dt, "cuda", monkeypatch)


@needs_module
@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.complex64, torch.float32, torch.bfloat16])
def test_module_takes_the_plain_calls(dt, monkeypatch):
    """the short way is the one that runs"""
    taken = []
    compiled = operators._compiled
    monkeypatch.setattr(operators, "_compiled", lambda call, *a: taken.append((call, compiled(call, *a))) or taken[-1][1])
    for name, call in _forms(dt, "cuda")[:7]:
        call()
    assert [c for c, ok in taken] == ["mix", "mix_8bit", "mix_backward", "rms_norm", "rms_norm", "rms_norm_backward", "clip_grad_norm"]
    assert all(ok for _, ok in taken)


def test_refusals_without_a_gpu():
    x, W = torch.zeros(4, 10), torch.zeros(6, 4)
    with pytest.raises(TypeError, match="on the GPU"):
        tf.mix(x, W)
    with pytest.raises(ValueError, match="one column per channel"):
        tf.mix(x, W.t())
    with pytest.raises(TypeError, match="float64"):
        tf.rms_norm(x.double(), torch.ones(4))
    with pytest.raises(ValueError, match="channels"):
        tf.mix(x[0], W)
    L = operators._lib()
    # refused before any GPU call; the pointers are never looked at
    assert L.turbofno_mix(7, 10, 6, 4, 1, 10, 1, None, None, 0, 0, None, 0, 1, 10, None) == 1 and b"type" in L.turbofno_last_error_string()
    assert L.turbofno_mix(0, -1, 6, 4, 1, 10, 1, None, None, 0, 0, None, 0, 1, 10, None) == 1
    assert L.turbofno_mix(0, 10, 6, 4, 1, 9, 1, None, None, 0, 0, None, 0, 1, 10, None) == 1 and b"between channels" in L.turbofno_last_error_string()
    assert L.turbofno_mix(0, 10, 70000, 4, 1, 10, 1, None, None, 0, 0, None, 0, 1, 10, None) == 2
    assert L.turbofno_mix(0, 0, 6, 4, None, 0, None, None, None, 0, 0, None, 0, None, 0, None) == 1 and b"W is null" in L.turbofno_last_error_string()
    assert L.turbofno_rms_norm(1, 10, 4, 1, 10, None, 0, None, 1e-6, None, 0, 1, 10, None, None) == 1 and b"gain" in L.turbofno_last_error_string()
    assert L.turbofno_clip_grad_norm(-1, None, None, None, None, 1.0, 1, 1, 1 << 20, None) == 1
    assert L.turbofno_clip_grad_norm(0, None, None, None, None, 1.0, 1, None, 0, None) == 3
    assert tf.mix_weight_grad_workspace_bytes(64, 64, 1 << 20, torch.complex64) > 0
    assert tf.rms_norm_backward_workspace_bytes(64, 1 << 20, torch.bfloat16) > 0
