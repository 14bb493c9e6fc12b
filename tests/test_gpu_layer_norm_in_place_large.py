"""Layer norm in place where a launch has several rows of blocks and strips lie side by side on an XCD: the residual replaced by the sum, x by the result, once each."""
import pytest
import torch

import turbofno_amd as tf
from operators_reference import randn
from test_gpu_layer_norm import rng_of

pytestmark = pytest.mark.gpu

# more than 2^22 strips of 256 real columns, in rows that do not end with a cache line
SIZES = [("bf16", 2, (1 << 31) + 333), ("c64", 3, (1 << 29) + 5)]


@pytest.mark.parametrize("kind,K,P", SIZES)
@pytest.mark.parametrize("form", ["norm", "dropout", "8bit"])
def test_once_each(kind, K, P, form):
    dt = torch.complex64 if kind == "c64" else torch.bfloat16
    wide = torch.complex64 if kind == "c64" else torch.float32
    gain, bias = 1 + 0.2 * randn((K,), torch.float32, 5), randn((K,), wide, 6)
    x, r = torch.empty((K, P), dtype=dt, device="cuda"), torch.empty((K, P), dtype=dt, device="cuda")
    step = 1 << 25
    for a in range(0, P, step):                         # patterns whose periods share nothing with strips
        n = min(step, P - a)
        t = torch.arange(a, a + n, device="cuda")
        for k in range(K):
            x[k, a:a + n] = ((t + 31 * k) % 1009).to(torch.float32) * 0.01 - 3
            r[k, a:a + n] = ((t + 17 * k) % 997).to(torch.float32) * 0.02 + 1
    parts = [slice(p, p + 5000) for p in (0, (1 << 28) - 77, P // 8 - 2000, P // 2 - 999, 5 * P // 8, P - 5000)]
    rng = rng_of()
    before = [(x[:, p].clone(), r[:, p].clone()) for p in parts]
    if form == "8bit":
        q, scale, s = tf.layer_norm_8bit(x, gain, bias, r, s=r)
    else:
        y, s, mean, rstd = tf.layer_norm(x, gain, bias, r, drop=0.3 if form == "dropout" else 0.0, rng=rng if form == "dropout" else None, s=r, y=x)
        assert y is x
    assert s is r
    # every position: the sum of what was there is a function of its place
    for a in range(0, P, step):
        n = min(step, P - a)
        t = torch.arange(a, a + n, device="cuda")
        for k in range(K):
            one = (((t + 31 * k) % 1009).to(torch.float32) * 0.01 - 3).to(dt)
            two = (((t + 17 * k) % 997).to(torch.float32) * 0.02 + 1).to(dt)
            if form == "dropout":                       # dropped, or lifted: the factor, the product and the sum round in fp32, then the result
                lifted = one.to(wide) / 0.7 + two.to(wide)
                off = torch.finfo(torch.float32 if kind == "c64" else dt).eps / 2 * 1.01 * lifted.abs() + 4 * 2.0 ** -24 * (one.abs().float() / 0.7 + two.abs().float())
                assert (((s[k, a:a + n].to(wide) - lifted).abs() <= off) | (s[k, a:a + n] == two)).all(), (a, k)
            else:
                assert torch.equal(s[k, a:a + n], (one.to(wide) + two.to(wide)).to(dt)), (a, k)
    if form != "dropout":
        for p, (one, two) in zip(parts, before):
            if form == "8bit":
                want = tf.layer_norm_8bit(one, gain, bias, two)
                assert torch.equal(q[:, p].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scale[:, p], want[1])
            else:
                want = tf.layer_norm(one, gain, bias, two)
                assert torch.equal(x[:, p], want[0]) and torch.equal(mean[p], want[2]) and torch.equal(rstd[p], want[3])
    del x, r, s
    torch.cuda.empty_cache()
