"""The kernels that the size rules of the layer norm and its gradient choose between, each at sizes that reach it, with and without a last strip that is not whole."""
import pytest
import torch

import turbofno_amd as tf
from layer_norm_reference import Backward, Forward, check_eight, rounded, within
from operators_reference import TYPES, randn
from test_gpu_layer_norm import SEED, operands, rng_of

pytestmark = pytest.mark.gpu

# channels and real columns: 32, 64, 128, 256, 512, 1024 and 2048 channels are held by one kernel or another; 2^17, 2^16, 8192, 4096 and 1024 columns part them; persistent
# blocks take several strips from 2^15 on
SIZES = [(20, 131080), (50, 131072), (50, 200003), (40, 1001), (100, 5002), (200, 6016), (100, 70001), (200, 65536), (400, 4004), (400, 9002), (400, 40007), (700, 1000), (700, 4002),
         (700, 9007), (1500, 3000), (1500, 5008), (2500, 902), (2500, 9008), (2500, 5003), (2100, 33001)]
CASES = [(kind, K, columns) for kind in TYPES for K, columns in SIZES]


def places(kind, columns):
    return (columns // (2 if kind == "c64" else 1),)


@pytest.mark.parametrize("kind,K,columns", CASES)
def test_forward(kind, K, columns):
    x, gain, bias, r = operands(kind, K, places(kind, columns), 1)
    for drop in (0.0, 0.3):
        y, s, mean, rstd = tf.layer_norm(x, gain, bias, r, drop=drop, rng=rng_of() if drop else None)
        E = Forward(x, gain, bias, r, drop=drop, rng=SEED)
        assert E.meaningful
        within(s, E.s, rounded(E.s, E.s_off, x.dtype), "s")
        within(mean, E.mean, E.mean_off, "mean")
        within(rstd, E.rstd, E.rstd_off, "rstd")
        within(y, E.y, rounded(E.y, E.y_off, x.dtype), "y")
        place = r.clone()
        assert torch.equal(tf.layer_norm(x, gain, bias, place, drop=drop, rng=rng_of() if drop else None, s=place)[0], y) and torch.equal(place, s)


@pytest.mark.parametrize("kind,K,columns", CASES)
def test_8bit(kind, K, columns):
    x, gain, bias, r = operands(kind, K, places(kind, columns), 2)
    q, scale, s = tf.layer_norm_8bit(x, gain, bias, r)
    E = Forward(x, gain, bias, r)
    check_eight(q, scale, E.y, E.y_off, "layer_norm_8bit")
    within(s, E.s, rounded(E.s, E.s_off, x.dtype), "s")


@pytest.mark.parametrize("kind,K,columns", CASES)
def test_gradient(kind, K, columns):
    x, gain, bias, gs = operands(kind, K, places(kind, columns), 3)
    gy = randn(x.shape, x.dtype, 12)
    _, s, mean, rstd = tf.layer_norm(x, gain, bias)
    for drop in (0.0, 0.3):
        run = lambda **k: tf.layer_norm_backward(gy, s, gain, mean, rstd, gs=gs, drop=drop, rng=rng_of() if drop else None, **k)  # noqa: E731
        gx, gr, ggain, gbias = run()
        E = Backward(gy, s, gain, mean, rstd, gs, drop, SEED)
        within(gr, E.gr, rounded(E.gr, E.gr_off, x.dtype), "gr")
        within(gx, E.gx, rounded(E.gx, E.gx_off, x.dtype), "gx")
        within(ggain, E.ggain, E.ggain_off, "ggain")
        within(gbias, E.gbias, E.gbias_off, "gbias")
        again = run()                                   # sums in a fixed order
        assert torch.equal(again[2], ggain) and torch.equal(again[3], gbias) and torch.equal(again[0], gx)
        del again, E


@pytest.mark.parametrize("form", ["norm", "8bit", "quantise", "gradient"])
def test_more_strips_than_a_launch_of_one_row_has_threads(form):
    """two channels of more than 2^31 positions: blocks behind the first 2^32 threads, offsets behind 2^32 bytes; the last positions against a call for them alone"""
    K, P, dt = 2, (1 << 31) + 333, torch.bfloat16
    x = torch.empty((K, P), dtype=dt, device="cuda")
    step = 1 << 28
    for a in range(0, P, step):                         # a pattern whose period shares nothing with strips
        part = x[:, a:a + step]
        part.copy_((torch.arange(a, a + part.shape[1], device="cuda") % 1009).to(torch.float32)[None] * torch.tensor([[0.01], [-0.003]], device="cuda") + 0.5)
    gain, bias = 1 + 0.2 * randn((K,), torch.float32, 5), randn((K,), torch.float32, 6)
    parts = [slice(0, 4096), slice((1 << 30) - 77, (1 << 30) + 1000), slice(P - 5000, P)]
    if form == "norm":
        y = torch.empty_like(x)
        _, _, mean, rstd = tf.layer_norm(x, gain, bias, y=y)
        for p in parts:
            want = tf.layer_norm(x[:, p].contiguous(), gain, bias)
            assert torch.equal(y[:, p], want[0]) and torch.equal(mean[p], want[2]) and torch.equal(rstd[p], want[3])
    elif form == "gradient":
        mean, rstd = torch.zeros(P, device="cuda"), torch.ones(P, device="cuda")
        gx = tf.layer_norm_backward(x, x, gain, mean, rstd)[0]
        for p in parts:
            assert torch.equal(gx[:, p], tf.layer_norm_backward(x[:, p].contiguous(), x[:, p].contiguous(), gain, mean[p].contiguous(), rstd[p].contiguous())[0])
    else:
        run = (lambda t: tf.layer_norm_8bit(t, gain, bias)[:2]) if form == "8bit" else tf.quantise_8bit
        q, scale = run(x)
        for p in parts:
            want = run(x[:, p].contiguous())
            assert torch.equal(q[:, p].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scale[:, p], want[1])
    del x
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind", TYPES)
def test_on_two_streams_at_once(kind):
    """forward and backward of two fields beside one another, each the result that it gives alone"""
    sets = [operands(kind, K, places(kind, columns), 70 + K) for K, columns in ((50, 131072), (400, 9002))]

    def step(x, gain, bias, r):
        y, s, mean, rstd = tf.layer_norm(x, gain, bias, r, drop=0.1, rng=rng)
        return (y, s) + tf.layer_norm_backward(y, s, gain, mean, rstd, gs=x, drop=0.1, rng=rng)
    rng = rng_of()
    want = [step(*o) for o in sets]
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for turn in range(3):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got.append((i, step(*sets[i])))
    torch.cuda.synchronize()
    for i, result in got:
        assert all(torch.equal(a, b) for a, b in zip(result, want[i]))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("K", [20, 50, 130])
def test_dropout_of_channels_far_apart(kind, K):
    """channels 2^25 values apart and more, where a lane's offset in a narrow strip would pass 32 bits"""
    dt, P = TYPES[kind], 300
    step = (1 << 25) + 13
    x, gain, bias, gs = operands(kind, K, (P,), 90)
    far = torch.empty((K - 1) * step + P, dtype=dt, device="cuda").as_strided((K, P), (step, 1))
    far.copy_(x)
    y, s, mean, rstd = tf.layer_norm(far, gain, bias, gs, drop=0.3, rng=rng_of())
    E = Forward(x, gain, bias, gs, drop=0.3, rng=SEED)
    within(s, E.s, rounded(E.s, E.s_off, dt), "s")
    within(y, E.y, rounded(E.y, E.y_off, dt), "y")
    gy = randn((K, P), dt, 91)
    far.copy_(s)
    gx, gr, ggain, gbias = tf.layer_norm_backward(gy, far, gain, mean, rstd, gs=gs, drop=0.3, rng=rng_of(), gx=far)
    E = Backward(gy, s, gain, mean, rstd, gs, 0.3, SEED)
    within(gr, E.gr, rounded(E.gr, E.gr_off, dt), "gr")
    within(gx, E.gx, rounded(E.gx, E.gx_off, dt), "gx")
    within(ggain, E.ggain, E.ggain_off, "ggain")
    within(gbias, E.gbias, E.gbias_off, "gbias")
    del far, gx
    torch.cuda.empty_cache()


@pytest.mark.parametrize("kind,K,columns", [(kind, K, columns) for kind in TYPES for K, columns in ((40, 1001), (200, 65537), (2500, 5003))])
def test_one_tensor_for_two_operands(kind, K, columns):
    """x its own residual, the gradient of y that of s too: what copies of them give"""
    x, gain, bias, _ = operands(kind, K, places(kind, columns), 100)
    want = tf.layer_norm(x, gain, bias, x.clone(), drop=0.2, rng=rng_of())
    got = tf.layer_norm(x, gain, bias, x, drop=0.2, rng=rng_of())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    back = lambda gs: tf.layer_norm_backward(x, want[1], gain, want[2], want[3], gs=gs, drop=0.2, rng=rng_of())  # noqa: E731
    assert all(torch.equal(a, b) for a, b in zip(back(x), back(x.clone())))
    assert torch.equal(tf.dropout(x, 0.2, rng_of(), residual=x), tf.dropout(x, 0.2, rng_of(), residual=x.clone()))


def test_two_graphs_in_turns():
    """two captured gradients of other sizes, each with its workspace, replayed in turns beside eager calls: the eager results"""
    sets = []
    for K, columns, seed in ((200, 30011, 110), (2500, 5003, 120)):
        x, gain, bias, gs = operands("bf16", K, places("bf16", columns), seed)
        _, s, mean, rstd = tf.layer_norm(x, gain, bias)
        call = lambda gy=x, s=s, gain=gain, mean=mean, rstd=rstd, gs=gs, **k: tf.layer_norm_backward(gy, s, gain, mean, rstd, gs=gs, **k)  # noqa: E731
        want = call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        sets.append((graph, got, want, call))
    for i in range(4):
        for graph, got, want, call in sets:
            for t in set(got):
                t.zero_()
            graph.replay()
        eager = [call() for _, _, _, call in sets]
        torch.cuda.synchronize()
        for (_, got, want, _), again in zip(sets, eager):
            assert all(torch.equal(a, b) and torch.equal(c, b) for a, b, c in zip(got, want, again)), i
