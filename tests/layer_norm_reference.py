"""Plain 64-bit forms of the layer norm, dropout and the products in 8 bits with scales by blocks, where their operands are, and bounds of their errors."""
import torch

from operators_reference import EPS32, rounding

BLOCK = 128


LOW = 0xFFFFFFFF


def wide(t):
    return t.detach().to(torch.complex128 if t.is_complex() else torch.float64)


def within(got, exact, bound, what=""):
    """|got - exact| <= bound for every element"""
    assert got.shape == exact.shape, what
    off = (wide(got) - exact).abs()
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert worst <= 0, "%s: %g over its bound (largest error %g)" % (what, worst, off.max().item())


def philox(counter, key):
    """Philox 4x32 with ten rounds: four int64 tensors of 32-bit numbers and a key of two words -> four of them. Products wrap around at 64 bits and lose none."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & LOW) ^ c[1] ^ k[0], b & LOW, ((a >> 32) & LOW) ^ c[3] ^ k[1], a & LOW]
        k = [(k[0] + 0x9E3779B9) & LOW, (k[1] + 0xBB67AE85) & LOW]
    return c


def kept(rng, K, positions, drop, device="cuda", first=0):
    """[K][positions] of truth values, for the positions from `first` on, a multiple of four"""
    seed, offset = (int(v) % 2 ** 64 for v in rng)
    q = torch.arange(-(-positions // 4), dtype=torch.int64, device=device)[None, :] + first // 4
    k = torch.arange(K, dtype=torch.int64, device=device)[:, None]
    each = torch.zeros((K, q.shape[1]), dtype=torch.int64, device=device)
    words = philox([each + (q & LOW), k + ((q >> 32) << 16), each + offset % 2 ** 32, each + offset // 2 ** 32], (seed % 2 ** 32, seed // 2 ** 32))
    return torch.stack(words, -1).reshape(K, -1)[:, :positions] >= min(round(drop * 2 ** 32), LOW)


def dropped(t, rng, drop):
    """dropout(t) of a [K][P] tensor in 64 bits"""
    return torch.where(kept(rng, *t.shape, drop, t.device), t / (1 - drop), torch.zeros_like(t)) if drop else t


def square(t):
    return t.real ** 2 + t.imag ** 2 if t.is_complex() else t * t


def along(a, b):
    """Re(conj(a) b)"""
    return (a.conj() * b).real if a.is_complex() else a * b


class Forward:
    """s, mean, rstd and y of the layer norm in 64 bits, and bounds of what 32 bits make of them before the last rounding"""

    def __init__(self, x, gain, bias=None, residual=None, eps=1e-6, drop=0.0, rng=None):
        X, K = dropped(wide(x).flatten(1), rng, drop), x.shape[0]
        R = wide(residual).flatten(1) if residual is not None else torch.zeros_like(X)
        G, B = wide(gain)[:, None], wide(bias)[:, None] if bias is not None else 0.0
        self.s = X + R
        # 1 / (1 - drop), its product and the sum: three roundings
        self.s_off = 3 * EPS32 * (X.abs() + R.abs()) if drop or residual is not None else torch.zeros(X.shape, dtype=torch.float64, device=X.device)
        self.mean = self.s.mean(0)
        # K + 3 roundings of a sum of magnitudes; so are the following sums
        self.mean_off = (K + 3) * EPS32 * self.s.abs().mean(0) + self.s_off.mean(0)
        d = self.s - self.mean
        variance = square(d).mean(0)
        off = self.s_off.amax(0) + self.mean_off
        variance_off = (K + 8) * EPS32 * variance + 2 * variance.sqrt() * off + off ** 2
        self.rstd = 1 / torch.sqrt(variance + eps)
        relative = 0.5 * variance_off / (variance + eps) * (1 + variance_off / (variance + eps)) + 4 * EPS32
        self.rstd_off = relative * self.rstd
        h = d * self.rstd
        self.y = h * G + B
        h_off = (self.s_off + self.mean_off) * self.rstd * (1 + relative) + h.abs() * (relative + 3 * EPS32)
        self.y_off = G.abs() * h_off + 2 * EPS32 * ((h * G).abs() + (B.abs() if bias is not None else 0.0))
        self.meaningful = relative.max().item() < 0.2               # the bounds are of first order


class Backward:
    """gr, gx, ggain and gbias in 64 bits from the operands as they are, and bounds of their errors before the last rounding"""

    def __init__(self, gy, s, gain, mean, rstd, gs=None, drop=0.0, rng=None):
        g, K = wide(gy).flatten(1), gy.shape[0]
        r, h = wide(rstd).flatten(), (wide(s).flatten(1) - wide(mean).flatten()) * wide(rstd).flatten()
        GG = g * wide(gain)[:, None]
        S = wide(gs).flatten(1) if gs is not None else torch.zeros_like(g)
        level, slope = GG.mean(0), along(h, GG).mean(0)
        inner = GG - level - h * slope
        self.gr = r * inner + S
        level_off = (K + 4) * EPS32 * GG.abs().mean(0)
        slope_off = (K + 8) * EPS32 * (h.abs() * GG.abs()).mean(0) * (2 if g.is_complex() else 1)
        inner_off = 5 * EPS32 * (GG.abs() + level.abs() + h.abs() * slope.abs()) + level_off + h.abs() * slope_off
        self.gr_off = r * inner_off + 3 * EPS32 * ((r * inner).abs() + S.abs())
        self.gx = dropped(self.gr, rng, drop)
        self.gx_off = self.gr_off / (1 - drop) + 3 * EPS32 * self.gx.abs()
        # a lane adds four columns of each of its strips, the lanes, the 512 blocks sixteen by sixteen and their sixteen sums follow
        chain = 4 * -(-g[0].numel() * (2 if g.is_complex() else 1) // (64 * 512)) + 6 + 32 + 16 + 8
        self.ggain = along(h, g).sum(1)
        self.ggain_off = chain * EPS32 * (h.abs() * g.abs()).sum(1) * (2 if g.is_complex() else 1)
        self.gbias = g.sum(1)
        self.gbias_off = chain * EPS32 * g.abs().sum(1)


def rounded(exact, off, dtype):
    """the bound after the rounding to the type of the result"""
    return off + 1.01 * rounding(dtype) * (exact.abs() + off)


def per_channel(scale, K):
    return scale.repeat_interleave(BLOCK, 0)[:K]


def check_eight(q, scale, exact, off, what):
    """q and scale of a field (64-bit [K][P], off by `off` in 32 bits) against its definition; q within half a step, 2^-4 of a number, 2^-10 below 2^-6"""
    K = exact.shape[0]
    parts = torch.view_as_real(exact) if exact.is_complex() else exact[..., None]
    got = q.detach().double().reshape(K, -1, parts.shape[-1])
    S = scale.detach().double().reshape(-(-K // BLOCK), -1)
    for b in range(S.shape[0]):
        rows = slice(b * BLOCK, min(K, (b + 1) * BLOCK))
        most, most_off = parts[rows].abs().amax((0, 2)), off[rows].amax(0)
        want = most / 448
        small = want < 2.0 ** -126
        assert ((S[b] - want).abs() <= most_off / 448 + 2 * EPS32 * want)[~small].all(), what + ": scale"
        assert (S[b][small] == 1).all() and (got[rows][:, small] == 0).all(), what + ": no scale"
        v = parts[rows] / S[b][None, :, None]
        bound = v.abs() * 2.0 ** -4 * (1 + 2.0 ** -10) + 2.0 ** -10 + (off[rows] / S[b])[..., None] * 1.1 + 4 * EPS32 * v.abs()
        assert ((got[rows] - v).abs() <= bound)[:, ~small].all(), "%s: q off by %g" % (what, ((got[rows] - v).abs() - bound)[:, ~small].max().item())


def quantised_weights(W):
    """[N][K](2) in e4m3 and scales [N / 128][K / 128]"""
    N, K = W.shape[:2]
    scale = torch.stack([torch.stack([t.abs().amax() for t in rows.split(BLOCK, 1)]) for rows in W.split(BLOCK, 0)]) / 448
    each = scale.repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]
    return (W / (each if W.dim() == 2 else each[..., None])).to(torch.float8_e4m3fn), scale


class Product:
    """z of the product in 64 bits from the operands as they are, and the sum of the magnitudes of its terms"""

    def __init__(self, xq, xscale, Wq, wscale, bias=None, residual=None):
        K, N, pair = xq.shape[0], Wq.shape[0], Wq.dim() == 3
        x, W = (t.detach().double() for t in (xq, Wq))
        x = x.reshape(K, -1, 2) if pair else x.reshape(K, -1)
        xs = per_channel(xscale.detach().double().reshape(-(-K // BLOCK), -1), K)
        ws = per_channel(wscale.detach().double(), N).t().contiguous()
        ws = per_channel(ws, K).t()
        x, W = (torch.view_as_complex(x) * xs, torch.view_as_complex(W) * ws) if pair else (x * xs, W * ws)
        self.z, self.sizes = W @ x, W.abs() @ x.abs() * (2 if pair else 1)
        self.more = torch.zeros_like(self.sizes)
        for t in (wide(bias)[:, None] if bias is not None else None, wide(residual).flatten(1) if residual is not None else None):
            if t is not None:
                self.z = self.z + t
                self.more = self.more + t.abs()
