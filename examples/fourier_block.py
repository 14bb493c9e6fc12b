"""A Fourier block as it is trained and served: the fused spectral layer with the operators around it, on fields x[channels][signals][samples], complex64.

    h = norm(x),  s = gelu(F^-1 R F h + W h + b)        spectral layer on the 64 lowest modes, pointwise product beside it
    m = norm(s + x),  y = s + x + W2 gelu(W1 m + b1) + b2

The gradients are written out: that of the spectral layer is the same layer with R^H, that of its weights a product of truncated spectra, a sum
over modes where the other products sum over positions. Training clips all gradients together; serving takes the wide product in 8 bits.

    python examples/fourier_block.py [--channels 64] [--hidden 128] [--signals 64] [--samples 256] [--steps 40] [--rate 2]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import turbofno_amd as tf  # noqa: E402

MODES = 64


def _randn(generator, shape, scale):
    return (torch.randn(shape, dtype=torch.complex64, generator=generator) * scale).cuda()


class FourierBlock:
    """`channels` a multiple of 64; parameters in self.parameters, by name."""

    def __init__(self, channels, hidden, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.parameters = {
            "gain1": torch.ones(channels, device="cuda"), "gain2": torch.ones(channels, device="cuda"),
            "R": _randn(g, (channels, channels), channels ** -0.5),
            "W": _randn(g, (channels, channels), channels ** -0.5), "b": _randn(g, (channels,), 0.1),
            "W1": _randn(g, (hidden, channels), channels ** -0.5), "b1": _randn(g, (hidden,), 0.1),
            "W2": _randn(g, (channels, hidden), hidden ** -0.5), "b2": _randn(g, (channels,), 0.1),
        }
        self.eight_bits = None

    def forward(self, x):
        """y, and what backward takes."""
        p = self.parameters
        h, _, rstd1 = tf.rms_norm(x, p["gain1"])
        u = tf.layer_1d(h, p["R"], alpha=1.0 / x.shape[-1])
        z = torch.empty_like(u)
        s = tf.mix(h, p["W"], bias=p["b"], residual=u, activation="gelu_tanh", z=z)
        m, t, rstd2 = tf.rms_norm(s, p["gain2"], residual=x)
        z1 = torch.empty((p["W1"].shape[0],) + x.shape[1:], dtype=x.dtype, device=x.device)
        v = tf.mix(m, p["W1"], bias=p["b1"], activation="gelu_tanh", z=z1)
        y = tf.mix(v, p["W2"], bias=p["b2"], residual=t)
        return y, (x, h, rstd1, z, m, t, rstd2, z1, v)

    def backward(self, gy, saved):
        """The gradient of x and, by name, those of the parameters."""
        p, g = self.parameters, {}
        x, h, rstd1, z, m, t, rstd2, z1, v = saved
        gv, g["W2"], g["b2"], gt = tf.mix_backward(gy, v, p["W2"])
        gm, g["W1"], g["b1"], _ = tf.mix_backward(gv, m, p["W1"], z=z1, activation="gelu_tanh")
        gt, g["gain2"] = tf.rms_norm_backward(gm, t, p["gain2"], rstd2, gs=gt)      # of s and, by the residual stream, of x
        gh, g["W"], g["b"], gu = tf.mix_backward(gt, h, p["W"], z=z, activation="gelu_tanh")
        g["R"] = self.spectral_weight_grad(gu, h)
        gh += tf.layer_1d(gu, p["R"].mH.contiguous(), alpha=1.0 / x.shape[-1])
        gx, g["gain1"] = tf.rms_norm_backward(gh, x, p["gain1"], rstd1, gs=gt)
        return gx, g

    @staticmethod
    def spectral_weight_grad(gu, h):
        """sum over signals and modes of F gu conj(F h): the gradient of R."""
        samples = h.shape[-1]

        def spectra(f):
            out = torch.empty(f.shape[:-1] + (MODES,), dtype=f.dtype, device=f.device)
            return tf.fft_stride_DY(f, out, 1, f.shape[0] * f.shape[1])

        gR, _ = tf.mix_weight_grad(spectra(gu), spectra(h))
        return gR / samples

    def train_step(self, x, target, rate, max_norm=1.0):
        """One step of gradient descent on |y - target|^2; (loss, norm of the gradients), on the GPU."""
        y, saved = self.forward(x)
        gy = (y - target) / y.numel()
        loss = 0.5 * torch.view_as_real(y - target).square().sum() / y.numel()
        _, g = self.backward(gy, saved)
        norm = tf.clip_grad_norm(list(g.values()), max_norm)
        for name, value in self.parameters.items():
            value.sub_(g[name], alpha=rate)
        return loss, norm

    def quantise(self):
        """W1 in 8 bits with a scale per row, laid out once for serving."""
        W1 = torch.view_as_real(self.parameters["W1"])
        scale = W1.abs().amax(dim=(1, 2)) / 448
        self.eight_bits = ((W1 / scale[:, None, None]).to(torch.float8_e4m3fn).contiguous(), scale)

    def serve(self, x):
        """forward with the norm's result and W1 in 8 bits."""
        p = self.parameters
        W1q, W1s = self.eight_bits
        h, _, _ = tf.rms_norm(x, p["gain1"])
        u = tf.layer_1d(h, p["R"], alpha=1.0 / x.shape[-1])
        s = tf.mix(h, p["W"], bias=p["b"], residual=u, activation="gelu_tanh", y=u)
        q, scale, t = tf.rms_norm_8bit(s, p["gain2"], residual=x, s=s)
        v = tf.mix_8bit(q, scale, W1q, W1s, bias=p["b1"], activation="gelu_tanh", dtype=x.dtype)
        return tf.mix(v, p["W2"], bias=p["b2"], residual=t, y=t)


def main():
    parser = argparse.ArgumentParser()
    for name, value in (("channels", 64), ("hidden", 128), ("signals", 64), ("samples", 256), ("steps", 40)):
        parser.add_argument("--" + name, type=int, default=value)
    parser.add_argument("--rate", type=float, default=2.0)
    args = parser.parse_args()
    g = torch.Generator().manual_seed(1)
    x = _randn(g, (args.channels, args.signals, args.samples), 1.0)
    target = FourierBlock(args.channels, args.hidden, seed=2).forward(x)[0]
    block = FourierBlock(args.channels, args.hidden)
    for step in range(args.steps):
        loss, norm = block.train_step(x, target, args.rate)
        if step % 10 == 0 or step == args.steps - 1:
            print("step %3d  loss %.5f  norm of the gradients %.5f" % (step, loss.item(), norm.item()), flush=True)
    block.quantise()
    y, q = block.forward(x)[0], block.serve(x)
    print("served in 8 bits: off by %.2g of the result" % ((q - y).norm() / y.norm()).item())


if __name__ == "__main__":
    main()
