"""The linear cross entropy in float64, and how far the library's outputs may be
from it: bounds by arithmetic, element by element.

With u = 2^-24 (half a step of fp32) a dot product of H terms in any order is
within 2·(H + 2)·u·Σ|h||w| of its exact value (the factor 2: the matrix units
may round each step towards zero), three-plane products within three times that
(six products a term, and the parts left out lie below u of each term).
The log-sum-exp moves by at most the largest error of its logits, plus the
rounding of the maximum in log2 units (|m|·u twice), the exponentials (each
2^-22 relative with its argument's rounding) and the additions (32 a lane, 6
steps over lanes, V/16384 tiles a lane: (64 + V/8192)·u).
"""
import torch

U = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


class Exact:
    """hidden, weight as the library gets them (any float type, CPU or GPU)."""

    def __init__(self, hidden, weight, labels, *, ignore_index=-100, label_smoothing=0.0):
        self.dtype = hidden.dtype
        h, w = hidden.double().cpu(), weight.double().cpu()
        y = labels.long().cpu()
        self.valid = y != ignore_index
        self.bad = self.valid & ((y < 0) | (y >= w.size(0)))
        h = torch.where(self.valid[:, None], h, torch.zeros((), dtype=torch.float64))
        self.h, self.w, self.a = h, w, label_smoothing
        self.y = torch.where(self.valid & ~self.bad, y, torch.zeros_like(y))
        n, v = h.size(0), w.size(0)
        self.x = h @ w.t()
        mags = h.abs() @ w.abs().t()
        planes = 3.0 if self.dtype == torch.float32 else 1.0
        self.dx = 2 * planes * (h.size(1) + 2) * U * mags          # error of a logit
        lse = torch.logsumexp(self.x, 1)
        top = self.x.abs().amax(1)
        self.dlse = self.dx.amax(1) + 2 * top * U + 2.0 ** -22 + (64 + v / 8192) * U + 2 * lse.abs() * U
        xy = self.x.gather(1, self.y[:, None])[:, 0]
        nll = lse - (1 - self.a) * xy
        self.dnll = self.dlse + self.dx.amax(1) + (lse.abs() + xy.abs()) * 2 * U
        if self.a:
            nll = nll - self.a * self.x.mean(1)
            self.dnll = self.dnll + self.a * (64 + v / 8192) * U * self.x.abs().mean(1) + self.a * self.dx.mean(1)
        zero = torch.zeros((), dtype=torch.float64)
        self.lse = torch.where(self.valid, lse, zero)
        self.nll = torch.where(self.valid, nll, zero)
        self.nll[self.bad] = float("nan")

    def check_losses(self, nll, lse):
        nll, lse = nll.double().cpu(), lse.double().cpu()
        keep = ~self.bad
        assert torch.isnan(nll[self.bad]).all()
        assert (nll[~self.valid] == 0).all() and (lse[~self.valid] == 0).all()
        e = (lse - self.lse).abs()
        assert (e <= self.dlse).all(), f"lse off by {e.max():.3g}, allowed {self.dlse[e.argmax()]:.3g}"
        e = (nll - self.nll).abs()[keep]
        assert (e <= self.dnll[keep]).all(), f"nll off by {e.max():.3g}"

    def gradients(self, gn, gl):
        """(grad_hidden, grad_weight, bound of each's error): the gradient of the
        logits d is off by its rounding and by its exponent's error, and the
        products by their additions and the rounding of the result."""
        zero = torch.zeros((), dtype=torch.float64)
        gn = zero if gn is None else gn.double().cpu()
        gl = zero if gl is None else gl.double().cpu()
        g1 = torch.where(self.valid, gn + gl, zero)
        g0 = torch.where(self.valid, gn + zero * gl, zero)
        n, v = self.x.shape
        p = torch.exp(self.x - torch.where(self.valid, self.lse, torch.logsumexp(self.x, 1))[:, None]) * g1[:, None]
        hot = torch.zeros_like(p)
        hot[torch.arange(n), self.y] = (1 - self.a) * g0
        d = p - (g0 * self.a / v)[:, None] - hot
        u = ROUND[self.dtype]
        dd = u * d.abs() + p.abs() * (self.dx + self.dlse[:, None] + 2.0 ** -21 + 2 * self.x.abs() * U)
        dd = dd + 4 * U * (p.abs() + hot.abs() + (g0.abs() * self.a / v)[:, None])
        out = []
        planes = 3.0 if self.dtype == torch.float32 else 1.0
        for a, da, b in ((d, dd, self.w), (d.t(), dd.t(), self.h)):
            r = a @ b
            bound = (da + 2 * planes * (a.size(1) + 2) * U * a.abs()) @ b.abs()
            out.append((r, bound * 1.01 + u * (r.abs() + bound) + 1e-37))
        return out

    def check_gradients(self, gh, gw, gn, gl):
        (rh, bh), (rw, bw) = self.gradients(gn, gl)
        for name, got, ref, bound in (("grad_hidden", gh, rh, bh), ("grad_weight", gw, rw, bw)):
            if got is None:
                continue
            assert got.dtype == self.dtype and got.shape == ref.shape
            e = (got.double().cpu() - ref).abs()
            bad = ~(e <= bound)
            assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} off, the first at "
                                   f"{bad.nonzero()[0].tolist()}, largest {e.max():.3g} (values {ref.abs().max():.3g})")
        assert gh is None or (gh[~self.valid.to(gh.device)] == 0).all()
