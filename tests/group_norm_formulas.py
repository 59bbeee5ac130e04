"""Group norm with an activation in float64: the definition for autograd, and its derivatives written out (which also say
what a backward pass that has x in 8 bits computes, and how large the terms of each sum are).

The size of a sum's term is that of what it is computed from: a difference is off by units of 2^-24 of its operands, which
may cancel (v - <v> - h <v h>, x - mean, 1 + z (1 - s), 2 + z (1 - 2 s)), so magnitudes are added in its place."""
import torch


def silu(z):
    return z * torch.sigmoid(z)


def _grouped(t, groups):
    return t.reshape(t.shape[0], -1, groups, t.shape[-1] // groups)


def _mean(t):
    return t.mean((1, 3), keepdim=True)


def definition(x, groups, w, b, eps, activation):
    X = _grouped(x, groups)
    c = X - _mean(X)
    z = (c / torch.sqrt(_mean(c * c) + eps)).reshape(x.shape)
    z = z if w is None else z * w
    z = z if b is None else z + b
    return silu(z) if activation else z


class Derivatives:
    """First and second derivatives of the group norm of x, with `value` in x's place within the normalised values."""

    def __init__(self, x, groups, w, b, eps, activation, g, value=None):
        x, g = x.double(), g.double()
        self.shape, self.groups = x.shape, groups
        X = _grouped(x, groups)
        mean = _mean(X)
        self.r = 1.0 / torch.sqrt(_mean((X - mean) ** 2) + eps)
        self.h = ((X if value is None else _grouped(value.double(), groups)) - mean) * self.r
        one = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device)
        self.w = (one if w is None else w.double()).view(groups, -1)
        b = (0 * one if b is None else b.double()).view(groups, -1)
        z = self.h * self.w + b
        self.hm = ((X if value is None else _grouped(value.double(), groups)).abs() + mean.abs()) * self.r
        zm = self.hm * self.w.abs() + b.abs()
        s = torch.sigmoid(z)
        self.slope = s * (1 + z * (1 - s)) if activation else torch.ones_like(z)
        self.bend = s * (1 - s) * (2 + z * (1 - 2 * s)) if activation else torch.zeros_like(z)
        self.g = _grouped(g, groups)
        self.slopem = s * (1 + zm * (1 - s)) if activation else self.slope
        self.bendm = s * (1 - s) * (2 + zm * (1 - 2 * s).abs()) if activation else self.bend
        self.ga = self.g * self.slope

    def _channels(self, t):
        return t.sum((0, 1)).reshape(-1)

    def first(self):
        """(dx, dw, db), and the sums of the magnitudes of dw's and db's terms."""
        u = self.ga * self.w
        dx = self.r * (u - _mean(u) - self.h * _mean(u * self.h))
        gm = self.g.abs() * self.slopem
        return ((dx.reshape(self.shape), self._channels(self.ga * self.h), self._channels(self.ga)),
                (self._channels(gm * self.hm), self._channels(gm)))

    def second(self, v, vw=None, vb=None):
        """Gradients of <v, dx> + <vw, dw> + <vb, db> by x, g, w and b, and the magnitudes of the last two's terms."""
        h, r, ga, w = self.h, self.r, self.ga, self.w
        v = _grouped(v.double(), self.groups)
        zero = torch.zeros_like(w)
        vw = zero if vw is None else vw.double().view(w.shape)
        vb = zero if vb is None else vb.double().view(w.shape)
        u = ga * w
        pv = r * (v - _mean(v) - h * _mean(v * h))
        e = w * pv + h * vw + vb
        zz = e * self.g * self.bend
        t = ga * vw + zz * w - r * (_mean(v * h) * u + _mean(u * h) * v)
        q = _mean(u * v) - _mean(u) * _mean(v) - _mean(u * h) * _mean(v * h)
        dx = r * (t - _mean(t) - h * _mean(t * h)) - r * r * q * h
        pm = r * (v.abs() + _mean(v.abs()) + self.hm * _mean(v.abs() * self.hm))
        zm = (w.abs() * pm + self.hm * vw.abs() + vb.abs()) * self.g.abs() * self.bendm
        return ((dx.reshape(self.shape), (e * self.slope).reshape(self.shape), self._channels(ga * pv + zz * h),
                 self._channels(zz)),
                (self._channels(self.g.abs() * self.slopem * pm + zm * self.hm), self._channels(zm)))
