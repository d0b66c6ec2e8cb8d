"""Float64 values with a bound on how far a computation in fewer bits may be from them.

``Bounded(v, e)``: the computed value lies within ``e`` of ``v``. Products of n terms summed in float32 in any order add
at most n 2^-24 of the sum of the terms' magnitudes (n - 1 additions and one rounding of each product, first order,
doubled for matrix units that truncate inside a step); a rounding to a type adds eps / 2 of the value, and half of the
smallest subnormal."""

import torch

U = 2.0 ** -23  # twice float32's half step


class Bounded:
    def __init__(self, v, e=None):
        self.v = v.double()
        self.e = torch.zeros_like(self.v) if e is None else e

    def __matmul__(self, o):
        n = self.v.shape[-1]
        a, b = self.v.abs() + self.e, o.v.abs() + o.e
        e = self.v.abs() @ o.e + self.e @ b + n * U * (a @ b)
        return Bounded(self.v @ o.v, e)

    def __add__(self, o):
        v = self.v + o.v
        return Bounded(v, self.e + o.e + U * (self.v.abs() + o.v.abs() + self.e + o.e))

    def times(self, s):
        """Times a float32 number or tensor."""
        s = s.double() if isinstance(s, torch.Tensor) else s
        m = abs(s) if not isinstance(s, torch.Tensor) else s.abs()
        return Bounded(self.v * s, m * (self.e + U * (self.v.abs() + self.e)))

    def sum(self, dim):
        n = self.v.shape[dim]
        return Bounded(self.v.sum(dim), self.e.sum(dim) + n * U * (self.v.abs() + self.e).sum(dim))

    def round(self, dtype, floor=0.0):
        """Rounded to ``dtype``; ``floor``: an absolute error instead of the smallest subnormal's half."""
        f = torch.finfo(dtype)
        tiny = f.tiny * f.eps / 2
        return Bounded(self.v, self.e + f.eps / 2 * (self.v.abs() + self.e) + (floor if isinstance(floor, torch.Tensor)
                                                                               else max(floor, tiny)))

    @property
    def T(self):
        return Bounded(self.v.transpose(-1, -2), self.e.transpose(-1, -2))

    def __getitem__(self, at):
        return Bounded(self.v[at], self.e[at])

    def check(self, got, what=""):
        got = got.double()
        assert got.shape == self.v.shape, (what, got.shape, self.v.shape)
        assert torch.isfinite(got).all(), f"{what}: not finite"
        off = (got - self.v).abs() - self.e
        assert (off <= 0).all(), f"{what}: {off.max().item():.3g} beyond the bound at {int(off.argmax())}"
