"""The feed-forward products in 64 bits, and bounds on what their kernels may be off by.

A sum of n products held in 32 bits is off by at most n 2^-23 times the sum of the magnitudes (each addition by at
most one unit in the last place, whatever the order and whether it rounds or truncates); the gate's functions are good to
2^-20 of their value; a rounding to the storage type is off by half a step of it."""
import math

import torch

import clblas_amd as cb

DTYPES = {cb.Type.F32: torch.float32, cb.Type.F16: torch.float16, cb.Type.BF16: torch.bfloat16}
SUM = 2.0 ** -23
FUNC = 2.0 ** -20


def half_step(dtype, x):
    """Largest rounding error of values of magnitude |x| in dtype (subnormals included)."""
    f = torch.finfo(dtype)
    return x.abs() * (f.eps / 2) + f.smallest_normal * f.eps / 2


class Buf:
    """A rows x cols matrix inside a larger buffer of known values: `off` elements before it, `ld` from row to row."""

    def __init__(self, rows, cols, dtype, off=0, pad=0, values=None, fill=7):
        self.off, self.ld, self.rows, self.cols = off, cols + pad, rows, cols
        self.fill = fill
        self.flat = torch.full((off + rows * self.ld + 16,), fill, dtype=dtype, device="cuda")
        self.mat = torch.as_strided(self.flat, (rows, cols), (self.ld, 1), off)
        if values is not None:
            self.mat.copy_(values.to(dtype))

    def args(self):
        return self.flat, self.off, self.ld

    def surroundings_untouched(self):
        """Whether everything outside the matrix still has its value."""
        rest = self.flat.clone()
        torch.as_strided(rest, (self.rows, self.cols), (self.ld, 1), self.off).fill_(self.fill)
        return bool((rest == self.fill).all())


def normal(rows, cols, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(rows, cols, generator=g) * std


def whole(rows, cols, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, (rows, cols), generator=g).to(torch.int8)


def scales(n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.rand(n, generator=g) * 0.02 + 1e-3


def act(gate, g):
    if gate == cb.Gate.Silu:
        return g * torch.sigmoid(g)
    if gate == cb.Gate.Gelu:
        return g * 0.5 * torch.special.erfc(-g * math.sqrt(0.5))
    return g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))


def slope(gate, g):
    if gate == cb.Gate.Gelu:
        return 0.5 * torch.special.erfc(-g * math.sqrt(0.5)) + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    z, dz = g, torch.ones_like(g)
    if gate == cb.Gate.GeluTanh:
        c = 2 * math.sqrt(2 / math.pi)
        z, dz = c * (g + 0.044715 * g ** 3), c * (1 + 3 * 0.044715 * g ** 2)
    return torch.sigmoid(z) + g * torch.sigmoid(z) * torch.sigmoid(-z) * dz


def gated_want(gate, g, u, eg, eu):
    """H and its error before the last rounding, from G, U and theirs.  |act'| and |act''| stay below 1.13 and 1."""
    h = act(gate, g) * u
    err = u.abs() * (1.13 * eg + eg * eg) + act(gate, g).abs() * eu + 1.13 * eg * eu + h.abs() * FUNC + g.abs() * u.abs() * 2.0 ** -24
    return h, err


def close(got, want, err, dtype):
    """Asserts |got - want| <= err + one rounding of a value that is off by err."""
    got = got.double()
    bound = err + half_step(dtype, want.abs() + err)
    top = torch.finfo(dtype).max
    over = want.abs() + bound > top  # may round to infinity
    bad = ((got - want).abs() > bound) & ~over
    assert not bool(bad.any()), "worst excess %.3g of bound" % float(((got - want).abs() / bound)[~over].max())
    assert not bool(torch.isnan(got).any())
