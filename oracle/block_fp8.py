"""The 8-bit block format and its products from their definitions, in float64 on the CPU (test infrastructure)."""
import numpy as np
import torch

_POW = torch.tensor([2.0 ** i for i in range(-400, 400)], dtype=torch.float64)


def _pow2(e):
    return _POW[e.long() + 400]


def exponents(x, rows):
    """x [R, C] (any float type, CPU) -> integer exponents [ceil(R/rows), ceil(C/128)] of its blocks: the smallest e >= -127 with
    max|x| <= 448 * 2^e over the finite values."""
    x = x.double()
    R, C = x.shape
    x = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))
    x = torch.nn.functional.pad(x, (0, -C % 128, 0, -R % rows))
    amax = x.view(x.shape[0] // rows, rows, x.shape[1] // 128, 128).amax((1, 3))
    e = torch.full(amax.shape, -127, dtype=torch.int64)
    for _ in range(400):
        low = 448.0 * _pow2(e) < amax
        if not bool(low.any()):
            break
        e = e + low.long()
    return e


def e4m3(v):
    """float64 -> the nearest e4m3 value, ties to even, |v| <= 448 (non-finite: NaN)."""
    ex = torch.frexp(v)[1].clamp(min=-5)
    step = _pow2(torch.where(torch.isfinite(v), ex, torch.zeros_like(ex)) - 4)
    q = torch.round(v / step) * step
    return torch.where(torch.isfinite(v), q, torch.full_like(v, float("nan")))


def quantize(x, rows):
    """-> (values the 8-bit matrix stands for divided by their scales [R, C padded], exponents)."""
    e = exponents(x, rows)
    R, C = x.shape
    x = torch.nn.functional.pad(x.double(), (0, -C % 128))
    per = e.repeat_interleave(rows, 0)[:R].repeat_interleave(128, 1)
    return e4m3(x / _pow2(per)), e


def stands_for(x, rows):
    q, e = quantize(x, rows)
    return (q * _pow2(e.repeat_interleave(rows, 0)[:x.shape[0]].repeat_interleave(128, 1)))[:, :x.shape[1]]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Operand:
    """An 8-bit matrix [R, C]: v, the values it stands for, and m, the magnitude its exponents say (|v| rounded up to e4m3's smallest normal
    times the block's scale: what a product of two values is aligned by)."""

    def __init__(self, x, rows):
        self.v = stands_for(x, rows)
        s = _pow2(exponents(x, rows).repeat_interleave(rows, 0)[:x.shape[0]].repeat_interleave(128, 1))[:, :x.shape[1]]
        self.m = torch.maximum(self.v.abs(), s * 2.0 ** -6)

    def t(self):
        o = object.__new__(Operand)
        o.v, o.m = self.v.t().contiguous(), self.m.t().contiguous()
        return o


def product(a, b):
    return a.v @ b.v.t()


def product_bound(a, b, exact, dtype):
    """Error bound of an engine product of exact 8-bit values.

    float32 results: every partial sum rounds by at most one step, 2^-23 of a magnitude below sum |a b|.
    16-bit results come from the 8-bit matrix instruction, which adds eight consecutive products at a time, each cut off (towards zero) at
    2^-13 of 2^E, E the largest exponent sum among the eight: below 8 * 2^-13 * max m_a m_b per eight, next to the same fp32 sums.
    Then half a step of the output type and its smallest subnormal."""
    mag = a.v.abs() @ b.v.abs().t()
    out = a.v.shape[1] * 2.0 ** -23 * mag + half_step(dtype) * exact.abs() * (1 + 2.0 ** -10) + float(np.finfo(np.float32).tiny) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    if dtype != torch.float32:
        pad = -a.v.shape[1] % 8
        ma, mb = torch.nn.functional.pad(a.m, (0, pad)), torch.nn.functional.pad(b.m, (0, pad))
        cut = torch.zeros_like(exact)
        for k in range(0, ma.shape[1], 8):
            largest = torch.zeros_like(exact)
            for j in range(8):
                largest = torch.maximum(largest, ma[:, k + j, None] * mb[None, :, k + j])
            cut += largest
        out = out + 8 * 2.0 ** -13 * cut * (1 + half_step(dtype))
    return out
