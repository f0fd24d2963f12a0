"""FP64 definition of the gated feed-forward block, and how far its kernels may be off.

`bounds` are elementwise and hold for any inputs: half a step of the type for every rounding to it (`a`, the two
projections' gradients, the results), 2^-16 for the projections that are kept of 16-bit inputs (24 bits of FP32), and a
2^-24 per addition of a product's depth for the FP32 sums, each carried on by the magnitudes that it meets.  Of inputs of FP32
a product is off by at most 4 more units of 2^-24, and additions are counted twice over for the six products of parts.

`norms` hold for large random inputs: roundings are independent of what they round, so a relative error keeps its size
through a product, and a result is off by at most half a step for each of the two roundings on its way (of FP32: 16
units and 4 times the square root of the depth's additions).
"""

from __future__ import annotations

import math

import torch

from layer_reference import FLOOR, HALF_STEP, U32


def _activation(name, g):
    """(value, slope, a bound of the second derivative)"""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s)), 0.5
    phi = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
    density = torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    return g * phi, phi + g * density, 0.8


def feed_forward(x, gate_up, down, activation, grad):
    """((out, dx, dgate_up, ddown), bounds, norms)"""
    dtype = x.dtype
    u16, wide = HALF_STEP[dtype], dtype == torch.float32
    kept = 0.0 if wide else 2.0**-16
    floor = FLOOR[dtype]
    x, w, wd = (t.double().reshape(-1, t.shape[-1]) for t in (x, gate_up, down))
    grad = grad.double().reshape(-1, wd.shape[0])
    rows, width, hidden, out_width = x.shape[0], x.shape[1], wd.shape[1], wd.shape[0]

    def sums(depth):
        return ((2 * depth + 16) if wide else (depth + 8)) * U32

    both = x @ w.T
    g, u = both.chunk(2, -1)
    off_both = sums(width) * (x.abs() @ w.abs().T)
    off_g, off_u = off_both.chunk(2, -1)
    value, slope, bend = _activation(activation, g)
    evaluated = (16 + 2 * g.abs() + g * g) * U32  # roundings of the exponential's argument and what follows
    off_value = slope.abs() * off_g + bend * off_g.square() + evaluated * value.abs() + 4 * U32 * g.abs()
    a = value * u
    off_a = value.abs() * off_u + u.abs() * off_value + off_u * off_value + 4 * U32 * a.abs()
    off_a16 = off_a + u16 * (a.abs() + off_a) + floor
    out = a @ wd.T
    bound_out = off_a16 @ wd.abs().T + sums(hidden) * ((a.abs() + off_a16) @ wd.abs().T)

    # from the projections that are kept
    off_g, off_u = off_g + kept * g.abs(), off_u + kept * u.abs()
    off_value = slope.abs() * off_g + bend * off_g.square() + evaluated * value.abs() + 4 * U32 * g.abs()
    off_slope = bend * off_g + evaluated * (1 + g.abs())
    da = grad @ wd
    off_da = sums(out_width) * (grad.abs() @ wd.abs())
    da_most, u_most = da.abs() + off_da, u.abs() + off_u
    dg, du = da * u * slope, da * value
    off_dg = off_da * u_most * (slope.abs() + off_slope) + da_most * (off_u * (slope.abs() + off_slope) + u.abs() * off_slope)
    off_du = off_da * (value.abs() + off_value) + da.abs() * off_value
    d, off_d = torch.cat((dg, du), -1), torch.cat((off_dg, off_du), -1)
    off_d = off_d + 4 * U32 * d.abs()
    off_d = off_d + u16 * (d.abs() + off_d) + floor
    off_a = value.abs() * off_u + u_most * off_value + 4 * U32 * a.abs()
    off_a = off_a + u16 * (a.abs() + off_a) + floor
    most = d.abs() + off_d
    dx, dw, dwd = d @ w, d.T @ x, grad.T @ a
    k = 16 * U32  # the parts' sums
    bound_x = off_d @ w.abs() + (sums(2 * hidden) + k) * (most @ w.abs())
    bound_w = off_d.T @ x.abs() + (sums(rows) + k) * (most.T @ x.abs())
    bound_wd = grad.abs().T @ off_a + (sums(rows) + k) * (grad.abs().T @ (a.abs() + off_a))

    def norm(*depths):
        return sum((16 + 4 * math.sqrt(n)) * U32 for n in depths) + (0.0 if wide else 2 * u16)

    return ((out, dx, dw, dwd), (bound_out, bound_x, bound_w, bound_wd),
            (norm(width, hidden), norm(width, out_width, 2 * hidden), norm(width, out_width, rows), norm(width, rows)))


__all__ = ["feed_forward"]
