"""Rows in 8 bits, RMS norm with a residual, the SwiGLU product and the linear over 8-bit rows with adapters, in 64 bits on the
host, and how far a computation in fewer bits may be off.  Written from the definitions."""

from __future__ import annotations

import torch

from oracle.attention import HALF_STEP

UNIT = 2.0**-24  # half a step of fp32, relative
TOP, LEAST = 448.0, 2.0**-100


def eight_bits(y, wrong):
    """y [rows, width] in 64 bits, known to `wrong` (relative) -> (scales, bound, values before their rounding, bound)."""
    scales = (y.abs().amax(-1) / TOP).clamp(min=LEAST)
    values = y / scales[:, None]
    # max / 448 rounds once, and so does the quotient by it; e4m3 keeps four bits (2^-4 of the value) down to steps of 2^-9
    off = values.abs() * (2 * wrong + 4 * UNIT)
    most = wrong.amax(-1) if torch.is_tensor(wrong) else wrong
    return scales, scales * (most + 2 * UNIT), values, off + (values.abs() + off) * 2.0**-4 + 2.0**-10


def add_rms_norm(x, weight, residual=None, eps=1e-6):
    """(sum in the element type, norm in 64 bits, relative bound of its error in fp32)."""
    total = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    s = total.double()
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * weight.double()
    # the sum of squares: at most 32 or width / 1024 in a thread's chain, then six and sixteen additions over lanes and wavefronts, halved by the
    # root; the squares, quotient, eps and root (4), weight and factor (2)
    chain = max(32, x.size(1) / 1024 + 8) + 24
    return total, y, (chain / 2 + 6) * UNIT


def silu_mul(gate_up):
    """(product in 64 bits, relative bound of its error in fp32)."""
    g, u = gate_up.double().chunk(2, dim=-1)
    # exp's argument rounds once after its product with log2 e (|g| 2 units), exp2 and the quotient to two units each, sum and products to one
    return g * torch.sigmoid(g) * u, (3 * g.abs() + 10) * UNIT


def linear(x, x_scales, w, w_scales, bias=None, a=(), b=(), columns=None, slots=None, dtype=torch.bfloat16):
    """(y in 64 bits, bound of its error with `dtype` outputs)."""
    x, w = x.double() * x_scales.double()[:, None], w.double() * w_scales.double()[:, None]
    k = x.size(1)
    y, size = x @ w.T, x.abs() @ w.abs().T
    # K additions and a few products in fp32; and the matrix instruction lines the products of eight neighbours along K up to the largest of them before it adds them, and
    # drops what lies more than 13 bits below that one's leading bit (found with powers of two: beside 2^8, 2^-5 counts and 2^-6 does not, beside 2^16, 2^2 does not; one place to the right, in the
    # next eight, all do that fp32 holds): seven numbers of less than 2^-13 of the largest, for every eight
    most = torch.zeros_like(size)
    for first in range(0, k, 8):
        of = torch.zeros_like(size)
        for i in range(first, min(first + 8, k)):
            of = torch.maximum(of, x[:, i, None].abs() * w[:, i].abs())
        most += of
    bound = size * (k + 8) * UNIT + 7 * 2.0**-13 * most
    if bias is not None:
        y = y + bias.double()
    first = 0
    for i, (a_of, b_of) in enumerate(zip(a, b)):
        n, rank = b_of.shape[1:]
        first = first if columns is None else columns[i]
        for t, s in enumerate(slots.tolist()):
            if not 0 <= s < a_of.size(0):
                continue
            aa, bb = a_of[s].double(), b_of[s].double()
            h, h_size = aa @ x[t], aa.abs() @ x[t].abs()
            y[t, first : first + n] += bb @ h
            # h: K additions; it is two bf16 numbers, 2^-16 of it, and fp16's B two as well, of whose four products with h three are taken, 2^-16 once more; then rank additions
            rounded = 2.0**-16 if dtype == torch.bfloat16 else 2 * 2.0**-16
            bound[t, first : first + n] += bb.abs() @ ((h_size * (k + 8) * UNIT) * (1 + rounded) + h.abs() * (rounded + (rank + 8) * 2 * UNIT))
            size[t, first : first + n] += bb.abs() @ h.abs()
        first += n
    # the sum's own additions (of wavefronts, slices, bias), then the result's rounding
    bound = bound + size * 40 * UNIT + y.abs() * UNIT
    return y, bound + (y.abs() + bound) * HALF_STEP[dtype] + (2.0**-25 if dtype == torch.float16 else 0.0)
