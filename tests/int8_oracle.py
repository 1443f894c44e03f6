"""Layers in 8-bit integers in 64 bits, from the definition: s = amax / 127, q = round(127 x / amax), y = s_x s_w sum(q_x q_w)."""
import torch


def rows(x: torch.Tensor):
    """(q fp64 [M, K], s fp32 [M]); the quotient in 64 bits: 127 x is exact there, and no quotient that is not a tie rounds to one."""
    x = x.double()
    amax = x.abs().amax(-1)
    safe = torch.where(amax > 0, amax, torch.ones_like(amax))
    q = torch.round(127.0 * x / safe[:, None])
    return q, (amax / 127.0).float()      # (a quotient in 64 bits: dividing an fp32 tensor by a number multiplies by its reciprocal)


def products(q, s, w, ws):
    """fp64 [M, N] from values (whole numbers in any type) and fp32 scales."""
    return (q.double() @ w.double().t()) * s.double()[:, None] * ws.double()[None]


def gated(y):
    g, u = y[:, 0::2], y[:, 1::2]
    return g * torch.sigmoid(g) * u


U = 2.0 ** -24          # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the distance between the smallest numbers of the type."""
    return {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}[dtype]


def bound(y, dtype, residual=None, extra=None):
    """How far a plain or residual result may be from y (fp64, without the residual): the sum to fp32 and two scales, three roundings, one more for the residual's
    addition, then half a step of the result's type.  `extra`: what y itself may be off."""
    off = 3.1 * U * y.abs() + (extra if extra is not None else 0.0)
    total = y
    if residual is not None:
        total = y + residual.double()
        off = off + 1.1 * U * (total.abs() + off)
    return off + half_step(dtype) * (total.abs() + off) + smallest(dtype), total


def bound_gated(y, dtype, extra=None):
    """silu(g) u: g and u are off by 3 roundings (and `extra`); the exponential by two steps (four roundings) of its own and |g| times what g is off; the
    sum adds a rounding, the quotient at most two steps (four).  |d silu / dg| <= 1.1."""
    g, u = y[:, 0::2], y[:, 1::2]
    r = gated(y)
    eg = 3.1 * U * g.abs() + (extra[:, 0::2] if extra is not None else 0.0)
    eu = 3.1 * U * u.abs() + (extra[:, 1::2] if extra is not None else 0.0)
    silu = g * torch.sigmoid(g)
    # d silu / silu = dg / g + (1 - sigmoid) dg, and 9 roundings of the chain
    es = 9.0 * U * silu.abs() + eg * (torch.sigmoid(g) + silu.abs() * (1 - torch.sigmoid(g))) * 1.01
    # a reciprocal of 2^126 and more may be taken as 0 (fp32's smallest normal number is 2^-126): from 1 + exp(-g) = 2^126 on, the sigmoid is less than 2^-126, and g u times
    # that is lost
    off = es * u.abs() + silu.abs() * eu + es * eu + 1.1 * U * r.abs() + 2.0 ** -126 * (g * u).abs()
    return off + half_step(dtype) * (r.abs() + off) + smallest(dtype), r


def bound_relu2(y, dtype):
    """relu(y)^2: y is off by three roundings, its square by twice that (and the square of it) and a rounding of its own."""
    r = y.clamp(min=0)
    off = (2 * 3.1 + 0.01 + 1.1) * U * r * r + smallest(torch.float32)
    return off + half_step(dtype) * (r * r + off) + smallest(dtype), r * r
