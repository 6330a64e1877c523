"""Plain 64-bit rotation, storage in 8 and 4 bits, and the error each may have.

The kernels round each product and sum of the rotation to fp32 (2^-24 of it) and
the result once to its type (half a step).  What is stored in few bits is the
nearest value to a quotient in fp32: half a step of the value's grid, and as much
beyond the midpoint as the errors before it can move it.
"""
from __future__ import annotations

import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def rotate(x, positions, table, *, interleaved=False, transpose=False):
    """(values, bound before the last rounding) of x (rows, heads, dim) in float64."""
    x, half = x.double().clone(), table.shape[1] // 2
    angle = table.double()[positions]
    c, s = angle[:, None, :half], angle[:, None, half:] * (-1 if transpose else 1)
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y, z = x[..., a], x[..., b]
    out, bound = x.clone(), torch.zeros_like(x)
    out[..., a], out[..., b] = y * c - z * s, z * c + y * s
    bound[..., a] = 2.0 ** -23 * ((y * c).abs() + (z * s).abs())
    bound[..., b] = 2.0 ** -23 * ((z * c).abs() + (y * s).abs())
    return out, bound + 2.0 ** -140


def rounding(values, dtype):
    """Half a step of dtype at each value."""
    if dtype == torch.float64:
        return torch.zeros_like(values)
    info = torch.finfo(dtype)
    return (values.abs() * info.eps / 2).clamp(min=info.smallest_normal * info.eps / 2)


def check_rows(got, want, bound, dtype):
    """got (of dtype, read as float64) is want within bound and one rounding."""
    room = bound + rounding(want.abs() + bound, dtype)
    err = (got.double() - want).abs()
    assert torch.isfinite(err).all() and (err <= room).all(), (err / room).max()


def check_e4m3(got, want, bound, factor):
    """got e4m3 stands for want / factor, to the nearest, at most 448."""
    g, y = got.double(), (want / factor).clamp(-448, 448)
    step = torch.exp2((torch.frexp(g.abs().clamp(min=2.0 ** -6)).exponent - 4).double())
    # next to a power of two the values below it are half as far apart: half a step of the upper side bounds both
    room = step / 2 * (1 + 2.0 ** -20) + bound / factor + y.abs() * 2.0 ** -23
    err = (g - y).abs()
    assert torch.isfinite(err).all() and (err <= room).all(), (err / room).max()


def unpack(rows, heads, dim):
    """(codes' values, scales) of e2m1 rows (..., bytes) in float64: (..., heads, dim) and (..., heads, dim / 16)."""
    n = heads * dim // 2
    low, high = rows[..., :n] & 15, rows[..., :n] >> 4
    code = torch.stack([low, high], -1).flatten(-2).long()
    value = E2M1[code % 8] * torch.where(code >= 8, -1.0, 1.0).double()
    scale = rows[..., n:n + heads * dim // 16].contiguous().view(torch.float8_e4m3fn).double()
    return value.view(*rows.shape[:-1], heads, dim), scale.view(*rows.shape[:-1], heads, dim // 16)


def values(rows, heads, dim, factor=1.0):
    """What e2m1 rows stand for."""
    value, scale = unpack(rows, heads, dim)
    return value * scale.repeat_interleave(16, -1) * factor


def check_e2m1(rows, want, bound, factor):
    """Rows (n, bytes) hold want (n, heads, dim): scales next to max / 6, codes next to the values over them."""
    heads, dim = want.shape[1:]
    value, scale = unpack(rows, heads, dim)
    groups = want.unflatten(-1, (-1, 16))
    big, slack = groups.abs().amax(-1), bound.unflatten(-1, (-1, 16)).amax(-1)
    ideal = (big / (6 * factor)).clamp(max=448)
    step = torch.exp2((torch.frexp(scale.clamp(min=2.0 ** -6)).exponent - 4).double())
    room = step / 2 * (1 + 2.0 ** -20) + slack / factor + ideal * 2.0 ** -22
    assert ((scale - ideal).abs() <= room).all(), ((scale - ideal).abs() / room).max()
    unit = (scale * factor).repeat_interleave(16, -1)
    y = torch.where(unit > 0, want / unit.clamp(min=1e-300), 0.0).clamp(-6, 6)
    a = value.abs()
    half = torch.where(a < 2, 0.25, torch.where(a < 4, 0.5, 1.0)).double()  # half a step above the code; below it, less
    slack = torch.where(unit > 0, bound / unit.clamp(min=1e-300), 0.0)
    room = half * (1 + 2.0 ** -20) + slack + y.abs() * 2.0 ** -22
    assert ((value - y).abs() <= room).all(), ((value - y).abs() / room).max()
    # below a code whose neighbours are nearer downwards
    down = (y.abs() < a) & ((a == 2) | (a == 4))
    room = torch.where(a == 2, 0.25, 0.5) + slack + y.abs() * 2.0 ** -22
    assert ((a - y.abs())[down] <= room[down]).all()


def pack(x, heads, dim):
    """Rows of e2m1 bytes for x (n, heads, dim) on the CPU: nearest codes with scales next to max / 6."""
    g = x.double().unflatten(-1, (-1, 16))
    scale = (g.abs().amax(-1) / 6).clamp(max=448).float().to(torch.float8_e4m3fn)
    y = g / scale.double().clamp(min=2.0 ** -9).unsqueeze(-1)
    code = (y.abs().unsqueeze(-1) - E2M1).abs().argmin(-1) + torch.where(y < 0, 8, 0)
    code = code.view(x.shape[0], -1).to(torch.uint8)
    size = -(-heads * dim * 9 // 256) * 16
    rows = torch.zeros((x.shape[0], size), dtype=torch.uint8)
    n = heads * dim // 2
    rows[:, :n] = code[:, 0::2] | code[:, 1::2] << 4
    rows[:, n:n + heads * dim // 16] = scale.view(torch.uint8).view(x.shape[0], -1)
    return rows
