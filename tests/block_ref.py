"""Block-scaled rows in 64 bits: what data and scales stand for, and whether they are the rounding of given values.

Elements and scales are checked as roundings: a result computed from values that are known to a relative `slack` has to be the
rounding of a value inside that interval, so nothing but a value next to a border between two codes may take either."""
import math

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
BLOCK = {"mxfp8": 32, "mxfp4": 32, "nvfp4": 16}


def grid_of(fmt):
    """the element values of a format from 0 up, a code each"""
    if fmt != "mxfp8":
        return torch.tensor(E2M1, dtype=torch.float64)
    return torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()


def nearest(v, grid):
    """codes of the nearest grid values to |v|, ties to the even code, beyond the last saturated"""
    grid = grid.to(v.device)
    mid = (grid[1:] + grid[:-1]) / 2
    a = v.abs().contiguous()
    up = torch.bucketize(a, mid, right=True)          # midpoints up to a, itself among them
    tie = (up > 0) & (a == mid[(up - 1).clamp(min=0)])
    return torch.where(tie & (up % 2 == 1), up - 1, up)


def unpack(data, fmt):
    """element codes [rows, K] (sign above the magnitude's bits)"""
    data = data.view(torch.uint8)
    if fmt == "mxfp8":
        return data
    return torch.stack((data & 15, data >> 4), -1).reshape(data.shape[0], -1)


def elements(data, fmt):
    codes = unpack(data, fmt)
    bits = 7 if fmt == "mxfp8" else 3
    grid = torch.cat((grid_of(fmt), torch.tensor([math.nan], dtype=torch.float64)))[: 1 << bits].to(codes.device)
    v = grid[(codes & ((1 << bits) - 1)).long()]
    return torch.where(codes >> bits != 0, -v, v)


def scale_values(scales, fmt):
    raw = scales.view(torch.uint8)
    if fmt == "nvfp4":
        return raw.view(torch.float8_e4m3fn).double()
    return torch.where(raw == 255, math.nan, torch.exp2(raw.double() - 127.0))


def values(data, scales, fmt, g=1.0):
    e = elements(data, fmt)
    return (e.view(e.shape[0], -1, BLOCK[fmt]) * (scale_values(scales, fmt) * g).unsqueeze(-1)).reshape(e.shape)


def _scale_codes(most, fmt, g):
    if fmt == "nvfp4":
        return nearest((most / (6.0 * g)).clamp(max=448.0), grid_of("mxfp8"))
    exponent = torch.frexp(most).exponent - 1 - (8 if fmt == "mxfp8" else 2) + 127
    return torch.where(most == 0, 0, exponent.clamp(0, 254))


def assert_quantised(data, scales, want, fmt, g=1.0, slack=0.0, tiny=0.0):
    """data, scales are the quantised form of `want` [rows, N] (64 bits), known to a relative `slack` and an absolute `tiny`;
    columns behind N are zeros"""
    b = BLOCK[fmt]
    codes = unpack(data, fmt)
    rows, k = codes.shape
    v = torch.zeros((rows, k), dtype=torch.float64, device=want.device)
    v[:, : want.shape[1]] = want
    v = v.view(rows, k // b, b)
    most = v.abs().amax(-1)
    lost = ~torch.isfinite(v).all(-1)
    raw = scales.view(torch.uint8).to(torch.int64)
    assert torch.equal(raw[lost], torch.full_like(raw[lost], 0x7F if fmt == "nvfp4" else 0xFF))
    low = _scale_codes((most * (1 - slack) - tiny).clamp(min=0), fmt, g)
    high = _scale_codes(most * (1 + slack) + tiny, fmt, g)
    fine = ~lost
    assert bool(((raw >= low) & (raw <= high))[fine].all()), "scales"
    codes = codes.view(rows, k // b, b).to(torch.int64)
    sign_bit = 128 if fmt == "mxfp8" else 8
    assert int(codes[lost].abs().sum()) == 0
    unit = scale_values(scales, fmt) * g
    unit = torch.where(unit == 0, math.inf, unit).unsqueeze(-1)
    grid = grid_of(fmt)
    # nvfp4 multiplies by the f32 reciprocal of scale * g: two roundings more, and one of the product
    slack = slack + (3 * 2.0 ** -24 if fmt == "nvfp4" else 0.0)
    lo = nearest(((v.abs() * (1 - slack) - tiny).clamp(min=0)) / unit, grid)
    hi = nearest((v.abs() * (1 + slack) + tiny) / unit, grid)
    got = codes & (sign_bit - 1)
    ok = (got >= lo) & (got <= hi) & ((got == 0) | ((codes & sign_bit != 0) == (v < 0)))
    assert bool(ok[fine].all()), f"{int((~ok[fine]).sum())} elements of {int(ok[fine].numel())}"


def buffers(rows, k, fmt, device, extra_rows=0):
    """data and scales for rows of K values, filled with a pattern that is no result, and `extra_rows` rows behind them"""
    data = torch.full((rows + extra_rows, k if fmt == "mxfp8" else k // 2), 0xA5, dtype=torch.uint8, device=device)
    return data, torch.full((rows + extra_rows, k // BLOCK[fmt]), 0xA5, dtype=torch.uint8, device=device)


def padded(n, fmt):
    return -(-n // BLOCK[fmt]) * BLOCK[fmt]
