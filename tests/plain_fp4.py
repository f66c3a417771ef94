"""Rows held in microscaled 4-bit floating point, restated in float64 from the definition: blocks of 32 values, a block's scale
the smallest power of two X with max|x| <= 7 X (2^-127 at least), every x / X to the nearest of the format's values, ties to the
code with an even number, to 6 beyond.  Codes: low half of a byte first.  Scales: tiles of 128 rows x 4 blocks in 512 bytes."""

import math

import torch

GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def scale_exponents(x):
    """[R, blocks] exponents of the scales of float64 rows; a block that holds a value that is not finite: 128 (NaN)."""
    r, k = x.shape
    blocks = -(-k // 32)
    top = torch.nn.functional.pad(x.double(), (0, blocks * 32 - k)).view(r, blocks, 32).abs().amax(-1)
    part, e = torch.frexp(top)  # top = part 2^e with 1/2 <= part < 1, and 7 2^n = 7/8 2^(n + 3)
    n = torch.where(part > 0.875, e - 2, e - 3)
    n = torch.where(top == 0, torch.full_like(n, -127), n).clamp(min=-127)
    return torch.where(torch.isfinite(top), n, torch.full_like(n, 128)).int()


def round_with(x, exponents):
    """What float64 rows are rounded to with these scales, float64."""
    r, k = x.shape
    unit = torch.ldexp(torch.ones(exponents.shape, dtype=torch.float64), exponents)
    unit = torch.where(exponents == 128, torch.full_like(unit, math.nan), unit).repeat_interleave(32, dim=1)[:, :k]
    q = (x.double() / unit).abs()
    grid = torch.tensor(GRID, dtype=torch.float64)
    best = torch.zeros_like(q)
    far = torch.full_like(q, math.inf)
    for n in (0, 2, 4, 6, 1, 3, 5, 7):  # the even codes first: a tie stays with them
        d = (q - grid[n]).abs()
        best, far = torch.where(d < far, grid[n], best), torch.minimum(d, far)
    best = torch.where(q > 6, grid[7], best)
    return torch.copysign(best, x.double()) * unit


def rounded(x):
    return round_with(x, scale_exponents(x))


def read(codes, scales, width):
    """The values that codes and scales stand for, float64 on the CPU, and the scales' bytes [R, blocks]."""
    codes, scales = codes.cpu(), scales.cpu()
    r, blocks = codes.shape[0], -(-width // 32)
    nibbles = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(r, -1)
    grid = torch.tensor(GRID + [-g for g in GRID], dtype=torch.float64)
    i, j = torch.arange(r)[:, None], torch.arange(blocks)[None, :]
    byte = scales.reshape(scales.shape[0], scales.shape[1], 512)[i // 128, j // 4, 16 * (i % 32) + 4 * (i % 128 // 32) + j % 4]
    unit = torch.ldexp(torch.ones(r, blocks, dtype=torch.float64), byte.int() - 127)
    unit = torch.where(byte == 255, torch.full_like(unit, math.nan), unit)
    return (grid[nibbles.int()] * unit.repeat_interleave(32, dim=1))[:, :width], byte


def between(x, slack):
    """For float64 rows known to within ``slack`` (absolute, per value): the lowest and highest value that each may be rounded
    to, with a block's scale that of either end."""
    lo, hi = x - slack, x + slack
    ends = [scale_exponents((x.abs() - slack).clamp(min=0)), scale_exponents(x.abs() + slack)]
    all_of = [round_with(v, e) for v in (lo, hi) for e in ends]
    return torch.stack(all_of).amin(0), torch.stack(all_of).amax(0)
