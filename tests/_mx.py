"""Microscaled blocks in 64 bits, plainly: the tests' references for 4-bit and 8-bit elements."""

import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [i * 2.0 ** -9 for i in range(8)] + [(8 + i % 8) * 2.0 ** (i // 8 - 9) for i in range(119)]


def rounded(x, grid, top):
    """x [rows, k] (finite): each block of 32 on its scaled grid, ties to the even code; (values, exponents [rows, blocks])."""
    grid = torch.tensor(grid, dtype=torch.float64, device=x.device)
    rows, k = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -k % 32)).view(rows, -1, 32)
    e = (torch.frexp(b.abs().amax(-1, keepdim=True)).exponent - 1 - top).clamp_min(-127)
    e = torch.where(b.abs().amax(-1, keepdim=True) == 0, torch.full_like(e, -127), e)
    y = torch.ldexp(b.abs(), -e)
    mid = (grid[1:] + grid[:-1]) / 2
    up, down = torch.bucketize(y, mid, right=True), torch.bucketize(y, mid)
    q = torch.copysign(grid[torch.where(up % 2 == 0, up, down)], b)
    return torch.ldexp(q, e).view(rows, -1)[:, :k], e[:, :, 0]


def four(x):
    return rounded(x, E2M1, 2)[0]


def eight(x):
    return rounded(x, E4M3, 8)[0]


def unpack(codes, scales, k):
    """The values of codes and scale tiles, element by element by the documented addresses."""
    rows = codes.shape[0]
    c = torch.stack((codes & 15, codes >> 4), -1).view(rows, -1).long()
    grid = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=codes.device)
    r = torch.arange(rows, device=codes.device)[:, None]
    b = torch.arange(c.shape[1], device=codes.device)[None, :] // 32
    at = (r // 128 * scales.shape[1] + b // 8) * 1024 + b % 8 // 4 * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4
    s = scales.flatten()[at].int()
    v = torch.ldexp(grid[c], s - 127)
    return torch.where(s == 255, torch.full_like(v, float("nan")), v)[:, :k]
