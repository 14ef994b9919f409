"""A row of a cache in 4 bits, from the definition: 32 columns share 2^(x - 127), x the least of 7 .. 252 for which none is above 6 times it;
a column is the nearest of 0 0.5 1 1.5 2 3 4 6 times it (of two as near the one of even place), with its sign.  A NaN or an infinity
makes all 32 NaN (x = 255)."""
import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def pack(x):
    """[..., D] -> codes [..., D / 2] and scales [..., D / 32], uint8."""
    x = x.double()
    g = x.unflatten(-1, (-1, 32))
    bad = ~g.isfinite().all(-1)
    g = torch.where(bad[..., None], torch.zeros_like(g), g)
    most = g.abs().amax(-1)
    scale = torch.full(most.shape, 7, dtype=torch.int64, device=x.device)
    for i in range(7, 252):
        scale = torch.where(most > 6.0 * 2.0 ** (i - 127), i + 1, scale)
    y = g / 2.0 ** (scale - 127).double()[..., None]
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    far = (y.abs()[..., None] - grid).abs()
    near = far.amin(-1, keepdim=True)
    place = torch.arange(8, device=x.device)
    # of the nearest, the one of even place (two of them are neighbours)
    code = torch.where(far == near, place + 8 * (place % 2), 100).amin(-1) % 8
    code = code + 8 * torch.signbit(y).long()
    code = code.flatten(-2)
    packed = (code[..., ::2] + 16 * code[..., 1::2]).to(torch.uint8)
    return packed, torch.where(bad, 255, scale).to(torch.uint8)


def values(codes, scales):
    """What they stand for, in float64."""
    b = codes.long()
    code = torch.stack((b % 16, b // 16), -1).flatten(-2)
    grid = torch.tensor(GRID + tuple(-z for z in GRID), dtype=torch.float64, device=codes.device)
    size = 2.0 ** (scales.double() - 127)
    size = torch.where(scales == 255, torch.full_like(size, float("nan")), size)
    return grid[code] * size.repeat_interleave(32, -1)
