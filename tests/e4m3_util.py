"""The 8-bit row format from its definition, in 64 bits and on the CPU or the GPU alike."""
import torch

D = 128
CODE = {torch.float16: 0, torch.bfloat16: 1}
LARGEST = {torch.float16: 1.875 * 2.0 ** 15, torch.bfloat16: 1.875 * 2.0 ** 127}
# magnitudes of the codes 0 .. 126
GRID = torch.tensor([(1 + m / 8) * 2.0 ** (e - 7) if e else m / 8 * 2.0 ** -6 for e in range(16) for m in range(8)][:127],
                    dtype=torch.float64)


def scales_of(x):
    """Bytes of the scales of rows x [..., 128]: by trying every exponent, 255 where the row is not finite."""
    top = x.double().abs().amax(dim=-1)
    bad = ~torch.isfinite(x.double()).all(dim=-1)
    steps = 448.0 * torch.pow(2.0, torch.arange(-126, 121, dtype=torch.float64, device=x.device))
    byte = 1 + (top[..., None] > steps).sum(dim=-1)
    return torch.where(bad, 255, byte).to(torch.uint8)


def hold(x, largest):
    """Rows x [..., 128] of any float type as (codes, scale bytes), both uint8: every element goes to the nearest code, of
    two as near the even one."""
    byte = scales_of(x)
    bad = byte == 255
    y = torch.where(bad[..., None], 0.0, x.double().clamp(-largest, largest))
    y = y / torch.pow(2.0, byte.double() - 127)[..., None].masked_fill(bad[..., None], 1.0)
    grid = GRID.to(x.device)
    at = torch.bucketize(y.abs(), grid).clamp(1, 126)    # grid[at - 1] < |y| <= grid[at]
    below, above = y.abs() - grid[at - 1], grid[at] - y.abs()
    code = torch.where((below < above) | ((below == above) & (at % 2 == 1)), at - 1, at)
    code = torch.where(y.abs() == 0.0, 0, code)
    sign = (torch.signbit(x.double()) & ~bad[..., None]).long() * 128
    return (code + sign).to(torch.uint8), byte


def values(codes, byte):
    """What codes [..., 128] and scale bytes stand for, in 64 bits."""
    scale = torch.pow(2.0, byte.double() - 127)
    scale = torch.where(byte == 255, float("nan"), scale)
    magnitude = torch.cat([GRID, torch.tensor([float("nan")], dtype=torch.float64)]).to(codes.device)[(codes & 127).long()]
    return torch.where(codes >= 128, -magnitude, magnitude) * scale[..., None]


def norm_rope(x, rope, at, eps):
    """Key rows x [tokens, sequences, heads, 128] as the cache write normalises and rotates them, in 32 bits with one rounding
    an operation: squares added in order by eights, the sixteen sums as a tree.  at: positions [tokens, sequences]."""
    x = x.float()
    s = torch.zeros(x.shape[:-1] + (16,), dtype=torch.float32, device=x.device)
    for e in range(8):
        q = x[..., e::8]
        s = s + q * q
    while s.shape[-1] > 1:
        s = s[..., 0::2] + s[..., 1::2]
    y = x * (1.0 / ((s / 128.0).sqrt() + torch.tensor(eps, dtype=torch.float32, device=x.device)))
    turn = rope.float()[at][:, :, None]
    a, b, c, d = y[..., 0::2], y[..., 1::2], turn[..., 0::2], turn[..., 1::2]
    return torch.stack([a * c - b * d, a * d + b * c], dim=-1).flatten(-2)


def rope_table(positions, dtype):
    rate = 1.0e6 ** (-2.0 * torch.arange(D // 2, dtype=torch.float64) / D)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * rate
    return torch.stack([angle.cos(), angle.sin()], dim=-1).view(positions, D).to(dtype)


def rows(gen, shape, dtype, spread=1.0):
    """Random rows [..., 128] whose magnitudes differ from row to row."""
    x = torch.randn((*shape, D), generator=gen, dtype=torch.float32) * torch.randn((*shape, 1), generator=gen).mul_(spread).exp_()
    return x.to(dtype)
