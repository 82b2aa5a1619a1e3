"""MXFP4 in 64 bits, from the format's definition, for the tests: a value is (-1)^s 2^(e-1) (1 + f/2), or f/2 where e is 0, times
2^(byte - 127) of its block of 32; byte 255 makes the block NaN."""
import torch

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def scale_bytes(k):
    return (k // 32 + 15) // 16 * 16


def values(codes, scales):
    """codes u8 [.., K/2], scales u8 [.., stride] -> float64 [.., K]"""
    codes, scales = codes.cpu(), scales.cpu()
    nibble = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    v = VALUES[nibble & 7] * torch.where(nibble >= 8, -1.0, 1.0).double()
    byte = scales[..., : v.shape[-1] // 32].long().repeat_interleave(32, -1)
    return torch.where(byte == 255, torch.full_like(v, float("nan")), v * torch.exp2((byte - 127).double()))


def quantize(x):
    """fp16 [rows, K] -> (codes, scales) on the CPU, block by block: the nearest value by its distance, ties to the even code."""
    x = x.cpu().double()
    rows, k = x.shape
    blocks = x.view(rows, k // 32, 32)
    top = blocks.abs().amax(-1)
    finite = torch.isfinite(top)
    safe = torch.where(finite & (top > 0), top, torch.ones_like(top))
    exponent = torch.frexp(safe)[1].long() - 3  # floor(log2(top)) - 2
    byte = torch.where(finite, torch.where(top > 0, exponent + 127, torch.full_like(exponent, 127)), torch.full_like(exponent, 255))
    scaled = torch.where(finite[..., None], blocks, torch.zeros_like(blocks)).abs() / torch.exp2(exponent.double())[..., None]
    away = (scaled[..., None] - VALUES).abs()
    # of two nearest codes the even one: an odd code's distance counts as a hair more (next to a tie, which is at 0.25 or above, fp16
    # numbers are 2^-13 apart)
    code = (away + torch.tensor([0.0, 1.0] * 4, dtype=torch.float64) * 2.0**-40).argmin(-1)
    code = torch.where(finite[..., None], code + 8 * torch.signbit(blocks), torch.zeros_like(code)).view(rows, k // 2, 2).to(torch.uint8)
    scales = torch.full((rows, scale_bytes(k)), 127, dtype=torch.uint8)
    scales[:, : k // 32] = byte.to(torch.uint8)
    return code[..., 0] | code[..., 1] << 4, scales


def product(a, w):
    """(A . W^T, sum of the products' magnitudes) of value matrices in 64 bits"""
    return a @ w.T, a.abs() @ w.abs().T


def silu(g):
    return g * torch.sigmoid(g)


def tolerance(y, magnitude, k):
    """How far fp16(fp32 sum) may be from y.  The sum is added up in at most K/32 + 16 steps (an MFMA takes 64 values or more, up to 16
    partial sums meet behind it), each off by at most one unit of fp32 in the last place of what has been added so far -- which
    never exceeds the sum of the magnitudes -- : 2^-23 of it a step; then half a step of fp16, 2^-11 of y, or of its smallest number."""
    return (k // 32 + 16) * 2.0**-23 * magnitude + 2.0**-11 * y.abs() * 1.001 + 2.0**-25


def gated(g, u, g_mag, u_mag, k):
    """(SiLU(g) u, its tolerance) from the exact products: the fp32 errors of either factor (SiLU's slope is below 1.1), 2^-18 of the
    result for exp, the division and two products in fp32 (exp's argument is rounded: 2^-24 |g| below 2^-20 for |g| < 16, beyond that SiLU
    is g or next to nothing), half a step of fp16."""
    steps = (k // 32 + 16) * 2.0**-23
    y = silu(g) * u
    return y, 1.1 * steps * g_mag * (u.abs() + steps * u_mag) + silu(g).abs() * steps * u_mag + 2.0**-18 * y.abs() + 2.0**-11 * y.abs() * 1.001 + 2.0**-25
