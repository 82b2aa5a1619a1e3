"""Block-scaled 8-bit floating point in 64 bits, from the format's definition, for the tests: (-1)^s 2^(e-7) (1 + f/8), or 2^-6 f/8 where e is 0; e = 15, f = 7
is NaN; times the fp32 scale of a block of 128 along K (for weights 128 x 128)."""
import torch


def _table():
    v = []
    for bits in range(128):
        e, f = bits >> 3, bits & 7
        v.append(float("nan") if bits == 127 else f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7))
    return torch.tensor(v + [-x for x in v], dtype=torch.float64)


VALUES = _table()


def blocks(size):
    return (size + 127) // 128


def decode(codes):
    return VALUES[codes.cpu().view(torch.uint8).long()]


def row_values(codes, scales):
    """codes [M, K], scales [ceil(K/128), M] -> float64 [M, K]"""
    return decode(codes) * scales.cpu().double().t().repeat_interleave(128, 1)[:, : codes.shape[1]]


def weight_values(codes, scales, n):
    """codes [.., parts * n, K], scales [.., parts * ceil(n/128), ceil(K/128)] -> float64 [.., parts * n, K]"""
    v = decode(codes)
    parts = v.shape[-2] // n
    s = scales.cpu().double().unflatten(-2, (parts, blocks(n))).repeat_interleave(128, -2)[..., :n, :].flatten(-3, -2)
    return v * s.repeat_interleave(128, -1)[..., : v.shape[-1]]


def _codes(q):
    """The nearest value's code, by distance among all of them, ties to the even code"""
    magnitudes = VALUES[:127]
    at = torch.searchsorted(magnitudes, q.abs().clamp(max=448.0))
    low, high = (at - 1).clamp(min=0), at.clamp(max=126)
    below, above = q.abs() - magnitudes[low], magnitudes[high] - q.abs()
    code = torch.where((below < above) | ((below == above) & (low % 2 == 0)), low, high)
    code = torch.where(magnitudes[high] == q.abs(), high, torch.where(q.abs() >= 448, torch.full_like(high, 126), code))
    return (code + 128 * torch.signbit(q)).to(torch.uint8)


def quantize(x, block_rows=1):
    """[N, K] -> (codes u8 [N, K], scales f32 [blocks of N, blocks of K]): both quotients rounded to fp32"""
    x = x.cpu().double()
    n, k = x.shape
    v = torch.nn.functional.pad(x, (0, -k % 128, 0, -n % block_rows)).view(-1, block_rows, blocks(k), 128)
    top = v.abs().amax((1, 3))
    fine = torch.isfinite(top)
    scales = torch.where(fine, (top.clamp(min=2.0 ** -64) / 448), float("nan")).float()
    # (a quotient of two fp32 numbers rounded to 64 bits, then to fp32, is the one rounded to fp32 at once)
    q = torch.where(fine[:, None, :, None], v / scales.double()[:, None, :, None], 0.0).float().double()
    return _codes(q).view(-1, blocks(k) * 128)[:n, :k].contiguous(), scales


def largest_of_eight(v):
    """[.., K] -> [.., ceil(K/8)]: the largest magnitude of each eight values"""
    return torch.nn.functional.pad(v.abs(), (0, -v.shape[-1] % 8)).unflatten(-1, (-1, 8)).amax(-1)


def product(a, w, n, gate=False, bias=None, residual=None):
    """a [M, K], w [N or 2N, K] as values -> (y, bound on its error: see test_gpu_fp8)"""
    y, size = a @ w.t(), a.abs() @ w.abs().t()
    bound = (130 + blocks(a.shape[1])) * 2.0 ** -23 * size + 8 * 2.0 ** -13 * (largest_of_eight(a) @ largest_of_eight(w).t())
    if gate:
        g, u, dg, du = y[:, :n], y[:, n:], bound[:, :n], bound[:, n:]
        s = g * torch.sigmoid(g)
        y, bound = s * u, 1.1 * dg * (u.abs() + du) + s.abs() * du + (s * u).abs() * (g.abs() + dg + 8) * 2.0 ** -22
    for more in (bias, residual):
        if more is not None:
            more = more.cpu().double()
            bound = bound + 2.0 ** -23 * (y.abs() + bound + more.abs())
            y = y + more
    return y, bound
