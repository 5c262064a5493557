"""The cache in 4 and 8 bits by its definition: the nearest code to each element, what
codes stand for, and where they lie in a page."""
import torch

GRID = {4: [0, 0.5, 1, 1.5, 2, 3, 4, 6],
        8: [m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]}
LIMIT = {4: 7.0, 8: 448.0}
P2 = torch.tensor([0.0] + [2.0 ** (b - 127) for b in range(1, 255)] + [float("nan")], dtype=torch.float64)


def page_bytes(d, bits):
    return 64 * d * bits // 8 + 2 * d


def quantise(x, bits):
    """(codes, scale bytes) of rows x [..., d]: each group's smallest power of two that
    takes its largest magnitude to the limit, then the nearest code, ties to the even one."""
    x = x.double().unflatten(-1, (-1, 32))
    grid = torch.tensor(GRID[bits], dtype=torch.float64)
    big = x.abs().amax(-1, keepdim=True)
    b = (big > LIMIT[bits] * P2[1:255]).sum(-1, keepdim=True) + 1
    b = torch.where(big == 0, 0, b)
    b = torch.where(big <= 1.75 * 2.0 ** 127, b, 255)
    a = torch.where((b == 0) | (b == 255), 0.0, x.abs() / P2[b.clamp(1, 254)])
    mid = (grid[1:] + grid[:-1]) / 2
    at = torch.bucketize(a, mid)
    tie = (at < len(mid)) & (a == mid[at.clamp_max(len(mid) - 1)])
    at = torch.where(tie & (at % 2 == 1), at + 1, at)
    at = at + torch.where((b != 0) & (b != 255) & x.signbit(), 2 ** (bits - 1), 0)
    return at.flatten(-2).to(torch.uint8), b.squeeze(-1).to(torch.uint8)


def values(codes, b, bits):
    """What they stand for, in 64 bits (a code of e4m3 that is no number: NaN)."""
    grid = torch.tensor(GRID[bits] + [float("nan")] * (bits == 8), dtype=torch.float64)
    v = torch.cat((grid, -grid))[codes.long()]
    return (v.unflatten(-1, (-1, 32)) * P2[b.long()][..., None]).flatten(-2)


def _byte(x, lane):
    return (x // 16 * 64 + lane) * 16 + x % 16


def places(d, bits, keys):
    """Of a page's tokens and elements: each code's byte [64, d], whether it is the byte's
    high half (4 bits), and each group's byte [64, d / 32]."""
    j, t, g = torch.arange(64)[:, None], torch.arange(d)[None], torch.arange(d // 32)[None]
    base = 64 * d * bits // 8
    if keys:
        mt, l16 = 2 * (j // 32) + j // 4 % 2, 4 * (j % 32 // 8) + j % 4
        at = _byte((mt * (d // 4) + t % (d // 4)) * bits // 8, l16 + 16 * (t // (d // 4)))
        return at, (t % 2 == 1).expand(64, d), base + (l16 + 16 * g) * 4 + mt
    at = _byte(j // 32 * (d * bits // 16) + (t // 16 * 8 + j % 8) * bits // 8, t % 16 + 16 * (j % 32 // 8))
    return at, (j % 2 == 1).expand(64, d), base + (j // 8 * (d // 32) + g) * 8 + j % 8


def write(page, slots, codes, b, bits, keys):
    """Tokens `slots` [n] of one KV head's page (a view of its bytes): codes [n, d], b [n, d / 32]."""
    at, high, sc = places(codes.shape[1], bits, keys)
    at, high, sc = at[slots], high[slots], sc[slots]
    page[sc] = b
    if bits == 8:
        page[at] = codes
        return
    for half in (False, True):
        where, c = at[high == half], codes[high == half]
        page[where] = (page[where] & 15) | (c << 4) if half else (page[where] & 240) | c


def rows(page, bits, d, keys):
    """A KV head's page (or pages [..., bytes]) as values [..., 64, d]."""
    at, high, sc = places(d, bits, keys)
    c = page[..., at]
    if bits == 4:
        c = torch.where(high, c >> 4, c & 15)
    return values(c, page[..., sc], bits)
