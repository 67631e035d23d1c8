"""Microscaled floating point in 64 bits, written from the formats: tables of the elements' values, nearest by comparison."""
import torch

E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8)][:127]
TABLE = {4: torch.tensor(E2M1, dtype=torch.float64), 8: torch.tensor(E4M3, dtype=torch.float64)}


def nearest_code(a, table):
    """Index of the entry nearest to ``a >= 0``, ties to the even index."""
    hi = torch.searchsorted(table, a).clamp(1, len(table) - 1)
    lo = hi - 1
    dlo, dhi = (a - table[lo]).abs(), (table[hi] - a).abs()
    return torch.where((dhi < dlo) | ((dhi == dlo) & (hi % 2 == 0)), hi, lo)


def blocks(x, bits):
    """x [M, K] on any device -> (codes [M, K] with the sign in the top bit, scale bytes [M, K/32], values [M, K]), on the CPU in 64 bits.
    The scale is found by trying every power of two."""
    b = x.detach().cpu().double().reshape(x.shape[0], x.shape[1] // 32, 32)
    table = TABLE[bits]
    finite = torch.isfinite(b).all(-1)
    a = torch.where(finite, b.abs().amax(-1), torch.zeros(b.shape[:2], dtype=torch.float64))
    limits = table[-1] * 2.0 ** torch.arange(-127, 128, dtype=torch.float64)
    byte = torch.searchsorted(limits, a)                      # the first power that holds the largest value
    scale = 2.0 ** (byte.double() - 127)
    u = torch.where(finite.unsqueeze(-1), b, torch.zeros_like(b)) / scale.unsqueeze(-1)
    code = nearest_code(u.abs(), table)
    value = torch.copysign(table[code], u) * scale.unsqueeze(-1)
    value = torch.where(finite.unsqueeze(-1), value, torch.full_like(value, float("nan")))
    code = code + (len(table) + (bits == 8)) * (torch.signbit(u)).long()
    return code.reshape(x.shape), torch.where(finite, byte, torch.full_like(byte, 255)), value.reshape(x.shape)


def pack4(code):
    c = code.reshape(*code.shape[:-1], code.shape[-1] // 2, 2).to(torch.uint8)
    return c[..., 0] | (c[..., 1] << 4)


def random_weight(n, k, gen, spread=3):
    """Any codes, scales of a few powers of two: (packed [N, K/2], scales [N, K/32], values [N, K] in 64 bits)."""
    code = torch.randint(0, 16, (n, k), generator=gen)
    byte = torch.randint(127 - spread, 128 + spread, (n, k // 32), generator=gen)
    v = TABLE[4][code & 7] * torch.where(code > 7, -1.0, 1.0).double() * (2.0 ** (byte.double() - 127)).repeat_interleave(32, dim=1)
    return pack4(code), byte.to(torch.uint8), v


def gated(h, limit, alpha=1.702):
    g, u = h.chunk(2, -1)
    if limit:
        g, u = torch.where(g > limit, torch.full_like(g, limit), g), u.clamp(-limit, limit)
        return (u + 1) * g / (1 + torch.exp(-alpha * g))
    return g / (1 + torch.exp(-g)) * u
