"""Blocks of 32 numbers that share a power of two, in 64 bits and without the library: what the microscaled tests compare with."""
import torch

GRID = {4: [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0],
        8: [m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127]}
LARGEST = {4: 2, 8: 8}      # exponent of the largest number


def split(v):
    """[.., C] -> [.., blocks, 32], the last one filled with zeros."""
    pad = -v.shape[-1] % 32
    return torch.nn.functional.pad(v, (0, pad)).unflatten(-1, (-1, 32))


def exponent_bytes(v, bits):
    """float64 [.., C] -> [.., blocks]: exponent of the largest magnitude less the format's, biased; 255 where there is no number."""
    b = split(v)
    top = b.abs().amax(-1)
    power = torch.frexp(top).exponent - 1
    e = torch.where(top > 0, (power - LARGEST[bits] + 127).clamp(min=0), 0)
    return torch.where(b.isfinite().all(-1), e, 255)


def codes(v, bits, e=None):
    """(codes [.., C] int64 with the sign as their highest bit, exponent bytes); e: given bytes."""
    e = exponent_bytes(v, bits) if e is None else e
    grid = torch.tensor(GRID[bits], dtype=torch.float64)
    border = (grid[1:] + grid[:-1]) / 2
    t = split(v) * torch.exp2(127.0 - e.double()).unsqueeze(-1)
    a = t.abs().contiguous()
    c = torch.searchsorted(border, a)
    at = c.clamp(max=len(border) - 1)
    c = torch.where((c < len(border)) & (a == border[at]) & (c % 2 == 1), c + 1, c)
    c = c + torch.signbit(t) * (8 if bits == 4 else 128)
    c = torch.where(e.unsqueeze(-1) == 255, 0, c)
    return c.flatten(-2)[..., :v.shape[-1]], e


def numbers(c, e, bits):
    """codes and bytes -> float64 [.., C]."""
    half = 8 if bits == 4 else 128
    grid = torch.tensor(GRID[bits] + [float("nan")] * (half - len(GRID[bits])), dtype=torch.float64)
    v = grid[c % half] * torch.where(c >= half, -1.0, 1.0)
    unit = torch.where(e == 255, float("nan"), torch.exp2(e.double() - 127))
    return (split(v) * unit.unsqueeze(-1)).flatten(-2)[..., :c.shape[-1]]


def pack(c, bits):
    """codes -> the tensor that the library takes."""
    if bits == 4:
        return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)
    return c.to(torch.uint8).view(torch.float8_e4m3fn)


def unpack(q):
    """the library's tensor (on the CPU) -> codes."""
    if q.dtype == torch.uint8:
        return torch.stack((q & 15, q >> 4), -1).flatten(-2).to(torch.int64)
    return q.view(torch.uint8).to(torch.int64)


def random_rows(gen, rows, cols, bits, spread=3):
    """(codes, bytes) of random rows whose blocks' exponents differ by up to `spread`."""
    v = torch.randn(rows, cols, generator=gen, dtype=torch.float64)
    v = (split(v) * torch.exp2(torch.randint(-spread, spread + 1, (rows, -(-cols // 32), 1), generator=gen).double())).flatten(-2)[..., :cols]
    return codes(v, bits)
