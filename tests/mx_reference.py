"""MX matrices and the token sort in 64 bits, written from their definitions, for the tests of the
operators (torch, any device)."""
import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
E4M3 = torch.tensor([m / 8 * 2.0**-6 for m in range(8)]
                    + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)][:-1], dtype=torch.float64)


def pow2(e):
    """2^e in f64, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def pad(n, to):
    return -(-n // to) * to


def quantise(x, fmt):
    """(codes [rows, padded cols], scale bytes [rows, blocks], values) of an f64 matrix that holds f32 values."""
    rows, cols = x.shape
    grid = (E2M1 if fmt == "e2m1" else E4M3).to(x.device)
    emax, sign_bit = (2, 8) if fmt == "e2m1" else (8, 128)
    wide = torch.zeros(rows, pad(cols, 128), dtype=torch.float64, device=x.device)
    wide[:, :cols] = x
    b = wide.view(rows, -1, 32)
    finite = torch.isfinite(b).all(dim=2, keepdim=True)
    b = torch.where(finite, b, torch.zeros_like(b))
    amax = b.abs().amax(dim=2, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax).exponent.long() - 1 - emax, torch.full_like(amax, -127, dtype=torch.long)).clamp(-127, 127)
    a = (b.abs() / pow2(e)).contiguous()
    mid = (grid[1:] + grid[:-1]) / 2
    lo = torch.searchsorted(mid, a)
    tie = (lo < mid.numel()) & (mid[lo.clamp(max=mid.numel() - 1)] == a)
    at = torch.where(tie & (lo % 2 == 1), lo + 1, lo)
    values = torch.where(finite, torch.copysign(grid[at], b) * pow2(e), torch.full_like(b, float("nan")))
    codes = torch.where(finite, at + sign_bit * torch.signbit(b).long(), torch.zeros_like(at))
    byte = torch.where(finite, e + 127, torch.full_like(e, 255)).squeeze(2)
    blocks = -(-cols // 32)
    return codes.view(rows, -1), byte[:, :blocks], values.view(rows, -1)[:, :cols]


def layout(codes, byte, fmt):
    """(data, scales) as the library lays them out."""
    c = codes.to(torch.uint8)
    data = c if fmt == "e4m3" else c[:, 0::2] | (c[:, 1::2] << 4)
    scales = torch.zeros(byte.shape[0], pad(byte.shape[1], 16), dtype=torch.uint8, device=byte.device)
    scales[:, : byte.shape[1]] = byte.to(torch.uint8)
    return data.contiguous(), scales


def values(data, scales, cols, fmt):
    """What data and scales stand for, in f64."""
    d = data.long()
    if fmt == "e2m1":
        d = torch.stack((d % 16, d // 16), dim=-1).flatten(-2)
        v = E2M1.to(d.device)[d % 8] * torch.where(d >= 8, -1.0, 1.0).double()
    else:
        grid = torch.cat((E4M3, torch.tensor([float("nan")], dtype=torch.float64))).to(d.device)
        v = grid[d % 128] * torch.where(d >= 128, -1.0, 1.0).double()
    s = torch.where(scales == 255, torch.full(scales.shape, float("nan"), dtype=torch.float64, device=scales.device), pow2(scales.long() - 127))
    s = s[..., : d.shape[-1] // 32].repeat_interleave(32, dim=-1)
    return (v * s)[..., :cols]


def sort_plan(idx, experts):
    """(offsets, at) of the stable counting sort, pair by pair."""
    flat = idx.reshape(-1).tolist()
    order = sorted((p for p, e in enumerate(flat) if 0 <= e < experts), key=lambda p: (flat[p], p))
    at = [-1] * len(flat)
    for row, p in enumerate(order):
        at[p] = row
    offsets = [sum(0 <= f < e for f in flat) for e in range(experts + 1)]
    return torch.tensor(offsets, dtype=torch.int32), torch.tensor(at, dtype=torch.int32).view(idx.shape)
