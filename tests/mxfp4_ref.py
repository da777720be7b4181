"""Rows in 4-bit floats with a power-of-two scale per 32 elements, from their definitions in 64 bits, for the tests."""
import torch

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
LOWEST = -100


def width(K):
    return 4 * -(-K // 128)


def values(packed, scale):
    """Codes [.., K / 2] and scale bytes [.., >= K / 32] -> values in 64 bits."""
    codes = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2)
    K = codes.shape[-1]
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=packed.device)
    s = scale[..., :K // 32].double()
    unit = torch.where(s == 255, float("nan"), torch.exp2(s - 127))
    return table[codes.long()] * unit.repeat_interleave(32, dim=-1)


def quantize(v):
    """fp64 rows -> (packed codes, scale bytes): the smallest power of two of which 7 reach the block's magnitude, the nearest code (ties to the
    even one, at most 6)."""
    rows, K = v.shape
    b = v.view(rows, K // 32, 32)
    a = b.abs().amax(dim=2)
    bad = ~torch.isfinite(a)
    a = torch.where(bad, 1.0, a)
    m, e = torch.frexp(a)
    e = torch.where(m > 0.875, e + 1, e) - 3
    e = torch.where(a > 0, e, LOWEST).clamp(min=LOWEST)
    assert bool(((a <= 7 * torch.exp2(e.double())) & ((a > 3.5 * torch.exp2(e.double())) | (e == LOWEST))).all())
    q = torch.where(bad.unsqueeze(2), 0.0, b / torch.exp2(e.double()).unsqueeze(2))
    levels = torch.tensor(E2M1, dtype=torch.float64, device=v.device)
    mids = (levels[1:] + levels[:-1]) / 2
    c = torch.bucketize(q.abs().contiguous(), mids)  # the number of borders below: a tie stays with the lower code
    tie = (q.abs().unsqueeze(-1) == mids).any(dim=-1)
    c = torch.where(tie & (c % 2 == 1), c + 1, c)
    c = (c + 8 * torch.signbit(q)).to(torch.uint8).view(rows, K)
    scale = torch.zeros(rows, width(K), dtype=torch.uint8, device=v.device)
    scale[:, :K // 32] = torch.where(bad, 255, e + 127).to(torch.uint8)
    return c[:, 0::2] | (c[:, 1::2] << 4), scale
