"""The 8-bit expert path and the balance loss from their definitions in 64 bits, for the tests."""
import torch

BLOCK = 128
FLOOR = 2.0 ** -100


def e4m3(codes):
    """uint8 / float8 codes -> their values in 64 bits."""
    return codes.view(torch.float8_e4m3fn).double()


def spread(scale, dim, n):
    return scale.double().repeat_interleave(BLOCK, dim=dim).narrow(dim, 0, n)


def quantize(v):
    """fp64 rows -> (codes as uint8, scale in 64 bits), ties to even, a non-finite block: scale NaN and codes 0."""
    rows, K = v.shape
    b = torch.nn.functional.pad(v, (0, -K % BLOCK)).view(rows, -1, BLOCK)
    a = b.abs().amax(dim=2)
    bad = ~torch.isfinite(a)
    a = torch.where(bad, 1.0, a.clamp(min=FLOOR))
    q = torch.where(bad.unsqueeze(2), 0.0, b * 448 / a.unsqueeze(2))
    m, e = torch.frexp(q.abs())
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    r = torch.copysign(torch.round(q.abs() / step) * step, q)  # (a representable value: the conversion below is exact)
    codes = r.float().to(torch.float8_e4m3fn).view(torch.uint8).reshape(rows, -1)[:, :K]
    return codes.contiguous(), torch.where(bad, float("nan"), a / 448)


def bounds(counts, group_list_type, M):
    """[start, end) of every expert's rows, clamped into 0 .. M and made monotone."""
    ends, at = [], 0
    for c in counts:
        at = max(at, min(M, at + c if group_list_type else c))
        ends.append(at)
    return list(zip([0] + ends[:-1], ends))


def grouped(x, x_scale, w, w_scale, ranges):
    """(product, sum of the magnitudes of its terms) in 64 bits; rows of no expert are 0."""
    M, K = x.shape
    G, _, N = w.shape
    xv = e4m3(x) * spread(x_scale, 1, K)
    y = torch.zeros(M, N, dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(y)
    for g, (a, b) in enumerate(ranges):
        if a < b:
            wv = e4m3(w[g]) * spread(spread(w_scale[g], 0, K), 1, N)
            y[a:b] = xv[a:b] @ wv
            mag[a:b] = xv[a:b].abs() @ wv.abs()
    return y, mag


def sum_error(mag, K):
    """What fp32 sums of K terms may be off: every addition and scaling by a unit in the last place (2^-23: sums may be cut off
    instead of rounded) of the magnitudes' sum."""
    return (BLOCK + -(-K // BLOCK) + 4) * 2.0 ** -23 * mag


def balance(logits, idx, seq_list, mask, grad_loss):
    """(loss [S], counts [S, E], gradient [T, E]) in 64 bits."""
    z = logits.detach().double().requires_grad_()
    T, E = z.shape
    k = idx.shape[1]
    ends = [T] if seq_list is None else seq_list.tolist()
    losses, counts = [], []
    for a, b in zip([0] + ends[:-1], ends):
        rows = torch.arange(a, max(a, b), device=z.device)
        if mask is not None:
            rows = rows[mask[rows]]
        zr = z[rows]
        some = (zr != -float("inf")).any(dim=1, keepdim=True)
        p = torch.where(some, torch.softmax(torch.where(some, zr, 0.0), dim=1), 0.0)
        i = idx[rows].long().reshape(-1)
        c = torch.bincount(i[(i >= 0) & (i < E)], minlength=E)
        n = rows.numel()
        losses.append(E / (k * n * n) * (c.double() * p.sum(dim=0)).sum() if n else z.sum() * 0)
        counts.append(c)
    loss = torch.stack(losses)
    (grad,) = torch.autograd.grad(loss, z, grad_loss.double(), allow_unused=True)
    return loss.detach(), torch.stack(counts), torch.zeros_like(z) if grad is None else grad
