"""The sort of the (token, j) pairs by expert and the rows' way to the experts and back, from their definitions in 64 bits, for the tests."""
import torch


def sort(idx, E):
    """(counts, token_of, slot), pair after pair."""
    T, k = idx.shape
    rows = [[] for _ in range(E)]
    for p, e in enumerate(idx.reshape(-1).tolist()):
        if 0 <= e < E:
            rows[e].append(p)
    order = [p for r in rows for p in r]
    slot = [-1] * (T * k)
    for at, p in enumerate(order):
        slot[p] = at
    token_of = [p // k for p in order] + [-1] * (T * k - len(order))
    as_int = dict(dtype=torch.int32, device=idx.device)
    return (torch.tensor([len(r) for r in rows], dtype=torch.int64, device=idx.device), torch.tensor(token_of, **as_int).view(-1),
            torch.tensor(slot, **as_int).view(T, k))


def picked(rows, slot):
    """rows[slot] in 64 bits, [T, k, H], zero where a pair was dropped."""
    v = rows.double()[slot.clamp(min=0).long()]
    return torch.where((slot >= 0).unsqueeze(2), v, 0.0)


def dispatch(x, token_of):
    v = x[token_of.clamp(min=0).long()]
    return torch.where((token_of >= 0).unsqueeze(1), v, torch.zeros_like(v))


def weight_of_rows(weight, slot):
    w = torch.zeros(slot.numel(), dtype=torch.float64, device=slot.device)
    w[slot[slot >= 0].long()] = weight.double()[slot >= 0]
    return w


def half_step(dtype):
    return torch.finfo(dtype).eps / 2
