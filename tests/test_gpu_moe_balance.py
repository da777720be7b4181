"""The router's balance loss, its counts and its gradient against their definitions in 64 bits, and against differences."""
import pytest
import torch

import ascend_kernel_b200 as ak
from tests import fp8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _router(T, E, k, dtype, seed=0):
    gen = _gen(seed)
    logits = (torch.randn(T, E, generator=gen, device=DEV) * 2 + torch.randn(E, generator=gen, device=DEV)).to(dtype)
    idx = logits.float().topk(k, dim=1).indices.to(torch.int32) if T else torch.zeros(0, k, dtype=torch.int32, device=DEV)
    return logits, idx


def _check(logits, idx, seq_list=None, mask=None, seed=0):
    S = 1 if seq_list is None else seq_list.numel()
    g = torch.rand(S, generator=_gen(seed), device=DEV) + 0.5
    leaf = logits.clone().requires_grad_()
    loss, counts = ak.moe_balance_loss(leaf, idx, seq_list, mask)
    (grad,) = torch.autograd.grad(loss, leaf, g)
    want, want_counts, want_grad = R.balance(logits, idx, seq_list, mask, g)
    T, E = logits.shape
    assert loss.dtype == torch.float32 and grad.dtype == logits.dtype and counts.dtype == torch.int64
    assert torch.equal(counts, want_counts)
    # A probability: the difference of two logits, its product with log2(e), the power of two (2 units), the sum over E experts
    # (a lane's 32 and five steps at most) and the reciprocal: the first two scale with the exponent's size, 2 * 126 at most where
    # the result is not flushed.  The sum over a sequence's tokens: one rounding for each of the at most T / (32 * 148) + 1 tokens a
    # warp adds up, and some more joining.  All terms are positive, so the relative errors carry over to the loss.
    z = logits.float().masked_fill(~torch.isfinite(logits.float()), 0)
    span = float((z.amax(dim=1) - z.amin(dim=1)).clamp(max=126).max()) if T else 0.0
    rel_p = (2 * span + 50) * 2.0 ** -24
    rel = rel_p + (T / 4736 + 64) * 2.0 ** -24
    assert bool(((loss.double() - want).abs() <= rel * want + 1e-38).all()), (loss.double() - want, rel * want)
    # The gradient p F' with F' = F - sum F p: p's error, and F's own sum's
    seq = torch.zeros(T, dtype=torch.long, device=DEV) if seq_list is None else torch.searchsorted(seq_list, torch.arange(T, device=DEV), right=True)
    inside = seq < S
    seq = seq.clamp(max=S - 1)
    n = torch.stack([((seq == s) & inside & (mask if mask is not None else inside)).sum() for s in range(S)]).clamp(min=1)
    f = want_counts.double() * E / (idx.shape[1] * n.unsqueeze(1)) - 1
    zz = logits.double()
    some = (zz != -float("inf")).any(dim=1, keepdim=True)
    p = torch.where(some, torch.softmax(torch.where(some, zz, 0.0), dim=1), 0.0)
    size = (f.abs()[seq] + (f.abs()[seq] * p).sum(dim=1, keepdim=True)) * p * (g.double() / n)[seq].unsqueeze(1)
    # (the 64-bit form takes the difference of F + 1: about E <= 1024 roundings of 2^-53 of that, which is all there is where F is 0)
    oracle = 2.0 ** -42 * p * ((1 + f.abs())[seq].amax(dim=1, keepdim=True) * (g.double() / n)[seq].unsqueeze(1))
    bound = oracle + (2 * rel_p + 50 * 2.0 ** -24) * size + torch.finfo(logits.dtype).eps / 2 * want_grad.abs() * (1 + 1e-3) + 1e-38
    assert bool(((grad.double() - want_grad).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (7, 4, 4), (100, 60, 6), (509, 64, 2), (333, 257, 8), (64, 1024, 32),
                                   (1000, 1000, 3), (41, 1021, 5), (4096, 256, 8), (9000, 160, 6), (130, 96, 1)])
def test_one_sequence(T, E, k, dtype):
    _check(*_router(T, E, k, dtype, seed=T + E))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ends", [[1], [0], [0, 0, 5], [300, 300, 301, 333], [10, 20, 30, 40, 50, 60, 70], [333], [200], [1, 2, 3, 4]])
def test_sequences(ends, dtype):
    """Empty ones, ones that end inside a CTA's range, tokens behind the last."""
    logits, idx = _router(333, 64, 4, dtype, seed=len(ends))
    _check(logits, idx, torch.tensor(ends, dtype=torch.int64, device=DEV))


def test_many_sequences():
    gen = _gen(5)
    logits, idx = _router(6000, 128, 8, torch.bfloat16)
    ends = torch.randint(0, 6001, (700,), generator=gen, device=DEV).sort().values
    _check(logits, idx, ends)


@pytest.mark.parametrize("kept", [0.0, 0.5, 1.0])
def test_masked_tokens(kept):
    """Masked rows hold anything, NaN too; a sequence may have no token left."""
    logits, idx = _router(200, 64, 2, torch.float32, seed=3)
    mask = torch.rand(200, generator=_gen(4), device=DEV) < kept
    mask[50:90] = False
    seq_list = torch.tensor([50, 90, 180], dtype=torch.int64, device=DEV)
    dirty = torch.where(mask.unsqueeze(1), logits, float("nan"))
    leaf = dirty.clone().requires_grad_()
    loss, counts = ak.moe_balance_loss(leaf, idx, seq_list, mask)
    loss.sum().backward()
    want, want_counts, want_grad = R.balance(logits, idx, seq_list, mask, torch.ones(3, device=DEV))
    assert torch.equal(counts, want_counts) and bool(loss.detach()[1] == 0)
    # (fp32: a few dozen roundings of 2^-24)
    assert bool(((loss.double() - want).abs() <= 2.0 ** -17 * want).all())
    assert bool((leaf.grad[~mask] == 0).all()) and bool((leaf.grad[180:] == 0).all())
    assert bool(((leaf.grad.double() - want_grad).abs() <= 2.0 ** -17 * 64 / 20).all())
    _check(logits, idx, seq_list, mask)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("E,k", [(4, 2), (16, 16), (32, 3), (40, 5), (64, 32), (68, 4), (72, 8), (128, 6), (136, 1), (512, 4), (520, 2)])
def test_every_width_of_a_row(E, k, dtype):
    """Rows of 8, 16 and 32 lanes and of several loads a lane, with sequences that end inside a warp's tokens and a mask."""
    T = 403
    logits, idx = _router(T, E, k, dtype, seed=E)
    ends = torch.tensor([1, 34, 34, 291, 399], dtype=torch.int64, device=DEV)
    mask = torch.rand(T, generator=_gen(E + 1), device=DEV) < 0.7
    _check(logits, idx, ends, mask, seed=3)


def test_experts_that_are_masked_out_and_rows_without_any():
    for lowest in (-float("inf"), torch.finfo(torch.bfloat16).min):
        logits, idx = _router(50, 24, 2, torch.bfloat16, seed=6)
        logits[:, 5] = lowest
        logits[7, :] = lowest
        logits[8, 1:] = lowest
        if lowest == -float("inf"):
            _check(logits, idx)
        else:  # differences that overflow, and a row of equal logits
            leaf = logits.clone().requires_grad_()
            loss, _ = ak.moe_balance_loss(leaf, idx)
            loss.sum().backward()
            want, _, want_grad = R.balance(logits, idx, None, None, torch.ones(1, device=DEV))
            assert bool(((loss.double() - want).abs() <= 2.0 ** -17 * want).all())
            assert bool(((leaf.grad.double() - want_grad).abs() <= 2.0 ** -8 * want_grad.abs() + 2.0 ** -17).all())


def test_a_nan_or_infinite_logit_is_not_hidden():
    for bad in (float("nan"), float("inf")):
        logits, idx = _router(40, 16, 2, torch.float32, seed=7)
        logits[21, 3] = bad
        seq_list = torch.tensor([20, 40], dtype=torch.int64, device=DEV)
        leaf = logits.clone().requires_grad_()
        loss, _ = ak.moe_balance_loss(leaf, idx, seq_list)
        loss.sum().backward()
        assert bool(torch.isfinite(loss[0])) and bool(torch.isnan(loss[1]))
        assert bool(torch.isnan(leaf.grad[21]).all()) and bool(torch.isfinite(leaf.grad[:21]).all()) and bool(torch.isfinite(leaf.grad[22:]).all())


def test_dropped_pairs_and_the_same_expert_twice():
    logits, idx = _router(30, 8, 3, torch.float32, seed=8)
    idx[3, 1], idx[4, 0], idx[5, 2] = -1, 8, 2 ** 31 - 1
    idx[6, :] = 2
    _check(logits, idx)


def test_gradient_against_differences():
    logits, idx = _router(12, 6, 2, torch.float32, seed=9)
    seq_list = torch.tensor([5, 12], dtype=torch.int64, device=DEV)
    w = torch.tensor([0.7, -1.3], device=DEV)
    leaf = logits.clone().requires_grad_()
    (ak.moe_balance_loss(leaf, idx, seq_list)[0] * w).sum().backward()
    step = 2.0 ** -6
    for t in range(12):
        for e in range(6):
            up, down = logits.clone(), logits.clone()
            up[t, e] += step
            down[t, e] -= step
            d = [(ak.moe_balance_loss(z, idx, seq_list)[0].double() * w.double()).sum() for z in (up, down)]
            # the losses are good to about 2^-20, the third derivative is at most of the size 6 / n, n >= 5
            assert abs(float((d[0] - d[1]) / (2 * step)) - float(leaf.grad[t, e])) <= 2.0 ** -20 * 4 / step + 2 * step ** 2


def test_an_even_load_keeps_its_digits():
    """Counts that differ by a few of many: the gradient is a small difference of numbers near 1."""
    T, E, k = 8192, 16, 2
    gen = _gen(10)
    logits = torch.randn(T, E, generator=gen, device=DEV) * 0.1
    idx = torch.stack([torch.arange(T, device=DEV) % E, (torch.arange(T, device=DEV) + 1) % E], dim=1).to(torch.int32)
    idx[0, 0] = 5
    _check(logits, idx)


def test_no_tokens():
    logits, idx = _router(0, 16, 2, torch.bfloat16)
    leaf = logits.requires_grad_()
    loss, counts = ak.moe_balance_loss(leaf, idx, torch.tensor([0, 0], dtype=torch.int64, device=DEV))
    loss.sum().backward()
    assert loss.tolist() == [0, 0] and int(counts.sum()) == 0 and leaf.grad.shape == (0, 16)


def test_an_invalid_list_is_cut_and_reported():
    logits, idx = _router(50, 16, 2, torch.float32, seed=11)
    leaf = logits.requires_grad_()
    loss, counts = ak.moe_balance_loss(leaf, idx, torch.tensor([20, 70], dtype=torch.int64, device=DEV))
    loss.sum().backward()
    assert ak.last_status(clear=True) == (1, 1)
    assert int(counts[1].sum()) == 60  # cut to the 50 tokens there are
    ak.moe_balance_loss(leaf, idx, torch.tensor([30, 20, 50], dtype=torch.int64, device=DEV))
    assert ak.last_status(clear=True) == (1, 1)


def test_the_same_bits_each_time():
    logits, idx = _router(5000, 256, 8, torch.bfloat16, seed=12)
    first = ak.moe_balance_loss(logits, idx)[0]
    for _ in range(5):
        assert torch.equal(ak.moe_balance_loss(logits, idx)[0], first)


def test_behind_the_router_in_a_captured_graph():
    """Route, loss and gradient of one step in a graph, replayed on other logits."""
    def step(z):
        idx, weight, counts, _, _ = ak.ops.moe_route(z.detach(), 4)
        leaf = z.detach().requires_grad_()
        loss, seen = ak.moe_balance_loss(leaf, idx)
        (g,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
        return loss.detach(), seen, counts, g

    a, b = (_router(300, 32, 4, torch.bfloat16, seed=s)[0] for s in (13, 14))
    want = step(b)
    assert torch.equal(want[1][0], want[2])
    buf = a.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(buf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(buf)
    buf.copy_(b)
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_offsets_behind_31_bits():
    """More than 2^31 logits: the last sequence against a call on its tokens alone."""
    T, E, tail = 2 ** 21 + 77, 1024, 500
    logits = torch.randn(T, E, device=DEV, dtype=torch.bfloat16, generator=_gen(15))
    idx = torch.randint(0, E, (T, 2), generator=_gen(16), device=DEV).to(torch.int32)
    g = torch.tensor([0.0, 1.0], device=DEV)
    leaf = logits.requires_grad_()
    loss, counts = ak.moe_balance_loss(leaf, idx, torch.tensor([T - tail, T], dtype=torch.int64, device=DEV))
    (grad,) = torch.autograd.grad(loss, leaf, g)
    end = logits.detach()[-tail:].clone().requires_grad_()
    want, want_counts = ak.moe_balance_loss(end, idx[-tail:].contiguous())
    (want_grad,) = torch.autograd.grad(want, end, g[1:])
    assert torch.equal(counts[1], want_counts[0]) and torch.equal(grad[-tail:], want_grad) and not bool(grad[:1000].any())
    # (the sums of the probabilities in another order: one rounding for each of 500 tokens at most)
    assert abs(float(loss[1].detach()) - float(want.detach())) <= 500 * 2.0 ** -24 * float(want.detach())


def test_second_derivative_is_refused():
    logits, idx = _router(10, 8, 2, torch.float32)
    leaf = logits.requires_grad_()
    loss, _ = ak.moe_balance_loss(leaf, idx)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss.sum(), leaf, create_graph=True)


def test_upstream_gradients_of_every_kind():
    """An expanded gradient (of a sum), none at all, one of another loss beside it, logits that are no leaf."""
    logits, idx = _router(40, 16, 2, torch.float32, seed=17)
    seq_list = torch.tensor([10, 40], dtype=torch.int64, device=DEV)
    leaf = logits.clone().requires_grad_()
    loss, counts = ak.moe_balance_loss(leaf * 1.0, idx, seq_list)
    (loss.sum() + (leaf * 2).sum()).backward()
    _, _, want = R.balance(logits, idx, seq_list, None, torch.ones(2, device=DEV))
    # (the gradients are at most 16 / 10, good to some 2^-18 of that, and 2 is added)
    assert bool(((leaf.grad.double() - 2 - want).abs() <= 2.0 ** -16).all())
    assert not counts.requires_grad
    with torch.no_grad():
        assert not ak.moe_balance_loss(leaf, idx, seq_list)[0].requires_grad


def test_refusals():
    logits, idx = _router(20, 16, 2, torch.float32)
    mask, seqs = torch.ones(20, dtype=torch.bool, device=DEV), torch.tensor([20], dtype=torch.int64, device=DEV)
    for args in [(logits.half(), idx), (logits[:, ::2], idx), (logits.cpu(), idx), (logits, idx.long()), (logits, idx[:10]),
                 (logits, idx, seqs.int()), (logits, idx, seqs[:0]), (logits, idx, None, mask[:5]), (logits, idx, None, mask.int()),
                 (torch.zeros(4, 1025, device=DEV), torch.zeros(4, 1, dtype=torch.int32, device=DEV)),
                 (logits, torch.zeros(20, 17, dtype=torch.int32, device=DEV))]:
        with pytest.raises(RuntimeError):
            ak.moe_balance_loss(*args)
