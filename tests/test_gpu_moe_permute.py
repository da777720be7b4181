"""The sort of the (token, j) pairs by expert, the rows of the sorted pairs and the weighted sum on the way back, with their gradients,
against their definitions in 64 bits."""
import pytest
import torch

import ascend_kernel_b200 as ak
from ascend_kernel_b200 import _abi, cinfer_ascendc, ops
from tests import permute_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _idx(T, E, k, gen, dropped=0.0):
    idx = torch.rand(T, max(E, k), generator=gen, device=DEV).topk(k, dim=1).indices.to(torch.int32)
    if dropped:
        idx[torch.rand(T, k, generator=gen, device=DEV) < dropped] = -1
    return idx


def _same(got, want):
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


# ---- the sort -------------------------------------------------------------------------------------


@pytest.mark.parametrize("T,E,k,dropped", [(0, 5, 2, 0), (1, 1, 1, 0), (1, 256, 8, 0), (37, 256, 8, 0.2), (31, 7, 3, 0), (33, 1024, 32, 0.1),
                                           (509, 64, 2, 1.0), (4096, 60, 1, 0), (513, 8, 8, 0.5), (8192, 257, 8, 0), (8200, 1024, 8, 0.03),
                                           (9000, 1, 1, 0.3), (40001, 16, 1, 0.0), (20011, 384, 4, 0.05), (40000, 1000, 8, 0.0)])
def test_sort_is_stable(T, E, k, dropped):
    """One block of few warps or many, and several (over 4096 pairs)."""
    idx = _idx(T, E, k, _gen(T + E), dropped)
    _same(ak.moe_sort(idx, E), R.sort(idx, E))


def test_sort_over_the_largest_blocks():
    """More pairs than 128 blocks of 4096: a warp's part is no whole number of batches."""
    gen = _gen(1)
    T, E, k = 70003, 256, 8
    idx = torch.randint(-2, E + 3, (T, k), generator=gen, device=DEV).to(torch.int32)
    counts, token_of, slot = ak.moe_sort(idx, E)
    key = torch.where((idx < 0) | (idx >= E), E, idx).reshape(-1)
    at, order = key.sort(stable=True)
    n = int((key < E).sum())
    assert torch.equal(counts, torch.bincount(key, minlength=E + 1)[:E])
    assert torch.equal(token_of, torch.where(at < E, order // k, -1).to(torch.int32))
    want = torch.empty(T * k, dtype=torch.int32, device=DEV)
    want[order] = torch.where(at < E, torch.arange(T * k, device=DEV), -1).to(torch.int32)
    assert torch.equal(slot.view(-1), want) and int((slot >= 0).sum()) == n


def test_one_expert_named_by_every_pair_and_the_ends_of_the_range():
    idx = torch.full((3000, 4), 5, dtype=torch.int32, device=DEV)
    idx[0, 0], idx[1, 1], idx[2, 2], idx[7, 3] = -2 ** 31, 2 ** 31 - 1, 6, 0
    _same(ak.moe_sort(idx, 6), R.sort(idx, 6))


def test_sort_of_the_router_s_own_choice_agrees_with_it_but_for_the_order_inside_an_expert():
    logits = torch.randn(300, 32, generator=_gen(2), device=DEV).to(torch.bfloat16)
    idx, _, counts, token_of, slot = ops.moe_route(logits, 4)
    c, t, s = ak.moe_sort(idx, 32)
    assert torch.equal(c, counts)
    ends = counts.cumsum(0).tolist()
    for a, b in zip([0] + ends[:-1], ends):
        assert torch.equal(t[a:b], token_of[a:b].sort().values)


def test_sort_refusals():
    idx = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    for bad, E in ((idx.long(), 4), (idx.view(-1), 4), (idx.T, 4), (idx, 0), (idx, 1025), (idx.cpu(), 4),
                   (torch.zeros(4, 33, dtype=torch.int32, device=DEV), 64)):
        with pytest.raises(RuntimeError):
            ak.moe_sort(bad, E)


# ---- rows -----------------------------------------------------------------------------------------

ROWS = [(1, 4, 1, 8), (1, 8, 8, 7168), (3, 5, 2, 64), (37, 256, 8, 1000), (50, 40, 9, 264), (21, 64, 32, 2056), (700, 16, 2, 136), (5, 8, 3, 40000)]


@pytest.mark.parametrize("T,E,k,H", ROWS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dropped", [0.0, 0.3])
def test_dispatch(T, E, k, H, dtype, dropped):
    gen = _gen(T + H)
    _, token_of, slot = ak.moe_sort(_idx(T, E, k, gen, dropped), E)
    x = torch.randn(T, H, generator=gen, device=DEV).to(dtype).requires_grad_()
    rows = ak.moe_dispatch(x, token_of, slot)
    assert torch.equal(rows, R.dispatch(x.detach(), token_of))
    g = torch.randn(T * k, H, generator=gen, device=DEV).to(dtype)
    (grad,) = torch.autograd.grad(rows, x, g)
    terms = R.picked(g, slot)
    # k - 1 additions in fp32, one rounding
    err = k * 2.0 ** -24 * terms.abs().sum(dim=1)
    want = terms.sum(dim=1)
    assert grad.dtype == dtype
    assert bool(((grad.double() - want).abs() <= err + R.half_step(dtype) * (want.abs() + err)).all())


@pytest.mark.parametrize("T,E,k,H", ROWS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dropped", [0.0, 0.3])
def test_combine(T, E, k, H, dtype, dropped):
    gen = _gen(T + H + 1)
    _, token_of, slot = ak.moe_sort(_idx(T, E, k, gen, dropped), E)
    y = torch.randn(T * k, H, generator=gen, device=DEV).to(dtype).requires_grad_()
    w = torch.randn(T, k, generator=gen, device=DEV).requires_grad_()
    out = ak.moe_combine(y, w, token_of, slot)
    terms = R.picked(y.detach(), slot)
    wt = w.detach().double().unsqueeze(2) * terms
    err = k * 2.0 ** -24 * wt.abs().sum(dim=1)
    want = wt.sum(dim=1)
    assert out.dtype == dtype
    assert bool(((out.double() - want).abs() <= err + R.half_step(dtype) * (want.abs() + err)).all())

    g = torch.randn(T, H, generator=gen, device=DEV).to(dtype)
    grad_y, grad_w = torch.autograd.grad(out, (y, w), g)
    want = R.dispatch(g.double(), token_of) * R.weight_of_rows(w.detach(), slot).unsqueeze(1)
    # a product in fp32 and its rounding to the type
    assert bool(((grad_y.double() - want).abs() <= (2.0 ** -24 + R.half_step(dtype) * (1 + 2.0 ** -24)) * want.abs()).all())
    prod = terms * g.double().unsqueeze(1)
    # H products in fp32, each fused with an addition: less than H roundings of a partial sum
    assert bool(((grad_w.double() - prod.sum(dim=2)).abs() <= H * 2.0 ** -24 * prod.abs().sum(dim=2)).all())
    assert bool((grad_w[slot < 0] == 0).all())


def test_only_one_of_the_gradients():
    gen = _gen(5)
    _, token_of, slot = ak.moe_sort(_idx(40, 8, 2, gen), 8)
    y = torch.randn(80, 64, generator=gen, device=DEV)
    w = torch.rand(40, 2, generator=gen, device=DEV)
    g = torch.randn(40, 64, generator=gen, device=DEV)
    ya, wa = y.clone().requires_grad_(), w.clone().requires_grad_()
    both = torch.autograd.grad(ak.moe_combine(ya, wa, token_of, slot), (ya, wa), g)
    yb, wb = y.clone().requires_grad_(), w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(ak.moe_combine(yb, w, token_of, slot), yb, g)[0], both[0])
    assert torch.equal(torch.autograd.grad(ak.moe_combine(y, wb, token_of, slot), wb, g)[0], both[1])
    assert not ak.moe_combine(y, w, token_of, slot).requires_grad


def test_gradients_against_differences():
    """fp32 central differences of a weighted sum of the way there and back: both sums are linear in x and in the weights, so a difference over a step of
    1 has no error but the roundings: (2 k + H) of them in a result of the terms' magnitude."""
    gen = _gen(6)
    T, E, k, H = 6, 4, 2, 16
    _, token_of, slot = ak.moe_sort(_idx(T, E, k, gen, 0.2), E)
    x = torch.randn(T, H, generator=gen, device=DEV).requires_grad_()
    w = torch.rand(T, k, generator=gen, device=DEV).requires_grad_()
    scale = torch.randn(T * k, H, generator=gen, device=DEV)
    g = torch.randn(T, H, generator=gen, device=DEV)

    def f(x, w):
        return ak.moe_combine(ak.moe_dispatch(x, token_of, slot) * scale, w, token_of, slot)

    gx, gw = torch.autograd.grad(f(x, w), (x, w), g)
    for leaf, grad in ((x, gx), (w, gw)):
        for i in range(leaf.numel()):
            d = torch.zeros_like(leaf).view(-1)
            d[i] = 1
            d = d.view_as(leaf)
            args = [(x + s * d, w) if leaf is x else (x, w + s * d) for s in (1, -1)]
            diff = ((f(*args[0]).double() - f(*args[1]).double()) * g.double()).sum() / 2
            assert abs(float(diff.detach() - grad.view(-1)[i])) <= (2 * k + H) * 2.0 ** -24 * 64 * 8


def test_non_finite_values_stay_with_their_rows():
    idx = torch.tensor([[0, 1], [1, -1], [0, 2]], dtype=torch.int32, device=DEV)
    _, token_of, slot = ak.moe_sort(idx, 3)
    y = torch.ones(6, 8, device=DEV)
    y[slot[0, 0]] = float("inf")
    y[5] = float("nan")  # the dropped pair's place: in no sum
    w = torch.tensor([[1.0, 2.0], [3.0, float("nan")], [0.5, 0.5]], device=DEV)
    out = ak.moe_combine(y, w, token_of, slot)
    assert bool(torch.isinf(out[0]).all()) and torch.equal(out[1], torch.full((8,), 3.0, device=DEV)) and torch.equal(out[2], torch.ones(8, device=DEV))


def test_no_tokens():
    _, token_of, slot = ak.moe_sort(torch.zeros(0, 3, dtype=torch.int32, device=DEV), 4)
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    before = ops.LAUNCHES
    rows = ak.moe_dispatch(x, token_of, slot)
    w = torch.zeros(0, 3, device=DEV, requires_grad=True)
    out = ak.moe_combine(rows, w, token_of, slot)
    gx, gw = torch.autograd.grad(out, (x, w), out.detach())
    assert rows.shape == (0, 64) and out.shape == (0, 64) and gx.shape == x.shape and gw.shape == w.shape
    assert ops.LAUNCHES == before


def test_results_of_the_route_are_taken_as_they_are():
    gen = _gen(7)
    x = torch.randn(100, 256, generator=gen, device=DEV).to(torch.bfloat16)
    idx, w, counts, token_of, slot = ops.moe_route(torch.randn(100, 16, generator=gen, device=DEV).to(torch.bfloat16), 3)
    rows = ak.moe_dispatch(x, token_of, slot)
    assert torch.equal(rows, ak.gather_rows(x, token_of))
    assert torch.equal(ak.moe_combine(rows, w, token_of, slot), ak.combine(rows, slot, w))


def test_row_refusals():
    _, token_of, slot = ak.moe_sort(torch.zeros(4, 2, dtype=torch.int32, device=DEV), 4)
    x, y, w = torch.zeros(4, 16, device=DEV), torch.zeros(8, 16, device=DEV), torch.zeros(4, 2, device=DEV)
    for args in ((x.half(), token_of, slot), (x[:, :12], token_of, slot), (x[:, :12].contiguous(), token_of, slot), (x[:3], token_of, slot),
                 (x, token_of.long(), slot), (x, token_of[:7], slot), (x, token_of, slot.view(-1)), (x, token_of, slot.cpu()), (x.view(-1), token_of, slot)):
        with pytest.raises(RuntimeError):
            ak.moe_dispatch(*args)
    for args in ((x, w, token_of, slot), (y, w.double(), token_of, slot), (y, w[:3], token_of, slot), (y, w.T, token_of, slot),
                 (y.half(), w, token_of, slot), (y, w, slot, slot)):
        with pytest.raises(RuntimeError):
            ak.moe_combine(*args)


def test_twice_differentiated_is_refused():
    _, token_of, slot = ak.moe_sort(torch.zeros(4, 2, dtype=torch.int32, device=DEV), 4)
    x = torch.ones(4, 8, device=DEV, requires_grad=True)
    w = torch.ones(4, 2, device=DEV, requires_grad=True)
    rows = ak.moe_dispatch(x, token_of, slot)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(rows.sum(), x, create_graph=True)
    out = ak.moe_combine(torch.ones(8, 8, device=DEV), w, token_of, slot)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(out.sum(), w, create_graph=True)


def test_two_streams_a_replayed_graph_and_a_broadcast_gradient():
    gen = _gen(8)
    T, E, k, H = 9000, 64, 8, 64  # (a sort with scratch)
    idx = _idx(T, E, k, gen)
    assert _abi.lib.b200moe_moe_sort_scratch_bytes(T, E, k) > 0
    x = torch.randn(T, H, generator=gen, device=DEV)
    w = torch.rand(T, k, generator=gen, device=DEV)

    def run():
        c, t, s = ak.moe_sort(idx, E)
        return c, t, s, ak.moe_combine(ak.moe_dispatch(x, t, s), w, t, s)

    want = run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            got.append(run())
    torch.cuda.synchronize()
    for g in got:
        _same(g, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    idx.copy_(_idx(T, E, k, gen))
    graph.replay()
    torch.cuda.synchronize()
    _same(out, run())
    # (the gradient of a sum has strides of zero)
    xr = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(ak.moe_dispatch(xr, want[1], want[2]).sum(), xr)
    assert torch.equal(gx, torch.full_like(gx, k))


def test_a_backward_pass_in_a_graph():
    gen = _gen(9)
    _, token_of, slot = ak.moe_sort(_idx(64, 8, 2, gen, 0.1), 8)
    x = torch.randn(64, 128, generator=gen, device=DEV).to(torch.bfloat16).requires_grad_()
    w = torch.rand(64, 2, generator=gen, device=DEV).requires_grad_()

    def step():
        out = ak.moe_combine(ak.moe_dispatch(x, token_of, slot), w, token_of, slot)
        return (out.detach(),) + torch.autograd.grad(out, (x, w), torch.ones_like(out))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(torch.randn(64, 128, generator=gen, device=DEV))
    graph.replay()
    torch.cuda.synchronize()
    _same(out, step())


def test_launches_and_the_drop_in_module():
    gen = _gen(10)
    idx = _idx(100, 8, 2, gen)
    before = ops.LAUNCHES
    c, t, s = ak.moe_sort(idx, 8)
    x = torch.randn(100, 64, generator=gen, device=DEV).requires_grad_()
    w = torch.rand(100, 2, generator=gen, device=DEV)
    out = ak.moe_combine(ak.moe_dispatch(x, t, s), w, t, s)
    assert ops.LAUNCHES - before == 3
    (grad,) = torch.autograd.grad(out.sum(), x)
    assert ops.LAUNCHES - before == 5
    before = ops.LAUNCHES
    ak.moe_sort(torch.zeros(9000, 8, dtype=torch.int32, device=DEV), 8)
    assert ops.LAUNCHES - before == 2
    before = ops.LAUNCHES
    _same(cinfer_ascendc.moe_sort(idx, 8), (c, t, s))
    out2 = cinfer_ascendc.moe_combine(cinfer_ascendc.moe_dispatch(x, t, s), w, t, s)
    assert torch.equal(out2, out) and torch.equal(torch.autograd.grad(out2.sum(), x)[0], grad)
    assert ops.LAUNCHES == before


def test_rows_behind_31_bits():
    """Offsets of more than 2^31 bytes and elements."""
    T, k, H = 40000, 8, 7168
    idx = torch.arange(T * k, device=DEV).to(torch.int32).remainder(256).view(T, k)
    _, token_of, slot = ak.moe_sort(idx, 256)
    x = torch.arange(T, device=DEV).remainder(251).to(torch.bfloat16).unsqueeze(1).expand(T, H).contiguous()
    rows = ak.moe_dispatch(x, token_of, slot)
    assert rows.numel() > 2 ** 31
    step = 50000
    for r in range(0, T * k, step):
        assert bool((rows[r:r + step] == (token_of[r:r + step] % 251).to(torch.bfloat16).unsqueeze(1)).all())
    w = torch.full((T, k), 0.125, device=DEV)
    assert torch.equal(ak.moe_combine(rows, w, token_of, slot), x)


def test_a_gradient_that_is_not_aligned():
    gen = _gen(11)
    _, token_of, slot = ak.moe_sort(_idx(30, 8, 2, gen), 8)
    x = torch.randn(30, 64, generator=gen, device=DEV).requires_grad_()
    w = torch.rand(30, 2, generator=gen, device=DEV).requires_grad_()
    rows = ak.moe_dispatch(x, token_of, slot)
    g = torch.randn(60 * 64 + 1, generator=gen, device=DEV)[1:].view(60, 64)
    assert g.data_ptr() % 16 != 0
    assert torch.equal(torch.autograd.grad(rows, x, g, retain_graph=True)[0], torch.autograd.grad(rows, x, g.clone())[0])
    out = ak.moe_combine(rows.detach(), w, token_of, slot)
    g = torch.randn(30 * 64 + 1, generator=gen, device=DEV)[1:].view(30, 64)
    assert torch.equal(torch.autograd.grad(out, w, g, retain_graph=True)[0], torch.autograd.grad(out, w, g.clone())[0])
