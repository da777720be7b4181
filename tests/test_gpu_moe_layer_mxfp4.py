"""The MoE layer on 4-bit floating-point experts, and its pass on another router's choice: the operators one after the other."""
import pytest
import torch

import ascend_kernel_b200 as ak
from ascend_kernel_b200 import ops
from ascend_kernel_b200.moe_layer import GraphedLayer, MoELayer
from tests import mxfp4_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _bytes(shape, gen):
    return torch.randint(0, 256, shape, generator=gen, device=DEV).to(torch.uint8)


def _layer(E, H, I, k, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    middle = lambda K: 125 - (K.bit_length() - 1) // 2  # noqa: E731  (rows of about unit norm)

    def weights(N, K):
        return _bytes((E, N, K // 2), gen), torch.randint(middle(K) - 1, middle(K) + 2, (E, N, K // 32), generator=gen, device=DEV).to(torch.uint8)

    (w13, s13), (w2, s2) = weights(2 * I, H), weights(H, I)
    return MoELayer(w13, s13, None, w2, s2, None, E, k, weight_format="mxfp4"), gen


def _experts(layer, x, counts, token_of):
    q, s = ak.mxfp4_quantize_rows(x, token_of)
    n = q.shape[0]
    h, hs = torch.zeros(n, layer.inter // 2, dtype=torch.uint8, device=DEV), torch.zeros(n, layer.inter // 32, dtype=torch.uint8, device=DEV)
    y = torch.zeros(n, layer.hidden, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_mxfp4(q, s, layer.w13, layer.s13, counts, h, output_scale=hs, group_list_type=1, gate_up_silu=True)
    ak.grouped_gemm_mxfp4(h, hs, layer.w2, layer.s2, counts, y, group_list_type=1)
    return y


@pytest.mark.parametrize("T,E,H,I,k", [(1, 8, 256, 128, 2), (37, 16, 384, 256, 4), (300, 8, 1024, 384, 2), (4, 4, 128, 128, 4)])
def test_pass_is_the_operators(T, E, H, I, k):
    layer, gen = _layer(E, H, I, k)
    x = torch.randn(T, H, generator=gen, device=DEV).to(torch.bfloat16)
    logits = torch.randn(T, E, generator=gen, device=DEV).to(torch.bfloat16)
    got = layer.forward(x, logits)
    # (the order of an expert's rows is arbitrary and changes no row's result)
    idx, wts, counts, token_of, slot = ops.moe_route(logits, k)
    assert torch.equal(got, ak.combine(_experts(layer, x, counts, token_of), slot, wts))
    # the same choice handed in
    assert torch.equal(layer.forward_routed(x, idx, wts), got)
    layer.read_status()


def test_pass_is_the_layer_up_to_its_quantisation():
    """Against the layer in 64 bits with unquantised rows.  A value is off by at most a quarter of itself when it is quantised (half a step of its binade,
    one bit behind the first), evenly spread 1 / 4 / sqrt(3) = 14.4 %; x passes a product of two sums (gate and up), silu(gate) * up one:
    sqrt(2 + 1) * 14.4 % = 25 % of the result's norm at most, and a third of that again for values in a block's last binade, whose steps are no smaller."""
    T, E, H, I, k = 64, 8, 512, 256, 2
    layer, gen = _layer(E, H, I, k, seed=1)
    x = torch.randn(T, H, generator=gen, device=DEV).to(torch.bfloat16)
    logits = torch.randn(T, E, generator=gen, device=DEV).to(torch.bfloat16)
    got = layer.forward(x, logits).double()
    idx, wts, _, _, _ = ops.moe_route(logits, k)
    want = torch.zeros_like(got)
    for e in range(E):
        g, u = (x.double() @ R.values(layer.w13[e], layer.s13[e]).T).chunk(2, dim=1)
        y = (g * torch.sigmoid(g) * u) @ R.values(layer.w2[e], layer.s2[e]).T
        want += y * (wts * (idx == e)).sum(dim=1, keepdim=True).double()
    assert float((got - want).norm() / want.norm()) <= 0.25 * 4 / 3


def test_graphed_pass():
    layer, gen = _layer(8, 256, 128, 2, seed=2)
    graphed = GraphedLayer(layer, 24)
    for _ in range(3):
        x = torch.randn(24, 256, generator=gen, device=DEV).to(torch.bfloat16)
        logits = torch.randn(24, 8, generator=gen, device=DEV).to(torch.bfloat16)
        assert torch.equal(graphed(x, logits), layer.forward(x, logits))


@pytest.mark.parametrize("fmt", ["mxfp4", "int8", "fp8"])
def test_routed_pass_with_dropped_pairs(fmt):
    """Dropped pairs have no part, an expert may be named twice, and a token of dropped pairs alone gives zeros."""
    T, E, H, I, k = 40, 8, 256, 256, 2
    gen = torch.Generator(device=DEV).manual_seed(3)
    if fmt == "mxfp4":
        layer, _ = _layer(E, H, I, k, seed=3)
    elif fmt == "int8":
        w13, w2 = _bytes((E, H, 2 * I), gen).view(torch.int8), _bytes((E, I, H), gen).view(torch.int8)
        s13, s2 = [(torch.rand(E, n, generator=gen, device=DEV) * 1e-3).to(torch.bfloat16) for n in (2 * I, H)]
        layer = MoELayer(w13, s13, None, w2, s2, None, E, k)
    else:
        w13, w2 = [(torch.randn(E, *n, generator=gen, device=DEV) * 110).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) for n in ((H, 2 * I), (I, H))]
        s13, s2 = [torch.full((E, *n), 2.0 ** -11, device=DEV) for n in ((H // 128, 2 * I // 128), (I // 128, H // 128))]
        layer = MoELayer(w13, s13, None, w2, s2, None, E, k, weight_format="fp8")
    x = torch.randn(T, H, generator=gen, device=DEV).to(torch.bfloat16)
    idx = torch.randint(0, E, (T, k), generator=gen, device=DEV).to(torch.int32)
    idx[3], idx[5, 0], idx[6, 1] = -1, E, -7
    idx[9, 0] = idx[9, 1] = 2
    wts = torch.rand(T, k, generator=gen, device=DEV)
    got = layer.forward_routed(x, idx, wts)
    assert bool((got[3] == 0).all())
    # pair by pair, every row a pass of its own
    one = torch.ones(T, 1, device=DEV)
    want = torch.zeros(T, H, dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(want)
    for j in range(k):
        y = layer.forward_routed(x, idx[:, j:j + 1].contiguous(), one).double()
        want += wts[:, j:j + 1].double() * y
        mag += (wts[:, j:j + 1].double() * y).abs()
    # the same rows may be summed in another order where a call is cut in another way, and are rounded to bf16 then: one more half step each
    assert bool(((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * mag + 1e-30).all())
    layer.read_status()


def test_refusals():
    layer, gen = _layer(4, 256, 128, 2)
    w = (layer.w13, layer.s13, None, layer.w2, layer.s2, None, 4, 2)
    for change in ({2: layer.s13}, {0: layer.w13[:, :, :64].contiguous()}, {1: layer.s13[:, :, :4].contiguous()}, {4: layer.s2[:, :128].contiguous()}):
        args = list(w)
        for i, v in change.items():
            args[i] = v
        with pytest.raises((ValueError, AssertionError)):
            MoELayer(*args, weight_format="mxfp4")
    with pytest.raises(ValueError):
        MoELayer(*w, weight_format="nvfp4")
    x = torch.zeros(3, 256, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError):
        layer.forward_routed(x, torch.zeros(3, 2, dtype=torch.int64, device=DEV), torch.zeros(3, 2, device=DEV))


def test_launches():
    layer, gen = _layer(4, 256, 128, 2)
    x = torch.randn(5, 256, generator=gen, device=DEV).to(torch.bfloat16)
    idx = torch.zeros(5, 2, dtype=torch.int32, device=DEV)
    wts = torch.ones(5, 2, device=DEV)
    before = ops.LAUNCHES
    layer.forward_routed(x, idx, wts)
    assert ops.LAUNCHES - before == 5  # sort, quantisation, two products, combine


def test_rows_that_come_through_the_exchange():
    """exchange="p2p" with one rank: the rows are quantised where they arrive, in a buffer with room for more.  How an expert's rows are cut goes by their number
    alone, so the results have the same bits."""
    E, H, I, k = 8, 256, 128, 2
    layer, gen = _layer(E, H, I, k, seed=4)
    p2p = MoELayer(layer.w13, layer.s13, None, layer.w2, layer.s2, None, E, k, weight_format="mxfp4", exchange="p2p", max_tokens=64)
    try:
        for T in (64, 7, 50):
            x = torch.randn(T, H, generator=gen, device=DEV).to(torch.bfloat16)
            logits = torch.randn(T, E, generator=gen, device=DEV).to(torch.bfloat16)
            assert torch.equal(layer.forward(x, logits), p2p.forward(x, logits))
        p2p.read_status()
    finally:
        p2p.px.close()


def test_trained_beside_the_pass():
    """A step as it would be used: the sort of a router's choice, the rows to plain experts and back, and the gradients of all of them, beside
    the balance loss of the same choice."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    T, E, H, k = 60, 6, 64, 2
    x = torch.randn(T, H, generator=gen, device=DEV).requires_grad_()
    router = (torch.randn(H, E, generator=gen, device=DEV) * 0.2).requires_grad_()
    experts = (torch.randn(E, H, H, generator=gen, device=DEV) * H ** -0.5).requires_grad_()
    logits = x @ router
    prob, chosen = torch.softmax(logits, dim=1).topk(k, dim=1)
    idx = chosen.to(torch.int32)
    counts, token_of, slot = ak.moe_sort(idx, E)
    rows = ak.moe_dispatch(x, token_of, slot)
    y = torch.cat([r @ w for r, w in zip(rows.split(counts.tolist()), experts)])
    out = ak.moe_combine(y, prob, token_of, slot)
    loss, pairs = ak.moe_balance_loss(logits, idx)
    assert torch.equal(pairs[0], counts)
    g = torch.randn(T, H, generator=gen, device=DEV)
    got = torch.autograd.grad((out * g).sum() + 0.1 * loss.sum(), (x, router, experts))
    # the same in 64 bits, every expert on every token
    x64, r64, e64 = [t.detach().double().requires_grad_() for t in (x, router, experts)]
    lg = x64 @ r64
    p = torch.softmax(lg, dim=1)
    on = torch.zeros(T, E, dtype=torch.float64, device=DEV).scatter_(1, chosen, 1.0)
    out64 = torch.einsum("te,teh->th", p * on, torch.einsum("th,ehj->tej", x64, e64))
    loss64 = E / (k * T * T) * (counts.double() * p.sum(dim=0)).sum()
    want = torch.autograd.grad((out64 * g.double()).sum() + 0.1 * loss64, (x64, r64, e64))
    assert float((out.detach().double() - out64.detach()).norm() / out64.detach().norm()) <= 1e-3
    for a, b in zip(got, want):
        # (torch's own products may run in tf32: 2^-11 a factor, of some ten in a row)
        assert float((a.double() - b).norm() / b.norm()) <= 10 * 2.0 ** -11
