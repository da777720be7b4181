"""The MoE layer on 8-bit floating-point experts: its pass is the operators one after the other, and it is the layer."""
import pytest
import torch

import ascend_kernel_b200 as ak
from ascend_kernel_b200.moe_layer import GraphedLayer, MoELayer
from tests import fp8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _layer(E, H, I, k, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def weights(K, N):
        w = (torch.randn(E, K, N, generator=gen, device=DEV) * 110).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        return w, (torch.rand(E, K // 128, N // 128, generator=gen, device=DEV) + 0.5) * (K ** -0.5 / 110)

    (w13, s13), (w2, s2) = weights(H, 2 * I), weights(I, H)
    return MoELayer(w13, s13, None, w2, s2, None, E, k, weight_format="fp8"), gen


def _operators(layer, x, logits):
    idx, wts, counts, token_of, slot = ak.ops.moe_route(logits, layer.top_k)
    q, s = ak.fp8_quantize_rows(x, token_of)
    n = q.shape[0]
    h = torch.empty(n, layer.inter, dtype=torch.uint8, device=DEV)
    hs = torch.empty(n, layer.inter // 128, device=DEV)
    y = torch.empty(n, layer.hidden, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_fp8_block(q, s, layer.w13, layer.s13, counts, h, output_scale=hs, group_list_type=1, gate_up_silu=True)
    ak.grouped_gemm_fp8_block(h, hs, layer.w2, layer.s2, counts, y, group_list_type=1)
    return ak.combine(y, slot, wts)


@pytest.mark.parametrize("T,E,H,I,k", [(1, 8, 256, 128, 2), (37, 16, 384, 256, 4), (300, 8, 1024, 384, 2), (4, 4, 128, 128, 4)])
def test_pass_is_the_operators(T, E, H, I, k):
    layer, gen = _layer(E, H, I, k)
    x = torch.randn(T, H, generator=gen, device=DEV).to(torch.bfloat16)
    logits = torch.randn(T, E, generator=gen, device=DEV).to(torch.bfloat16)
    got = layer.forward(x, logits)
    # (the order of an expert's rows is arbitrary and changes no row's result)
    assert torch.equal(got, _operators(layer, x, logits))
    layer.read_status()


def test_pass_is_the_layer_up_to_its_quantisation():
    """Against the layer in 64 bits with unquantised rows.  x and silu(gate) * up are each rounded to three bits behind the first: off
    by at most 2^-4, evenly spread 2^-4 / sqrt(3) = 3.6 % of a value; two such roundings, of which the first passes a product of two sums
    (gate and up), make sqrt(2 + 1) * 3.6 % = 6.3 % of the result's norm at most."""
    T, E, H, I, k = 64, 8, 512, 256, 2
    layer, gen = _layer(E, H, I, k, seed=1)
    x = torch.randn(T, H, generator=gen, device=DEV).to(torch.bfloat16)
    logits = torch.randn(T, E, generator=gen, device=DEV).to(torch.bfloat16)
    got = layer.forward(x, logits).double()
    idx, wts, _, _, _ = ak.ops.moe_route(logits, k)
    want = torch.zeros_like(got)
    for e in range(E):
        w13 = R.e4m3(layer.w13[e]) * R.spread(R.spread(layer.s13[e], 0, H), 1, 2 * I)
        w2 = R.e4m3(layer.w2[e]) * R.spread(R.spread(layer.s2[e], 0, I), 1, H)
        g, u = (x.double() @ w13).chunk(2, dim=1)
        y = (g * torch.sigmoid(g) * u) @ w2
        want += y * (wts * (idx == e)).sum(dim=1, keepdim=True).double()
    assert float((got - want).norm() / want.norm()) <= 0.063 + 2.0 ** -7


def test_graphed_pass():
    layer, gen = _layer(8, 256, 128, 2, seed=2)
    graphed = GraphedLayer(layer, 24)
    for _ in range(3):
        x = torch.randn(24, 256, generator=gen, device=DEV).to(torch.bfloat16)
        logits = torch.randn(24, 8, generator=gen, device=DEV).to(torch.bfloat16)
        assert torch.equal(graphed(x, logits), layer.forward(x, logits))


def test_router_trained_beside_the_pass():
    """A step as it would be used: the pass, and the balance loss of the same routing with its gradient."""
    layer, gen = _layer(8, 256, 128, 2, seed=3)
    x = torch.randn(50, 256, generator=gen, device=DEV).to(torch.bfloat16)
    router = (torch.randn(256, 8, generator=gen, device=DEV) * 0.1).to(torch.bfloat16).requires_grad_()
    logits = x @ router
    out = layer.forward(x, logits.detach())
    idx, _, counts, _, _ = ak.ops.moe_route(logits.detach(), 2)
    loss, seen = ak.moe_balance_loss(logits, idx)
    loss.sum().backward()
    want, _, want_grad = R.balance(logits, idx, None, None, torch.ones(1, device=DEV))
    assert torch.equal(seen[0], counts) and bool(torch.isfinite(out).all())
    dense = x.double().t() @ want_grad
    # bf16 gradients of the logits (2^-8), a bf16 product with fp32 sums and a bf16 result: two roundings of the terms' magnitudes
    mag = x.double().abs().t() @ want_grad.abs()
    assert bool(((router.grad.double() - dense).abs() <= (2.0 ** -8 + 2.0 ** -12) * mag + 2.0 ** -8 * dense.abs() + 1e-9).all())


def test_rows_that_come_through_the_exchange():
    """exchange="p2p" with one rank: the rows are quantised where they arrive, in a buffer with room for more."""
    E, H, I, k = 8, 256, 128, 2
    layer, gen = _layer(E, H, I, k, seed=4)
    p2p = MoELayer(layer.w13, layer.s13, None, layer.w2, layer.s2, None, E, k, weight_format="fp8", exchange="p2p", max_tokens=64)
    try:
        for T in (64, 7, 50):
            x = torch.randn(T, H, generator=gen, device=DEV).to(torch.bfloat16)
            logits = torch.randn(T, E, generator=gen, device=DEV).to(torch.bfloat16)
            a, b = layer.forward(x, logits).double(), p2p.forward(x, logits).double()
            # Another number of rows may cut the k range otherwise: sums that differ by some 2^-20 at most. Where one lies at a border it
            # moves a result to the next bf16 value (2^-8), or one of a row's I codes by a step (2^-3, of a row 2^-3 / sqrt(I) < 2^-6.4).
            assert float((a - b).norm() / a.norm()) <= 2.0 ** -6
        p2p.read_status()
    finally:
        p2p.px.close()


def test_refusals():
    layer, _ = _layer(4, 128, 128, 2)
    for change in (dict(o13=layer.s13), dict(w13=layer.w13[:, :, :128]), dict(w2=layer.w2.to(torch.int16))):
        args = dict(w13=layer.w13, s13=layer.s13, o13=None, w2=layer.w2, s2=layer.s2, o2=None)
        args.update(change)
        with pytest.raises(ValueError):
            MoELayer(*args.values(), 4, 2, weight_format="fp8")
