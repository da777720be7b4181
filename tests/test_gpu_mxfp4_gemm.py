"""The grouped product of 4-bit rows and 4-bit experts, and the form whose epilogue quantises silu(gate) * up, against their
definitions in 64 bits."""
import pytest
import torch

import ascend_kernel_b200 as ak
from ascend_kernel_b200 import cinfer_ascendc, ops
from tests import mxfp4_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _bytes(shape, gen):
    return torch.randint(0, 256, shape, generator=gen, device=DEV).to(torch.uint8)


def _scales(rows, K, low, high, gen):
    s = torch.zeros(*rows, R.width(K), dtype=torch.uint8, device=DEV)
    s[..., :K // 32] = torch.randint(low, high + 1, (*rows, K // 32), generator=gen, device=DEV).to(torch.uint8)
    return s


def _problem(counts, K, N, spare=0, seed=0, low=126, high=127):
    """Codes of all values.  A product is a multiple of 1/4 of the product of the smallest scales and at most 36 times that of the largest: with
    scales of two neighbouring powers for each operand, sums of K <= 7168 terms are whole multiples of a quantum and below 36 * 4 * 4 * 7168
    < 2^22 of them, so fp32 holds every partial sum exactly, in whatever order they are made."""
    gen = _gen(seed)
    G, M = len(counts), sum(counts) + spare
    return (_bytes((M, K // 2), gen), _scales((M,), K, low, high, gen), _bytes((G, N, K // 2), gen), _scales((G, N), K, low, high, gen),
            torch.tensor(counts, dtype=torch.int64, device=DEV))


def _ranges(counts):
    ends, at = [], 0
    for c in counts:
        ends.append((at, at + c))
        at += c
    return ends


def _product(x, xs, w, ws, ranges):
    xv = R.values(x, xs)
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device=DEV)
    for g, (a, b) in enumerate(ranges):
        if a < b:
            y[a:b] = xv[a:b] @ R.values(w[g], ws[g]).T
    return y


def _check_gate_up(codes, scale, y, ranges):
    """y is exact in fp32 (see _problem).  exp, the division and the products cost some roundings of silu(g) * u."""
    I = y.shape[1] // 2
    g, u = y[:, :I], y[:, I:]
    h = g * torch.sigmoid(g) * u
    eh = 16 * 2.0 ** -23 * (1 + g.abs()) * h.abs() + 2.0 ** -126 * (1 + u.abs())
    for a, b in ranges:
        if a == b:
            continue
        unit = torch.exp2(scale[a:b].double() - 127)
        hb, eb = h[a:b].view(b - a, -1, 32), eh[a:b].view(b - a, -1, 32)
        top, etop = hb.abs().amax(dim=2), eb.amax(dim=2)
        assert bool((top - etop <= 7 * unit).all())
        assert bool(((top + etop > 3.5 * unit) | (scale[a:b] == 27)).all())
        v = R.values(codes[a:b], scale[a:b]).view_as(hb)
        q = (hb.abs() + eb) / unit.unsqueeze(2)
        half = torch.where(q < 2, 0.25, torch.where(q < 4, 0.5, 1.0)) * unit.unsqueeze(2)
        assert bool(((v - hb).abs() <= eb + half).all())


SHAPES = [([1], 32, 16), ([3], 64, 48), ([16], 96, 128), ([17, 0, 5], 128, 144), ([0, 0, 2], 160, 272), ([33, 64, 1, 0], 256, 512), ([100], 288, 400),
          ([128, 129], 512, 256), ([191, 192, 193], 544, 384), ([385, 7], 1024, 640), ([1] * 40, 2048, 1024), ([0, 700, 0, 40, 3], 2080, 528),
          ([5, 150], 7168, 272), ([1000, 0, 24], 256, 2048)]


@pytest.mark.parametrize("counts,K,N", SHAPES)
def test_product_is_exact_and_rounded_once(counts, K, N):
    x, xs, w, ws, gl = _problem(counts, K, N, spare=3, seed=K + N)
    out = torch.full((x.shape[0], N), -7.0, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_mxfp4(x, xs, w, ws, gl, out, group_list_type=1)
    want = _product(x, xs, w, ws, _ranges(counts)).float().to(torch.bfloat16)
    want[sum(counts):] = -7.0  # rows of no expert are left as they were
    assert torch.equal(out, want)
    again = torch.full_like(out, -7.0)
    ak.grouped_gemm_mxfp4(x, xs, w, ws, gl.cumsum(0), again)
    assert torch.equal(again, want)
    ak.check_status()


@pytest.mark.parametrize("counts,K,I", [([1], 32, 128), ([3, 0, 18], 160, 256), ([130], 256, 384), ([64, 200, 1], 544, 128), ([33] * 9, 1024, 640),
                                        ([1] * 8, 7168, 256), ([500, 0, 3], 512, 2048)])
def test_gate_up(counts, K, I):
    x, xs, w, ws, gl = _problem(counts, K, 2 * I, spare=5, seed=K + I, low=122, high=123)
    M = x.shape[0]
    out, scale = torch.full((M, I // 2), 0x5A, dtype=torch.uint8, device=DEV), torch.full((M, I // 32), 77, dtype=torch.uint8, device=DEV)
    ak.grouped_gemm_mxfp4(x, xs, w, ws, gl, out, output_scale=scale, group_list_type=1, gate_up_silu=True)
    _check_gate_up(out, scale, _product(x, xs, w, ws, _ranges(counts)), _ranges(counts))
    n = sum(counts)
    assert bool((out[n:] == 0x5A).all()) and bool((scale[n:] == 77).all())
    ak.check_status()


def test_scales_over_their_whole_range():
    """Every scale byte but 0 and 255 on either side, a single term each: exact products between 2^-126 and 2^127 in bf16."""
    n = 254
    x = torch.zeros(n, 16, dtype=torch.uint8, device=DEV)
    x[:, 0] = 2  # 1 at k = 0
    xs = torch.zeros(n, 4, dtype=torch.uint8, device=DEV)
    xs[:, 0] = torch.arange(1, 255, device=DEV)
    w = torch.zeros(1, 256, 16, dtype=torch.uint8, device=DEV)
    w[:, :, 0] = 3  # 1.5
    ws = torch.zeros(1, 256, 4, dtype=torch.uint8, device=DEV)
    ws[0, :254, 0] = torch.arange(1, 255, device=DEV)
    ws[0, 254:, 0] = 127
    out = torch.empty(n, 256, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_mxfp4(x, xs, w, ws, torch.tensor([n], device=DEV), out, group_list_type=1)
    want = 1.5 * torch.exp2(xs[:, :1].double() - 127) * torch.exp2(ws[0, :, 0].double() - 127)
    fits = (want < 2.0 ** 127) & (want >= 2.0 ** -126)
    assert torch.equal(out.double()[fits], want[fits])


def test_scales_that_are_not_numbers_stay_with_their_row_and_column():
    x, xs, w, ws, gl = _problem([40, 30], 320, 272, seed=5)
    xs[7, 3], xs[50, 0] = 255, 255
    ws[0, 33, 9], ws[1, 271, 1] = 255, 255
    out = torch.empty(70, 272, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_mxfp4(x, xs, w, ws, gl, out, group_list_type=1)
    bad = torch.zeros(70, 272, dtype=torch.bool, device=DEV)
    bad[7], bad[50] = True, True
    bad[:40, 33], bad[40:, 271] = True, True
    assert torch.equal(torch.isnan(out), bad)
    xs2, ws2 = xs.clone(), ws.clone()
    xs2[xs2 == 255], ws2[ws2 == 255] = 127, 127
    want = _product(x, xs2, w, ws2, _ranges([40, 30])).float().to(torch.bfloat16)
    assert torch.equal(out[~bad], want[~bad])


def test_gate_up_of_rows_that_are_not_finite():
    x, xs, w, ws, gl = _problem([20], 128, 512, seed=6, low=122, high=123)
    ok, ok_scale = torch.empty(20, 128, dtype=torch.uint8, device=DEV), torch.empty(20, 8, dtype=torch.uint8, device=DEV)
    ak.grouped_gemm_mxfp4(x, xs, w, ws, gl, ok, output_scale=ok_scale, group_list_type=1, gate_up_silu=True)
    xs[3, 1] = 255
    ws[0, 256 + 70, 0] = 255  # an up column: its block of 32
    out, scale = torch.empty_like(ok), torch.empty_like(ok_scale)
    ak.grouped_gemm_mxfp4(x, xs, w, ws, gl, out, output_scale=scale, group_list_type=1, gate_up_silu=True)
    bad = torch.zeros(20, 8, dtype=torch.bool, device=DEV)
    bad[3], bad[:, 2] = True, True
    assert torch.equal(scale == 255, bad)
    codes = out.view(20, 8, 16)
    assert bool((codes[bad] == 0).all()) and torch.equal(codes[~bad], ok.view(20, 8, 16)[~bad]) and torch.equal(scale[~bad], ok_scale[~bad])


def test_rows_of_a_longer_buffer_and_scales_at_any_word():
    x, xs, w, ws, gl = _problem([9, 14], 96, 32, seed=7)
    out = torch.empty(23, 32, dtype=torch.bfloat16, device=DEV)
    room = torch.full((30, 4), 255, dtype=torch.uint8, device=DEV)
    room[3:26] = xs
    ak.grouped_gemm_mxfp4(x, room[3:26], w, ws, gl, out, group_list_type=1)
    assert torch.equal(out, _product(x, xs, w, ws, _ranges([9, 14])).float().to(torch.bfloat16))


@pytest.mark.parametrize("lists,kind", [([5, 3, 20], 0), ([4, -1, 9], 1), ([12, 30, 1], 1), ([-5, 7, 40], 0)])
def test_invalid_lists_are_clamped_and_reported(lists, kind):
    from tests.fp8_ref import bounds

    x, xs, w, ws, _ = _problem([7, 7, 6], 128, 144, seed=8)
    gl = torch.tensor(lists, dtype=torch.int64, device=DEV)
    out = torch.full((20, 144), -7.0, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_mxfp4(x, xs, w, ws, gl, out, group_list_type=kind)
    code, at = ak.last_status(clear=True)
    assert code == 1
    ends, pos = [], 0
    for c in lists:
        end = pos + max(c, 0) if kind else max(pos, c)
        ends.append((pos, min(end, 20)))
        pos = min(end, 20)
    want = _product(x, xs, w, ws, ends).float().to(torch.bfloat16)
    want[pos:] = -7.0
    assert torch.equal(out, want)
    assert ak.last_status() == (0, 0)


def test_refusals_and_no_rows():
    x, xs, w, ws, gl = _problem([4, 4], 128, 256, seed=9)
    out = torch.empty(8, 256, dtype=torch.bfloat16, device=DEV)
    codes, scale = torch.empty(8, 64, dtype=torch.uint8, device=DEV), torch.empty(8, 4, dtype=torch.uint8, device=DEV)
    good = dict(x=x, x_scale=xs, weight=w, weight_scale=ws, group_list=gl, output=out, group_list_type=1)
    gated = good | dict(output=codes, output_scale=scale, gate_up_silu=True)
    ak.grouped_gemm_mxfp4(**good)
    ak.grouped_gemm_mxfp4(**gated)
    for base, change in [(good, dict(x=x.float())), (good, dict(x_scale=xs[:, :3])), (good, dict(x_scale=xs[:7])), (good, dict(weight=w[:, :, :48].contiguous())),
                         (good, dict(weight_scale=ws[:1])), (good, dict(group_list=gl.int())), (good, dict(group_list=gl[:1])), (good, dict(output=out.float())),
                         (good, dict(output=out[:7])), (good, dict(output_scale=scale)), (good, dict(group_list_type=2)), (good, dict(x=x.cpu())),
                         (gated, dict(output_scale=None)), (gated, dict(output=out)), (gated, dict(output_scale=scale.float())), (gated, dict(output=codes[:, :32]))]:
        with pytest.raises(RuntimeError):
            ak.grouped_gemm_mxfp4(**(base | change))
    before = ops.LAUNCHES
    ak.grouped_gemm_mxfp4(x[:0], xs[:0], w, ws, torch.zeros(2, dtype=torch.int64, device=DEV), out[:0], group_list_type=1)
    assert ops.LAUNCHES == before
    # rows, but none of an expert
    out.fill_(3)
    ak.grouped_gemm_mxfp4(x, xs, w, ws, torch.zeros(2, dtype=torch.int64, device=DEV), out, group_list_type=1)
    assert bool((out == 3).all())


def test_two_streams_a_replayed_graph_and_the_drop_in_module():
    counts = [200, 3, 0, 60]
    x, xs, w, ws, gl = _problem(counts, 512, 768, seed=10)
    M = x.shape[0]

    def run(module=ak):
        out = torch.zeros(M, 768, dtype=torch.bfloat16, device=DEV)
        h, hs = torch.zeros(M, 192, dtype=torch.uint8, device=DEV), torch.zeros(M, 12, dtype=torch.uint8, device=DEV)
        module.grouped_gemm_mxfp4(x, xs, w, ws, gl, out, group_list_type=1)
        module.grouped_gemm_mxfp4(x, xs, w, ws, gl, h, output_scale=hs, group_list_type=1, gate_up_silu=True)
        return out, h, hs

    want = run()
    assert torch.equal(want[0], _product(x, xs, w, ws, _ranges(counts)).float().to(torch.bfloat16))
    results = [run(cinfer_ascendc)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for st in streams:
        with torch.cuda.stream(st):
            results.append(run())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results.append(run())
    graph.replay()
    torch.cuda.synchronize()
    for r in results:
        for a, b in zip(r, want):
            assert torch.equal(a, b)
    ak.check_status()
    cinfer_ascendc.check_status()


def test_experts_behind_31_bits():
    G, K, N = 256, 7168, 4096
    gen = _gen(11)
    counts = [0] * G
    counts[0], counts[100], counts[200], counts[255] = 2, 3, 1, 4
    w = torch.empty(G, N, K // 2, dtype=torch.uint8, device=DEV)
    for g in range(0, G, 32):
        w[g:g + 32] = _bytes((32, N, K // 2), gen)
    ws = _scales((G, N), K, 126, 127, gen)
    x, xs = _bytes((10, K // 2), gen), _scales((10,), K, 126, 127, gen)
    gl = torch.tensor(counts, dtype=torch.int64, device=DEV)
    out = torch.zeros(10, N, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_mxfp4(x, xs, w, ws, gl, out, group_list_type=1)
    assert torch.equal(out, _product(x, xs, w, ws, _ranges(counts)).float().to(torch.bfloat16))


def test_the_operators_together():
    """Sorted by given ids, quantised on the way, both projections, and the weighted sum: the layer's result from the quantised values in 64 bits."""
    gen = _gen(12)
    T, E, k, H, I = 50, 8, 2, 256, 128
    x = torch.randn(T, H, generator=gen, device=DEV).to(torch.bfloat16)
    idx = torch.rand(T, E, generator=gen, device=DEV).topk(k, dim=1).indices.to(torch.int32)
    idx[5, 1] = -1
    wts = torch.rand(T, k, generator=gen, device=DEV)
    w13, s13 = _bytes((E, 2 * I, H // 2), gen), _scales((E, 2 * I), H, 120, 122, gen)
    w2, s2 = _bytes((E, H, I // 2), gen), _scales((E, H), I, 121, 123, gen)
    counts, token_of, slot = ak.moe_sort(idx, E)
    q, qs = ak.mxfp4_quantize_rows(x, token_of)
    h, hs = torch.zeros(T * k, I // 2, dtype=torch.uint8, device=DEV), torch.zeros(T * k, I // 32, dtype=torch.uint8, device=DEV)
    y = torch.zeros(T * k, H, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_mxfp4(q, qs, w13, s13, counts, h, output_scale=hs, group_list_type=1, gate_up_silu=True)
    ak.grouped_gemm_mxfp4(h, hs, w2, s2, counts, y, group_list_type=1)
    out = ak.moe_combine(y, wts, token_of, slot)
    ranges = _ranges(counts.tolist())
    want_q, want_qs = R.quantize(torch.where((token_of >= 0).unsqueeze(1), x[token_of.clamp(min=0).long()].double(), 0.0))
    assert torch.equal(q, want_q) and torch.equal(qs, want_qs)
    y64 = _product(h, hs, w2, s2, ranges)
    want = torch.zeros(T, H, dtype=torch.float64, device=DEV)
    mag = torch.zeros_like(want)
    for t in range(T):
        for j in range(k):
            if slot[t, j] >= 0:
                want[t] += wts[t, j].double() * y64[slot[t, j]]
                mag[t] += wts[t, j].double() * y64[slot[t, j]].abs()
    # y is rounded to bf16, the sum once more; fp32 sums of I terms before (2^-23 of 64 + I magnitudes at most, far below)
    terms = R.values(h, hs).abs().sum(dim=1).max() * R.values(w2, s2).abs().max()
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * (mag + want.abs() * 1.01) + (I + 64) * 2.0 ** -23 * k * terms).all())
    ak.check_status()


def test_rows_that_come_through_a_prefix_of_other_kernels():
    """Quantisation, product and quantised product right behind one another on a stream, again and again: each starts beside the end of the one before
    it and may not read what that has not written."""
    gen = _gen(13)
    T, E, k, H, I = 300, 16, 4, 1024, 512
    w13, s13 = _bytes((E, 2 * I, H // 2), gen), _scales((E, 2 * I), H, 119, 121, gen)
    w2, s2 = _bytes((E, H, I // 2), gen), _scales((E, H), I, 120, 122, gen)
    h, hs = torch.zeros(T * k, I // 2, dtype=torch.uint8, device=DEV), torch.zeros(T * k, I // 32, dtype=torch.uint8, device=DEV)
    q, qs = torch.zeros(T * k, H // 2, dtype=torch.uint8, device=DEV), torch.zeros(T * k, H // 32, dtype=torch.uint8, device=DEV)
    y = torch.zeros(T * k, H, dtype=torch.bfloat16, device=DEV)
    xs = [torch.randn(T, H, generator=gen, device=DEV).to(torch.bfloat16) for _ in range(6)]
    idx = [torch.rand(T, E, generator=gen, device=DEV).topk(k, dim=1).indices.to(torch.int32) for _ in range(6)]
    wts = torch.rand(T, k, generator=gen, device=DEV)

    def run(i):
        counts, token_of, slot = ak.moe_sort(idx[i], E)
        ak.mxfp4_quantize_rows(xs[i], token_of, codes=q, scale=qs)
        ak.grouped_gemm_mxfp4(q, qs, w13, s13, counts, h, output_scale=hs, group_list_type=1, gate_up_silu=True)
        ak.grouped_gemm_mxfp4(h, hs, w2, s2, counts, y, group_list_type=1)
        return ak.moe_combine(y, wts, token_of, slot)

    alone = []
    for i in range(6):
        alone.append(run(i))
        torch.cuda.synchronize()
    for _ in range(5):
        got = [run(i) for i in range(6)]
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            assert torch.equal(a, b)
    ak.check_status()


@pytest.mark.parametrize("G", [1, 300, 1024])
def test_one_expert_and_as_many_as_there_can_be(G):
    gen = _gen(G)
    K, N = 64, 32
    counts = [0] * G
    for g in torch.randint(0, G, (40,), generator=gen, device=DEV).tolist():
        counts[g] += 1
    counts[0] += 200
    x, xs, w, ws, gl = _problem(counts, K, N, seed=G)
    out = torch.zeros(sum(counts), N, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_mxfp4(x, xs, w, ws, gl, out, group_list_type=1)
    assert torch.equal(out, _product(x, xs, w, ws, _ranges(counts)).float().to(torch.bfloat16))
