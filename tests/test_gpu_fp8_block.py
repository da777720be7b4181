"""Rows and experts in e4m3 with scales per block of 128: quantisation, the grouped product, and the product whose epilogue
quantises silu(gate) * up, against their definitions in 64 bits."""
import pytest
import torch

import ascend_kernel_b200 as ak
from ascend_kernel_b200 import _abi
from tests import fp8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _codes(shape, gen):
    return (torch.randn(shape, generator=gen, device=DEV) * 110).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _problem(counts, K, N, spare=0, seed=0):
    gen = _gen(seed)
    G, M = len(counts), sum(counts) + spare
    KB, NB = -(-K // 128), -(-N // 128)
    x, w = _codes((M, K), gen), _codes((G, K, N), gen)
    xs = (torch.rand(M, KB, generator=gen, device=DEV) + 0.5) * (2 / 110)
    ws = (torch.rand(G, KB, NB, generator=gen, device=DEV) + 0.5) * (K ** -0.5 / 110)
    return x, xs, w, ws, torch.tensor(counts, dtype=torch.int64, device=DEV)


def _check_product(out, x, xs, w, ws, ranges):
    y, mag = R.grouped(x, xs, w, ws, ranges)
    bound = R.sum_error(mag, x.shape[1])
    bound = bound + 2.0 ** -8 * (y.abs() + bound) + 2.0 ** -134  # one rounding to bf16
    off = (out.double() - y).abs()
    for a, b in ranges:
        assert bool((off[a:b] <= bound[a:b]).all()), f"rows {a}..{b}: {float((off[a:b] / bound[a:b]).max())} of the bound"


def _check_gate_up(codes, scale, x, xs, w, ws, ranges):
    y, mag = R.grouped(x, xs, w, ws, ranges)
    e = R.sum_error(mag, x.shape[1])
    I = y.shape[1] // 2
    g, u, eg, eu = y[:, :I], y[:, I:], e[:, :I], e[:, I:]
    h = g * torch.sigmoid(g) * u
    # |silu'| <= 1.1 and |silu(g)| <= |g|; exp, the division and the products cost some roundings
    eh = 1.1 * eg * u.abs() + (g.abs() + eg) * eu + 1.1 * eg * eu + 16 * 2.0 ** -23 * (1 + g.abs()) * h.abs()
    a = h.abs().view(h.shape[0], -1, 128).amax(dim=2)
    ea = eh.view(h.shape[0], -1, 128).amax(dim=2)
    for r0, r1 in ranges:
        off = (scale[r0:r1].double() * 448 - a[r0:r1].clamp(min=R.FLOOR)).abs()
        assert bool((off <= ea[r0:r1] + 2.0 ** -22 * a[r0:r1] + 1e-44).all())
        # the value that is stored is the nearest one: half a step of e4m3, or of its subnormals
        s = R.spread(scale[r0:r1], 1, I)
        v = R.e4m3(codes[r0:r1]) * s
        half = torch.maximum(2.0 ** -4 * (h[r0:r1].abs() + eh[r0:r1]), 2.0 ** -10 * s)
        assert bool(((v - h[r0:r1]).abs() <= eh[r0:r1] + half * (1 + 2.0 ** -20)).all())


# ---- quantisation ---------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,K", [(1, 16), (1, 128), (3, 144), (7, 1024), (130, 2064), (33, 7168), (2, 8208)])
def test_quantised_rows_are_the_definitions_bit_for_bit(rows, K):
    gen = _gen(rows + K)
    x = (torch.randn(rows, K, generator=gen, device=DEV) * torch.exp2(torch.randint(-30, 30, (rows, K), generator=gen, device=DEV).float() / 6)).to(torch.bfloat16)
    codes, scale = ak.fp8_quantize_rows(x)
    want, want_scale = R.quantize(x.double())
    assert torch.equal(codes, want)
    assert torch.equal(scale, want_scale.float())


def test_every_pair_of_significands_ties_included():
    """All significands of a block's largest magnitude against all of the others, at the distances where e4m3 rounds: the codes are those of
    the exact quotient."""
    a = torch.arange(128, 256, device=DEV, dtype=torch.float64)
    rows = []
    for shift in range(0, 20):
        v = torch.arange(0, 256, device=DEV, dtype=torch.float64) * 2.0 ** -shift
        for half in (v[:128], v[128:]):
            b = half.unsqueeze(0).repeat(128, 1).clone()
            b = torch.where(b > a.unsqueeze(1), 0.0, b)
            b[:, 0] = a
            rows.append(b)
    x64 = torch.cat(rows)
    for power in (0, -40, 70, -96):
        x = (x64 * 2.0 ** power).to(torch.bfloat16)
        assert torch.equal(x.double(), x64 * 2.0 ** power)
        codes, scale = ak.fp8_quantize_rows(x)
        want, want_scale = R.quantize(x.double())
        assert torch.equal(codes, want) and torch.equal(scale, want_scale.float())


def test_extreme_blocks():
    x = torch.zeros(9, 256, dtype=torch.bfloat16, device=DEV)
    top, tiny = torch.finfo(torch.bfloat16).max, 2.0 ** -133
    x[1, :] = top
    x[2, 3], x[2, 4] = top, -top
    x[3, 5] = tiny  # below the floor: zeros
    x[4, 7], x[4, 8] = 2.0 ** -100, -(2.0 ** -101)
    x[5, 130] = float("inf")
    x[5, 0] = 3
    x[6, 0] = float("nan")
    x[6, 200] = -2
    x[7, :] = -0.0
    x[8, 127], x[8, 128] = -1, 2.0 ** -20
    codes, scale = ak.fp8_quantize_rows(x)
    want, want_scale = R.quantize(x.double())
    assert torch.equal(torch.isnan(scale), torch.isnan(want_scale))
    assert torch.equal(torch.nan_to_num(scale), torch.nan_to_num(want_scale.float()))
    assert torch.equal(R.e4m3(codes), R.e4m3(want))  # (-0 and 0 alike)
    assert torch.isnan(scale[5, 1]) and not torch.isnan(scale[5, 0]) and torch.isnan(scale[6, 0]) and not torch.isnan(scale[6, 1])


def test_gathered_rows_and_indexes_outside():
    gen = _gen(3)
    x = torch.randn(17, 400, generator=gen, device=DEV).to(torch.bfloat16)
    index = torch.tensor([16, 0, 0, 5, -1, 17, 2 ** 31 - 1, 3], dtype=torch.int32, device=DEV)
    codes, scale = ak.fp8_quantize_rows(x, index)
    rows = torch.where(((index >= 0) & (index < 17)).unsqueeze(1), x[index.clamp(0, 16).long()].float(), 0.0)
    want, want_scale = R.quantize(rows.double())
    assert torch.equal(codes, want) and torch.equal(scale, want_scale.float())


def test_rows_quantised_once_and_gathered_have_the_same_bits():
    """A long call whose index names rows again and again takes two passes: indexes outside x, blocks that are not finite, a short last block."""
    gen = _gen(4)
    T, n_rows, K = 64, 40000, 1360
    assert _abi.lib.b200moe_fp8_quantize_rows_scratch_bytes(T, n_rows, K, 1) > 0
    x = torch.randn(T, K, generator=gen, device=DEV).to(torch.bfloat16)
    x[3, 200], x[5, K - 1] = float("nan"), float("inf")
    index = torch.randint(-1, T + 1, (n_rows,), generator=gen, device=DEV).to(torch.int32)
    codes, scale = ak.fp8_quantize_rows(x, index)
    once, once_scale = ak.fp8_quantize_rows(x)
    at = index.clamp(0, T - 1).long()
    inside = ((index >= 0) & (index < T)).unsqueeze(1)
    want_scale = torch.where(inside, once_scale[at], torch.tensor(2.0 ** -100 / 448, device=DEV))
    assert torch.equal(codes, torch.where(inside, once[at], torch.zeros_like(codes)))
    assert torch.equal(torch.nan_to_num(scale), torch.nan_to_num(want_scale)) and torch.equal(torch.isnan(scale), torch.isnan(want_scale))


def test_quantise_into_given_tensors_and_no_rows():
    x = torch.randn(4, 128, device=DEV).to(torch.bfloat16)
    codes = torch.empty(4, 128, dtype=torch.float8_e4m3fn, device=DEV)
    scale = torch.empty(4, 1, device=DEV)
    assert ak.fp8_quantize_rows(x, codes=codes, scale=scale)[0] is codes
    assert torch.equal(codes.view(torch.uint8), R.quantize(x.double())[0])
    c, s = ak.fp8_quantize_rows(x[:0])
    assert tuple(c.shape) == (0, 128) and tuple(s.shape) == (0, 1)
    c, s = ak.fp8_quantize_rows(x[:0], torch.zeros(3, dtype=torch.int32, device=DEV))  # no row to take: zeros
    assert int(c.sum()) == 0


# ---- the grouped product --------------------------------------------------------------------------

SHAPES = [
    # counts per expert, K, N, rows behind the last
    ([1], 16, 16, 0),
    ([1], 128, 128, 0),
    ([3], 144, 144, 5),
    ([0, 1, 0, 17, 0], 256, 272, 0),
    ([16, 15, 2], 400, 112, 3),
    ([33, 0, 64, 1], 384, 512, 9),
    ([128, 129], 512, 384, 0),
    ([255, 256, 257], 272, 256, 1),
    ([300, 1, 0, 40], 2048, 640, 130),
    ([8] * 40, 640, 1280, 0),
    ([1, 0] * 32, 1152, 256, 7),
    ([700], 896, 400, 0),
    ([1], 7168, 256, 0),
    ([2, 1, 0, 5], 4112, 2064, 2),
]


@pytest.mark.parametrize("counts,K,N,spare", SHAPES)
@pytest.mark.parametrize("kind", [0, 1])
def test_grouped_product(counts, K, N, spare, kind):
    x, xs, w, ws, gl = _problem(counts, K, N, spare)
    out = torch.full((x.shape[0], N), 7.0, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl if kind else gl.cumsum(0), out, group_list_type=kind)
    used = sum(counts)
    assert bool((out[used:] == 7).all())
    _check_product(out, x, xs, w, ws, R.bounds(counts, 1, x.shape[0]))
    assert ak.last_status() == (0, 0)


@pytest.mark.parametrize("counts,K,N,spare", [s for s in SHAPES if s[2] % 256 == 0])
def test_gate_up(counts, K, N, spare):
    x, xs, w, ws, gl = _problem(counts, K, N, spare, seed=1)
    ws = ws * 3  # gates of both signs and some size
    codes = torch.full((x.shape[0], N // 2), 9, dtype=torch.uint8, device=DEV)
    scale = torch.full((x.shape[0], N // 256), 7.0, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, codes, output_scale=scale, group_list_type=1, gate_up_silu=True)
    used = sum(counts)
    assert bool((codes[used:] == 9).all()) and bool((scale[used:] == 7).all())
    _check_gate_up(codes, scale, x, xs, w, ws, R.bounds(counts, 1, x.shape[0]))


def test_no_rows():
    x, xs, w, ws, gl = _problem([0, 0], 256, 512)
    out, codes = torch.empty(0, 512, dtype=torch.bfloat16, device=DEV), torch.empty(0, 256, dtype=torch.uint8, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, out, group_list_type=1)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, codes, output_scale=torch.empty(0, 2, device=DEV), group_list_type=1, gate_up_silu=True)
    x, xs, w, ws, gl = _problem([0, 0], 256, 512, spare=5)  # rows, but none of an expert's
    out = torch.full((5, 512), 7.0, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, out, group_list_type=1)
    assert bool((out == 7).all())


def test_many_uneven_experts():
    gen = _gen(11)
    counts = (torch.rand(96, generator=gen, device=DEV) ** 4 * 500).int().tolist()
    x, xs, w, ws, gl = _problem(counts, 656, 512, 0, seed=2)
    out = torch.empty(x.shape[0], 512, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, out, group_list_type=1)
    _check_product(out, x, xs, w, ws, R.bounds(counts, 1, x.shape[0]))


def test_the_same_call_twice_gives_the_same_bits():
    x, xs, w, ws, gl = _problem([1, 5, 0, 2], 2048, 1024, 0, seed=5)
    outs = []
    for _ in range(3):
        out = torch.empty(8, 1024, dtype=torch.bfloat16, device=DEV)
        ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, out, group_list_type=1)
        outs.append(out)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_a_bad_row_stays_its_own_and_the_next_experts_rows_too():
    """NaN codes, NaN and infinite scales of one row; the rows around it, of the same tile, of the next expert's and behind the last."""
    counts, K, N = [5, 4], 400, 272
    x, xs, w, ws, gl = _problem(counts, K, N, 4, seed=6)
    clean = torch.zeros(13, N, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, clean, group_list_type=1)
    x[2, 17] = 0x7F
    x[9:] = 0xFF
    xs[6, 1] = float("nan")
    xs[7, 0] = float("inf")
    out = torch.zeros_like(clean)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, out, group_list_type=1)
    assert bool(torch.isnan(out[2]).all()) and bool(torch.isnan(out[6]).all())
    assert not bool(torch.isfinite(out[7]).any())
    for r in (0, 1, 3, 4, 5, 8, 9, 10, 11, 12):
        assert torch.equal(out[r], clean[r])


def test_a_bad_row_leaves_its_neighbours_codes_alone():
    """The same of the quantised product: a NaN row, and NaN rows behind the last one of a tile."""
    counts, K, N = [5, 3], 400, 512
    x, xs, w, ws, gl = _problem(counts, K, N, 5, seed=23)

    def run():
        codes, scale = torch.zeros(13, N // 2, dtype=torch.uint8, device=DEV), torch.zeros(13, N // 256, device=DEV)
        ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, codes, output_scale=scale, group_list_type=1, gate_up_silu=True)
        return codes, scale

    codes, scale = run()
    x[2, 17], x[8:] = 0x7F, 0xFF
    got, got_scale = run()
    assert bool(torch.isnan(got_scale[2]).all()) and not bool(got[2].any())
    for r in (0, 1, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12):
        assert torch.equal(got[r], codes[r]) and torch.equal(got_scale[r], scale[r])


def test_nan_weights_stay_in_their_column_and_expert():
    counts, K, N = [3, 3, 3], 144, 272  # (K ends inside a block: what follows belongs to the next expert)
    x, xs, w, ws, gl = _problem(counts, K, N, 0, seed=7)
    clean = torch.zeros(9, N, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, clean, group_list_type=1)
    w[1, :, 5] = 0x7F
    out = torch.zeros_like(clean)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, out, group_list_type=1)
    assert bool(torch.isnan(out[3:6, 5]).all())
    out[3:6, 5] = clean[3:6, 5]
    assert torch.equal(out, clean)


def test_gate_up_blocks_that_are_not_finite():
    x, xs, w, ws, gl = _problem([4], 256, 512, 0, seed=8)
    w[0, 3, 256 + 130] = 0x7F  # an up column of the second block
    codes = torch.empty(4, 256, dtype=torch.uint8, device=DEV)
    scale = torch.empty(4, 2, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, codes, output_scale=scale, group_list_type=1, gate_up_silu=True)
    assert bool(torch.isnan(scale[:, 1]).all()) and bool(torch.isfinite(scale[:, 0]).all())
    assert int(codes[:, 128:].max()) == 0
    x.zero_()
    w[0, 3, 256 + 130] = 0
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, codes, output_scale=scale, group_list_type=1, gate_up_silu=True)
    assert bool((R.e4m3(codes) == 0).all()) and bool((scale == 2.0 ** -100 / 448).all())


def test_extreme_gates():
    """Gates of a size where exp overflows or vanishes: silu is 0 or the gate itself."""
    x = torch.full((2, 16), 0x38, dtype=torch.uint8, device=DEV)  # ones
    xs = torch.tensor([[1.0], [-1.0]], device=DEV)
    w = torch.full((1, 16, 256), 0x38, dtype=torch.uint8, device=DEV)
    ws = torch.tensor([[[50.0, 1.0]]], device=DEV)  # gates of +-800, up of +-16
    codes = torch.empty(2, 128, dtype=torch.uint8, device=DEV)
    scale = torch.empty(2, 1, device=DEV)
    gl = torch.tensor([2], dtype=torch.int64, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, codes, output_scale=scale, group_list_type=1, gate_up_silu=True)
    assert bool((R.e4m3(codes[0]) * float(scale[0]) - 12800).abs().max() <= 12800 * 2.0 ** -22)
    # (compared as fp32, which the quotient is rounded to)
    assert bool((R.e4m3(codes[1]) == 0).all()) and bool((scale[1] == torch.tensor(2.0 ** -100 / 448, device=DEV)).all())


def test_an_invalid_group_list_is_cut_and_reported():
    x, xs, w, ws, _ = _problem([4, 4], 128, 128, 0, seed=9)
    out = torch.full((8, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, torch.tensor([6, 100], dtype=torch.int64, device=DEV), out, group_list_type=1)
    _check_product(out, x, xs, w, ws, [(0, 6), (6, 8)])
    assert ak.last_status(clear=True) == (1, 1)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, torch.tensor([0, 0], dtype=torch.int64, device=DEV), out, group_list_type=1)
    assert ak.last_status() == (0, 0)


def test_a_captured_chain_replayed_beside_another():
    """quantise -> gate/up -> down in two graphs captured on one stream, replayed on two at once, on new inputs."""
    I, H, G = 256, 512, 3
    gen = _gen(12)
    w13, w2 = _codes((G, H, 2 * I), gen), _codes((G, I, H), gen)
    s13 = (torch.rand(G, H // 128, 2 * I // 128, generator=gen, device=DEV) + 0.5) * (H ** -0.5 / 110)
    s2 = (torch.rand(G, I // 128, H // 128, generator=gen, device=DEV) + 0.5) * (I ** -0.5 / 110)
    gl = torch.tensor([2, 30, 9], dtype=torch.int64, device=DEV)
    index = torch.randint(0, 20, (41,), generator=gen, device=DEV).to(torch.int32)

    def chain(x):
        q, s = ak.fp8_quantize_rows(x, index)
        h = torch.empty(41, I, dtype=torch.uint8, device=DEV)
        hs = torch.empty(41, I // 128, device=DEV)
        y = torch.empty(41, H, dtype=torch.bfloat16, device=DEV)
        ak.grouped_gemm_fp8_block(q, s, w13, s13, gl, h, output_scale=hs, group_list_type=1, gate_up_silu=True)
        ak.grouped_gemm_fp8_block(h, hs, w2, s2, gl, y, group_list_type=1)
        return y

    xs = [torch.randn(20, H, generator=gen, device=DEV).to(torch.bfloat16) for _ in range(4)]
    want = [chain(x) for x in xs]
    inputs = [xs[0].clone(), xs[1].clone()]
    graphs, outs = [], []
    for x in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(chain(x))
        graphs.append(g)
    inputs[0].copy_(xs[2])
    inputs[1].copy_(xs[3])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[2]) and torch.equal(outs[1], want[3])


def test_a_captured_call_that_deals_out_its_tiles_is_replayed():
    """Tiles of many waves are drawn from a counter, which every replay has to clear: 256 experts, 2560 and 2 x 1280 columns."""
    G, K, N = 256, 144, 2560
    x, xs, w, ws, gl = _problem([1, 3] * (G // 2), K, N, 4, seed=24)
    M = x.shape[0]

    def run():
        out, codes = torch.zeros(M, N, dtype=torch.bfloat16, device=DEV), torch.zeros(M, N // 2, dtype=torch.uint8, device=DEV)
        scale = torch.zeros(M, N // 256, device=DEV)
        ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, out, group_list_type=1)
        ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, codes, output_scale=scale, group_list_type=1, gate_up_silu=True)
        return out, codes, scale

    graph = torch.cuda.CUDAGraph()
    run()
    with torch.cuda.graph(graph):
        got = run()
    for counts in ([1, 3] * (G // 2), [0, 2] * (G // 2), [M] + [0] * (G - 1)):
        gl.copy_(torch.tensor(counts))
        want = run()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        _check_product(got[0], x, xs, w, ws, R.bounds(counts, 1, M))


@pytest.mark.parametrize("G", [1023, 1024])
def test_as_many_experts_as_there_may_be(G):
    """Most of them without rows; the last one has some."""
    K, N = 160, 256
    counts = [0] * G
    for g, c in ((0, 2), (500, 33), (G - 1, 170)):
        counts[g] = c
    x, xs, w, ws, gl = _problem(counts, K, N, 1, seed=25)
    out = torch.full((x.shape[0], N), 7.0, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, out, group_list_type=1)
    assert bool((out[-1] == 7).all())
    _check_product(out, x, xs, w, ws, R.bounds(counts, 1, x.shape[0]))


def test_inputs_that_are_misaligned_are_refused():
    x, xs, w, ws, gl = _problem([2, 2], 128, 128)
    out = torch.empty(4, 128, dtype=torch.bfloat16, device=DEV)
    off = torch.empty(4 * 128 + 8, dtype=torch.uint8, device=DEV)[8:].view(4, 128)
    with pytest.raises(RuntimeError):
        ak.grouped_gemm_fp8_block(off, xs, w, ws, gl, out)
    half = torch.empty(4 * 128 + 4, dtype=torch.bfloat16, device=DEV)[4:].view(4, 128)
    with pytest.raises(RuntimeError):
        ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, half)
    with pytest.raises(RuntimeError):
        ak.fp8_quantize_rows(half)


def test_refusals():
    x, xs, w, ws, gl = _problem([2, 2], 256, 256)
    out = torch.empty(4, 256, dtype=torch.bfloat16, device=DEV)
    ok = dict(x=x, x_scale=xs, weight=w, weight_scale=ws, group_list=gl, output=out)
    codes, scale = torch.empty(4, 128, dtype=torch.uint8, device=DEV), torch.empty(4, 1, device=DEV)
    bad = [
        dict(x=x.cpu()), dict(x=x[:, ::2]), dict(x=x.float()), dict(x=x[:, :128].contiguous()), dict(x_scale=xs[:, :1].contiguous()),
        dict(x_scale=xs.double()), dict(weight=w[0]), dict(weight_scale=ws.half()), dict(group_list=gl.int()), dict(group_list=gl[:1]),
        dict(output=out.float()), dict(output=out[:3]), dict(output_scale=scale), dict(gate_up_silu=True),
        dict(gate_up_silu=True, output=codes), dict(gate_up_silu=True, output=codes, output_scale=scale.double()),
        dict(group_list_type=2),
    ]
    for change in bad:
        with pytest.raises(RuntimeError):
            ak.grouped_gemm_fp8_block(**{**ok, **change})
    with pytest.raises(RuntimeError):  # N is no multiple of 256
        ak.grouped_gemm_fp8_block(x, xs, w[:, :, :128].contiguous(), ws[:, :, :1].contiguous(), gl, codes[:, :64].contiguous(),
                                  output_scale=scale, gate_up_silu=True)
    xb = torch.zeros(4, 256, dtype=torch.bfloat16, device=DEV)
    for args in [(xb.float(),), (xb[0],), (xb[:, :8].contiguous(),), (xb, torch.zeros(4, dtype=torch.int64, device=DEV)),
                 (xb, None, torch.empty(3, 256, dtype=torch.uint8, device=DEV)), (xb, None, None, torch.empty(4, 1, device=DEV)), (xb.cpu(),)]:
        with pytest.raises(RuntimeError):
            ak.fp8_quantize_rows(*args)


def test_offsets_behind_31_bits():
    """Results and codes of more than 2^31 elements: the rows at the end against the same rows of a short call."""
    gen = _gen(20)
    M, K, N, tail = 300_000, 128, 7168, 300
    assert M * N > 2 ** 31
    x, w = _codes((M, K), gen), _codes((1, K, N), gen)
    xs, ws = torch.rand(M, 1, generator=gen, device=DEV) + 0.5, torch.rand(1, 1, N // 128, generator=gen, device=DEV) / 1000
    out = torch.empty(M, N, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, torch.tensor([M], dtype=torch.int64, device=DEV), out, group_list_type=1)
    short = torch.empty(tail, N, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_fp8_block(x[-tail:].contiguous(), xs[-tail:].contiguous(), w, ws, torch.tensor([tail], dtype=torch.int64, device=DEV),
                              short, group_list_type=1)
    assert torch.equal(out[-tail:], short)
    codes, scale = ak.fp8_quantize_rows(out)
    want, want_scale = ak.fp8_quantize_rows(out[-tail:].contiguous())
    assert torch.equal(codes[-tail:], want) and torch.equal(scale[-tail:], want_scale)


def test_on_another_stream():
    x, xs, w, ws, gl = _problem([5, 40, 2], 512, 1024, 0, seed=21)
    want = torch.empty(47, 1024, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, want, group_list_type=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [torch.empty_like(want) for _ in range(8)]
    for i, out in enumerate(outs):  # two streams side by side
        with torch.cuda.stream(side if i & 1 else torch.cuda.current_stream()):
            ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, out, group_list_type=1)
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out, want)


def test_cuts_of_the_columns_give_the_same_products():
    """Few rows go through stages of two blocks of columns, many through stages of one, few tiles through parts of the k range: a row's
    result differs by the order of its fp32 sums at most."""
    K, N = 1280, 1024
    x, xs, w, ws, _ = _problem([200], K, N, 0, seed=22)
    many = torch.empty(200, N, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_fp8_block(x, xs, w, ws, torch.tensor([200], dtype=torch.int64, device=DEV), many, group_list_type=1)
    few = torch.empty(40, N, dtype=torch.bfloat16, device=DEV)
    ak.grouped_gemm_fp8_block(x[:40].contiguous(), xs[:40].contiguous(), w, ws, torch.tensor([40], dtype=torch.int64, device=DEV), few,
                              group_list_type=1)
    for out, rows in ((many, 200), (few, 40)):
        _check_product(out, x[:rows], xs[:rows], w, ws, [(0, rows)])
