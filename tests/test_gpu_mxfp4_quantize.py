"""Rows of bf16 quantised to e2m1 with a power-of-two scale per 32 elements: bit for bit the definition."""
import pytest
import torch

import ascend_kernel_b200 as ak
from ascend_kernel_b200 import _abi, cinfer_ascendc, ops
from tests import mxfp4_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _check(x, codes, scale):
    want, want_scale = R.quantize(x.double())
    assert torch.equal(scale, want_scale)
    assert torch.equal(codes & 0x77, want & 0x77)
    # (a zero's sign is the value's own)
    assert torch.equal(codes, want)


@pytest.mark.parametrize("rows,K", [(1, 32), (1, 128), (3, 160), (7, 1024), (130, 2080), (33, 7168), (2, 8224), (5, 96), (1, 20000)])
def test_quantised_rows_are_the_definition(rows, K):
    gen = _gen(rows + K)
    x = (torch.randn(rows, K, generator=gen, device=DEV) * torch.exp2(torch.randint(-30, 30, (rows, K), generator=gen, device=DEV).float() / 6)).to(torch.bfloat16)
    _check(x, *ak.mxfp4_quantize_rows(x))


def test_every_significand_against_every_border():
    """Every bf16 of six binades beside every largest magnitude of one: all ties and all scales are among them."""
    a = torch.arange(128, 256, dtype=torch.float64, device=DEV)
    small = torch.cat([torch.arange(128, 256, dtype=torch.float64, device=DEV) * 2.0 ** -s for s in range(6)])  # 768 = 31 to a block
    small = torch.nn.functional.pad(small, (0, -small.numel() % 31)).view(-1, 31)
    block = torch.cat([a.view(-1, 1, 1).expand(-1, small.shape[0], 1), small.unsqueeze(0).expand(a.numel(), -1, -1)], dim=2)
    block = torch.where(block > a.view(-1, 1, 1), a.view(-1, 1, 1), block)
    x64 = torch.cat([block, -block], dim=1).reshape(a.numel(), -1)
    for power in (0, -40, 70, 119, -100, -106):
        x = (x64 * 2.0 ** power).to(torch.bfloat16)
        assert torch.equal(x.double(), x64 * 2.0 ** power)
        _check(x, *ak.mxfp4_quantize_rows(x))


def test_extreme_blocks():
    x = torch.zeros(10, 64, dtype=torch.bfloat16, device=DEV)
    top, tiny = torch.finfo(torch.bfloat16).max, 2.0 ** -133
    x[1, :] = top
    x[2, 3], x[2, 4] = top, -top
    x[3, 5] = tiny
    x[4, 7], x[4, 8] = 2.0 ** -98, -(2.0 ** -101)
    x[5, 40], x[5, 0] = float("inf"), 3
    x[6, 0], x[6, 50] = float("nan"), -2
    x[7, :] = -0.0
    x[8, 31], x[8, 32] = -7, 7.0625
    x[9, 0] = -float("inf")
    codes, scale = ak.mxfp4_quantize_rows(x)
    _check(x, codes, scale)
    assert scale[5].tolist() == [126, 255, 0, 0] and scale[6, 0] == 255 and scale[8].tolist() == [127, 128, 0, 0] and scale[0].tolist() == [27, 27, 0, 0]


def test_gathered_rows_and_indexes_outside():
    x = torch.randn(17, 416, generator=_gen(3), device=DEV).to(torch.bfloat16)
    index = torch.tensor([16, 0, 0, 5, -1, 17, 2 ** 31 - 1, 3, -2 ** 31], dtype=torch.int32, device=DEV)
    rows = torch.where(((index >= 0) & (index < 17)).unsqueeze(1), x[index.clamp(0, 16).long()].float(), 0.0)
    _check(rows, *ak.mxfp4_quantize_rows(x, index))


@pytest.mark.parametrize("K", [1376, 1408])
def test_rows_quantised_once_and_gathered_have_the_same_bits(K):
    gen = _gen(4)
    T, n_rows = 64, 40000
    assert _abi.lib.b200moe_mxfp4_quantize_rows_scratch_bytes(T, n_rows, K, 1) > 0
    x = torch.randn(T, K, generator=gen, device=DEV).to(torch.bfloat16)
    x[3, 200], x[5, K - 1] = float("nan"), float("inf")
    index = torch.randint(-1, T + 1, (n_rows,), generator=gen, device=DEV).to(torch.int32)
    codes, scale = ak.mxfp4_quantize_rows(x, index)
    rows = torch.cat([x, torch.zeros_like(x[:1])])
    once, once_scale = ak.mxfp4_quantize_rows(rows)
    at = torch.where((index >= 0) & (index < T), index, T).long()
    assert torch.equal(codes, once[at]) and torch.equal(scale, once_scale[at])


def test_given_outputs_no_rows_and_refusals():
    x = torch.randn(6, 64, generator=_gen(5), device=DEV).to(torch.bfloat16)
    want = ak.mxfp4_quantize_rows(x)
    room, room_scale = torch.zeros(8, 32, dtype=torch.uint8, device=DEV), torch.zeros(8, 4, dtype=torch.uint8, device=DEV)
    got = ak.mxfp4_quantize_rows(x, codes=room[1:7], scale=room_scale[1:7])  # (a scale that is aligned to 4 bytes alone)
    assert got[0].data_ptr() == room[1:7].data_ptr() and torch.equal(room[1:7], want[0]) and torch.equal(room_scale[1:7], want[1])
    assert int(room[0].sum() + room[7].sum() + room_scale[0].sum() + room_scale[7].sum()) == 0
    before = ops.LAUNCHES
    codes, scale = ak.mxfp4_quantize_rows(x, torch.zeros(0, dtype=torch.int32, device=DEV))
    assert codes.shape == (0, 32) and scale.shape == (0, 4) and ops.LAUNCHES == before
    for args, kw in (((x.float(),), {}), ((x[:, :48].contiguous(),), {}), ((x[:, :32],), {}), ((x, torch.zeros(2, dtype=torch.int64, device=DEV)), {}),
                     ((x,), dict(codes=room)), ((x,), dict(scale=room_scale)), ((x,), dict(scale=room_scale[1:7].to(torch.int8))), ((x.view(-1),), {})):
        with pytest.raises(RuntimeError):
            ak.mxfp4_quantize_rows(*args, **kw)
    for a, b in zip(cinfer_ascendc.mxfp4_quantize_rows(x), want):
        assert torch.equal(a, b)


def test_read_back_by_the_dequantisation_of_the_same_format():
    x = torch.randn(9, 256, generator=_gen(6), device=DEV).to(torch.bfloat16)
    codes, scale = ak.mxfp4_quantize_rows(x)
    out = torch.empty_like(x)
    ak.fp4_dequant(codes, scale, out)
    assert torch.equal(out.double(), R.values(codes, scale))
    # half a step of the value's binade: a quarter of the value, or of the smallest step of the block
    unit = torch.exp2(scale.double() - 127).repeat_interleave(32, dim=1)
    assert bool(((out.double() - x.double()).abs() <= torch.maximum(0.25 * x.double().abs(), 0.25 * unit)).all())


def test_a_replayed_graph_and_two_streams():
    gen = _gen(7)
    T, K = 64, 1408
    x = torch.randn(T, K, generator=gen, device=DEV).to(torch.bfloat16)
    index = torch.randint(0, T, (40000,), generator=gen, device=DEV).to(torch.int32)
    ak.mxfp4_quantize_rows(x, index)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        codes, scale = ak.mxfp4_quantize_rows(x, index)
    x.copy_(torch.randn(T, K, generator=gen, device=DEV))
    graph.replay()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for st in streams:
        with torch.cuda.stream(st):
            got.append(ak.mxfp4_quantize_rows(x, index))
    torch.cuda.synchronize()
    for g in got:
        assert torch.equal(g[0], codes) and torch.equal(g[1], scale)
