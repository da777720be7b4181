"""Findings of the operators that have no workspace of status words (the 8-bit product, the balance loss): whose they are, and what a
status call waits for."""
import pytest
import torch

import ascend_kernel_b200 as ak
from ascend_kernel_b200 import cinfer_ascendc
from tests.test_gpu_fp8_block import _problem

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _bad_product(m, at=1):
    """A product whose group list names more rows than there are, expert ``at`` the first of them."""
    x, xs, w, ws, _ = _problem([4, 4, 4], 128, 128, 0, seed=9)
    counts = [0, 0, 0]
    counts[at] = 100
    gl = torch.tensor(counts, dtype=torch.int64).pin_memory().to(DEV, non_blocking=True)
    out = torch.zeros(12, 128, dtype=torch.bfloat16, device=DEV)
    m.grouped_gemm_fp8_block(x, xs, w, ws, gl, out, group_list_type=1)


def _bad_loss(m, at):
    """A balance loss whose list of sequences leaves the tokens at sequence ``at``."""
    logits = torch.randn(20, 8, device=DEV)
    ends = [5, 10, 20]
    ends[at] = 21 if at == 2 else 30
    m.moe_balance_loss(logits, torch.zeros(20, 2, dtype=torch.int32, device=DEV), torch.tensor(ends[:at + 1], dtype=torch.int64, device=DEV), None)


def test_a_status_call_does_not_wait_for_streams_that_ran_nothing():
    side, busy = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        _bad_product(ak, 2)
        _bad_product(cinfer_ascendc, 1)
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(3_000_000_000)  # well over a second
        done.record()
    with torch.cuda.stream(side):
        got = ak.last_status(), tuple(cinfer_ascendc.last_status())
        early = not done.query()
    torch.cuda.synchronize()
    assert got == ((1, 2), (1, 1))
    assert early, "the status calls waited for a stream of somebody else's"
    ak.last_status(clear=True)
    cinfer_ascendc.last_status(True)


def test_a_status_call_while_a_stream_is_captured():
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        _bad_product(ak, 1)
    torch.cuda.synchronize()
    graph, buf = torch.cuda.CUDAGraph(), torch.zeros(8, device=DEV)
    with torch.cuda.graph(graph, stream=other, capture_error_mode="relaxed"):
        buf.add_(1)
        got = ak.last_status()
        buf.add_(1)
    graph.replay()
    torch.cuda.synchronize()
    assert got == (1, 1) and buf.tolist() == [2.0] * 8
    assert ak.last_status(clear=True) == (1, 1)


def test_each_binding_has_its_own():
    """Whoever clears takes its own findings only."""
    _bad_product(ak, 2)
    assert tuple(cinfer_ascendc.last_status(True)) == (0, 0)
    assert ak.last_status() == (1, 2)
    _bad_loss(cinfer_ascendc, 0)
    assert ak.last_status(clear=True) == (1, 2)
    assert tuple(cinfer_ascendc.last_status()) == (1, 0)
    assert ak.last_status() == (0, 0)
    with pytest.raises(RuntimeError, match="status"):
        cinfer_ascendc.check_status()
    cinfer_ascendc.check_status()
    ak.check_status()


def test_findings_of_a_side_stream_and_of_replays():
    """A call captured on one stream and replayed on another; the first call on its stream is the captured one."""
    x, xs, w, ws, gl = _problem([4, 4], 128, 128, 0, seed=9)
    out = torch.zeros(8, 128, dtype=torch.bfloat16, device=DEV)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, out, group_list_type=1)
    assert ak.last_status() == (0, 0)
    graph.replay()
    assert ak.last_status() == (0, 0)
    gl[1] = 50
    graph.replay()
    assert ak.last_status() == (1, 1)
    graph.replay()
    assert ak.last_status(clear=True) == (1, 1)
    gl[1] = 4
    graph.replay()
    assert ak.last_status() == (0, 0)


def _bad_gemm(m, at):
    """The same of an operator that keeps its findings in its stream's workspace."""
    x = torch.zeros(12, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(3, 64, 256, dtype=torch.int8, device=DEV)
    s = torch.ones(3, 256, dtype=torch.bfloat16, device=DEV)
    counts = [0, 0, 0]
    counts[at] = 100
    offset = torch.zeros(0, device=DEV) if m is cinfer_ascendc else None
    m.grouped_gemm(x, w, s, offset, torch.tensor(counts, device=DEV), "int8", torch.zeros(12, 256, dtype=torch.bfloat16, device=DEV),
                   group_list_type=1)


@pytest.mark.parametrize("m", [ak, cinfer_ascendc], ids=["mirror", "drop-in"])
def test_clearing_takes_what_is_returned(m):
    """Two operators that keep their findings in different places, and the second one's on two streams: each is reported once."""
    side = torch.cuda.Stream()
    _bad_gemm(m, 0)
    _bad_product(m, 1)
    with torch.cuda.stream(side):
        _bad_product(m, 2)
    got = [tuple(m.last_status(clear=True)) for _ in range(4)]
    assert got[0] == (1, 0) and sorted(got[1:3]) == [(1, 1), (1, 2)] and got[3] == (0, 0)
    _bad_gemm(m, 0)
    _bad_product(m, 1)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="status"):
            m.check_status()
    m.check_status()
