"""ops.LAUNCHES against the kernels that the 8-bit operators and the balance loss launch, as the profiler of torch sees them."""
import pytest
import torch

import ascend_kernel_b200 as ak
from ascend_kernel_b200 import _abi, ops
from tests.test_gpu_fp8_block import _problem

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _launched(fn, counted):
    fn()
    before = ops.LAUNCHES
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as p:
        fn()
        torch.cuda.synchronize()
    seen = [e.name for e in p.events() if e.device_type == torch.autograd.DeviceType.CUDA and "b200moe" in e.name]
    assert ops.LAUNCHES - before == counted
    assert len(seen) in (0, counted), seen  # (0: no tracing of kernels on this host)


@pytest.mark.parametrize("K,counted", [(256, 1), (2048, 2)])
@pytest.mark.parametrize("gate_up", [False, True])
def test_products(K, counted, gate_up):
    """Few tiles of a long k range are cut in parts, which a second kernel adds."""
    x, xs, w, ws, gl = _problem([1, 5], K, 512)
    assert (_abi.lib.b200moe_grouped_gemm_fp8_block_workspace_bytes(6, K, 512, 2, int(gate_up)) > 256) == (counted == 2)
    if gate_up:
        out, scale = torch.empty(6, 256, dtype=torch.uint8, device=DEV), torch.empty(6, 2, device=DEV)
    else:
        out, scale = torch.empty(6, 512, dtype=torch.bfloat16, device=DEV), None
    _launched(lambda: ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, out, output_scale=scale, group_list_type=1, gate_up_silu=gate_up), counted)


@pytest.mark.parametrize("rows,counted", [(0, 0), (64, 1), (40000, 2)])
def test_quantisation(rows, counted):
    x = torch.randn(64, 1360, device=DEV).to(torch.bfloat16)
    index = torch.randint(0, 64, (rows,), device=DEV).to(torch.int32)
    _launched(lambda: ak.fp8_quantize_rows(x, index), counted)


@pytest.mark.parametrize("T,forward,backward", [(0, 1, 0), (100, 2, 1)])
def test_balance_loss(T, forward, backward):
    logits = torch.randn(T, 16, device=DEV).requires_grad_()
    idx = torch.zeros(T, 2, dtype=torch.int32, device=DEV)

    def both():
        loss, _ = ak.moe_balance_loss(logits, idx)
        torch.autograd.grad(loss.sum(), logits)

    with torch.no_grad():
        _launched(lambda: ak.moe_balance_loss(logits, idx), forward)
    _launched(both, forward + backward)


def test_a_backward_pass_on_another_thread_and_one_of_the_drop_in_module():
    from ascend_kernel_b200 import cinfer_ascendc

    logits = torch.randn(50, 16, device=DEV).requires_grad_()
    idx = torch.zeros(50, 2, dtype=torch.int32, device=DEV)
    loss, _ = ak.moe_balance_loss(logits, idx)
    theirs, _ = cinfer_ascendc.moe_balance_loss(logits, idx)
    before = ops.LAUNCHES
    theirs.sum().backward()
    assert ops.LAUNCHES == before
    loss.sum().backward()  # (the engine runs it on a thread of its own)
    assert ops.LAUNCHES == before + 1
