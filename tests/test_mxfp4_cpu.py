"""What the product of 4-bit rows and experts refuses, through the C ABI: nothing is launched, so no device is needed."""
import pytest
import torch

from ascend_kernel_b200 import _abi, ops

lib = _abi.lib
A = 1 << 20  # an aligned address that is never read
OK, NULL, SHAPE, ALIGN, WS, ARG = 0, 2, 3, 4, 5, 6


def _gemm(x=A, xs=A, w=A, ws=A, gl=A, out=A, os=A, M=4, K=256, N=256, G=2, kind=1, gu=0):
    return lib.b200moe_grouped_gemm_mxfp4(x, xs, w, ws, gl, out, os, M, K, N, G, kind, gu, None, None)


@pytest.mark.parametrize("change,code", [
    (dict(M=-1), SHAPE), (dict(K=16), SHAPE), (dict(K=0), SHAPE), (dict(K=48), SHAPE), (dict(N=24), SHAPE), (dict(N=0), SHAPE), (dict(G=0), SHAPE),
    (dict(G=1025), SHAPE), (dict(M=1 << 40), SHAPE), (dict(gu=1, N=128), SHAPE), (dict(gu=1, N=384), SHAPE), (dict(kind=2), ARG),
    (dict(gu=2), ARG), (dict(x=None), NULL), (dict(xs=None), NULL), (dict(w=None), NULL), (dict(ws=None), NULL), (dict(gl=None), NULL),
    (dict(out=None), NULL), (dict(gu=1, os=None), NULL), (dict(x=A + 8), ALIGN), (dict(w=A + 4), ALIGN), (dict(out=A + 2), ALIGN),
    (dict(xs=A + 1), ALIGN), (dict(ws=A + 2), ALIGN), (dict(gu=1, os=A + 1), ALIGN), (dict(M=0, x=None, out=None), OK),
])
def test_refusals(change, code):
    assert _gemm(**change) == code


@pytest.mark.parametrize("big", [1 << 30, 1 << 46, 1 << 58, 1 << 62, (1 << 63) - 1, -(1 << 63)])
def test_sizes_whose_products_leave_64_bits(big):
    for change in (dict(M=big), dict(K=big), dict(N=big), dict(G=big)):
        assert _gemm(**change) == SHAPE


def test_python_refuses_host_tensors():
    b = torch.zeros(4, 64, dtype=torch.uint8)
    with pytest.raises(RuntimeError):
        ops.grouped_gemm_mxfp4(b, b, b.view(1, 4, 64), b, torch.zeros(1, dtype=torch.int64), torch.zeros(4, 16, dtype=torch.bfloat16))
