"""What the 8-bit expert path and the balance loss refuse, through the C ABI: nothing is launched, so no device is needed."""
import pytest
import torch

from ascend_kernel_b200 import _abi, ops

lib = _abi.lib
A = 1 << 20  # an aligned address that is never read
OK, NULL, SHAPE, ALIGN, WS, ARG = 0, 2, 3, 4, 5, 6


def _gemm(x=A, xs=A, w=A, ws=A, gl=A, out=A, os=A, M=4, K=256, N=256, G=2, kind=1, gu=0, work=A, nbytes=1 << 40):
    return lib.b200moe_grouped_gemm_fp8_block(x, xs, w, ws, gl, out, os, M, K, N, G, kind, gu, work, nbytes, None)


@pytest.mark.parametrize("change,code", [
    (dict(M=-1), SHAPE), (dict(K=8), SHAPE), (dict(K=0), SHAPE), (dict(N=24), SHAPE), (dict(N=0), SHAPE), (dict(G=0), SHAPE),
    (dict(G=1025), SHAPE), (dict(M=1 << 40), SHAPE), (dict(gu=1, N=128), SHAPE), (dict(gu=1, N=384), SHAPE), (dict(kind=2), ARG),
    (dict(gu=2), ARG), (dict(x=None), NULL), (dict(xs=None), NULL), (dict(w=None), NULL), (dict(ws=None), NULL), (dict(gl=None), NULL),
    (dict(out=None), NULL), (dict(gu=1, os=None), NULL), (dict(x=A + 8), ALIGN), (dict(w=A + 4), ALIGN), (dict(out=A + 2), ALIGN),
    (dict(work=None), WS), (dict(nbytes=0), WS), (dict(M=0, x=None, out=None), OK),
])
def test_grouped_gemm_refusals(change, code):
    assert _gemm(**change) == code


@pytest.mark.parametrize("args,code", [
    ((A, None, A, A, 4, 4, 24), SHAPE), ((A, None, A, A, 4, 4, 0), SHAPE), ((A, None, A, A, 3, 4, 128), SHAPE),
    ((A, None, A, A, -1, 0, 128), SHAPE), ((A, A, A, A, 4, 1 << 40, 128), SHAPE), ((None, None, A, A, 4, 4, 128), NULL),
    ((A, None, None, A, 4, 4, 128), NULL), ((A, None, A, None, 4, 4, 128), NULL), ((A + 2, None, A, A, 4, 4, 128), ALIGN),
    ((A, None, A + 8, A, 4, 4, 128), ALIGN), ((None, None, None, None, 0, 0, 128), OK),
])
def test_quantize_refusals(args, code):
    assert lib.b200moe_fp8_quantize_rows(*args, None, 0, None) == code


def _loss(logits=A, f32=0, idx=A, seqs=A, mask=None, T=8, E=16, k=2, S=2, loss=A, counts=A, load=A, inv=A, scratch=A, nbytes=1 << 40):
    return lib.b200moe_moe_balance_loss(logits, f32, idx, seqs, mask, T, E, k, S, loss, counts, load, inv, scratch, nbytes, None)


@pytest.mark.parametrize("change,code", [
    (dict(T=-1), SHAPE), (dict(E=0), SHAPE), (dict(E=1025), SHAPE), (dict(k=0), SHAPE), (dict(k=33, E=64), SHAPE), (dict(k=17), SHAPE),
    (dict(S=0), SHAPE), (dict(S=65536), SHAPE), (dict(seqs=None), SHAPE), (dict(T=1 << 30), SHAPE), (dict(f32=2), ARG),
    (dict(logits=None), NULL), (dict(idx=None), NULL), (dict(loss=None), NULL), (dict(counts=None), NULL), (dict(load=None), NULL),
    (dict(inv=None), NULL), (dict(scratch=None), WS), (dict(nbytes=64), WS), (dict(scratch=A + 4), ALIGN),
])
def test_balance_loss_refusals(change, code):
    assert _loss(**change) == code


@pytest.mark.parametrize("change,code", [
    (dict(logits=None), NULL), (dict(load=None), NULL), (dict(inv=None), NULL), (dict(g=None), NULL), (dict(out=None), NULL),
    (dict(seqs=None), SHAPE), (dict(E=2000), SHAPE), (dict(f32=-1), ARG), (dict(T=0, logits=None), OK),
])
def test_balance_gradient_refusals(change, code):
    c = dict(logits=A, f32=0, seqs=A, mask=None, load=A, inv=A, g=A, T=8, E=16, S=2, out=A, **{})
    c.update(change)
    assert lib.b200moe_moe_balance_loss_grad(*c.values(), None) == code


def test_scratch_holds_a_row_for_every_piece():
    """Pieces are numbered range + sequence, so there are at most ranges + sequences of them."""
    for T, S in ((0, 1), (1, 1), (17, 3), (4096, 7), (100000, 65535)):
        for E in (1, 7, 256, 1024):
            chunk = max(32, -(-T // 148))
            rows = -(-T // chunk) + S
            assert lib.b200moe_moe_balance_scratch_bytes(T, E, S) >= rows * (8 * E + 4)


@pytest.mark.parametrize("big", [1 << 30, 1 << 46, 1 << 58, 1 << 59, 1 << 62, (1 << 63) - 1, -(1 << 63)])
def test_sizes_whose_products_leave_64_bits(big):
    """(2^58 rows of 16 columns of four bytes are 2^64, which is 0: such a product must not be divided by.)"""
    for gu in (0, 1):
        assert lib.b200moe_grouped_gemm_fp8_block_workspace_bytes(big, 256, 16, 2, gu) == 256
        assert lib.b200moe_grouped_gemm_fp8_block_workspace_bytes(4, big, 256, 2, gu) == 256
        assert lib.b200moe_grouped_gemm_fp8_block_workspace_bytes(4, 256, big, 2, gu) == 256
    for change in (dict(M=big), dict(K=big), dict(N=big), dict(G=big)):
        assert _gemm(**change) == SHAPE
    for sizes in ((big, 64, 128), (4, big, 128), (4, 64, big), (big, big, big)):
        assert lib.b200moe_fp8_quantize_rows_scratch_bytes(*sizes, 1) == 0
        assert lib.b200moe_fp8_quantize_rows(A, A, A, A, *sizes, None, 0, None) == SHAPE
    assert lib.b200moe_moe_balance_scratch_bytes(big, 16, 1) == 0
    assert _loss(T=big) == SHAPE and _loss(T=big, k=16) == SHAPE and _loss(S=big) == SHAPE and _loss(E=big) == SHAPE


def test_scratch_of_the_quantisation_is_aligned():
    assert lib.b200moe_fp8_quantize_rows(A, A, A, A, 64, 1 << 20, 128, A + 8, 1 << 40, None) == ALIGN


def test_python_refuses_host_tensors():
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        ops.fp8_quantize_rows(x)
    with pytest.raises(RuntimeError):
        ops.moe_balance_loss(x, torch.zeros(4, 2, dtype=torch.int32))
