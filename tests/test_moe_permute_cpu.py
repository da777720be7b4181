"""What the sort by expert, the rows' way to the experts and back and the quantisation to 4 bits refuse, through the C ABI: nothing is
launched, so no device is needed."""
import pytest
import torch

from ascend_kernel_b200 import _abi, ops

lib = _abi.lib
A = 1 << 20  # an aligned address that is never read
OK, NULL, SHAPE, ALIGN, WS, ARG = 0, 2, 3, 4, 5, 6


def _sort(idx=A, T=8, E=16, k=2, counts=A, token_of=A, slot=A, scratch=A, nbytes=1 << 40):
    return lib.b200moe_moe_sort(idx, T, E, k, counts, token_of, slot, scratch, nbytes, None)


@pytest.mark.parametrize("change,code", [
    (dict(T=-1), SHAPE), (dict(E=0), SHAPE), (dict(E=1025), SHAPE), (dict(k=0), SHAPE), (dict(k=33), SHAPE), (dict(T=1 << 30), SHAPE),
    (dict(T=1 << 62), SHAPE), (dict(idx=None), NULL), (dict(counts=None), NULL), (dict(token_of=None), NULL), (dict(slot=None), NULL),
    (dict(T=0, counts=None), NULL), (dict(T=1 << 20, scratch=None), WS), (dict(T=1 << 20, nbytes=16), WS), (dict(T=1 << 20, scratch=A + 4), ALIGN),
])
def test_sort_refusals(change, code):
    assert _sort(**change) == code


@pytest.mark.parametrize("big", [1 << 30, 1 << 46, 1 << 62, (1 << 63) - 1, -(1 << 63), -1])
def test_sort_scratch_of_absurd_sizes(big):
    assert lib.b200moe_moe_sort_scratch_bytes(big, 16, 2) == 0
    assert lib.b200moe_moe_sort_scratch_bytes(4, big, 2) == 0
    assert lib.b200moe_moe_sort_scratch_bytes(4, 16, big) == 0
    assert _sort(T=big) == SHAPE and _sort(E=big) == SHAPE and _sort(k=big) == SHAPE


def test_sort_scratch_holds_the_counts_of_every_block():
    for T, E, k in ((1, 1, 1), (512, 256, 8), (513, 256, 8), (4096, 256, 8), (4097, 256, 8), (65536, 1024, 8), (1 << 25, 7, 31)):
        pairs = T * k
        blocks = 1 if pairs <= 4096 else min(128, -(-pairs // 1024))
        assert lib.b200moe_moe_sort_scratch_bytes(T, E, k) == (0 if blocks == 1 else 4 * E * 128)


def _rows(name, **change):
    c = {"dispatch": dict(x=A, f32=0, token_of=A, slot=A, rows=A), "dispatch_grad": dict(g=A, f32=0, slot=A, x=A),
         "combine": dict(y=A, f32=0, w=A, slot=A, out=A),
         "combine_grad": dict(y=A, f32=0, w=A, token_of=A, slot=A, g=A, gy=A, gw=A)}[name]
    c |= dict(T=8, k=2, H=64)
    assert set(change) <= set(c)
    c.update(change)
    return getattr(lib, "b200moe_moe_" + name)(*c.values(), None)


@pytest.mark.parametrize("name,tensors,aligned", [
    ("dispatch", ["x", "token_of", "slot", "rows"], ["x", "rows"]), ("dispatch_grad", ["g", "slot", "x"], ["g", "x"]),
    ("combine", ["y", "w", "slot", "out"], ["y", "out"]), ("combine_grad", ["y", "w", "token_of", "slot", "g"], ["y", "g", "gy"])])
def test_row_refusals(name, tensors, aligned):
    for change in (dict(T=-1), dict(k=0), dict(k=33), dict(H=0), dict(H=12), dict(H=1 << 40), dict(T=1 << 30), dict(T=1 << 62), dict(H=-8)):
        assert _rows(name, **change) == SHAPE
    assert _rows(name, f32=2) == ARG
    for t in tensors:
        assert _rows(name, **{t: None}) == NULL
    for t in aligned:
        assert _rows(name, **{t: A + 8}) == ALIGN
    assert _rows(name, T=0, **{t: None for t in tensors}) == OK


def test_a_gradient_that_nobody_wants():
    assert _rows("combine_grad", gy=None, gw=None) == OK


@pytest.mark.parametrize("args,code", [
    ((A, None, A, A, 4, 4, 48), SHAPE), ((A, None, A, A, 4, 4, 0), SHAPE), ((A, None, A, A, 3, 4, 128), SHAPE),
    ((A, None, A, A, -1, 0, 128), SHAPE), ((A, A, A, A, 4, 1 << 40, 128), SHAPE), ((None, None, A, A, 4, 4, 128), NULL),
    ((A, None, None, A, 4, 4, 128), NULL), ((A, None, A, None, 4, 4, 128), NULL), ((A + 2, None, A, A, 4, 4, 128), ALIGN),
    ((A, None, A + 8, A, 4, 4, 128), ALIGN), ((A, None, A, A + 2, 4, 4, 128), ALIGN), ((None, None, None, None, 0, 0, 128), OK),
])
def test_quantise_refusals(args, code):
    assert lib.b200moe_mxfp4_quantize_rows(*args, None, 0, None) == code


@pytest.mark.parametrize("big", [1 << 30, 1 << 46, 1 << 58, 1 << 62, (1 << 63) - 1, -(1 << 63)])
def test_quantise_absurd_sizes(big):
    for sizes in ((big, 64, 128), (4, big, 128), (4, 64, big), (big, big, big)):
        assert lib.b200moe_mxfp4_quantize_rows_scratch_bytes(*sizes, 1) == 0
        assert lib.b200moe_mxfp4_quantize_rows(A, A, A, A, *sizes, None, 0, None) == SHAPE


def test_quantise_scratch_is_aligned():
    assert lib.b200moe_mxfp4_quantize_rows_scratch_bytes(64, 1 << 20, 128, 1) == 64 * 68
    assert lib.b200moe_mxfp4_quantize_rows(A, A, A, A, 64, 1 << 20, 128, A + 8, 1 << 40, None) == ALIGN


def test_python_refuses_host_tensors():
    x = torch.zeros(4, 128, dtype=torch.bfloat16)
    i = torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: ops.moe_sort(i, 4), lambda: ops.moe_dispatch(x, i.view(-1), i), lambda: ops.mxfp4_quantize_rows(x),
                 lambda: ops.moe_combine(x, torch.zeros(2, 2), i.view(-1), i)):
        with pytest.raises(RuntimeError):
            call()


def test_routed_pass_is_for_one_rank():
    from ascend_kernel_b200.moe_layer import MoELayer

    layer = object.__new__(MoELayer)
    layer.world, layer.px = 2, None
    with pytest.raises(RuntimeError, match="one rank"):
        layer.forward_routed(None, None, None)
    layer.world, layer.px = 1, object()
    with pytest.raises(RuntimeError, match="one rank"):
        layer.forward_routed(None, None, None)
