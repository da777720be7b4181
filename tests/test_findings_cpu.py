"""The C entries around the pairs of words that keep findings: refusals, which need no device."""
import ctypes

import pytest

from ascend_kernel_b200 import _abi

lib = _abi.lib
A = 1 << 20  # an address that is never read
NULL, SHAPE, ARG = 2, 3, 6


def test_pairs_outside_are_refused():
    p = ctypes.c_void_p()
    for pair in (-1, 1024, 1 << 30):
        assert lib.b200moe_findings_pair(pair, ctypes.byref(p)) == ARG
    assert lib.b200moe_findings_pair(0, None) == NULL


def test_reading_refuses_null():
    out = (ctypes.c_int32 * 2)()
    assert lib.b200moe_read_findings_at(None, out, 0, None) == NULL
    assert lib.b200moe_read_findings_at(A, None, 0, None) == NULL
    assert lib.b200moe_read_findings(None, 0, None) == NULL


@pytest.mark.parametrize("findings", [None, A])
def test_the_entries_that_take_a_pair_refuse_what_the_others_do(findings):
    assert lib.b200moe_grouped_gemm_fp8_block_findings(A, A, A, A, A, A, A, 4, 8, 256, 2, 1, 0, A, 1 << 40, findings, None) == SHAPE
    assert lib.b200moe_grouped_gemm_fp8_block_findings(None, A, A, A, A, A, A, 4, 256, 256, 2, 1, 0, A, 1 << 40, findings, None) == NULL
    assert lib.b200moe_moe_balance_loss_findings(A, 0, A, None, None, 8, 16, 2, 2, A, A, A, A, A, 1 << 40, findings, None) == SHAPE
    assert lib.b200moe_moe_balance_loss_findings(A, 2, A, A, None, 8, 16, 2, 2, A, A, A, A, A, 1 << 40, findings, None) == ARG
