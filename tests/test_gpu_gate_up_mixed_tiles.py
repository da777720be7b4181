"""The gate/up product where a pair's consecutive tiles differ in size and a tile has so few blocks of k that the epilogue's groups
may be a tile apart: scales and codes against the 64-bit definition, and the same bits each time."""
import pytest
import torch

import ascend_kernel_b200 as ak
from tests import fp8_ref as R
from tests.test_gpu_fp8_block import _check_gate_up, _problem

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("K,most", [(128, 64), (256, 64), (512, 64), (128, 128), (256, 96), (256, 128), (128, 160), (384, 160)])
def test_tiles_of_every_size_side_by_side(K, most):
    G, N = 256, 1024  # two tiles an expert at least: seven waves of the pairs
    rows = torch.randint(1, most + 1, (G,), generator=torch.Generator().manual_seed(K + most))
    rows[::2] = rows[::2].clamp(max=32)  # (a tile of 32 rows beside every larger one)
    rows[1] = most
    counts = rows.tolist()
    x, xs, w, ws, gl = _problem(counts, K, N, 3, seed=K)
    ws = ws * 3
    M = x.shape[0]

    def run():
        codes, scale = torch.zeros(M, N // 2, dtype=torch.uint8, device=DEV), torch.zeros(M, N // 256, device=DEV)
        ak.grouped_gemm_fp8_block(x, xs, w, ws, gl, codes, output_scale=scale, group_list_type=1, gate_up_silu=True)
        return codes, scale

    codes, scale = run()
    _check_gate_up(codes, scale, x, xs, w, ws, R.bounds(counts, 1, M))
    for _ in range(20):
        again, again_scale = run()
        assert torch.equal(again, codes) and torch.equal(again_scale, scale)
    assert ak.last_status() == (0, 0)
