"""The sort by expert at numbers of experts around the shared memory that a launch has without asking for more (48 KB, of which
34 counts an expert are dynamic and the warps' sums static)."""
import os
import subprocess
import sys

import pytest
import torch

import ascend_kernel_b200 as ak
from tests import permute_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SIZES = [(100, 4), (2000, 4)]  # one block, and two kernels


def check(E, T, k):
    gen = torch.Generator(device=DEV).manual_seed(E + T)
    idx = torch.randint(-1, E + 1, (T, k), generator=gen, device=DEV).to(torch.int32)
    idx[0, 0], idx[T - 1, k - 1] = E - 1, E - 1
    for a, b in zip(ak.moe_sort(idx, E), R.sort(idx, E)):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


@pytest.mark.parametrize("E", [360, 361, 362])
def test_first_call_of_a_process(E):
    """What a kernel was granted once it keeps, so that a larger number of experts before would hide a launch that does not ask."""
    call = f"from tests.test_gpu_moe_sort_experts import SIZES, check\nfor s in SIZES: check({E}, *s)"
    r = subprocess.run([sys.executable, "-c", call], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


@pytest.mark.parametrize("E", [257, 300, 352, 353, 359, 384, 512, 1023])
def test_more_experts_than_a_small_block_has_threads(E):
    for s in SIZES:
        check(E, *s)
