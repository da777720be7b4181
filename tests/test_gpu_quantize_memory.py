"""A quantisation whose results have their place already needs no further memory: where there is none for the scratch of the two-pass
form, every row of the result is quantised.  In a process of its own, whose allocator holds nothing else."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = r"""
import torch
import ascend_kernel_b200 as ak
from ascend_kernel_b200 import _abi, ops

T, k, K = 4096, 4, 7168
gen = torch.Generator(device="cuda").manual_seed(1)
x = torch.randn(T, K, generator=gen, device="cuda").to(torch.bfloat16)
index = torch.randint(0, T, (T * k,), generator=gen, device="cuda").to(torch.int32)
assert _abi.lib.b200moe_fp8_quantize_rows_scratch_bytes(T, T * k, K, 1) > 16 << 20
want, want_scale = ak.fp8_quantize_rows(x, index)
codes, scale = torch.empty_like(want), torch.empty_like(want_scale)
torch.cuda.synchronize()
torch.cuda.empty_cache()
before = ops.LAUNCHES
# 4 MB more than there is now: room for nothing of the scratch's size
torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (4 << 20)) / torch.cuda.get_device_properties(0).total_memory)
try:
    torch.empty(16 << 20, dtype=torch.uint8, device="cuda")
    raise SystemExit("there is room")
except torch.cuda.OutOfMemoryError:
    pass
ak.fp8_quantize_rows(x, index, codes, scale)
torch.cuda.set_per_process_memory_fraction(1.0)
assert ops.LAUNCHES == before + 1
assert torch.equal(codes, want) and torch.equal(scale, want_scale)
print("done")
"""


def test_no_room_for_the_scratch():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("done"), r.stderr[-2000:]
