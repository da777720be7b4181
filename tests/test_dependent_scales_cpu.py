"""The 8-bit product starts beside the end of the kernel before it, which may be the one that writes its scales (the gate/up product's,
the quantisation's): it reads them with ordinary loads.  ``__ldg`` is defined for data that nothing writes while the kernel is there; no run
on a device can show the difference."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ascend_kernel_b200", "csrc")


def test_scales_are_read_with_ordinary_loads():
    text = open(os.path.join(CSRC, "grouped_gemm_fp8_block.cu")).read()
    assert "launch_dependent(kernel, grid" in text
    assert re.findall(r"(\w+)\(ws \+ ", text) == ["__ldca"] and re.findall(r"(\w+)\(xs \+ ", text) == ["__ldca"]
    assert "__ldg(" not in text and "ldg_stream(" not in text


def test_gathered_rows_are_read_with_ordinary_loads():
    text = open(os.path.join(CSRC, "fp8_quantize.cu")).read()
    kernel = text[text.index("gather_kernel(const uint4*"):text.index("static bool sizes_ok")]
    assert "grid_dep_wait();" in kernel
    # (the index was there before the quantisation began, which is launched the usual way)
    assert set(re.findall(r"__ldg\((\w+)", kernel)) == {"index"}
