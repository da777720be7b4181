"""What no run of the 4-bit product can show, read from its source: it starts beside the end of the kernel before it, which may be the one that writes its
scales, so it reads them with ordinary loads; and the second CTA of a pair ends behind every arrival that a commit of the first one's sends it."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ascend_kernel_b200", "csrc")


def _kernel():
    text = open(os.path.join(CSRC, "grouped_gemm_mxfp4.cu")).read()
    return text, text[text.index("grouped_kernel(const __grid_constant__"):text.index("static bool sizes_ok")]


def test_scales_are_read_with_ordinary_loads():
    text, kernel = _kernel()
    assert "launch_dependent(kernel" in text
    assert kernel.index("grid_dep_wait();") < kernel.index("load_row_starts(")
    loads = re.findall(r"c\.v\[b\](?:\.\w)? = (\w+)\(", kernel)
    assert len(loads) == 6 and set(loads) == {"make_uint4", "__ldca"}
    assert "__ldg(" not in text and "ldg_stream(" not in text


def test_gathered_rows_are_read_with_ordinary_loads():
    text = open(os.path.join(CSRC, "mxfp4_quantize.cu")).read()
    kernel = text[text.index("gather_kernel(const uint4*"):text.index("static bool sizes_ok")]
    assert "grid_dep_wait();" in kernel
    # (the index was there before the quantisation began, which is launched the usual way)
    assert set(re.findall(r"__ldg\((\w+)", kernel)) == {"index"}


def test_every_commit_has_arrived_before_a_cta_of_the_pair_ends():
    _, kernel = _kernel()
    committed = set(re.findall(r"umma_commit_pair\(ptx::smem_u32\(&sy->(\w+)\[", kernel))
    assert committed == {"s_empty", "empty", "d_full", "drain"}
    # the epilogue warps of both CTAs wait for every tile
    assert "wait(&sy->d_full[buf], ph" in kernel
    # the loading warp of both waits for the stages that it filled last, the scale warps for the chunks that they wrote last
    loads = kernel[kernel.index("if (warp == kWarpLoad)"):kernel.index("} else if (warp < kWarpMma0 + kBlocks && rank == 0)")]
    assert re.search(r"for \(uint32_t i = it; ok && i < it \+ \(uint32_t\)n_slots; \+\+i\) \{\s*if \(i >= \(uint32_t\)n_slots\) ok = wait\(&sy->empty\[slot\], ph \^ 1", loads)
    scales = kernel[kernel.index("const auto put = "):kernel.index("setmaxnreg.inc")]
    assert re.search(r"for \(uint32_t i = n < 2 \? n : 2; ok && i > 0; --i\) \{.*?ok = wait\(&sy->s_empty\[cb\], cph \^ 1", scales, re.S)
    # the first CTA's MMA warps and the second's idle ones
    assert "mbar_wait(ptx::smem_u32(&sy->drain[u]), 0)" in kernel
    end = kernel[kernel.rindex("__syncthreads();"):]
    wait = end.index("if (rank != 0 && warp >= kWarpMma0 && warp < kWarpMma0 + kBlocks) (void)ptx::mbar_wait(ptx::smem_u32(&sy->drain[warp - kWarpMma0]), 0);")
    assert wait < end.index("ptx::cluster_sync();")


def test_registers_of_the_roles_are_those_of_the_launch():
    """A split whose sum is above the launch's total would wait for ever: 128 registers (65536 / 512 threads) for each of the 16 warps."""
    _, kernel = _kernel()
    split = [int(n) for n in re.findall(r"setmaxnreg\.(?:dec|inc)\.sync\.aligned\.u32 (\d+);", kernel)]
    assert len(split) == 3 and split[0] < 128 and split[1] < 128 < split[2]
    assert 4 * split[0] + 4 * split[1] + 8 * split[2] <= 16 * 128 and all(n % 8 == 0 for n in split)
