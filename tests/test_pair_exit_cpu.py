"""The pair kernel's second CTA takes part in commits that the first one issues (a multicast arrive on barriers of both).  It may not end
before they have arrived: shared memory that has passed to another block would get them.  No run can show that, so the source is read:
every barrier that a commit arrives on is waited for in both CTAs before the last cluster barrier."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ascend_kernel_b200", "csrc")


def test_every_commit_has_arrived_before_a_cta_of_the_pair_ends():
    text = open(os.path.join(CSRC, "grouped_gemm_fp8_block.cu")).read()
    kernel = text[text.index("grouped_kernel(const __grid_constant__"):text.index("// The parts of a split k range")]
    committed = set(re.findall(r"umma_commit_pair\(ptx::smem_u32\(&sy->(\w+)\[", kernel))
    assert committed == {"t_full", "empty", "drain"}
    # the epilogue warps of both CTAs take every buffer
    assert "wait(&sy->t_full[e.buf], e.ph" in text
    # the loading warp of both CTAs, whose role is not under a test of the rank, waits for the stages that it filled last
    loads = kernel[kernel.index("if (warp == kWarpLoad)"):kernel.index("} else if (warp == kWarpScale)")]
    tail = loads[loads.index("while (ok) {"):]
    assert re.search(r"for \(uint32_t i = it; ok && i < it \+ \(uint32_t\)n_slots; \+\+i\) \{\s*if \(i >= \(uint32_t\)n_slots\) ok = wait\(&sy->empty\[slot\], ph \^ 1", tail)
    # the first CTA's MMA warps and the second's idle ones
    assert "mbar_wait(ptx::smem_u32(&sy->drain[turn]), 0)" in kernel
    end = kernel[kernel.rindex("__syncthreads();"):]
    wait = end.index("if (rank != 0 && (warp == kWarpMma0 || warp == kWarpMma0 + 1)) (void)ptx::mbar_wait(ptx::smem_u32(&sy->drain[warp - kWarpMma0]), 0);")
    assert wait < end.index("ptx::cluster_sync();")
