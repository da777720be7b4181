// Python module `cinfer_ascendc`: the operator names and keyword arguments of the reference's
// extension (pybind.cpp:13-32 of the reference; GroupedGemm at grouped_gemm/src/grouped_gemm.h:12-16,
// GroupedSoftGemv at grouped_soft_gemv/src/grouped_soft_gemv.h:12-14), bound to the B200 kernels
// through the C ABI of include/b200moe.h.  This file only unpacks tensors: device/dtype/shape
// checks, the current CUDA stream, a workspace from torch's caching allocator, status -> exception.
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/extension.h>

#include <algorithm>
#include <atomic>
#include <cstdio>
#include <map>
#include <mutex>
#include <stdexcept>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "../../../include/b200moe.h"

namespace {

int compute_type_of(const std::string& s) {
    if (s == "fp8") return B200MOE_CT_FP8;
    if (s == "fp4") return B200MOE_CT_FP4;
    if (s == "int8") return B200MOE_CT_INT8;
    if (s == "int4") return B200MOE_CT_INT4;
    if (s == "bf16") return B200MOE_CT_BF16;
    // same report as the reference binding for an unknown computeType
    std::printf("Invalid compute type: %s. Supported: \"fp4\", \"fp8\", \"int8\", \"int4\", \"bf16\"\n", s.c_str());
    throw std::runtime_error("Host tiling failed!");
}

int layout_of(const std::string& s) {
    if (s == "ascend") return B200MOE_LAYOUT_ASCEND;
    if (s == "canonical") return B200MOE_LAYOUT_CANONICAL;
    throw std::runtime_error("weight_layout must be \"ascend\" or \"canonical\"");
}

void check_tensor(const at::Tensor& t, const char* name) {
    TORCH_CHECK(t.defined(), name, " is undefined");
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (there is no CPU path)");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

void raise_on(int rc, const char* what) {
    if (rc != B200MOE_OK) {
        std::printf("%s failed. ERROR: %d (%s)\n", what, rc, b200moe_strerror(rc));
        throw std::runtime_error(std::string(what) + ": " + b200moe_strerror(rc));
    }
}

struct Dims {
    int64_t M, K, N, G;
};

// One persistent workspace per (device, stream).  The reference binding keeps a process-wide,
// never-freed workspace map as well (grouped_gemm/src/grouped_gemm.cpp:91-120); this one is guarded by
// a mutex, and it exists for a second reason: words 4 / 5 of a workspace keep the first device-side
// finding (invalid group list, expired wait) of every call that used it, so last_status() can report
// at the caller's synchronisation point what no asynchronous call can report by itself.
// A captured CUDA graph keeps the address of the workspace its calls got.  So a workspace that became too small is
// kept, not freed, or replays would write into memory that has become somebody else's.  The first one holds what
// every operator needs whatever its sizes (the split GEMV's 4.9 MB is the largest such part) and a larger one is at
// least twice its predecessor, so the kept ones of a stream are together no larger than the one in use.  Findings of
// replays land in the kept ones, so the status calls read those too.
std::mutex g_ws_mutex;
using StreamKey = std::pair<int, void*>;
std::map<StreamKey, at::Tensor> g_workspaces;
std::vector<std::pair<StreamKey, at::Tensor>> g_kept_workspaces;
constexpr size_t kFirstWorkspace = size_t(8) << 20;

at::Tensor workspace_for(const at::Tensor& like, size_t bytes, void* stream) {
    std::lock_guard<std::mutex> lock(g_ws_mutex);
    const StreamKey key((int)like.get_device(), stream);
    auto it = g_workspaces.find(key);
    if (it == g_workspaces.end() || (size_t)it->second.numel() < bytes) {
        const bool first = it == g_workspaces.end();
        const size_t size = std::max(bytes, first ? kFirstWorkspace : 2 * (size_t)it->second.numel());
        at::Tensor fresh = at::empty({(int64_t)size}, like.options().dtype(at::kByte));
        fresh.slice(0, 0, B200MOE_STATUS_BYTES).zero_();  // (the operators clear what else they start from)
        if (!first) {
            fresh.slice(0, 16, 24).copy_(it->second.slice(0, 16, 24));
            g_kept_workspaces.emplace_back(key, it->second);
        }
        g_workspaces[key] = fresh;
        return fresh;
    }
    return it->second;
}

// The operators without a workspace of status words keep their findings in pairs of words of the library's, one for each of the two
// bindings and every stream that they were called on: like the workspaces, so that a status call waits for those streams
// alone and clears what its own binding found.  (Should a device run out of pairs, the streams that come last share one.)
enum Binding { kDropIn, kMirror };  // this module, and the package's functions of the same names
struct FindingWords {
    Binding binding;
    int device;
    void* stream;
    int32_t* words;
};
std::vector<FindingWords> g_findings;  // (guarded by g_ws_mutex)

// for the current device
int32_t* findings_for(Binding binding, int device, void* stream) {
    std::lock_guard<std::mutex> lock(g_ws_mutex);
    int used = 0;
    for (const auto& f : g_findings) {
        if (f.binding == binding && f.device == device && f.stream == stream) return f.words;
        used += f.device == device;
    }
    int32_t* words = nullptr;
    const int rc = b200moe_findings_pair(std::min(used + 1, B200MOE_FINDINGS_PAIRS - 1), &words);
    TORCH_CHECK(rc == B200MOE_OK, "findings_pair: ", b200moe_strerror(rc));
    g_findings.push_back({binding, device, stream, words});
    return words;
}

// Whether work may be queued on the stream now (not while it is captured: what is recorded there has not run).
bool may_wait_for(void* stream) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &status) == cudaSuccess) return status == cudaStreamCaptureStatusNone;
    (void)cudaGetLastError();
    return false;
}

// The first finding of a binding's calls on the current device.  Waits for the streams that they ran on and, since replays of
// captured calls run where the caller says, for the caller's own; only where there were such calls.  `clear` takes the finding
// that is returned and leaves the others to the calls that follow.  g_ws_mutex is held.
std::pair<int, int> read_findings(Binding binding, int device, bool clear) {
    std::pair<int, int> found{0, 0};
    bool waited = false;
    for (const auto& f : g_findings) {
        if (f.binding != binding || f.device != device) continue;
        if (!waited) {
            waited = true;
            const auto own = c10::cuda::getCurrentCUDAStream().stream();
            if (may_wait_for(own)) TORCH_CHECK(cudaStreamSynchronize(own) == cudaSuccess, "cudaStreamSynchronize failed");
        }
        if (!may_wait_for(f.stream)) continue;
        int32_t out[2] = {0, 0};
        int rc = b200moe_read_findings_at(f.words, out, 0, f.stream);
        if (rc == B200MOE_OK && found.first == 0 && out[0] != 0) {
            found = {out[0], out[1]};
            if (clear) rc = b200moe_read_findings_at(f.words, out, 1, f.stream);
        }
        TORCH_CHECK(rc == B200MOE_OK, "read_findings: ", b200moe_strerror(rc));
    }
    return found;
}

// What the package's own functions found on a device, for its status calls (which know its workspaces).
std::pair<int, int> MirrorFindings(int64_t device, bool clear) {
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
    std::lock_guard<std::mutex> lock(g_ws_mutex);
    return read_findings(kMirror, (int)device, clear);
}

std::pair<int, int> LastStatus(bool clear) {
    std::lock_guard<std::mutex> lock(g_ws_mutex);
    int dev = 0;
    TORCH_CHECK(cudaGetDevice(&dev) == cudaSuccess, "cudaGetDevice failed");
    std::pair<int, int> found{0, 0};
    auto read = [&](const StreamKey& key, const at::Tensor& ws) {
        if (key.first != dev) return;
        int32_t out[2] = {0, 0};
        const int rc = b200moe_read_sticky_status(ws.data_ptr(), out, clear ? 1 : 0, key.second);
        TORCH_CHECK(rc == B200MOE_OK, "read_sticky_status: ", b200moe_strerror(rc));
        if (found.first == 0 && out[0] != 0) found = {out[0], out[1]};
    };
    for (auto& kv : g_workspaces) read(kv.first, kv.second);
    for (auto& kv : g_kept_workspaces) read(kv.first, kv.second);
    // and what the operators without a workspace of status words found
    const auto kept = read_findings(kDropIn, dev, clear && found.first == 0);
    return found.first != 0 ? found : kept;
}

void CheckStatus() {
    const auto st = LastStatus(true);
    if (st.first != 0)
        throw std::runtime_error("b200moe device status " + std::to_string(st.first) + " (detail " +
                                 std::to_string(st.second) + "): " +
                                 (st.first == 1 ? "a group_list was invalid, rows were clamped"
                                                : "a bounded wait inside a kernel expired, results are incomplete"));
}

Dims dims_of(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& group_list, const at::Tensor& output,
             int ct) {
    TORCH_CHECK(x.scalar_type() == at::kBFloat16 && output.scalar_type() == at::kBFloat16,
                "x and output must be bfloat16");
    TORCH_CHECK(group_list.scalar_type() == at::kLong, "group_list must be int64");
    TORCH_CHECK(x.dim() == 2 && weight.dim() == 3 && output.dim() == 2, "expected x [M,K], weight [G,K,N], output [M,N]");
    if (ct == B200MOE_CT_BF16) {
        TORCH_CHECK(weight.scalar_type() == at::kBFloat16, "weight must be bfloat16 for computeType bf16");
    } else {
        TORCH_CHECK(weight.element_size() == 1, "weight must be a 1-byte container (uint8 / int8)");
    }
    Dims d{x.size(0), x.size(1), weight.size(2), weight.size(0)};
    if (ct == B200MOE_CT_FP4 || ct == B200MOE_CT_INT4) d.N *= 2;  // two codes per byte
    TORCH_CHECK(weight.size(1) == d.K && output.size(0) == d.M && output.size(1) == d.N && group_list.numel() == d.G,
                "shape mismatch between x, weight, output and group_list");
    return d;
}

void check_scale(const at::Tensor& s, int ct, const Dims& d, const char* name) {
    if (ct == B200MOE_CT_FP8) {
        TORCH_CHECK(s.scalar_type() == at::kFloat && s.numel() == d.G * (d.K / 128) * (d.N / 128), name,
                    " must be float32 [G, K/128, N/128]");
    } else if (ct == B200MOE_CT_FP4) {
        TORCH_CHECK(s.scalar_type() == at::kBFloat16 && s.numel() == d.G * (d.K / 16) * d.N, name,
                    " must be bfloat16 [G, K/16, N]");
    } else if (ct == B200MOE_CT_INT8) {
        TORCH_CHECK(s.scalar_type() == at::kBFloat16 && s.numel() == d.G * d.N, name, " must be bfloat16 [G, N]");
    } else {
        TORCH_CHECK(s.scalar_type() == at::kBFloat16 && s.numel() == d.G * (d.K / 128) * d.N, name,
                    " must be bfloat16 [G, K/128, N]");
    }
}

void GroupedGemm(at::Tensor x, at::Tensor weight, at::Tensor antiquantScaleOptional,
                 at::Tensor antiquantOffsetOptional, at::Tensor groupListOptional, const std::string& computeType,
                 at::Tensor output, int64_t group_list_type, const std::string& weight_layout) {
    const int ct = compute_type_of(computeType);
    const int layout = layout_of(weight_layout);
    check_tensor(x, "x"); check_tensor(weight, "weight");
    check_tensor(groupListOptional, "groupListOptional"); check_tensor(output, "output");
    const Dims d = dims_of(x, weight, groupListOptional, output, ct);
    const void* scale_ptr = nullptr;  // bf16: the matmul phase alone, no scale
    if (ct != B200MOE_CT_BF16) {
        check_tensor(antiquantScaleOptional, "antiquantScaleOptional");
        check_scale(antiquantScaleOptional, ct, d, "antiquantScaleOptional");
        scale_ptr = antiquantScaleOptional.data_ptr();
    }
    const void* offset = nullptr;  // fp8 / fp4: accepted and ignored, as in the reference kernel
    if ((ct == B200MOE_CT_INT8 || ct == B200MOE_CT_INT4) && antiquantOffsetOptional.defined() &&
        antiquantOffsetOptional.numel() > 0) {
        check_tensor(antiquantOffsetOptional, "antiquantOffsetOptional");
        check_scale(antiquantOffsetOptional, ct, d, "antiquantOffsetOptional");
        offset = antiquantOffsetOptional.data_ptr();
    }
    c10::cuda::CUDAGuard guard(x.device());
    auto stream = c10::cuda::getCurrentCUDAStream();
    const size_t ws_bytes = b200moe_grouped_gemm_workspace_bytes(d.M, d.K, d.N, d.G, ct, layout);
    at::Tensor ws = workspace_for(x, ws_bytes, stream.stream());
    // int4 without offsets: scratch for the one-pass kernel, from the caching allocator and back to it; without it the two-pass kernel runs
    const size_t scratch_bytes = b200moe_grouped_gemm_scratch_bytes(d.M, d.K, d.N, d.G, ct, offset != nullptr);
    at::Tensor scratch;
    if (scratch_bytes > 0) {
        try {
            scratch = at::empty({(int64_t)scratch_bytes}, x.options().dtype(at::kByte));
        } catch (const c10::OutOfMemoryError&) {
        }
    }
    raise_on(b200moe_grouped_gemm_scratch(x.data_ptr(), weight.data_ptr(), scale_ptr, offset,
                                          groupListOptional.data_ptr<int64_t>(), output.data_ptr(), d.M, d.K, d.N, d.G, ct,
                                          (int)group_list_type, layout, ws.data_ptr(), ws_bytes,
                                          scratch.defined() ? scratch.data_ptr() : nullptr, scratch_bytes, stream.stream()),
             "grouped_gemm");
}

void GroupedSoftGemv(at::Tensor x, at::Tensor weight, at::Tensor scale, at::Tensor groupList,
                     const std::string& computeType, at::Tensor output, int64_t group_list_type,
                     const std::string& weight_layout, c10::optional<at::Tensor> offset_opt) {
    const int ct = compute_type_of(computeType);
    const int layout = layout_of(weight_layout);
    check_tensor(x, "x"); check_tensor(weight, "weight"); check_tensor(scale, "scale");
    check_tensor(groupList, "groupList"); check_tensor(output, "output");
    const Dims d = dims_of(x, weight, groupList, output, ct);
    check_scale(scale, ct, d, "scale");
    const void* offset = nullptr;
    if (offset_opt.has_value() && offset_opt->defined()) {
        TORCH_CHECK(ct == B200MOE_CT_INT8 || ct == B200MOE_CT_INT4, "offset is only defined for int8 / int4");
        check_tensor(*offset_opt, "offset");
        check_scale(*offset_opt, ct, d, "offset");
        offset = offset_opt->data_ptr();
    }
    c10::cuda::CUDAGuard guard(x.device());
    auto stream = c10::cuda::getCurrentCUDAStream();
    const size_t ws_bytes = b200moe_grouped_gemv_split_workspace_bytes(d.M, d.K, d.N, d.G, ct, layout);
    at::Tensor ws = workspace_for(x, ws_bytes, stream.stream());
    raise_on(b200moe_grouped_gemv(x.data_ptr(), weight.data_ptr(), scale.data_ptr(), offset,
                                  groupList.data_ptr<int64_t>(), output.data_ptr(), d.M, d.K, d.N, d.G, ct,
                                  (int)group_list_type, layout, ws.data_ptr(), ws_bytes, stream.stream()),
             "grouped_soft_gemv");
}

void Fp4Dequant(at::Tensor codes, c10::optional<at::Tensor> scale, at::Tensor output) {
    check_tensor(codes, "codes"); check_tensor(output, "output");
    TORCH_CHECK(codes.element_size() == 1 && output.scalar_type() == at::kBFloat16 &&
                output.numel() == 2 * codes.numel(), "codes: bytes [..., L/2]; output: bfloat16 [..., L]");
    const void* sp = nullptr;
    if (scale.has_value() && scale->defined()) {
        check_tensor(*scale, "scale");
        TORCH_CHECK(scale->element_size() == 1 && scale->numel() * 32 == output.numel(),
                    "scale: one e8m0 byte per 32 elements");
        sp = scale->data_ptr();
    }
    c10::cuda::CUDAGuard guard(codes.device());
    raise_on(b200moe_fp4_dequant(codes.data_ptr(), sp, output.data_ptr(), output.numel(),
                                 sp ? B200MOE_FP4_SCALE_E8M0_PER32 : B200MOE_FP4_SCALE_NONE,
                                 c10::cuda::getCurrentCUDAStream().stream()),
             "fp4_dequant");
}

void Fp4DequantBf16Scale(at::Tensor codes, at::Tensor scale, at::Tensor output, const std::string& weight_layout) {
    check_tensor(codes, "codes"); check_tensor(scale, "scale"); check_tensor(output, "output");
    TORCH_CHECK(codes.dim() == 3 && codes.element_size() == 1, "codes: bytes [G, K, N/2]");
    const int64_t G = codes.size(0), K = codes.size(1), N = 2 * codes.size(2);
    TORCH_CHECK(scale.scalar_type() == at::kBFloat16 && scale.numel() == G * (K / 16) * N, "scale: bfloat16 [G, K/16, N]");
    TORCH_CHECK(output.scalar_type() == at::kBFloat16 && output.numel() == G * K * N, "output: bfloat16 [G, K, N]");
    c10::cuda::CUDAGuard guard(codes.device());
    raise_on(b200moe_fp4_dequant_bf16_scale(codes.data_ptr(), scale.data_ptr(), output.data_ptr(), G, K, N,
                                            layout_of(weight_layout), c10::cuda::getCurrentCUDAStream().stream()),
             "fp4_dequant_bf16_scale");
}

void Fp8Dequant(at::Tensor codes, at::Tensor scale, at::Tensor output) {
    check_tensor(codes, "codes"); check_tensor(scale, "scale"); check_tensor(output, "output");
    TORCH_CHECK(codes.dim() == 3 && codes.element_size() == 1, "codes: uint8 [G, K, N]");
    const int64_t G = codes.size(0), K = codes.size(1), N = codes.size(2);
    TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.numel() == G * (K / 128) * (N / 128),
                "scale: float32 [G, K/128, N/128]");
    TORCH_CHECK(output.scalar_type() == at::kBFloat16 && output.numel() == G * K * N, "output: bfloat16 [G, K, N]");
    c10::cuda::CUDAGuard guard(codes.device());
    raise_on(b200moe_fp8_dequant(codes.data_ptr(), scale.data_ptr<float>(), output.data_ptr(), G, K, N,
                                 c10::cuda::getCurrentCUDAStream().stream()),
             "fp8_dequant");
}

at::Tensor PackWeightInt8(at::Tensor weight, bool gate_up) {
    check_tensor(weight, "weight");
    TORCH_CHECK(weight.dim() == 3 && weight.element_size() == 1, "weight: int8 [G, K, N]");
    at::Tensor out = at::empty_like(weight);
    c10::cuda::CUDAGuard guard(weight.device());
    raise_on(b200moe_pack_weight_int8(weight.data_ptr(), out.data_ptr(), weight.size(0), weight.size(1), weight.size(2),
                                      gate_up ? 1 : 0, c10::cuda::getCurrentCUDAStream().stream()),
             "pack_weight_int8");
    return out;
}

// grouped_gemm with computeType "int8" on weights from pack_weight_int8 (same keyword names; scale / offset in
// the original column order; gate_up_silu: output [M, N/2] = bf16(silu(gate) * up)).
void GroupedGemmPacked(at::Tensor x, at::Tensor weight, at::Tensor antiquantScaleOptional,
                       c10::optional<at::Tensor> antiquantOffsetOptional, at::Tensor groupListOptional, at::Tensor output,
                       int64_t group_list_type, bool gate_up_silu) {
    check_tensor(x, "x"); check_tensor(weight, "weight"); check_tensor(antiquantScaleOptional, "antiquantScaleOptional");
    check_tensor(groupListOptional, "groupListOptional"); check_tensor(output, "output");
    TORCH_CHECK(x.scalar_type() == at::kBFloat16 && output.scalar_type() == at::kBFloat16, "x and output must be bfloat16");
    TORCH_CHECK(groupListOptional.scalar_type() == at::kLong, "group_list must be int64");
    TORCH_CHECK(x.dim() == 2 && weight.dim() == 3 && weight.element_size() == 1, "expected x [M,K], packed weight [G,K,N]");
    Dims d{x.size(0), x.size(1), weight.size(2), weight.size(0)};
    TORCH_CHECK(weight.size(1) == d.K && output.size(0) == d.M && output.size(1) == (gate_up_silu ? d.N / 2 : d.N) &&
                groupListOptional.numel() == d.G, "shape mismatch between x, weight, output and group_list");
    check_scale(antiquantScaleOptional, B200MOE_CT_INT8, d, "antiquantScaleOptional");
    const void* offset = nullptr;
    if (antiquantOffsetOptional.has_value() && antiquantOffsetOptional->defined() && antiquantOffsetOptional->numel() > 0) {
        check_tensor(*antiquantOffsetOptional, "antiquantOffsetOptional");
        check_scale(*antiquantOffsetOptional, B200MOE_CT_INT8, d, "antiquantOffsetOptional");
        offset = antiquantOffsetOptional->data_ptr();
    }
    c10::cuda::CUDAGuard guard(x.device());
    auto stream = c10::cuda::getCurrentCUDAStream();
    const size_t ws_bytes = b200moe_grouped_gemm_workspace_bytes(d.M, d.K, d.N, d.G, B200MOE_CT_INT8, B200MOE_LAYOUT_CANONICAL);
    at::Tensor ws = workspace_for(x, ws_bytes, stream.stream());
    raise_on(b200moe_grouped_gemm_int8_packed(x.data_ptr(), weight.data_ptr(), antiquantScaleOptional.data_ptr(), offset,
                                              groupListOptional.data_ptr<int64_t>(), output.data_ptr(), d.M, d.K, d.N, d.G,
                                              (int)group_list_type, gate_up_silu ? 1 : 0, ws.data_ptr(), ws_bytes,
                                              stream.stream()),
             "grouped_gemm_packed");
}

at::Tensor Fp4ScaleFold(at::Tensor block_scale, at::Tensor global_scale) {
    check_tensor(block_scale, "block_scale"); check_tensor(global_scale, "global_scale");
    TORCH_CHECK(block_scale.dim() == 3 && block_scale.scalar_type() == at::kBFloat16, "block_scale: bfloat16 [G, N, K/16]");
    const int64_t G = block_scale.size(0), N = block_scale.size(1), KB = block_scale.size(2);
    TORCH_CHECK(global_scale.scalar_type() == at::kFloat && G > 0 &&
                (global_scale.numel() == G || global_scale.numel() == 2 * G), "global_scale: float32 [G, 1 or 2, 1]");
    at::Tensor out = at::empty({G, KB, N}, block_scale.options());
    c10::cuda::CUDAGuard guard(block_scale.device());
    raise_on(b200moe_fp4_scale_fold(block_scale.data_ptr(), global_scale.data_ptr<float>(), out.data_ptr(), G, N, KB,
                                    global_scale.numel() / G, c10::cuda::getCurrentCUDAStream().stream()),
             "fp4_scale_fold");
    return out;
}

// ---- rows and experts in 8-bit floats with a scale per block of 128, and the router's balance loss -----------------------

using OptionalTensor = c10::optional<at::Tensor>;

const at::Tensor* given(const OptionalTensor& t, const char* name, const at::Tensor& like) {
    if (!t.has_value() || !t->defined()) return nullptr;
    check_tensor(*t, name);
    TORCH_CHECK(t->device() == like.device(), name, " is on another device");
    return &*t;
}
void check_beside(const at::Tensor& t, const char* name, const at::Tensor& like) {
    check_tensor(t, name);
    TORCH_CHECK(t.device() == like.device(), name, " is on another device");
}
void check_e4m3(const at::Tensor& t, const char* name, int64_t dim) {
    TORCH_CHECK((t.scalar_type() == at::kByte || t.scalar_type() == at::kFloat8_e4m3fn) && t.dim() == dim, name, " must be ", dim,
                "-dimensional e4m3 codes (uint8 or float8_e4m3fn)");
}
void check_f32(const at::Tensor& t, const char* name, at::IntArrayRef shape) {
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.sizes() == shape, name, " must be float32 of shape ", shape, ", got ",
                t.scalar_type(), " ", t.sizes());
}
int64_t blocks_of(int64_t n) { return (n + 127) / 128; }

// (codes, scale, number of kernels launched)
std::tuple<at::Tensor, at::Tensor, int> QuantizeRows(const at::Tensor& x, const OptionalTensor& index_opt, const OptionalTensor& codes_opt,
                                                     const OptionalTensor& scale_opt) {
    check_tensor(x, "x");
    TORCH_CHECK(x.dim() == 2 && x.scalar_type() == at::kBFloat16, "x must be bfloat16 [T, K]");
    const at::Tensor* index = given(index_opt, "index", x);
    TORCH_CHECK(!index || (index->scalar_type() == at::kInt && index->dim() == 1), "index must be int32 [R]");
    const int64_t T = x.size(0), K = x.size(1), R = index ? index->numel() : T, KB = blocks_of(K);
    c10::cuda::CUDAGuard guard(x.device());
    const at::Tensor* codes_in = given(codes_opt, "codes", x);
    const at::Tensor* scale_in = given(scale_opt, "scale", x);
    at::Tensor codes = codes_in ? *codes_in : at::empty({R, K}, x.options().dtype(at::kByte));
    at::Tensor scale = scale_in ? *scale_in : at::empty({R, KB}, x.options().dtype(at::kFloat));
    check_e4m3(codes, "codes", 2);
    TORCH_CHECK(codes.size(0) == R && codes.size(1) == K, "codes must be [", R, ", ", K, "]");
    check_f32(scale, "scale", {R, KB});
    // scratch from the caching allocator and back to it; without it every row of the result is quantised
    size_t scratch_bytes = b200moe_fp8_quantize_rows_scratch_bytes(T, R, K, index != nullptr);
    at::Tensor scratch;
    if (scratch_bytes > 0) {
        try {
            scratch = at::empty({(int64_t)scratch_bytes}, x.options().dtype(at::kByte));
        } catch (const c10::OutOfMemoryError&) {
            scratch_bytes = 0;
        }
    }
    raise_on(b200moe_fp8_quantize_rows(x.data_ptr(), index ? index->data_ptr<int32_t>() : nullptr, codes.data_ptr(),
                                       scale.data_ptr<float>(), T, R, K, scratch_bytes > 0 ? scratch.data_ptr() : nullptr,
                                       scratch_bytes, c10::cuda::getCurrentCUDAStream().stream()),
             "fp8_quantize_rows");
    return {codes, scale, R == 0 ? 0 : scratch_bytes > 0 ? 2 : 1};
}

std::tuple<at::Tensor, at::Tensor> Fp8QuantizeRows(const at::Tensor& x, const OptionalTensor& index, const OptionalTensor& codes,
                                                   const OptionalTensor& scale) {
    const auto out = QuantizeRows(x, index, codes, scale);
    return {std::get<0>(out), std::get<1>(out)};
}

// The number of kernels launched.
template <Binding BINDING>
int ProductFp8Block(const at::Tensor& x, const at::Tensor& x_scale, const at::Tensor& weight, const at::Tensor& weight_scale,
                         const at::Tensor& group_list, const at::Tensor& output, const OptionalTensor& output_scale_opt,
                         int64_t group_list_type, bool gate_up_silu) {
    check_tensor(x, "x");
    check_beside(x_scale, "x_scale", x); check_beside(weight, "weight", x); check_beside(weight_scale, "weight_scale", x);
    check_beside(group_list, "group_list", x); check_beside(output, "output", x);
    const at::Tensor* output_scale = given(output_scale_opt, "output_scale", x);
    check_e4m3(x, "x", 2);
    check_e4m3(weight, "weight", 3);
    TORCH_CHECK(group_list.scalar_type() == at::kLong, "group_list must be int64");
    const int64_t M = x.size(0), K = x.size(1), G = weight.size(0), N = weight.size(2);
    TORCH_CHECK(weight.size(1) == K && group_list.numel() == G, "shape mismatch: x ", x.sizes(), ", weight ", weight.sizes(),
                ", group_list ", group_list.numel());
    check_f32(x_scale, "x_scale", {M, blocks_of(K)});
    check_f32(weight_scale, "weight_scale", {G, blocks_of(K), blocks_of(N)});
    if (gate_up_silu) {
        TORCH_CHECK(N % 256 == 0, "gate_up_silu needs N to be a multiple of 256");
        check_e4m3(output, "output", 2);
        TORCH_CHECK(output.size(0) == M && output.size(1) == N / 2 && output_scale, "output must be [", M, ", ", N / 2,
                    "], with an output_scale");
        check_f32(*output_scale, "output_scale", {M, N / 256});
    } else {
        TORCH_CHECK(output.scalar_type() == at::kBFloat16 && output.dim() == 2 && output.size(0) == M && output.size(1) == N &&
                    !output_scale, "output must be bfloat16 [", M, ", ", N, "], without output_scale");
    }
    TORCH_CHECK(group_list_type == 0 || group_list_type == 1, "group_list_type must be 0 or 1");
    c10::cuda::CUDAGuard guard(x.device());
    // a workspace for this call alone: two graphs captured on one stream may be replayed side by side
    const size_t bytes = b200moe_grouped_gemm_fp8_block_workspace_bytes(M, K, N, G, gate_up_silu ? 1 : 0);
    at::Tensor workspace = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    const auto stream = c10::cuda::getCurrentCUDAStream().stream();
    raise_on(b200moe_grouped_gemm_fp8_block_findings(x.data_ptr(), x_scale.data_ptr<float>(), weight.data_ptr(),
                                                     weight_scale.data_ptr<float>(), group_list.data_ptr<int64_t>(), output.data_ptr(),
                                                     output_scale ? output_scale->data_ptr<float>() : nullptr, M, K, N, G,
                                                     (int)group_list_type, gate_up_silu ? 1 : 0, workspace.data_ptr(), bytes,
                                                     findings_for(BINDING, x.get_device(), stream), stream),
             "grouped_gemm_fp8_block");
    // (a workspace with room for parts of the k range comes with the kernel that adds them)
    return M == 0 ? 0 : bytes > b200moe_grouped_gemm_fp8_block_workspace_bytes(0, K, N, G, gate_up_silu ? 1 : 0) ? 2 : 1;
}

void GroupedGemmFp8Block(const at::Tensor& x, const at::Tensor& x_scale, const at::Tensor& weight, const at::Tensor& weight_scale,
                         const at::Tensor& group_list, const at::Tensor& output, const OptionalTensor& output_scale,
                         int64_t group_list_type, bool gate_up_silu) {
    ProductFp8Block<kDropIn>(x, x_scale, weight, weight_scale, group_list, output, output_scale, group_list_type, gate_up_silu);
}

// Kernels that backward passes of the package's own functions launched: no caller of theirs sees one.
std::atomic<int64_t> g_mirror_backward_launches{0};

template <Binding BINDING>
struct BalanceLoss : torch::autograd::Function<BalanceLoss<BINDING>> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& idx,
                                                  const OptionalTensor& seq_opt, const OptionalTensor& mask_opt) {
        const at::Tensor* seq = given(seq_opt, "seq_list", logits);
        const at::Tensor* mask = given(mask_opt, "token_mask", logits);
        const int64_t T = logits.size(0), E = logits.size(1), S = seq ? seq->numel() : 1;
        c10::cuda::CUDAGuard guard(logits.device());
        const auto f32 = logits.options().dtype(at::kFloat);
        at::Tensor loss = at::empty({S}, f32), counts = at::empty({S, E}, f32.dtype(at::kLong));
        at::Tensor kept = at::empty({S * (E + 1)}, f32);  // the load per sequence and expert, and the reciprocals of the token numbers
        const size_t bytes = b200moe_moe_balance_scratch_bytes(T, E, S);
        at::Tensor scratch = at::empty({(int64_t)bytes}, f32.dtype(at::kByte));
        float* load = kept.data_ptr<float>();
        const auto stream = c10::cuda::getCurrentCUDAStream().stream();
        raise_on(b200moe_moe_balance_loss_findings(logits.data_ptr(), logits.scalar_type() == at::kFloat ? 1 : 0, idx.data_ptr<int32_t>(),
                                                   seq ? seq->data_ptr<int64_t>() : nullptr,
                                                   mask ? static_cast<const uint8_t*>(mask->data_ptr()) : nullptr, T, E, idx.size(1), S,
                                                   loss.data_ptr<float>(), counts.data_ptr<int64_t>(), load, load + S * E,
                                                   scratch.data_ptr(), bytes, findings_for(BINDING, logits.get_device(), stream),
                                                   stream),
                 "moe_balance_loss");
        ctx->save_for_backward({logits, seq ? *seq : at::Tensor(), mask ? *mask : at::Tensor(), kept});
        ctx->mark_non_differentiable({counts});
        return {loss, counts};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "moe_balance_loss is differentiable once");
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &logits = saved[0], &seq = saved[1], &mask = saved[2], &kept = saved[3];
        if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
        const int64_t T = logits.size(0), E = logits.size(1), S = kept.numel() / (E + 1);
        c10::cuda::CUDAGuard guard(logits.device());
        const at::Tensor g = grads[0].to(at::kFloat).contiguous();
        at::Tensor out = at::empty_like(logits);
        const float* load = kept.data_ptr<float>();
        raise_on(b200moe_moe_balance_loss_grad(logits.data_ptr(), logits.scalar_type() == at::kFloat ? 1 : 0,
                                               seq.defined() ? seq.data_ptr<int64_t>() : nullptr,
                                               mask.defined() ? static_cast<const uint8_t*>(mask.data_ptr()) : nullptr, load,
                                               load + S * E, g.data_ptr<float>(), T, E, S, out.data_ptr(),
                                               c10::cuda::getCurrentCUDAStream().stream()),
                 "moe_balance_loss (gradient)");
        if (T > 0 && BINDING == kMirror) ++g_mirror_backward_launches;
        return {out, at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

template <Binding BINDING>
std::tuple<at::Tensor, at::Tensor> MoeBalanceLoss(const at::Tensor& logits, const at::Tensor& idx, const OptionalTensor& seq_opt,
                                                  const OptionalTensor& mask_opt) {
    check_tensor(logits, "logits");
    check_beside(idx, "idx", logits);
    TORCH_CHECK(logits.dim() == 2 && (logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat),
                "logits must be bfloat16 or float32 [T, E]");
    const int64_t T = logits.size(0);
    TORCH_CHECK(idx.scalar_type() == at::kInt && idx.dim() == 2 && idx.size(0) == T, "idx must be int32 [", T, ", k]");
    const at::Tensor* seq = given(seq_opt, "seq_list", logits);
    TORCH_CHECK(!seq || (seq->scalar_type() == at::kLong && seq->dim() == 1), "seq_list must be int64 [S]");
    const at::Tensor* mask = given(mask_opt, "token_mask", logits);
    TORCH_CHECK(!mask || (mask->scalar_type() == at::kBool && mask->dim() == 1 && mask->size(0) == T), "token_mask must be bool [", T, "]");
    auto out = BalanceLoss<BINDING>::apply(logits, idx, seq_opt, mask_opt);
    return {out[0], out[1]};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    using namespace pybind11::literals;
    m.def("grouped_soft_gemv", &GroupedSoftGemv, "x"_a, "weight"_a, "scale"_a, "groupList"_a, "computeType"_a,
          "output"_a, "group_list_type"_a = 0, "weight_layout"_a = "ascend", "offset"_a = pybind11::none(),
          "GROUP GEMV.");
    m.def("grouped_gemm", &GroupedGemm, "x"_a, "weight"_a, "antiquantScaleOptional"_a, "antiquantOffsetOptional"_a,
          "groupListOptional"_a, "computeType"_a, "output"_a, "group_list_type"_a = 0, "weight_layout"_a = "ascend",
          "GROUP GEMM.");
    m.def("fp4_dequant", &Fp4Dequant, "codes"_a, "scale"_a, "output"_a, "FP4(e2m1) -> BF16.");
    m.def("fp4_dequant_bf16_scale", &Fp4DequantBf16Scale, "codes"_a, "scale"_a, "output"_a, "weight_layout"_a = "ascend",
          "FP4(e2m1) x bf16 scale per 16 k -> BF16 weights.");
    m.def("fp8_dequant", &Fp8Dequant, "codes"_a, "scale"_a, "output"_a, "FP8(e4m3) x fp32 scale per 128x128 -> BF16 weights.");
    m.def("pack_weight_int8", &PackWeightInt8, "weight"_a, "gate_up"_a = false,
          "int8 [G,K,N] -> the tile-packed order grouped_gemm_packed reads.");
    m.def("grouped_gemm_packed", &GroupedGemmPacked, "x"_a, "weight"_a, "antiquantScaleOptional"_a,
          "antiquantOffsetOptional"_a, "groupListOptional"_a, "output"_a, "group_list_type"_a = 0, "gate_up_silu"_a = false,
          "GROUP GEMM on int8 weights repacked once.");
    m.def("fp4_scale_fold", &Fp4ScaleFold, "block_scale"_a, "global_scale"_a, "Two-level FP4 scale fold.");
    m.def("fp8_quantize_rows", &Fp8QuantizeRows, "x"_a, "index"_a = pybind11::none(), "codes"_a = pybind11::none(),
          "scale"_a = pybind11::none(), "bf16 rows -> (e4m3 codes, fp32 scale per 128), optionally gathered by an index.");
    m.def("grouped_gemm_fp8_block", &GroupedGemmFp8Block, "x"_a, "x_scale"_a, "weight"_a, "weight_scale"_a, "group_list"_a, "output"_a,
          "output_scale"_a = pybind11::none(), "group_list_type"_a = 0, "gate_up_silu"_a = false,
          "GROUP GEMM on e4m3 rows and e4m3 weights with scales per block of 128.");
    m.def("moe_balance_loss", &MoeBalanceLoss<kDropIn>, "logits"_a, "idx"_a, "seq_list"_a = pybind11::none(), "token_mask"_a = pybind11::none(),
          "(balance loss per sequence, pairs per sequence and expert), differentiable in the logits.");
    // the package's functions of the same names: their findings are read by its status calls, their launches counted there
    m.def("_mirror_fp8_quantize_rows", &QuantizeRows);
    m.def("_mirror_grouped_gemm_fp8_block", &ProductFp8Block<kMirror>);
    m.def("_mirror_moe_balance_loss", &MoeBalanceLoss<kMirror>);
    m.def("_mirror_findings", &MirrorFindings);
    m.def("_mirror_backward_launches", []() { return g_mirror_backward_launches.load(); });
    m.def("last_status", [](bool clear) { return LastStatus(clear); }, "clear"_a = false,
          "(code, detail) of the first device-side finding since the status was last cleared.");
    m.def("check_status", &CheckStatus, "Raises if an operator call left a device-side finding (and clears it).");
}
