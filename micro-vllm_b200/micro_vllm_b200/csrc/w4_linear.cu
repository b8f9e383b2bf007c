// Plans and launches of the mma.sync product kernel (w4_linear.cuh).
#include <algorithm>
#include <cstdlib>
#include <mutex>

#include "mvq_host.cuh"

namespace mvq {
namespace {

// How a call is cut up (see w4_linear_kernel).
struct LinearPlan {
    int nb;       // tokens / 8 per pass over the records
    int ksplit;
    int cluster;
    int stages;
    int64_t x_chunks;
    size_t ring_bytes;
    size_t smem;
};

LinearPlan linear_plan(int64_t m, int64_t chunks, int64_t tiles, int kind, int record, int sms) {
    LinearPlan plan;
    plan.nb = m <= 8 || kind == kF32 ? 1 : m <= 16 ? 2 : 4;
    const int64_t tokens = std::min<int64_t>(m, 8 * plan.nb);
    const int64_t blocks = (m + 8 * plan.nb - 1) / (8 * plan.nb);
    const int64_t x_chunk = tokens * (kind == kF32 ? 768 : kind == kI8 ? 128 : 256);
    plan.ksplit = kWarps;
    plan.cluster = 1;
    plan.stages = 3;
#ifdef MVQ_TUNE
    if (getenv("KS")) plan.ksplit = atoi(getenv("KS"));
    if (getenv("CL")) plan.cluster = atoi(getenv("CL"));
    if (getenv("ST")) plan.stages = atoi(getenv("ST"));
    if (!getenv("CL"))
#endif
    while (plan.cluster < 8 && tiles * blocks * plan.cluster < 3 * static_cast<int64_t>(sms) &&
           chunks > kWarps * plan.cluster)
        plan.cluster *= 2;
    const int64_t run = (chunks + plan.cluster - 1) / plan.cluster;
    int64_t most = 32 * 1024;
#ifdef MVQ_TUNE
    if (getenv("XB")) most = atoi(getenv("XB"));
#endif
    plan.x_chunks = std::max<int64_t>(1, most / x_chunk / plan.ksplit) * plan.ksplit;
    plan.x_chunks = std::min<int64_t>(plan.x_chunks, (run + plan.ksplit - 1) / plan.ksplit * plan.ksplit);
    plan.ring_bytes = std::max<size_t>(plan.stages * record, plan.nb * 8 * kPartStride * 4);
    plan.ring_bytes = (plan.ring_bytes + 127) / 128 * 128;
    plan.smem = kWarps * plan.ring_bytes + plan.x_chunks * x_chunk;
    return plan;
}

template <int KIND, int NB, int GROUP, bool ZEROS>
int launch_linear(LinearParams p, const LinearPlan& plan, int device, void* stream) {
    auto kernel = w4_linear_kernel<KIND, NB, GROUP, ZEROS>;
    static std::mutex mutex;
    static bool ready[kMaxDevices];
    {
        std::lock_guard<std::mutex> lock(mutex);
        if (!ready[device]) {
            cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(kSmemMost));
            if (err == cudaSuccess)
                err = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                           static_cast<int>(cudaSharedmemCarveoutMaxShared));
            if (err != cudaSuccess) return cuda_fail(err, "cudaFuncSetAttribute");
            ready[device] = true;
        }
    }
    const int64_t blocks = (static_cast<int64_t>(p.m) + 8 * NB - 1) / (8 * NB);
    if (blocks > 65535) return fail(MVQ_ERR_UNSUPPORTED, "too many rows of x for one call");
    const int per_cta = kWarps / plan.ksplit;
    const int64_t ctas = (static_cast<int64_t>(p.tiles) + per_cta - 1) / per_cta * plan.cluster;
    if (ctas >= (int64_t(1) << 31)) return fail(MVQ_ERR_UNSUPPORTED, "too many weight rows for one call");
    p.cluster = plan.cluster;
    p.ksplit = plan.ksplit;
    p.stages = plan.stages;
    p.x_chunks = static_cast<int>(plan.x_chunks);
    p.ring_bytes = static_cast<int>(plan.ring_bytes);
    const dim3 grid(static_cast<unsigned>(ctas), static_cast<unsigned>(blocks));
    const cudaError_t err = launch(kernel, grid, kThreads, plan.smem, plan.cluster, stream, p);
    return err == cudaSuccess ? MVQ_OK : cuda_fail(err, "4-bit linear kernel launch");
}

template <int KIND, int NB>
int launch_linear_group(const LinearParams& p, const LinearPlan& plan, int group, bool zeros, int device,
                        void* stream) {
    switch (group * 2 + zeros) {
        case 64: return launch_linear<KIND, NB, 32, false>(p, plan, device, stream);
        case 65: return launch_linear<KIND, NB, 32, true>(p, plan, device, stream);
        case 128: return launch_linear<KIND, NB, 64, false>(p, plan, device, stream);
        case 129: return launch_linear<KIND, NB, 64, true>(p, plan, device, stream);
        case 256: return launch_linear<KIND, NB, 128, false>(p, plan, device, stream);
        default: return launch_linear<KIND, NB, 128, true>(p, plan, device, stream);
    }
}

template <int KIND>
int launch_linear_kind(const LinearParams& p, int group, bool zeros, int device, int sms, void* stream) {
    const LinearPlan plan = linear_plan(p.m, p.chunks, p.tiles, KIND, record_size(group, zeros), sms);
    if constexpr (KIND != kF32) {
        if (plan.nb == 4) return launch_linear_group<KIND, 4>(p, plan, group, zeros, device, stream);
        if (plan.nb == 2) return launch_linear_group<KIND, 2>(p, plan, group, zeros, device, stream);
    }
    return launch_linear_group<KIND, 1>(p, plan, group, zeros, device, stream);
}

}  // namespace

int launch_narrow(const LinearParams& p, int kind, int group, bool zeros, int device, int sms, void* stream) {
    switch (kind) {
        case kF32: return launch_linear_kind<kF32>(p, group, zeros, device, sms, stream);
        case kBF16: return launch_linear_kind<kBF16>(p, group, zeros, device, sms, stream);
        case kI8: return launch_linear_kind<kI8>(p, group, zeros, device, sms, stream);
        default: return launch_linear_kind<kF16>(p, group, zeros, device, sms, stream);
    }
}

}  // namespace mvq
