// Plans and launches of the mma.sync product kernel (w4_linear.cuh).
#include <algorithm>
#include <mutex>

#include "mvq_host.cuh"

namespace mvq {
namespace {

// How a call is cut up (see w4_linear_kernel).
struct LinearPlan {
    int ksplit, cluster, stages;
    int64_t x_bytes, x_chunks;
    size_t ring_bytes, smem;
};

// The cut with the least estimated time. A CTA costs `start` (its launch, x's
// part of its run, the joining of its sums) and its warps' chunks; an SM takes
// its share of the CTAs, and fewer than twelve warps on it do not hide a
// warp's own latency. The constants (us) are fitted to measured calls of 896 x
// 1152 to 8192 x 57344 at 1 to 8 tokens: at one token four warps per tile are
// best (3584 x 28672: 16.2 us, one warp per tile 17.7), at eight one warp per
// tile and clusters, which share the staged x (21.7 and 28 us). fp32 rows cost
// mostly their staging as three planes (3584 x 4608 at five tokens: one warp per
// tile in eights 11.3 us, four warps per tile in eights 14.3). Where few CTAs
// share an SM, x is staged in one turn or few: 14336 x 3584 in fp32 at eight
// tokens 25.4 us, 16 KB at a time 40.6.
LinearPlan linear_plan(int64_t m, int64_t chunks, int64_t tiles, int kind, int record, int sms) {
    const int64_t tokens = std::min<int64_t>(m, kTokens);
    const int64_t blocks = (m + kTokens - 1) / kTokens;
    const int64_t x_chunk = tokens * (kind == kF32 ? 768 : kind == kI8 ? 128 : 256);
    const double chunk = kind == kI8 ? 0.06 + 0.004 * tokens : kind == kF32 ? 0.09 : 0.11 + 0.007 * tokens;
    LinearPlan best = {};
    double least = 0.0;
    for (int ksplit = 1; ksplit <= kWarps; ksplit *= 2) {
        const int64_t groups = (tiles + kWarps / ksplit - 1) / (kWarps / ksplit);
        for (int cluster = 1; cluster <= 8 && cluster <= chunks; cluster *= 2) {
            const int64_t run = (chunks + cluster - 1) / cluster;
            const int64_t per_warp = (run + ksplit - 1) / ksplit;
            const double per_sm = static_cast<double>((groups * cluster * blocks + sms - 1) / sms);
            const double start = kind == kF32 ? 0.4 + 0.074 * tokens * run : 0.7 + 0.006 * tokens * run + 0.02 * tokens;
            const double busy = kWarps * std::min(per_sm, 4.0);
            const double time = per_sm * (start + kWarps * per_warp * chunk * std::max(1.0, 12.0 / busy)) +
                                (cluster > 1 ? kind == kF32 ? 0.15 * cluster : 0.6 : 0.0);
            if (best.cluster == 0 || time < least) {
                least = time;
                best.ksplit = ksplit;
                best.cluster = cluster;
                best.stages = per_sm >= 4.0 ? 2 : 3;  // four CTAs per SM, or deeper rings
                best.x_bytes = (per_sm >= 3.0 ? 16 : per_sm >= 2.0 ? 48 : 96) * 1024;
            }
        }
    }
    const int64_t run = (chunks + best.cluster - 1) / best.cluster;
    best.x_chunks = std::max<int64_t>(1, best.x_bytes / x_chunk / best.ksplit) * best.ksplit;
    best.x_chunks = std::min<int64_t>(best.x_chunks, (run + best.ksplit - 1) / best.ksplit * best.ksplit);
    best.ring_bytes = std::max<size_t>(best.stages * record, kTokens * kPartStride * 4);
    best.ring_bytes = (best.ring_bytes + 127) / 128 * 128;
    best.smem = kWarps * best.ring_bytes + best.x_chunks * x_chunk;
    return best;
}

template <int KIND, int GROUP, bool ZEROS>
int launch_linear(LinearParams p, const LinearPlan& plan, int device, void* stream) {
    auto kernel = w4_linear_kernel<KIND, GROUP, ZEROS>;
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
    const int64_t blocks = (static_cast<int64_t>(p.m) + kTokens - 1) / kTokens;
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

template <int KIND>
int launch_linear_group(const LinearParams& p, const LinearPlan& plan, int group, bool zeros, int device,
                        void* stream) {
    switch (group * 2 + zeros) {
        case 64: return launch_linear<KIND, 32, false>(p, plan, device, stream);
        case 65: return launch_linear<KIND, 32, true>(p, plan, device, stream);
        case 128: return launch_linear<KIND, 64, false>(p, plan, device, stream);
        case 129: return launch_linear<KIND, 64, true>(p, plan, device, stream);
        case 256: return launch_linear<KIND, 128, false>(p, plan, device, stream);
        default: return launch_linear<KIND, 128, true>(p, plan, device, stream);
    }
}

template <int KIND>
int launch_linear_kind(const LinearParams& p, int group, bool zeros, int device, int sms, void* stream) {
    const LinearPlan plan = linear_plan(p.m, p.chunks, p.tiles, KIND, record_size(group, zeros), sms);
    return launch_linear_group<KIND>(p, plan, group, zeros, device, stream);
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
