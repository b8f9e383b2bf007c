// Plans and launches of the tcgen05 product kernel (w4_wide.cuh), and the device status that its waits set.
#include <algorithm>
#include <cudaTypedefs.h>

#include <mutex>

#include "mvq_host.cuh"
#include "w4_wide.cuh"

namespace mvq {
namespace {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult status;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &status) == cudaSuccess &&
            status == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

// X as [m, k] in boxes of `rows` rows of 128 bytes, swizzled (e4m3 rows as they lie); what lies beyond reads as zero.
int x_map(const LinearParams& p, int kind, int rows, CUtensorMap* map) {
    auto encode = encode_fn();
    if (!encode) return fail(MVQ_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
    const int size = kind == kI8 || kind == kE4M3 ? 1 : 2;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(p.k), static_cast<cuuint64_t>(p.m)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(p.x_stride * size)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / size), static_cast<cuuint32_t>(rows)};
    const cuuint32_t steps[2] = {1, 1};
    const CUresult r = encode(map, size == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : kind == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                              2, const_cast<void*>(p.x), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              kind == kE4M3 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(MVQ_ERR_CUDA, "cuTensorMapEncodeTiled failed (CUresult %d)", static_cast<int>(r));
    return MVQ_OK;
}

constexpr int kClusterSizes = 6;
constexpr int kClusters[kClusterSizes] = {1, 2, 3, 4, 6, 8};

// What a call costs (us), by the tokens of a pass: fitted to 90 calls of 16 to
// 57344 weight rows, 896 to 14336 columns and 9 to 256 tokens, 9% off on average.
struct WideCosts {
    double start, round;          // of the call, and of each round of CTAs that fill the device
    double chunk, group;          // of a round's chunk, and of each of its groups after the first
    double alone, alone_group;    // the same of a CTA that has no second one beside it (16 and 32 tokens)
};
constexpr WideCosts wide_costs(int nt) {
    return nt == 16   ? WideCosts{3.8, 4.2, 0.44, 0.19, 0.35, 0.16}
           : nt == 32 ? WideCosts{4.5, 6.0, 0.49, 0.23, 0.44, 0.18}
           : nt == 64 ? WideCosts{1.6, 5.4, 0.43, 0.15, 0.0, 0.0}
                      : WideCosts{0.1, 7.3, 0.61, 0.27, 0.0, 0.0};
}

// CTAs that share a block of rows' columns, for passes of nt tokens: the kClusters
// number with the least estimated time; slots[i]: how many clusters of kClusters[i]
// the device holds at once. Both sides measured: 3584 x 28672 at 16 rows 22.7 us
// alone, 27.7 in pairs; 14336 x 3584 at 64 rows 52.0 alone, 20.2 in fours, 30.7 in
// eights, of which not all fit at once.
struct WidePlan {
    int nt, cluster;
    double time;
};
WidePlan wide_plan(int64_t blocks, int chunks, int groups, int nt, const int* slots) {
    const WideCosts cost = wide_costs(nt);
    WidePlan best = {nt, 1, 0.0};
    for (int i = 0; i < kClusterSizes; ++i) {
        const int c = kClusters[i];
        if (c > chunks || slots[i] <= 0) break;
        const double rounds = static_cast<double>((blocks + slots[i] - 1) / slots[i]);
        const int run = (chunks + c - 1) / c;
        double time = cost.start + 0.25 * (c - 1);
        if (nt <= 32 && 2 * blocks <= slots[i])
            time += run * (cost.alone + (groups - 1) * cost.alone_group);
        else
            time += rounds * (cost.round + run * (cost.chunk + (groups - 1) * cost.group));
        if (c == 1 || time < best.time) best.time = time, best.cluster = c;
    }
    return best;
}

template <int KIND, int NT, int GROUP, bool ZEROS>
struct Wide {
    using Shape = WideShape<KIND, NT, GROUP, ZEROS>;
    static_assert(Shape::kSmem <= kSmemMost, "shared memory");

    // `slots`: how many clusters of each kClusters size the device holds at once.
    static int prepare(int device, int sms, const int** slots) {
        static std::mutex mutex;
        static bool ready[kMaxDevices];
        static int held[kMaxDevices][kClusterSizes];
        std::lock_guard<std::mutex> lock(mutex);
        *slots = held[device];
        if (ready[device]) return MVQ_OK;
        auto kernel = w4_wide_kernel<KIND, NT, GROUP, ZEROS>;
        cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::kSmem);
        if (err == cudaSuccess)
            err = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                       static_cast<int>(cudaSharedmemCarveoutMaxShared));
        if (err != cudaSuccess) return cuda_fail(err, "cudaFuncSetAttribute");
        for (int i = 0; i < kClusterSizes; ++i) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(kClusters[i] * sms);
            cfg.blockDim = dim3(Shape::kThreads);
            cfg.dynamicSmemBytes = Shape::kSmem;
            cudaLaunchAttribute attr;
            attr.id = cudaLaunchAttributeClusterDimension;
            attr.val.clusterDim.x = kClusters[i];
            attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
            cfg.attrs = &attr;
            cfg.numAttrs = 1;
            err = cudaOccupancyMaxActiveClusters(&held[device][i], kernel, &cfg);
            if (err != cudaSuccess) return cuda_fail(err, "cudaOccupancyMaxActiveClusters");
            // It counts one CTA per SM for every kernel that allocates tensor memory, but two of 256
            // columns do run together (224 CTAs of 16 rows in 21.5 us; made for one per SM, 27.6).
            held[device][i] *= Shape::kCtas;
        }
        ready[device] = true;
        return MVQ_OK;
    }

    // Puts the plan for NT tokens per pass into `best` where its estimate is lower, or is the first (time 0).
    static int consider(const LinearParams& p, int device, int sms, WidePlan* best) {
        const int* slots;
        const int rc = prepare(device, sms, &slots);
        if (rc != MVQ_OK) return rc;
        const int64_t blocks = (static_cast<int64_t>(p.n) + kWideRows - 1) / kWideRows;
        const int64_t passes = (static_cast<int64_t>(p.m) + NT - 1) / NT;
        const WidePlan plan = wide_plan(blocks * passes, p.chunks, Shape::kGroups, NT, slots);
        if (best->time == 0.0 || plan.time < best->time) *best = plan;
        return MVQ_OK;
    }

    static int launch_plan(LinearParams p, int cluster, void* stream) {
        p.cluster = cluster;
        CUtensorMap map = {};
        if (p.x_units) {
            const int rc = x_map(p, KIND, NT, &map);
            if (rc != MVQ_OK) return rc;
        }
        const int64_t blocks = (static_cast<int64_t>(p.n) + kWideRows - 1) / kWideRows;
        const dim3 grid(static_cast<unsigned>(blocks * cluster), static_cast<unsigned>((p.m + NT - 1) / NT));
        const cudaError_t err = launch(w4_wide_kernel<KIND, NT, GROUP, ZEROS>, grid, Shape::kThreads, Shape::kSmem,
                                       cluster, stream, p, map);
        return err == cudaSuccess ? MVQ_OK : cuda_fail(err, "wide 4-bit linear kernel launch");
    }
};

// The tokens of a pass: as many as there are (16, 32, 64 or 128), or fewer where
// several passes over few weight rows fill the device better, by the estimates above.
// Both sides measured: 896 x 1152 at 128 rows 5.8 us in passes of 16, 8.6 in one;
// 12928 x 16 in fp16 with groups of 32 at 230 rows 16 in passes of 32, 23 in two;
// 3584 x 28672 at 128 rows 50.2 in one, 80.5 in passes of 32.
template <int KIND, int GROUP, bool ZEROS>
int launch_group(const LinearParams& p, int device, int sms, void* stream) {
    WidePlan plan = {};
    int rc = MVQ_OK;
    if (p.m > 64) rc = Wide<KIND, 128, GROUP, ZEROS>::consider(p, device, sms, &plan);
    if (rc == MVQ_OK && p.m > 32) rc = Wide<KIND, 64, GROUP, ZEROS>::consider(p, device, sms, &plan);
    if (rc == MVQ_OK && p.m > 16) rc = Wide<KIND, 32, GROUP, ZEROS>::consider(p, device, sms, &plan);
    if (rc == MVQ_OK) rc = Wide<KIND, 16, GROUP, ZEROS>::consider(p, device, sms, &plan);
    if (rc != MVQ_OK) return rc;
    switch (plan.nt) {
        case 16: return Wide<KIND, 16, GROUP, ZEROS>::launch_plan(p, plan.cluster, stream);
        case 32: return Wide<KIND, 32, GROUP, ZEROS>::launch_plan(p, plan.cluster, stream);
        case 64: return Wide<KIND, 64, GROUP, ZEROS>::launch_plan(p, plan.cluster, stream);
        default: return Wide<KIND, 128, GROUP, ZEROS>::launch_plan(p, plan.cluster, stream);
    }
}

template <int KIND>
int launch_kind(const LinearParams& p, int group, bool zeros, int device, int sms, void* stream) {
    switch (group * 2 + zeros) {
        case 64: return launch_group<KIND, 32, false>(p, device, sms, stream);
        case 65: return launch_group<KIND, 32, true>(p, device, sms, stream);
        case 128: return launch_group<KIND, 64, false>(p, device, sms, stream);
        case 129: return launch_group<KIND, 64, true>(p, device, sms, stream);
        case 256: return launch_group<KIND, 128, false>(p, device, sms, stream);
        default: return launch_group<KIND, 128, true>(p, device, sms, stream);
    }
}

}  // namespace

int launch_wide(const LinearParams& p, int kind, int group, bool zeros, int device, int sms, void* stream) {
    switch (kind) {
        case kBF16: return launch_kind<kBF16>(p, group, zeros, device, sms, stream);
        case kI8: return launch_kind<kI8>(p, group, zeros, device, sms, stream);
        case kE4M3: return launch_kind<kE4M3>(p, group, zeros, device, sms, stream);
        default: return launch_kind<kF16>(p, group, zeros, device, sms, stream);
    }
}

}  // namespace mvq

extern "C" {

int mvq_device_status(int32_t device, uint32_t* status) try {
    if (!status) return mvq::fail(MVQ_ERR_INVALID_ARGUMENT, "status must not be NULL");
    int current = 0;
    cudaError_t err = cudaGetDevice(&current);
    if (err == cudaSuccess) err = cudaSetDevice(device);
    if (err != cudaSuccess) return mvq::cuda_fail(err, "cudaSetDevice");
    unsigned value = 0;
    err = cudaMemcpyFromSymbol(&value, mv::g_device_status, sizeof(value));
    cudaSetDevice(current);
    if (err != cudaSuccess) return mvq::cuda_fail(err, "reading the device status");
    *status = value;
    return MVQ_OK;
} catch (...) {
    return mvq::fail(MVQ_ERR_CUDA, "unexpected C++ exception");
}

int mvq_clear_device_status(int32_t device) try {
    int current = 0;
    cudaError_t err = cudaGetDevice(&current);
    if (err == cudaSuccess) err = cudaSetDevice(device);
    if (err != cudaSuccess) return mvq::cuda_fail(err, "cudaSetDevice");
    const unsigned zero = 0;
    err = cudaMemcpyToSymbol(mv::g_device_status, &zero, sizeof(zero));
    cudaSetDevice(current);
    return err == cudaSuccess ? MVQ_OK : mvq::cuda_fail(err, "clearing the device status");
} catch (...) {
    return mvq::fail(MVQ_ERR_CUDA, "unexpected C++ exception");
}

int mvq_selftest_wait_timeout(uint64_t limit_ns, void* stream) try {
    if (limit_ns == 0 || limit_ns > 100000000ull)
        return mvq::fail(MVQ_ERR_INVALID_ARGUMENT, "limit_ns must be in (0, 100 ms]");
    mvq::wait_timeout_selftest_kernel<<<1, 32, 0, static_cast<cudaStream_t>(stream)>>>(limit_ns);
    const cudaError_t err = cudaGetLastError();
    return err == cudaSuccess ? MVQ_OK : mvq::cuda_fail(err, "self-test kernel launch");
} catch (...) {
    return mvq::fail(MVQ_ERR_CUDA, "unexpected C++ exception");
}

}  // extern "C"
