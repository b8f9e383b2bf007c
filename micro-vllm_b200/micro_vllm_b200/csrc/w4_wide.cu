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

// X as [m, k] in boxes of `rows` rows of 128 bytes, swizzled; what lies beyond reads as zero.
int x_map(const LinearParams& p, int kind, int rows, CUtensorMap* map) {
    auto encode = encode_fn();
    if (!encode) return fail(MVQ_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable from the driver");
    const int size = kind == kI8 ? 1 : 2;
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(p.k), static_cast<cuuint64_t>(p.m)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(p.x_stride * size)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / size), static_cast<cuuint32_t>(rows)};
    const cuuint32_t steps[2] = {1, 1};
    const CUresult r = encode(map, kind == kI8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : kind == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                              2, const_cast<void*>(p.x), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(MVQ_ERR_CUDA, "cuTensorMapEncodeTiled failed (CUresult %d)", static_cast<int>(r));
    return MVQ_OK;
}

constexpr int kClusters[] = {1, 2, 3, 4, 6, 8};

// CTAs that share a block of rows' columns: the kClusters number with the least
// estimated time (us); slots[i]: how many clusters of kClusters[i] the device holds
// at once. Fitted to calls of 896 x 1152 to 8192 x 57344: a call starts and ends in
// about five (with 64 tokens and one CTA per SM, ten); a chunk takes 0.33 us of a
// CTA alone on its SM, 0.22 of an SM with two, and up to 0.53 with 128 tokens; a
// cluster costs its barriers. Both sides measured: 3584 x 28672 at 16 rows 22.7 us
// alone, 27.7 in pairs; 14336 x 3584 at 64 rows 52.0 alone, 20.2 in fours, 30.7 in
// eights, of which not all fit at once.
int wide_cluster(int64_t blocks, int chunks, int nt, const int* slots) {
    int best = 1;
    double least = 0.0;
    for (int i = 0; i < 6; ++i) {
        const int c = kClusters[i];
        if (c > chunks || slots[i] <= 0) break;
        const double rounds = static_cast<double>((blocks + slots[i] - 1) / slots[i]);
        const int run = (chunks + c - 1) / c;
        double time = c > 1 ? 0.3 * c : 0.0;
        if (nt >= 64) time += rounds * (9.7 + run * (nt == 64 ? 0.38 : 0.53));
        else time += 5.2 + (2 * blocks <= slots[i] ? run * 0.33 : 2 * rounds * (3.0 + run * 0.22));
        if (c == 1 || time < least) least = time, best = c;
    }
    return best;
}

template <int KIND, int NT, int GROUP, bool ZEROS>
int launch_one(LinearParams p, int device, int sms, void* stream) {
    auto kernel = w4_wide_kernel<KIND, NT, GROUP, ZEROS>;
    using Shape = WideShape<KIND, NT, GROUP, ZEROS>;
    constexpr int kSmem = Shape::kSmem;
    static_assert(kSmem <= kSmemMost, "shared memory");
    static std::mutex mutex;
    static bool ready[kMaxDevices];
    static int slots[kMaxDevices][6];  // clusters of each kClusters size that the device holds at once
    {
        std::lock_guard<std::mutex> lock(mutex);
        if (!ready[device]) {
            cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
            if (err == cudaSuccess)
                err = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                           static_cast<int>(cudaSharedmemCarveoutMaxShared));
            if (err != cudaSuccess) return cuda_fail(err, "cudaFuncSetAttribute");
            for (int i = 0; i < 6; ++i) {
                cudaLaunchConfig_t cfg = {};
                cfg.gridDim = dim3(kClusters[i] * sms);
                cfg.blockDim = dim3(Shape::kThreads);
                cfg.dynamicSmemBytes = kSmem;
                cudaLaunchAttribute attr;
                attr.id = cudaLaunchAttributeClusterDimension;
                attr.val.clusterDim.x = kClusters[i];
                attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
                cfg.attrs = &attr;
                cfg.numAttrs = 1;
                err = cudaOccupancyMaxActiveClusters(&slots[device][i], kernel, &cfg);
                if (err != cudaSuccess) return cuda_fail(err, "cudaOccupancyMaxActiveClusters");
                // It counts one CTA per SM for every kernel that allocates tensor memory, but two of 256
                // columns do run together (224 CTAs of 16 rows in 21.5 us; made for one per SM, 27.6).
                slots[device][i] *= Shape::kCtas;
            }
            ready[device] = true;
        }
    }
    const int64_t blocks = (static_cast<int64_t>(p.n) + kWideRows - 1) / kWideRows;
    const int64_t passes = (static_cast<int64_t>(p.m) + NT - 1) / NT;
    p.cluster = wide_cluster(blocks * passes, p.chunks, NT, slots[device]);
    CUtensorMap map = {};
    if (p.x_units) {
        const int rc = x_map(p, KIND, NT, &map);
        if (rc != MVQ_OK) return rc;
    }
    const dim3 grid(static_cast<unsigned>(blocks * p.cluster), static_cast<unsigned>(passes));
    const cudaError_t err = launch(kernel, grid, Shape::kThreads, kSmem, p.cluster, stream, p, map);
    return err == cudaSuccess ? MVQ_OK : cuda_fail(err, "wide 4-bit linear kernel launch");
}

template <int KIND, int NT>
int launch_group(const LinearParams& p, int group, bool zeros, int device, int sms, void* stream) {
    switch (group * 2 + zeros) {
        case 64: return launch_one<KIND, NT, 32, false>(p, device, sms, stream);
        case 65: return launch_one<KIND, NT, 32, true>(p, device, sms, stream);
        case 128: return launch_one<KIND, NT, 64, false>(p, device, sms, stream);
        case 129: return launch_one<KIND, NT, 64, true>(p, device, sms, stream);
        case 256: return launch_one<KIND, NT, 128, false>(p, device, sms, stream);
        default: return launch_one<KIND, NT, 128, true>(p, device, sms, stream);
    }
}

template <int KIND>
int launch_tokens(const LinearParams& p, int group, bool zeros, int device, int sms, void* stream) {
    if (p.m <= 16) return launch_group<KIND, 16>(p, group, zeros, device, sms, stream);
    if (p.m <= 32) return launch_group<KIND, 32>(p, group, zeros, device, sms, stream);
    if (p.m <= 64) return launch_group<KIND, 64>(p, group, zeros, device, sms, stream);
    return launch_group<KIND, 128>(p, group, zeros, device, sms, stream);
}

}  // namespace

int launch_wide(const LinearParams& p, int kind, int group, bool zeros, int device, int sms, void* stream) {
    switch (kind) {
        case kBF16: return launch_tokens<kBF16>(p, group, zeros, device, sms, stream);
        case kI8: return launch_tokens<kI8>(p, group, zeros, device, sms, stream);
        default: return launch_tokens<kF16>(p, group, zeros, device, sms, stream);
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

}  // extern "C"
