// Plans and launches of the tcgen05 product kernel (w4_wide.cuh), and the device status that its waits set.
#include <algorithm>
#include <cstdlib>
#include <mutex>

#include "mvq_host.cuh"
#include "w4_wide.cuh"

namespace mvq {
namespace {

// CTAs that share a block of rows' columns: the number in 1..8 that fills whole
// rounds of the SMs best.
int wide_cluster(int64_t blocks, int chunks, int sms) {
#ifdef MVQ_TUNE
    if (getenv("CL")) return atoi(getenv("CL"));
#endif
    int best = 1;
    double most = 0.0;
    for (int c = 1; c <= 8 && c <= chunks; ++c) {
        const int64_t ctas = blocks * c;
        const int64_t rounds = (ctas + sms - 1) / sms;
        // The longest run of chunks, in each of the rounds.
        const double used = static_cast<double>(blocks) * chunks /
                            (static_cast<double>(rounds) * sms * ((chunks + c - 1) / c));
        if (used > most * 1.02) most = used, best = c;
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
    {
        std::lock_guard<std::mutex> lock(mutex);
        if (!ready[device]) {
            cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
            if (err == cudaSuccess)
                err = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                           static_cast<int>(cudaSharedmemCarveoutMaxShared));
            if (err != cudaSuccess) return cuda_fail(err, "cudaFuncSetAttribute");
            ready[device] = true;
        }
    }
    const int64_t blocks = (static_cast<int64_t>(p.n) + kWideRows - 1) / kWideRows;
    const int64_t passes = (static_cast<int64_t>(p.m) + NT - 1) / NT;
    if (passes > 65535) return fail(MVQ_ERR_UNSUPPORTED, "too many rows of x for one call");
    p.cluster = wide_cluster(blocks * passes, p.chunks, sms);
    const dim3 grid(static_cast<unsigned>(blocks * p.cluster), static_cast<unsigned>(passes));
    const cudaError_t err = launch(kernel, grid, Shape::kThreads, kSmem, p.cluster, stream, p);
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
