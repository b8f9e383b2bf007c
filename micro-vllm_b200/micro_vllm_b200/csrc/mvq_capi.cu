// C ABI of libmvquant.so (include/mvquant.h): argument checks, kernel choice, launches.
#include "mvquant.h"

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>

#include "mvq_host.cuh"
#include "quant_rows.cuh"

namespace mvq {

static thread_local char g_error[512];

int fail(int code, const char* fmt, ...) {
    va_list args;
    va_start(args, fmt);
    vsnprintf(g_error, sizeof(g_error), fmt, args);
    va_end(args);
    return code;
}

int cuda_fail(cudaError_t err, const char* what) {
    cudaGetLastError();  // reported here: not once more by whoever asks the runtime next
    return fail(MVQ_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
}

}  // namespace mvq

namespace {

using mvq::cuda_fail;
using mvq::fail;
using mvq::launch;
using mvq::kMaxDevices;

// Streaming multiprocessors of the current device (asked once per device).
int device_sms(int* device, int* sms) {
    static std::mutex mutex;
    static int known[kMaxDevices];
    cudaError_t err = cudaGetDevice(device);
    if (err != cudaSuccess) return cuda_fail(err, "cudaGetDevice");
    if (*device < 0 || *device >= kMaxDevices) return fail(MVQ_ERR_UNSUPPORTED, "device index %d out of range", *device);
    std::lock_guard<std::mutex> lock(mutex);
    if (known[*device] == 0) {
        int n = 0;
        err = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, *device);
        if (err != cudaSuccess) return cuda_fail(err, "cudaDeviceGetAttribute");
        known[*device] = n;
    }
    *sms = known[*device];
    return MVQ_OK;
}

bool float_dtype(int64_t d) { return d == MVQ_DTYPE_F32 || d == MVQ_DTYPE_F16 || d == MVQ_DTYPE_BF16; }
int64_t dtype_size(int64_t d) { return d == MVQ_DTYPE_F32 ? 4 : d == MVQ_DTYPE_F16 || d == MVQ_DTYPE_BF16 ? 2 : 1; }
uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }
bool off_element(const void* p, int64_t dtype) { return address(p) % dtype_size(dtype) != 0; }

// ------------------------------------------------------------------- weights

constexpr int64_t kMaxSize = int64_t(1) << 30;
// Rows of x per launch: a grid's 65535 blocks of the narrow kernel's eight.
constexpr int64_t kLaunchRows = int64_t(65535) * mvq::kTokens;

int check_weight(const void* records, int64_t n, int64_t k, int64_t group, int64_t scale_dtype) {
    if (!records) return fail(MVQ_ERR_INVALID_ARGUMENT, "records must not be NULL");
    if (address(records) % 16) return fail(MVQ_ERR_INVALID_ARGUMENT, "records must be 16-byte aligned");
    if (n <= 0 || k <= 0) return fail(MVQ_ERR_INVALID_ARGUMENT, "sizes must be positive");
    if (n > kMaxSize || k > kMaxSize) return fail(MVQ_ERR_UNSUPPORTED, "sizes must be at most 2^30");
    if (group != 32 && group != 64 && group != 128)
        return fail(MVQ_ERR_UNSUPPORTED, "group must be 32, 64 or 128");
    if (scale_dtype != MVQ_DTYPE_F16 && scale_dtype != MVQ_DTYPE_BF16)
        return fail(MVQ_ERR_INVALID_ARGUMENT, "scale_dtype must be MVQ_DTYPE_F16 or MVQ_DTYPE_BF16");
    return MVQ_OK;
}

// ---------------------------------------------------------------------- rows

// Threads and runs of eight per thread for rows of `width` elements.
struct RowShape {
    int threads;
    int held;      // runs of eight elements a thread holds: 1, 2, 4 or 8; 0: none, the row is read twice
    int per_cta;   // rows
};

// `vector`: rows that are read a run at a time; `most`: the most runs that a thread may hold; `norm`: the norm, not
// the gate.
RowShape row_shape(int64_t width, int64_t rows, int sms, bool vector, int most, bool norm) {
    const int64_t runs = (width + 7) / 8;
    // Few rows: a thread per run, which spreads the row's latency over the CTA.
    // Many rows: two runs a thread and CTAs of at most 512 threads (2048 rows of
    // 14336: 33.6 us, with at most 256 threads 37.9, with up to 1024 62), or eight
    // rows a CTA where a warp holds a row (8192 rows of 128: 3.4 us, a CTA each 8.9;
    // of 896: 9.9 and 10.6).
    int held = 1;
    if (rows > 2 * static_cast<int64_t>(sms)) {
        if (runs <= 32 * (most < 4 ? most : 4)) {
            while (runs > 32 * held) held *= 2;
            return {32, held, 8};
        }
        if (vector || !norm) {
            for (held = 2; held < most && runs > static_cast<int64_t>(held) * 512;) held *= 2;
        } else {
            // The norm by elements has registers for one run a thread: two spill (2000
            // rows of 4001 in bf16: 33.0 us, two runs 36.4; of 8191, where one run would
            // take 1024 threads: 74.7 and 70.6), and in 1024 threads are behind a row
            // that is read twice (1000 rows of 12001: 66.8 and 40.8). A warp that reads
            // a row twice is ahead of a CTA where there are enough of them (8000 rows
            // of 1001: 25.6 and 29.5; 1000 rows: 7.7 and 6.2).
            if (runs <= 128 && rows > 8 * static_cast<int64_t>(sms)) return {32, 0, 8};
            held = runs <= 512 ? 1 : 2;
        }
    }
    const auto threads = [&](int held) {
        return !vector && norm && held == 2 ? 512 : mvq::max_row_threads(held, norm);
    };
    while (held <= most && runs > static_cast<int64_t>(held) * threads(held)) held *= 2;
    if (held > most) return {threads(0), 0, 1};
    return {static_cast<int>(((runs + held - 1) / held + 31) / 32 * 32), held, 1};
}

template <typename T, int OUT, bool RUNS, template <typename, int, bool, int> class Kernel, typename P>
cudaError_t launch_row_held(const P& p, RowShape shape, int64_t rows, void* stream) {
    const dim3 grid(static_cast<unsigned>((rows + shape.per_cta - 1) / shape.per_cta));
    const dim3 block(shape.threads, shape.per_cta);
    switch (shape.held) {
        case 0: return launch(Kernel<T, OUT, RUNS, 0>::get(), grid, block, 0, 1, stream, p);
        case 1: return launch(Kernel<T, OUT, RUNS, 1>::get(), grid, block, 0, 1, stream, p);
        case 2: return launch(Kernel<T, OUT, RUNS, 2>::get(), grid, block, 0, 1, stream, p);
        default: break;
    }
    if constexpr (Kernel<T, OUT, RUNS, 1>::most() >= 4)
        if (shape.held == 4) return launch(Kernel<T, OUT, RUNS, 4>::get(), grid, block, 0, 1, stream, p);
    if constexpr (Kernel<T, OUT, RUNS, 1>::most() >= 8)
        if (shape.held == 8) return launch(Kernel<T, OUT, RUNS, 8>::get(), grid, block, 0, 1, stream, p);
    return cudaErrorInvalidConfiguration;  // a shape that no kernel was made for
}

template <typename T, int OUT, template <typename, int, bool, int> class Kernel, typename P>
cudaError_t launch_row_access(const P& p, bool runs, int64_t width, int64_t rows, int sms, void* stream) {
    using Runs = Kernel<T, OUT, true, 1>;
    using Elements = Kernel<T, OUT, false, 1>;
    const RowShape shape =
        row_shape(width, rows, sms, runs, runs ? Runs::most() : Elements::most(), Runs::norm());
    return runs ? launch_row_held<T, OUT, true, Kernel>(p, shape, rows, stream)
                : launch_row_held<T, OUT, false, Kernel>(p, shape, rows, stream);
}

template <int OUT, template <typename, int, bool, int> class Kernel, typename P>
cudaError_t launch_row_type(const P& p, int64_t dtype, bool runs, int64_t width, int64_t rows, int sms, void* stream) {
    if (dtype == MVQ_DTYPE_F32) return launch_row_access<float, OUT, Kernel>(p, runs, width, rows, sms, stream);
    if (dtype == MVQ_DTYPE_F16) return launch_row_access<__half, OUT, Kernel>(p, runs, width, rows, sms, stream);
    return launch_row_access<__nv_bfloat16, OUT, Kernel>(p, runs, width, rows, sms, stream);
}

template <typename T, int OUT, bool RUNS, int C>
struct NormKernel {
    static constexpr bool norm() { return true; }
    // Eight runs of fp32 spill: a row that is read twice is ahead of them (1024 rows of 14344 to e4m3 43.4 us, held
    // 57.9; in bf16 31.9 and 23.6).
    static constexpr int most() { return !RUNS ? 2 : sizeof(T) == 4 ? 4 : 8; }
    static auto get() { return mvq::add_rms_norm_kernel<T, OUT, RUNS, C>; }
};
template <typename T, int OUT, bool RUNS, int C>
struct SiluKernel {
    static constexpr bool norm() { return false; }
    static constexpr int most() { return RUNS ? 8 : 2; }
    static auto get() { return mvq::silu_mul_quant_kernel<T, OUT, RUNS, C>; }
};

int check_rows(int64_t rows, int64_t width, int64_t dtype) {
    if (rows <= 0 || width <= 0) return fail(MVQ_ERR_INVALID_ARGUMENT, "sizes must be positive");
    if (rows >= (int64_t(1) << 31) || width > kMaxSize)
        return fail(MVQ_ERR_UNSUPPORTED, "rows must be below 2^31 and at most 2^30 elements wide");
    if (!float_dtype(dtype))
        return fail(MVQ_ERR_INVALID_ARGUMENT, "dtype must be MVQ_DTYPE_F32, MVQ_DTYPE_F16 or MVQ_DTYPE_BF16");
    return MVQ_OK;
}

}  // namespace

extern "C" {

int mvq_abi_version(void) { return MVQ_ABI_VERSION; }

const char* mvq_last_error(void) { return mvq::g_error; }

int mvq_w4_linear(const MvqLinearArgs* a, void* stream) try {
    if (!a) return fail(MVQ_ERR_INVALID_ARGUMENT, "args must not be NULL");
    int rc = check_weight(a->records, a->n, a->k, a->group, a->scale_dtype);
    if (rc != MVQ_OK) return rc;
    if (!a->x || !a->out) return fail(MVQ_ERR_INVALID_ARGUMENT, "x and out must not be NULL");
    if (a->m <= 0) return fail(MVQ_ERR_INVALID_ARGUMENT, "sizes must be positive");
    if (a->m > kMaxSize) return fail(MVQ_ERR_UNSUPPORTED, "sizes must be at most 2^30");
    if (a->x_dtype < 0 || a->x_dtype > MVQ_DTYPE_E4M3)
        return fail(MVQ_ERR_INVALID_ARGUMENT, "x_dtype must be an MVQ_DTYPE_* value");
    if (!float_dtype(a->out_dtype))
        return fail(MVQ_ERR_INVALID_ARGUMENT, "out_dtype must be MVQ_DTYPE_F32, MVQ_DTYPE_F16 or MVQ_DTYPE_BF16");
    if (a->m > 1 && (a->x_stride_row < 0 || a->out_stride_row < a->n || (a->residual && a->residual_stride_row < 0)))
        return fail(MVQ_ERR_INVALID_ARGUMENT, "row strides must be nonnegative and out's rows must not overlap");
    if (off_element(a->x, a->x_dtype) || off_element(a->x_scale, MVQ_DTYPE_F32) || off_element(a->bias, a->out_dtype) ||
        off_element(a->residual, a->out_dtype) || off_element(a->out, a->out_dtype))
        return fail(MVQ_ERR_INVALID_ARGUMENT, "pointers must be aligned to their elements");
    int device, sms;
    rc = device_sms(&device, &sms);
    if (rc != MVQ_OK) return rc;
    const int64_t size = dtype_size(a->x_dtype);
    const int64_t run = size == 1 ? 8 : 16;  // bytes of a vector load of x
    mvq::LinearParams p = {};
    p.x_stride = a->x_stride_row;
    p.records = static_cast<const uint8_t*>(a->records);
    p.n = static_cast<int>(a->n);
    p.k = static_cast<int>(a->k);
    p.chunks = static_cast<int>((a->k + mvq::kChunk - 1) / mvq::kChunk);
    p.tiles = static_cast<int>((a->n + mvq::kTileRows - 1) / mvq::kTileRows);
    p.x_dtype = static_cast<int>(a->x_dtype);
    p.scale_bf16 = a->scale_dtype == MVQ_DTYPE_BF16;
    p.x_runs = a->k % 8 == 0 && address(a->x) % run == 0 && (a->m == 1 || a->x_stride_row * size % run == 0);
    p.bias = a->bias;
    p.residual_stride = a->residual_stride_row;
    p.out_stride = a->out_stride_row;
    p.out_dtype = static_cast<int>(a->out_dtype);
    // TMA wants 16-byte rows that do not overlap.
    p.x_units = size < 4 && address(a->x) % 16 == 0 && a->x_stride_row * size % 16 == 0 && a->x_stride_row >= a->k &&
                a->x_stride_row < (int64_t(1) << 38);
    const int kind = a->x_dtype == MVQ_DTYPE_E4M3 ? mvq::kF16 : static_cast<int>(a->x_dtype);
    const int group = static_cast<int>(a->group);
    // The mma.sync kernel for few rows: how many depends on the stream of the weights
    // beside what each row costs it, on the tcgen05 kernel's fixed part, which is
    // larger for e4m3 rows, and on the commit and the wait that each group costs that
    // kernel. Measured (us, tcgen05 and mma.sync):
    //   groups of 128, 16 bits  896 x 1152    three rows 4.4, 4.5   four 4.2, 4.8
    //                           3584 x 4608   three 7.5, 7.4        four 7.5, 8.0
    //                           14336 x 3584  four 15.0, 14.3       five 15.0, 15.3
    //                           3584 x 28672  seven 20.5, 20.3      eight 20.5, 21.8
    //                           8192 x 57344  eight 79, 68
    //                   int8    2048 x 2048   four 4.8, 4.8         five 4.8, 5.5
    //                           3584 x 4608   seven 7.2, 7.2        eight 7.3, 8.2
    //                           14336 x 3584  eight 14.8, 13.6
    //                   e4m3    2048 x 2048   four 6.5, 5.8         five 6.5, 7.2
    //                           3584 x 4608   seven 10.4, 9.6       eight 10.5, 10.6
    //                           14336 x 3584  eight 21.5, 20.0
    //   groups of 64, 16 bits   1536 x 2048   four 5.2, 5.2         five 5.2, 5.8
    //                           3584 x 4608   seven 9.3, 8.9        eight 9.2, 9.9
    //                           3584 x 28672  eight 25.8, 23.0      nine 25.9, 36.1
    //                   int8    3584 x 3584   seven 7.6, 7.5        eight 7.6, 8.6
    //                           3584 x 4608   eight 9.5, 9.0        nine 9.4, 10.8
    //   groups of 32, 16 bits   1536 x 2048   four 6.2, 5.5         five 6.2, 6.3
    //                           3584 x 3584   eight 10.0, 9.6       nine 9.9, 11.4
    //                           3584 x 28672  eight 37.7, 24.7      nine 37.7, 39.7
    const int64_t held = static_cast<int64_t>(p.chunks) * p.tiles;  // records
    const int few = held < 1000    ? (size == 1 || group < 128 ? 4 : 3)
                    : group == 32  ? 8
                    : group == 64  ? (held < 1800 ? (size == 1 ? 7 : 4) : size == 1 || held >= 8192 ? 8 : 7)
                    : size == 1    ? (held < 1800 ? 4 : held < 4096 ? 7 : 8)
                    : held < 4096  ? 3
                    : held < 8192  ? 4
                    : held < 32768 ? 7
                                   : 8;
    const int64_t out_size = dtype_size(a->out_dtype);
    for (int64_t m0 = 0; m0 < a->m; m0 += kLaunchRows) {
        p.m = static_cast<int>(a->m - m0 < kLaunchRows ? a->m - m0 : kLaunchRows);
        p.x = static_cast<const uint8_t*>(a->x) + m0 * a->x_stride_row * size;
        if (a->x_scale) p.x_scale = static_cast<const float*>(a->x_scale) + m0;
        if (a->residual)
            p.residual = static_cast<const uint8_t*>(a->residual) + m0 * a->residual_stride_row * out_size;
        p.out = static_cast<uint8_t*>(a->out) + m0 * a->out_stride_row * out_size;
        rc = kind == mvq::kF32 || p.m <= few
                 ? mvq::launch_narrow(p, kind, group, a->has_zeros != 0, device, sms, stream)
                 : mvq::launch_wide(p, p.x_dtype, group, a->has_zeros != 0, device, sms, stream);
        if (rc != MVQ_OK) return rc;
    }
    return MVQ_OK;
} catch (...) {
    return fail(MVQ_ERR_CUDA, "unexpected C++ exception");
}

int mvq_w4_dequantize(const MvqDequantizeArgs* a, void* stream) try {
    if (!a) return fail(MVQ_ERR_INVALID_ARGUMENT, "args must not be NULL");
    int rc = check_weight(a->records, a->n, a->k, a->group, a->scale_dtype);
    if (rc != MVQ_OK) return rc;
    if (!a->out) return fail(MVQ_ERR_INVALID_ARGUMENT, "out must not be NULL");
    if (!float_dtype(a->out_dtype))
        return fail(MVQ_ERR_INVALID_ARGUMENT, "out_dtype must be MVQ_DTYPE_F32, MVQ_DTYPE_F16 or MVQ_DTYPE_BF16");
    if (a->n > 1 && a->out_stride_row < a->k)
        return fail(MVQ_ERR_INVALID_ARGUMENT, "out's rows must not overlap");
    if (off_element(a->out, a->out_dtype))
        return fail(MVQ_ERR_INVALID_ARGUMENT, "pointers must be aligned to their elements");
    const int chunks = static_cast<int>((a->k + mvq::kChunk - 1) / mvq::kChunk);
    const int64_t total = (a->n + mvq::kTileRows - 1) / mvq::kTileRows * chunks;
    if (total >= (int64_t(1) << 31)) return fail(MVQ_ERR_UNSUPPORTED, "the weight is too large for one call");
    const int64_t size = dtype_size(a->out_dtype);
    const int runs = address(a->out) % 16 == 0 && (a->n == 1 || a->out_stride_row * size % 16 == 0);
    // A warp per 32 columns of a record.
    const dim3 grid(static_cast<unsigned>((4 * total + mvq::kDequantizeWarps - 1) / mvq::kDequantizeWarps));
    const int bytes = mvq::record_size(static_cast<int>(a->group), a->has_zeros != 0), bf16 = a->scale_dtype == MVQ_DTYPE_BF16;
    const uint8_t* records = static_cast<const uint8_t*>(a->records);
    const int group = static_cast<int>(a->group), zeros = a->has_zeros != 0;
    const int n = static_cast<int>(a->n), k = static_cast<int>(a->k);
    cudaError_t err;
    if (a->out_dtype == MVQ_DTYPE_F32)
        err = launch(mvq::w4_dequantize_kernel<float>, grid, 256, 0, 1, stream, records, total, chunks, bytes, group,
                     zeros, bf16, n, k, static_cast<float*>(a->out), a->out_stride_row, runs);
    else if (a->out_dtype == MVQ_DTYPE_F16)
        err = launch(mvq::w4_dequantize_kernel<__half>, grid, 256, 0, 1, stream, records, total, chunks, bytes, group,
                     zeros, bf16, n, k, static_cast<__half*>(a->out), a->out_stride_row, runs);
    else
        err = launch(mvq::w4_dequantize_kernel<__nv_bfloat16>, grid, 256, 0, 1, stream, records, total, chunks, bytes,
                     group, zeros, bf16, n, k, static_cast<__nv_bfloat16*>(a->out), a->out_stride_row, runs);
    return err == cudaSuccess ? MVQ_OK : cuda_fail(err, "4-bit dequantize kernel launch");
} catch (...) {
    return fail(MVQ_ERR_CUDA, "unexpected C++ exception");
}

int mvq_add_rms_norm(const MvqNormArgs* a, void* stream) try {
    if (!a) return fail(MVQ_ERR_INVALID_ARGUMENT, "args must not be NULL");
    int rc = check_rows(a->rows, a->hidden, a->dtype);
    if (rc != MVQ_OK) return rc;
    if (!a->x || !a->weight || !a->out) return fail(MVQ_ERR_INVALID_ARGUMENT, "x, weight and out must not be NULL");
    const bool eight = a->out_dtype == MVQ_DTYPE_I8 || a->out_dtype == MVQ_DTYPE_E4M3;
    if (!eight && a->out_dtype != a->dtype)
        return fail(MVQ_ERR_INVALID_ARGUMENT, "out_dtype must be dtype, MVQ_DTYPE_I8 or MVQ_DTYPE_E4M3");
    if (eight != (a->scales != nullptr))
        return fail(MVQ_ERR_INVALID_ARGUMENT, "8-bit outputs, and only those, come with scales");
    if (!(a->eps >= 0.0) || std::isinf(a->eps))
        return fail(MVQ_ERR_INVALID_ARGUMENT, "eps must be finite and nonnegative");
    if (a->rows > 1 && (a->x_stride_row < 0 || (a->residual && a->residual_stride_row < 0) ||
                        a->out_stride_row < a->hidden ||
                        (a->residual_out && a->residual_out_stride_row < a->hidden)))
        return fail(MVQ_ERR_INVALID_ARGUMENT, "row strides must be nonnegative and outputs' rows must not overlap");
    if (off_element(a->x, a->dtype) || off_element(a->residual, a->dtype) || off_element(a->weight, a->dtype) ||
        off_element(a->residual_out, a->dtype) || off_element(a->out, a->out_dtype) ||
        off_element(a->scales, MVQ_DTYPE_F32))
        return fail(MVQ_ERR_INVALID_ARGUMENT, "pointers must be aligned to their elements");
    int device, sms;
    rc = device_sms(&device, &sms);
    if (rc != MVQ_OK) return rc;
    const int64_t size = dtype_size(a->dtype);
    const bool one = a->rows == 1;  // strides that no row uses
    const uintptr_t wide = address(a->x) | address(a->residual) | address(a->weight) | address(a->residual_out) |
                           (one ? 0 : static_cast<uintptr_t>(a->x_stride_row * size) |
                                          (a->residual ? static_cast<uintptr_t>(a->residual_stride_row * size) : 0) |
                                          (a->residual_out ? static_cast<uintptr_t>(a->residual_out_stride_row * size) : 0));
    const int64_t out_run = eight ? 8 : 16;
    const bool runs = a->hidden % 8 == 0 && wide % 16 == 0 && address(a->out) % out_run == 0 &&
                      (one || a->out_stride_row * (eight ? 1 : size) % out_run == 0);
    mvq::NormParams p = {};
    p.rows = a->rows;
    p.x = a->x;
    p.x_stride = a->x_stride_row;
    p.residual = a->residual;
    p.residual_stride = a->residual_stride_row;
    p.weight = a->weight;
    p.out = a->out;
    p.out_stride = a->out_stride_row;
    p.scales = static_cast<float*>(a->scales);
    p.residual_out = a->residual_out;
    p.residual_out_stride = a->residual_out_stride_row;
    p.hidden = static_cast<int>(a->hidden);
    p.eps = static_cast<float>(a->eps);
    cudaError_t err;
    if (a->out_dtype == MVQ_DTYPE_I8)
        err = launch_row_type<mvq::kOutI8, NormKernel>(p, a->dtype, runs, a->hidden, a->rows, sms, stream);
    else if (a->out_dtype == MVQ_DTYPE_E4M3)
        err = launch_row_type<mvq::kOutE4M3, NormKernel>(p, a->dtype, runs, a->hidden, a->rows, sms, stream);
    else
        err = launch_row_type<mvq::kOutSame, NormKernel>(p, a->dtype, runs, a->hidden, a->rows, sms, stream);
    return err == cudaSuccess ? MVQ_OK : cuda_fail(err, "add-RMSNorm kernel launch");
} catch (...) {
    return fail(MVQ_ERR_CUDA, "unexpected C++ exception");
}

int mvq_silu_mul_quant(const MvqSiluArgs* a, void* stream) try {
    if (!a) return fail(MVQ_ERR_INVALID_ARGUMENT, "args must not be NULL");
    int rc = check_rows(a->rows, a->width, a->dtype);
    if (rc != MVQ_OK) return rc;
    if (!a->gate_up || !a->out || !a->scales)
        return fail(MVQ_ERR_INVALID_ARGUMENT, "gate_up, out and scales must not be NULL");
    if (a->out_dtype != MVQ_DTYPE_I8 && a->out_dtype != MVQ_DTYPE_E4M3)
        return fail(MVQ_ERR_INVALID_ARGUMENT, "out_dtype must be MVQ_DTYPE_I8 or MVQ_DTYPE_E4M3");
    if (a->rows > 1 && (a->stride_row < 0 || a->out_stride_row < a->width))
        return fail(MVQ_ERR_INVALID_ARGUMENT, "row strides must be nonnegative and out's rows must not overlap");
    if (off_element(a->gate_up, a->dtype) || off_element(a->scales, MVQ_DTYPE_F32))
        return fail(MVQ_ERR_INVALID_ARGUMENT, "pointers must be aligned to their elements");
    int device, sms;
    rc = device_sms(&device, &sms);
    if (rc != MVQ_OK) return rc;
    const int64_t size = dtype_size(a->dtype);
    const bool one = a->rows == 1;
    const bool runs = a->width % 8 == 0 && address(a->gate_up) % 16 == 0 && address(a->out) % 8 == 0 &&
                      (one || (a->stride_row * size % 16 == 0 && a->out_stride_row % 8 == 0));
    mvq::SiluParams p = {};
    p.rows = a->rows;
    p.gate_up = a->gate_up;
    p.stride = a->stride_row;
    p.out = a->out;
    p.out_stride = a->out_stride_row;
    p.scales = static_cast<float*>(a->scales);
    p.width = static_cast<int>(a->width);
    const cudaError_t err =
        a->out_dtype == MVQ_DTYPE_I8
            ? launch_row_type<mvq::kOutI8, SiluKernel>(p, a->dtype, runs, a->width, a->rows, sms, stream)
            : launch_row_type<mvq::kOutE4M3, SiluKernel>(p, a->dtype, runs, a->width, a->rows, sms, stream);
    return err == cudaSuccess ? MVQ_OK : cuda_fail(err, "SiLU-mul-quantize kernel launch");
} catch (...) {
    return fail(MVQ_ERR_CUDA, "unexpected C++ exception");
}

}  // extern "C"
