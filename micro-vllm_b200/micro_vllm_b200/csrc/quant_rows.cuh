// Row operations that end in 8 bits (or, for the norm, in the row's type):
//  * add_rms_norm: s = to_T(x + residual), y = weight * s * rsqrt(mean(s^2) + eps);
//  * silu_mul_quant: y = silu(g) * u of rows [g | u];
// with 8-bit outputs round(y / scale), scale = max|y| / top over the row.
//
// One pass over the row: the values stay in registers (fp32) between the
// reductions and the store, so each input is read once and each output written
// once. The norm's maximum needs no second pass over the data: max|y| =
// rsqrt(...) * max|weight * s|, so the sum of squares and the maximum are
// reduced together. One CTA per row.
#pragma once

#include <cuda_fp8.h>

#include "mv_device.cuh"

namespace mvq {

using mv::from_float;
using mv::to_float;

enum : int { kOutSame = 0, kOutI8 = 1, kOutE4M3 = 2 };

// Eight elements of a row. Runs: the eight at 8 c (one or two 16-byte
// accesses). Elements: the eight at `threads` apart, each checked, for rows
// that are not aligned or not a multiple of eight wide.
template <typename T, bool RUNS>
struct RowAccess {
    int width, threads;
    __device__ __forceinline__ int at(int j, int i) const {
        return RUNS ? 8 * (j * threads + static_cast<int>(threadIdx.x)) + i
                    : (8 * j + i) * threads + static_cast<int>(threadIdx.x);
    }
    __device__ __forceinline__ void load(const T* row, int j, float (&v)[8]) const {
        if constexpr (RUNS) {
            if (at(j, 0) < width) {
                __align__(16) T e[8];
#pragma unroll
                for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
                    reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(row + at(j, 0))[i];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = to_float<T>(e[i]);
                return;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = at(j, i) < width ? to_float<T>(row[at(j, i)]) : 0.0f;
        }
    }
    __device__ __forceinline__ void store(T* row, int j, const float (&v)[8]) const {
        if constexpr (RUNS) {
            if (at(j, 0) < width) {
                __align__(16) T e[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = from_float<T>(v[i]);
#pragma unroll
                for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
                    reinterpret_cast<uint4*>(row + at(j, 0))[i] = reinterpret_cast<const uint4*>(e)[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (at(j, i) < width) row[at(j, i)] = from_float<T>(v[i]);
        }
    }
    // Eight 8-bit values (already scaled).
    template <int OUT>
    __device__ __forceinline__ void store8(uint8_t* row, int j, const float (&v)[8]) const {
        uint32_t b[8];
        if constexpr (OUT == kOutI8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] = static_cast<uint32_t>(__float2int_rn(v[i])) & 0xffu;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(v[i], v[i + 1]), __NV_SATFINITE, __NV_E4M3);
                b[i] = two & 0xffu;
                b[i + 1] = two >> 8;
            }
        }
        if constexpr (RUNS) {
            if (at(j, 0) < width)
                *reinterpret_cast<uint2*>(row + at(j, 0)) =
                    make_uint2(b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24),
                               b[4] | (b[5] << 8) | (b[6] << 16) | (b[7] << 24));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (at(j, i) < width) row[at(j, i)] = static_cast<uint8_t>(b[i]);
        }
    }
};

// A maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Sum and maximum over the CTA; every thread gets both.
__device__ __forceinline__ float2 block_sum_max(float sum, float top) {
    __shared__ float2 part[32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    const int warps = blockDim.x >> 5;
    if (warps == 1) return make_float2(sum, top);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_float2(sum, top);
    __syncthreads();
    float2 all = part[0];
    for (int w = 1; w < warps; ++w) {
        all.x += part[w].x;
        all.y = max_nan(all.y, part[w].y);
    }
    return all;
}

// Scale of a row whose largest |y| is `amax`, and what takes a value v with
// y = v * amax / top_v to its 8-bit number: v * mul.x * mul.y. mul.x is a power
// of two that keeps top / top_v finite for tiny rows.
template <int OUT>
__device__ __forceinline__ float row_scale(float amax, float top_v, float2* mul) {
    constexpr float kTop = OUT == kOutI8 ? 127.0f : 448.0f;
    const float scale = amax < INFINITY ? amax / kTop : __int_as_float(0x7fffffff);
    const float up = top_v < 0x1p-100f ? 0x1p+100f : 1.0f;
    *mul = scale > 0.0f ? make_float2(up, kTop / (top_v * up)) : make_float2(0.0f, 0.0f);
    return scale;
}

template <int OUT>
__device__ __forceinline__ float scaled(float v, float2 mul) {
    // A row without a scale gives zeros, whatever its values (NaN and infinities among them).
    return mul.y == 0.0f ? 0.0f : v * mul.x * mul.y;
}

struct NormParams {
    const void* x;
    int64_t x_stride;
    const void* residual;
    int64_t residual_stride;
    const void* weight;
    void* out;
    int64_t out_stride;
    float* scales;
    void* residual_out;
    int64_t residual_out_stride;
    int hidden;
    float eps;
};

// Threads of a CTA at most, by the runs of eight a thread holds (0: it holds none and reads the row twice).
constexpr int max_row_threads(int held) { return held == 1 || held == 2 ? 1024 : 512; }

template <typename T, int OUT, bool RUNS, int C>
__global__ void __launch_bounds__(max_row_threads(C)) add_rms_norm_kernel(const NormParams p) {
    mv::wait_for_prior_grid();
    mv::allow_next_grid();
    const RowAccess<T, RUNS> at{p.hidden, static_cast<int>(blockDim.x)};
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* residual = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_stride : nullptr;
    T* residual_out = p.residual_out ? static_cast<T*>(p.residual_out) + row * p.residual_out_stride : nullptr;
    const T* weight = static_cast<const T*>(p.weight);
    T* out = static_cast<T*>(p.out) + row * p.out_stride;
    uint8_t* out8 = static_cast<uint8_t*>(p.out) + row * p.out_stride;
    const auto add = [&](int j, float (&v)[8]) {  // s of run j, x's values being in v
        if (!residual) return;
        float e[8];
        at.load(residual, j, e);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_float<T>(from_float<T>(__fadd_rn(v[i], e[i])));
    };
    const auto weigh = [&](int j, float (&v)[8]) {
        float w[8];
        at.load(weight, j, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= w[i];
    };
    float sum = 0.0f, top = 0.0f;
    const auto gather = [&](int j, float (&v)[8]) {  // v: x in, weight * s out
        add(j, v);
        if (residual_out) at.store(residual_out, j, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(v[i], v[i], sum);
        weigh(j, v);
        if (OUT != kOutSame) {
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(v[i]));
        }
    };
    const int turns = (p.hidden + 8 * static_cast<int>(blockDim.x) - 1) / (8 * static_cast<int>(blockDim.x));
    float v[C ? C : 1][8];
    if constexpr (C > 0) {
#pragma unroll
        for (int j = 0; j < C; ++j) at.load(x, j, v[j]);
#pragma unroll
        for (int j = 0; j < C; ++j) gather(j, v[j]);
    } else {
        for (int j = 0; j < turns; ++j) {
            at.load(x, j, v[0]);
            gather(j, v[0]);
        }
    }
    const float2 all = block_sum_max(sum, top);
    const float r = rsqrtf(all.x / static_cast<float>(p.hidden) + p.eps);
    float2 mul = make_float2(r, 1.0f);
    if constexpr (OUT != kOutSame) {
        const float scale = row_scale<OUT>(all.y * r, all.y, &mul);
        if (threadIdx.x == 0) p.scales[row] = scale;
    }
    const auto finish = [&](int j, float (&v)[8]) {
        if constexpr (OUT == kOutSame) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= r;
            at.store(out, j, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = scaled<OUT>(v[i], mul);
            at.template store8<OUT>(out8, j, v);
        }
    };
    if constexpr (C > 0) {
#pragma unroll
        for (int j = 0; j < C; ++j) finish(j, v[j]);
    } else {
        for (int j = 0; j < turns; ++j) {
            // The sum that this thread stored, where there is one: it may lie over x or the residual.
            at.load(residual_out ? residual_out : x, j, v[0]);
            if (!residual_out) add(j, v[0]);
            weigh(j, v[0]);
            finish(j, v[0]);
        }
    }
}

struct SiluParams {
    const void* gate_up;
    int64_t stride;
    void* out;
    int64_t out_stride;
    float* scales;
    int width;
};

template <typename T, int OUT, bool RUNS, int C>
__global__ void __launch_bounds__(max_row_threads(C)) silu_mul_quant_kernel(const SiluParams p) {
    mv::wait_for_prior_grid();
    mv::allow_next_grid();
    const RowAccess<T, RUNS> at{p.width, static_cast<int>(blockDim.x)};
    const int64_t row = blockIdx.x;
    const T* gate = static_cast<const T*>(p.gate_up) + row * p.stride;
    uint8_t* out = static_cast<uint8_t*>(p.out) + row * p.out_stride;
    float top = 0.0f;
    const auto value = [&](int j, float (&v)[8]) {
        float u[8];
        at.load(gate, j, v);
        at.load(gate + p.width, j, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fdividef(v[i], 1.0f + __expf(-v[i])) * u[i];
    };
    const auto measure = [&](const float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(v[i]));
    };
    const int turns = (p.width + 8 * static_cast<int>(blockDim.x) - 1) / (8 * static_cast<int>(blockDim.x));
    float v[C ? C : 1][8];
    if constexpr (C > 0) {
#pragma unroll
        for (int j = 0; j < C; ++j) {
            value(j, v[j]);
            measure(v[j]);
        }
    } else {
        for (int j = 0; j < turns; ++j) {
            value(j, v[0]);
            measure(v[0]);
        }
    }
    const float2 all = block_sum_max(0.0f, top);
    float2 mul;
    const float scale = row_scale<OUT>(all.y, all.y, &mul);
    if (threadIdx.x == 0) p.scales[row] = scale;
    const auto finish = [&](int j, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = scaled<OUT>(v[i], mul);
        at.template store8<OUT>(out, j, v);
    };
    if constexpr (C > 0) {
#pragma unroll
        for (int j = 0; j < C; ++j) finish(j, v[j]);
    } else {
        for (int j = 0; j < turns; ++j) {
            value(j, v[0]);
            finish(j, v[0]);
        }
    }
}

}  // namespace mvq
