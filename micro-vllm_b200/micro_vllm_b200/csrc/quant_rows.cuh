// Row operations that end in 8 bits (or, for the norm, in the row's type):
//  * add_rms_norm: s = to_T(x + residual), y = weight * s * rsqrt(mean(s^2) + eps);
//  * silu_mul_quant: y = silu(g) * u of rows [g | u];
// with 8-bit outputs round(y / scale), scale = max|y| / top over the row.
//
// One pass over the row: the values stay in registers (fp32) between the
// reductions and the store, so each input is read once and each output written
// once. The norm's maximum needs no second pass over the data: max|y| =
// rsqrt(...) * max|weight * s|, so the sum of squares and the maximum are
// reduced together. One CTA per row, or, for many narrow rows, one warp.
#pragma once

#include <cuda_fp8.h>

#include "mv_device.cuh"

namespace mvq {

using mv::from_float;
using mv::to_float;

enum : int { kOutSame = 0, kOutI8 = 1, kOutE4M3 = 2 };

// Two fp32 numbers rounded to a pair of T (the first in the low half), and back.
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    return mv::MmaOp<T>::pack(lo, hi);
}
template <typename T>
__device__ __forceinline__ float2 unpack_pair(uint32_t w) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    else
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

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
    // Eight elements as they lie in memory, so that several loads can be under way before one is used.
    struct Raw {
        uint4 w[sizeof(T) / 2];  // RUNS
        T e[RUNS ? 1 : 8];       // elements
    };
    __device__ __forceinline__ void fetch(const T* row, int j, Raw& r) const {
        if constexpr (RUNS) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
                r.w[i] = make_uint4(0, 0, 0, 0);
                if (at(j, 0) < width) r.w[i] = reinterpret_cast<const uint4*>(row + at(j, 0))[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) r.e[i] = at(j, i) < width ? row[at(j, i)] : from_float<T>(0.0f);
        }
    }
    __device__ __forceinline__ void expand(const Raw& r, float (&v)[8]) const {
        if constexpr (!RUNS) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_float<T>(r.e[i]);
        } else if constexpr (sizeof(T) == 4) {
            v[0] = __uint_as_float(r.w[0].x), v[1] = __uint_as_float(r.w[0].y), v[2] = __uint_as_float(r.w[0].z);
            v[3] = __uint_as_float(r.w[0].w), v[4] = __uint_as_float(r.w[1].x), v[5] = __uint_as_float(r.w[1].y);
            v[6] = __uint_as_float(r.w[1].z), v[7] = __uint_as_float(r.w[1].w);
        } else {
            const uint32_t words[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = unpack_pair<T>(words[i]);
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            }
        }
    }
    __device__ __forceinline__ void load(const T* row, int j, float (&v)[8]) const {
        Raw r;
        fetch(row, j, r);
        expand(r, v);
    }
    // Stores v rounded to T (if `row` is not null) and leaves the rounded values in v.
    __device__ __forceinline__ void round_store(T* row, int j, float (&v)[8]) const {
        if constexpr (RUNS && sizeof(T) == 2) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = pack_pair<T>(v[2 * i], v[2 * i + 1]);
                const float2 f = unpack_pair<T>(w[i]);
                v[2 * i] = f.x, v[2 * i + 1] = f.y;
            }
            if (row && at(j, 0) < width)
                *reinterpret_cast<uint4*>(row + at(j, 0)) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_float<T>(from_float<T>(v[i]));
            if (row) store(row, j, v);
        }
    }
    __device__ __forceinline__ void store(T* row, int j, const float (&v)[8]) const {
        if constexpr (RUNS) {
            if (at(j, 0) >= width) return;
            if constexpr (sizeof(T) == 4) {
                reinterpret_cast<float4*>(row + at(j, 0))[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4*>(row + at(j, 0))[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                *reinterpret_cast<uint4*>(row + at(j, 0)) = make_uint4(pack_pair<T>(v[0], v[1]), pack_pair<T>(v[2], v[3]),
                                                                       pack_pair<T>(v[4], v[5]), pack_pair<T>(v[6], v[7]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (at(j, i) < width) row[at(j, i)] = from_float<T>(v[i]);
        }
    }
    // Eight finite values, scaled already, as 8-bit numbers.
    template <int OUT>
    __device__ __forceinline__ void store8(uint8_t* row, int j, const float (&v)[8]) const {
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (OUT == kOutI8) {
                // 1.5 2^23 + v rounds v to an integer, whose low byte is the number's lowest.
                uint32_t b[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(v[4 * i + e] + 12582912.0f);
                w[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
            } else {
                uint16_t lo, hi;
                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(v[4 * i + 1]), "f"(v[4 * i]));
                asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(v[4 * i + 3]), "f"(v[4 * i + 2]));
                w[i] = static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
            }
        }
        if constexpr (RUNS) {
            if (at(j, 0) < width) *reinterpret_cast<uint2*>(row + at(j, 0)) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (at(j, i) < width) row[at(j, i)] = static_cast<uint8_t>(w[i >> 2] >> (8 * (i & 3)));
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

// What turns a row's values v (y = v * amax / top_v) into its 8-bit numbers: y /
// scale = v * (top / top_v), the factor as the sum of two fp32 numbers. With it the
// quotient is off by half of fp32's step, so that one that fp32 holds -- a tie
// between two 8-bit numbers among them -- comes out as it is; one rounded factor put
// one tie in 17 on the wrong side. `shift`: a power of two that v is multiplied by
// first where the factor's parts would leave fp32's range. A factor of zero: the row
// has no scale (zeros, or a NaN or an infinity among them).
struct RowScale {
    float scale, mul, rest, shift;
};
template <int OUT>
__device__ __forceinline__ RowScale row_scale(float amax, float top_v) {
    constexpr float kTop = OUT == kOutI8 ? 127.0f : 448.0f;
    RowScale s;
    s.scale = amax < INFINITY ? amax / kTop : __int_as_float(0x7fffffff);
    s.shift = top_v < 0x1p-80f ? 0x1p+80f : top_v > 0x1p+80f ? 0x1p-80f : 1.0f;
    top_v *= s.shift;
    s.mul = s.scale > 0.0f ? kTop / top_v : 0.0f;
    s.rest = s.scale > 0.0f ? fmaf(-s.mul, top_v, kTop) / top_v : 0.0f;
    return s;
}
__device__ __forceinline__ void apply_scale(const RowScale& s, float (&v)[8]) {
    if (s.mul == 0.0f || s.shift != 1.0f) {  // the same for the whole row
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = s.mul == 0.0f ? 0.0f : v[i] * s.shift;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf(v[i], s.mul, v[i] * s.rest);
}

struct NormParams {
    int64_t rows;
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

// Threads of a CTA at most, by the runs of eight a thread holds (0: it holds none and
// reads the row twice). With four runs the norm has registers for 448 threads to
// load all of a row at once (1024 rows of 14336: 18.9 us, bound to 512 threads 26.3);
// the gate runs better in more threads with fewer (2048 rows of 11008: 23.5 and 26.1).
constexpr int max_row_threads(int held, bool norm) {
    return held == 1 || held == 2 ? 1024 : held == 4 && norm ? 448 : 512;
}

template <typename T, int OUT, bool RUNS, int C>
__global__ void __launch_bounds__(max_row_threads(C, true)) add_rms_norm_kernel(const NormParams p) {
    mv::wait_for_prior_grid();
    mv::allow_next_grid();
    const RowAccess<T, RUNS> at{p.hidden, static_cast<int>(blockDim.x)};
    const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    if (row >= p.rows) return;  // with several rows per CTA, each has one warp and waits for no other
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* residual = p.residual ? static_cast<const T*>(p.residual) + row * p.residual_stride : nullptr;
    T* residual_out = p.residual_out ? static_cast<T*>(p.residual_out) + row * p.residual_out_stride : nullptr;
    const T* weight = static_cast<const T*>(p.weight);
    T* out = static_cast<T*>(p.out) + row * p.out_stride;
    uint8_t* out8 = static_cast<uint8_t*>(p.out) + row * p.out_stride;
    using Raw = typename RowAccess<T, RUNS>::Raw;
    const auto add = [&](int j, float (&v)[8], const Raw& r, T* to) {  // s of run j, x's values being in v
        if (!residual) return;
        float e[8];
        at.expand(r, e);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fadd_rn(v[i], e[i]);
        at.round_store(to, j, v);
    };
    const auto weigh = [&](const Raw& r, float (&v)[8]) {
        float w[8];
        at.expand(r, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= w[i];
    };
    float sum = 0.0f, top = 0.0f;
    const auto gather = [&](int j, float (&v)[8], const Raw& r, const Raw& w) {  // v: x in, weight * s out
        add(j, v, r, residual_out);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(v[i], v[i], sum);
        weigh(w, v);
        if (OUT != kOutSame) {
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(v[i]));
        }
    };
    const int turns = (p.hidden + 8 * static_cast<int>(blockDim.x) - 1) / (8 * static_cast<int>(blockDim.x));
    float v[C ? C : 1][8];
    if constexpr (C > 0) {
        Raw rx[C], rr[C], rw[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            at.fetch(x, j, rx[j]);
            if (residual) at.fetch(residual, j, rr[j]);
        }
#pragma unroll
        for (int j = 0; j < C; ++j) at.fetch(weight, j, rw[j]);
#pragma unroll
        for (int j = 0; j < C; ++j) {
            at.expand(rx[j], v[j]);
            gather(j, v[j], rr[j], rw[j]);
        }
    } else {
        for (int j = 0; j < turns; ++j) {
            Raw r, w;
            at.load(x, j, v[0]);
            if (residual) at.fetch(residual, j, r);
            at.fetch(weight, j, w);
            gather(j, v[0], r, w);
        }
    }
    const float2 all = block_sum_max(sum, top);
    const float r = rsqrtf(all.x / static_cast<float>(p.hidden) + p.eps);
    RowScale scale;
    if constexpr (OUT != kOutSame) {
        scale = row_scale<OUT>(all.y * r, all.y);
        if (threadIdx.x == 0) p.scales[row] = scale.scale;
    }
    const auto finish = [&](int j, float (&v)[8]) {
        if constexpr (OUT == kOutSame) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= r;
            at.store(out, j, v);
        } else {
            apply_scale(scale, v);
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
            Raw r;
            if (residual && !residual_out) {
                at.fetch(residual, j, r);
                add(j, v[0], r, nullptr);
            }
            at.fetch(weight, j, r);
            weigh(r, v[0]);
            finish(j, v[0]);
        }
    }
}

struct SiluParams {
    int64_t rows;
    const void* gate_up;
    int64_t stride;
    void* out;
    int64_t out_stride;
    float* scales;
    int width;
};

template <typename T, int OUT, bool RUNS, int C>
__global__ void __launch_bounds__(max_row_threads(C, false)) silu_mul_quant_kernel(const SiluParams p) {
    mv::wait_for_prior_grid();
    mv::allow_next_grid();
    const RowAccess<T, RUNS> at{p.width, static_cast<int>(blockDim.x)};
    const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    if (row >= p.rows) return;  // with several rows per CTA, each has one warp and waits for no other
    const T* gate = static_cast<const T*>(p.gate_up) + row * p.stride;
    uint8_t* out = static_cast<uint8_t*>(p.out) + row * p.out_stride;
    float top = 0.0f;
    const auto gated = [&](float (&v)[8], const float (&u)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // exp(-g) / 4 as a power of two and 4 / (1 + exp(-g)): the quarter keeps 1 + exp(-g) below
            // 2^126, where the reciprocal would be flushed to zero, for every g down to -88.72 (beyond
            // it fp32's exp(-g) is an infinity, and the value a zero here as there). The argument's
            // rounding makes the exponential off by about |g| 2^-24, the rest adds a few 2^-24
            // (measured: 9 2^-24 of the value for gates above -8, 66 at -80). expf and the division,
            // at 4 2^-24, took 2048 x 14336 from 33.1 us to 41.1; the argument in two parts, at 6, to 36.9.
            float e, d;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(v[i], -1.4426950408889634f, -2.0f)));
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(d) : "f"(0.25f + e));
            v[i] = v[i] * 0.25f * d * u[i];
        }
    };
    const auto value = [&](int j, float (&v)[8]) {
        float u[8];
        at.load(gate, j, v);
        at.load(gate + p.width, j, u);
        gated(v, u);
    };
    const auto measure = [&](const float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(v[i]));
    };
    const int turns = (p.width + 8 * static_cast<int>(blockDim.x) - 1) / (8 * static_cast<int>(blockDim.x));
    float v[C ? C : 1][8];
    if constexpr (C > 0) {
        typename RowAccess<T, RUNS>::Raw rg[C], ru[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            at.fetch(gate, j, rg[j]);
            at.fetch(gate + p.width, j, ru[j]);
        }
#pragma unroll
        for (int j = 0; j < C; ++j) {
            float u[8];
            at.expand(rg[j], v[j]);
            at.expand(ru[j], u);
            gated(v[j], u);
            measure(v[j]);
        }
    } else {
        for (int j = 0; j < turns; ++j) {
            value(j, v[0]);
            measure(v[0]);
        }
    }
    const float2 all = block_sum_max(0.0f, top);
    const RowScale scale = row_scale<OUT>(all.y, all.y);
    if (threadIdx.x == 0) p.scales[row] = scale.scale;
    const auto finish = [&](int j, float (&v)[8]) {
        apply_scale(scale, v);
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
