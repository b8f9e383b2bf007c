// Products with 4-bit weights: y = (x W^T) * x_scale + bias + residual for a
// few rows of x (mma.sync tiles, split over the columns of W), and W itself
// written out. The weight's record layout is in include/mvquant.h.
//
// Mathematics. W[n, k] = (code - zero) * scale per row n and group of k. The
// kernel never forms the scaled weight: within a group it sums x * (code -
// zero) -- code - zero is a small integer, exact in bf16, fp16 and int8 -- and
// then adds scale * sum to the row's fp32 accumulator. So the only rounding of
// 16-bit activations' results is the last one.
//
// What bounds it: the codes are read once, half a byte per weight, and each
// weight costs about 1.4 instructions to become a bf16 (shift, mask-xor,
// subtract on pairs), 1.1 an fp16, 0.4 an int8, against about 2.8 issue slots
// per weight at the copy bandwidth. The records hold the codes in the order of
// the A operand of mma.sync (16 weight rows x 16 or 32 columns), so a lane's 16
// bytes become four operand registers by masks and shifts alone, and both the
// 16-bit and the 8-bit instruction read the same records.
#pragma once

#include <cuda_fp8.h>

#include "mv_device.cuh"

namespace mvq {

using mv::from_float;
using mv::to_float;

constexpr int kTileRows = 64;
constexpr int kChunk = 128;
constexpr int kCodeBytes = kTileRows * kChunk / 2;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 4;
// Row stride of the partial sums [token][64 weight rows] in shared memory, in
// floats: 68 keeps the eight rows and four token pairs that a warp stores at
// once in different banks.
constexpr int kPartStride = 68;

struct LinearParams {
    const void* x;
    int64_t x_stride;
    const float* x_scale;
    const uint8_t* records;
    int n, k, m;
    int chunks;        // ceil(k / 128)
    int record_bytes;
    int has_zeros;
    int scale_bf16;
    int x_runs;        // x may be read 8 elements at a time: aligned rows, k a multiple of 8
    int cluster;       // CTAs that share a tile's columns
    const void* bias;
    const void* residual;
    int64_t residual_stride;
    void* out;
    int64_t out_stride;
    int out_dtype;
};

enum : int { kF32 = 0, kF16 = 1, kBF16 = 2, kI8 = 3, kE4M3 = 4 };

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}

// (a & mask) ^ bits in one instruction.
__device__ __forceinline__ uint32_t and_xor(uint32_t a, uint32_t mask, uint32_t bits) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(d) : "r"(a), "r"(mask), "r"(bits));
    return d;
}

__device__ __forceinline__ float2 scale_pair(uint32_t bits, int bf16) {
    if (bf16) return make_float2(__uint_as_float(bits << 16), __uint_as_float(bits & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&bits));
}

// Operand arithmetic of each activation type. A holds how a word of codes
// (rows g and g + 8 of a 16-row block, columns 4e..4e+3 of the lane's run of
// eight) becomes operand registers; kPlanes bf16 numbers make up one x.
template <int XT>
struct Act;

struct ActHalfBase {
    static constexpr int kRegs = 4;  // 32-bit registers of x per plane, 8-column run and token
};

template <>
struct Act<kBF16> : ActHalfBase {
    using T = __nv_bfloat16;
    static constexpr int kPlanes = 1;
    // (code - zero) / 2^11 from 128 + code (bf16 numbers from 128 to 255 have a
    // step of one): (128 + code) / 2^11 - (128 + zero) / 2^11, exact. The power
    // of two goes back into the scale; with it a group's sum of 128 products of
    // at most 15 stays below the largest |x|, so no x that is finite overflows.
    static constexpr float kScale = 2048.0f;
    __device__ __forceinline__ static uint32_t zero_low(int z) { return (0xbd80u + z) * 0x10001u; }
    __device__ __forceinline__ static uint32_t zero_high(int z) { return zero_low(z); }
    __device__ __forceinline__ static uint32_t sub(uint32_t a, uint32_t z) {
        const uint32_t step = 0x3a003a00u;  // 2^-11
        const __nv_bfloat162 d = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                         *reinterpret_cast<const __nv_bfloat162*>(&step),
                                         *reinterpret_cast<const __nv_bfloat162*>(&z));
        return *reinterpret_cast<const uint32_t*>(&d);
    }
    __device__ __forceinline__ static void weights(uint32_t w, uint32_t zl, uint32_t zh, uint32_t (&a)[4]) {
        a[0] = sub(and_xor(w, 0x000f000fu, 0x43084308u), zl);
        a[1] = sub(and_xor(w >> 4, 0x000f000fu, 0x43084308u), zh);
        a[2] = sub(and_xor(w >> 8, 0x000f000fu, 0x43084308u), zl);
        a[3] = sub(and_xor(w >> 12, 0x000f000fu, 0x43084308u), zh);
    }
    __device__ __forceinline__ static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        mv::MmaOp<__nv_bfloat16>::run(c, a, b0, b1);
    }
};

// fp32 x as the exact sum of three bf16 numbers (8 + 8 + 8 bits of its 24).
template <>
struct Act<kF32> : Act<kBF16> {
    using T = float;
    static constexpr int kPlanes = 3;
};

template <>
struct Act<kF16> : ActHalfBase {
    using T = __half;
    static constexpr int kPlanes = 1;
    static constexpr float kScale = 1.0f;
    // Low nibbles become 1024 + code (step one), high nibbles 1024 + 16 code,
    // then code - zero as (1024 + 16 code) / 16 - (64 + zero): all exact.
    __device__ __forceinline__ static uint32_t zero_low(int z) { return (0x6400u + z) * 0x10001u; }
    __device__ __forceinline__ static uint32_t zero_high(int z) { return (0xd400u + 16 * z) * 0x10001u; }
    __device__ __forceinline__ static uint32_t low(uint32_t w, uint32_t z) {
        const uint32_t v = and_xor(w, 0x000f000fu, 0x64086408u);
        const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&z));
        return *reinterpret_cast<const uint32_t*>(&d);
    }
    __device__ __forceinline__ static uint32_t high(uint32_t w, uint32_t z) {
        const uint32_t v = and_xor(w, 0x00f000f0u, 0x64806480u), sixteenth = 0x2c002c00u;
        const __half2 d = __hfma2(*reinterpret_cast<const __half2*>(&v), *reinterpret_cast<const __half2*>(&sixteenth),
                                  *reinterpret_cast<const __half2*>(&z));
        return *reinterpret_cast<const uint32_t*>(&d);
    }
    __device__ __forceinline__ static void weights(uint32_t w, uint32_t zl, uint32_t zh, uint32_t (&a)[4]) {
        a[0] = low(w, zl);
        a[1] = high(w, zh);
        a[2] = low(w >> 8, zl);
        a[3] = high(w >> 8, zh);
    }
    __device__ __forceinline__ static void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        mv::MmaOp<__half>::run(c, a, b0, b1);
    }
};

// e4m3 numbers are exact in fp16.
template <>
struct Act<kE4M3> : Act<kF16> {
    using T = __nv_fp8_storage_t;
};

template <>
struct Act<kI8> {
    using T = int8_t;
    static constexpr int kPlanes = 1;
    static constexpr int kRegs = 2;
};

__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight consecutive elements of a row of x as operand registers: columns k..k+7
// (zeros at and beyond `limit`), r[plane][...]. `runs`: one vector load.
template <int XT>
__device__ __forceinline__ void load_run(const typename Act<XT>::T* row, int k, int limit, bool runs,
                                         uint32_t (&r)[Act<XT>::kPlanes][Act<XT>::kRegs]) {
    if constexpr (XT == kBF16 || XT == kF16) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (runs) {
            if (k < limit) v = __ldg(reinterpret_cast<const uint4*>(row + k));
        } else {
            const uint16_t* e = reinterpret_cast<const uint16_t*>(row);
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = k + i < limit ? __ldg(e + k + i) : 0u;
            v = make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
        }
        r[0][0] = v.x, r[0][1] = v.y, r[0][2] = v.z, r[0][3] = v.w;
    } else if constexpr (XT == kF32) {
        float f[8];
        if (runs && k < limit) {
            const float4 lo = __ldg(reinterpret_cast<const float4*>(row + k));
            const float4 hi = __ldg(reinterpret_cast<const float4*>(row + k) + 1);
            f[0] = lo.x, f[1] = lo.y, f[2] = lo.z, f[3] = lo.w, f[4] = hi.x, f[5] = hi.y, f[6] = hi.z, f[7] = hi.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = k + i < limit ? __ldg(row + k + i) : 0.0f;
        }
        // Truncation to bf16 three times: x = b0 + b1 + b2 exactly. What is not
        // finite goes into b0 alone (a NaN may not lose its last bits to an infinity).
        uint32_t b[3][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool finite = fabsf(f[i]) < INFINITY;
            b[0][i] = (__float_as_uint(f[i]) | (f[i] != f[i] ? 0x00400000u : 0u)) & 0xffff0000u;
            const float rest = finite ? f[i] - __uint_as_float(b[0][i]) : 0.0f;
            b[1][i] = __float_as_uint(rest) & 0xffff0000u;
            b[2][i] = __float_as_uint(rest - __uint_as_float(b[1][i])) & 0xffff0000u;
        }
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i) r[p][i] = (b[p][2 * i] >> 16) | b[p][2 * i + 1];
    } else {
        uint2 v = make_uint2(0, 0);
        const uint8_t* e = reinterpret_cast<const uint8_t*>(row);
        if (runs) {
            if (k < limit) v = __ldg(reinterpret_cast<const uint2*>(e + k));
        } else {
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = k + i < limit ? __ldg(e + k + i) : 0u;
            v = make_uint2(h[0] | (h[1] << 8) | (h[2] << 16) | (h[3] << 24),
                           h[4] | (h[5] << 8) | (h[6] << 16) | (h[7] << 24));
        }
        if constexpr (XT == kI8) {  // the codes' byte order: 0, 2, 1, 3
            r[0][0] = __byte_perm(v.x, 0, 0x3120);
            r[0][1] = __byte_perm(v.y, 0, 0x3120);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t pair = (i < 2 ? v.x : v.y) >> (16 * (i & 1)) & 0xffffu;
                const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(pair), __NV_E4M3);
                r[0][i] = h.x | (static_cast<uint32_t>(h.y) << 16);
            }
        }
    }
}

__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int dtype) {
    if (dtype == kF32) return static_cast<const float*>(p)[i];
    if (dtype == kF16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void store_from_float(void* p, int64_t i, int dtype, float v) {
    if (dtype == kF32) static_cast<float*>(p)[i] = v;
    else if (dtype == kF16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
// A float of another CTA's shared memory (of the same cluster).
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
    uint32_t remote;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
    return v;
}

// One cluster of `cluster` CTAs per (tile of 64 weight rows, block of 8 NB
// tokens). The chunks of 128 columns are dealt to its 4 * cluster warps in
// turn; each warp streams its records through a ring of its own (cp.async, no
// barrier: the warp reads what its own lanes copied), sums all 64 rows for all
// its tokens, and the warps' partial sums meet in (distributed) shared memory,
// added in a fixed order.
template <int XT, int NB, int GROUP>
__global__ void __launch_bounds__(kThreads) w4_linear_kernel(const LinearParams p) {
    using A = Act<XT>;
    using T = typename A::T;
    constexpr int kGroupRuns = GROUP / 32;        // 32-column runs per group
    constexpr int kGroups = kChunk / GROUP;       // groups per chunk
    extern __shared__ __align__(128) uint8_t smem[];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const uint32_t rank = p.cluster > 1 ? cluster_rank() : 0;
    const int64_t tile = blockIdx.x / p.cluster;
    const int token0 = blockIdx.y * (8 * NB);
    const int step = kWarps * p.cluster;
    const int first = static_cast<int>(rank) * kWarps + warp;
    const int mine = p.chunks > first ? (p.chunks - first + step - 1) / step : 0;
    const uint8_t* base = p.records + tile * p.chunks * static_cast<int64_t>(p.record_bytes);
    const uint32_t ring = mv::smem_addr(smem) + warp * kStages * p.record_bytes;

    // The weights' first records come into L2 while the grid before drains. Its
    // writes are not visible yet, so nothing is read.
    for (int i = 0; i < kStages && i < mine; ++i) {
        const uint8_t* rec = base + static_cast<int64_t>(first + i * step) * p.record_bytes;
        for (int b = lane * 128; b < p.record_bytes; b += 32 * 128)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(rec + b));
    }
    mv::wait_for_prior_grid();
    mv::allow_next_grid();

    auto issue = [&](int i) {
        if (i < mine) {
            const uint8_t* rec = base + static_cast<int64_t>(first + i * step) * p.record_bytes;
            const uint32_t dst = ring + (i % kStages) * p.record_bytes;
            for (int b = lane * 16; b < p.record_bytes; b += 32 * 16) cp_async_16(dst + b, rec + b);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages; ++i) issue(i);

    const T* rows[NB];
    bool live[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int token = token0 + 8 * b + g;
        live[b] = token < p.m;
        rows[b] = static_cast<const T*>(p.x) + (live[b] ? token : 0) * p.x_stride;
    }

    float acc[4][NB][4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[r][b][e] = 0.0f;

    for (int i = 0; i < mine; ++i) {
        const int k0 = (first + i * step) * kChunk;
        uint32_t x[4][NB][A::kPlanes][A::kRegs];
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int b = 0; b < NB; ++b)
                load_run<XT>(rows[b], k0 + 32 * h + 8 * t, live[b] ? p.k : 0, p.x_runs, x[h][b]);
        cp_async_wait<kStages - 1>();
        __syncwarp();
        const uint32_t rec = ring + (i % kStages) * p.record_bytes;
        const uint32_t scales = rec + kCodeBytes + g * 16;
        const uint32_t zeros = rec + kCodeBytes + kGroups * 128 + g * 8;
#pragma unroll
        for (int rp = 0; rp < 2; ++rp) {  // 32 rows at a time
            if constexpr (XT == kI8) {
                int c[2][NB][4], sum[NB][4];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    if (h % kGroupRuns == 0) {
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int e = 0; e < 4; ++e) c[0][b][e] = c[1][b][e] = sum[b][e] = 0;
                    }
                    const uint4 w = lds128(rec + ((h * 2 + rp) * 32 + lane) * 16);
                    // A nibble (code - 8 in two's complement) in a byte's high half is 16 (code - 8).
                    const uint32_t a0[4] = {(w.x << 4) & 0xf0f0f0f0u, w.x & 0xf0f0f0f0u, (w.y << 4) & 0xf0f0f0f0u,
                                            w.y & 0xf0f0f0f0u};
                    const uint32_t a1[4] = {(w.z << 4) & 0xf0f0f0f0u, w.z & 0xf0f0f0f0u, (w.w << 4) & 0xf0f0f0f0u,
                                            w.w & 0xf0f0f0f0u};
                    const uint32_t ones[4] = {0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u};
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        mma_s8(c[0][b], a0, x[h][b][0][0], x[h][b][0][1]);
                        mma_s8(c[1][b], a1, x[h][b][0][0], x[h][b][0][1]);
                        if (p.has_zeros) mma_s8(sum[b], ones, x[h][b][0][0], x[h][b][0][1]);
                    }
                    if (h % kGroupRuns == kGroupRuns - 1) {
                        const int group = h / kGroupRuns;
                        const uint2 s = lds64(scales + group * 128 + rp * 8);
                        uint32_t z = 0;
                        if (p.has_zeros) z = lds32(zeros + group * 64 + rp * 4);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const float2 sc = scale_pair(q ? s.y : s.x, p.scale_bf16);
                            const int zl = 16 * static_cast<int8_t>(z >> (16 * q));
                            const int zh = 16 * static_cast<int8_t>(z >> (16 * q + 8));
                            const float lo = sc.x * 0.0625f, hi = sc.y * 0.0625f;
#pragma unroll
                            for (int b = 0; b < NB; ++b) {
                                // Below 2^24 (16 * 15 * 128 * 128): exact as floats.
                                float(&a)[4] = acc[2 * rp + q][b];
                                a[0] = fmaf(lo, static_cast<float>(c[q][b][0] - zl * sum[b][0]), a[0]);
                                a[1] = fmaf(lo, static_cast<float>(c[q][b][1] - zl * sum[b][1]), a[1]);
                                a[2] = fmaf(hi, static_cast<float>(c[q][b][2] - zh * sum[b][2]), a[2]);
                                a[3] = fmaf(hi, static_cast<float>(c[q][b][3] - zh * sum[b][3]), a[3]);
                            }
                        }
                    }
                }
            } else {
                float c[2][NB][4];
                uint32_t zl[2], zh[2];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    if (h % kGroupRuns == 0) {
                        uint32_t z = 0;
                        if (p.has_zeros) z = lds32(zeros + (h / kGroupRuns) * 64 + rp * 4);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            zl[q] = A::zero_low(8 + static_cast<int8_t>(z >> (16 * q)));
                            zh[q] = A::zero_high(8 + static_cast<int8_t>(z >> (16 * q + 8)));
#pragma unroll
                            for (int b = 0; b < NB; ++b)
#pragma unroll
                                for (int e = 0; e < 4; ++e) c[q][b][e] = 0.0f;
                        }
                    }
                    const uint4 w = lds128(rec + ((h * 2 + rp) * 32 + lane) * 16);
                    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t a[4];
                        A::weights(words[j], zl[j >> 1], zh[j >> 1], a);
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int pl = 0; pl < A::kPlanes; ++pl)
                                A::mma(c[j >> 1][b], a, x[h][b][pl][2 * (j & 1)], x[h][b][pl][2 * (j & 1) + 1]);
                    }
                    if (h % kGroupRuns == kGroupRuns - 1) {
                        const uint2 s = lds64(scales + (h / kGroupRuns) * 128 + rp * 8);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            float2 sc = scale_pair(q ? s.y : s.x, p.scale_bf16);
                            sc.x *= A::kScale, sc.y *= A::kScale;
#pragma unroll
                            for (int b = 0; b < NB; ++b) {
                                float(&a)[4] = acc[2 * rp + q][b];
                                a[0] = fmaf(sc.x, c[q][b][0], a[0]);
                                a[1] = fmaf(sc.x, c[q][b][1], a[1]);
                                a[2] = fmaf(sc.y, c[q][b][2], a[2]);
                                a[3] = fmaf(sc.y, c[q][b][3], a[3]);
                            }
                        }
                    }
                }
            }
        }
        __syncwarp();  // every lane has read the record before its stage is filled again
        issue(i + kStages);
    }
    cp_async_wait<0>();
    __syncwarp();

    // Partial sums [token][row] of each warp over its own ring.
    float* part = reinterpret_cast<float*>(smem + warp * kStages * p.record_bytes);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            float* at = part + (8 * b + 2 * t) * kPartStride + 16 * r + g;
            at[0] = acc[r][b][0];
            at[kPartStride] = acc[r][b][1];
            at[8] = acc[r][b][2];
            at[kPartStride + 8] = acc[r][b][3];
        }
    if (p.cluster > 1) cluster_barrier();
    else __syncthreads();

    const int tokens = min(8 * NB, p.m - token0);
    const int64_t row0 = tile * kTileRows;
    for (int e = rank * kThreads + threadIdx.x; e < tokens * kTileRows; e += kThreads * p.cluster) {
        const int token = e / kTileRows, row = e % kTileRows;
        if (row0 + row >= p.n) continue;
        float v = 0.0f;
        for (int c = 0; c < p.cluster; ++c)
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const uint32_t at = mv::smem_addr(smem) + w * kStages * p.record_bytes + (token * kPartStride + row) * 4;
                v += p.cluster > 1 ? ld_cluster(at, c) : __uint_as_float(lds32(at));
            }
        const int64_t out_row = token0 + token;
        if (p.x_scale) v *= p.x_scale[out_row];
        if (p.bias) v += load_as_float(p.bias, row0 + row, p.out_dtype);
        if (p.residual) v += load_as_float(p.residual, out_row * p.residual_stride + row0 + row, p.out_dtype);
        store_from_float(p.out, out_row * p.out_stride + row0 + row, p.out_dtype, v);
    }
    if (p.cluster > 1) cluster_barrier();  // no CTA leaves while another reads its shared memory
}

// W written out, rounded once: a warp per record, a lane's word pairs being
// eight consecutive columns of a row. Bound by the output's bytes.
template <typename T>
__global__ void __launch_bounds__(256)
w4_dequantize_kernel(const uint8_t* records, int64_t total, int chunks, int record_bytes, int group, int has_zeros,
                     int scale_bf16, int n, int k, T* out, int64_t out_stride, int runs) {
    mv::wait_for_prior_grid();
    mv::allow_next_grid();
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (id >= total) return;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t tile = id / chunks;
    const int k0 = static_cast<int>(id - tile * chunks) * kChunk;
    const uint8_t* rec = records + id * record_bytes;
    const int group_runs = group / 32, groups = kChunk / group;
    for (int h = 0; h < 4; ++h) {
        const int gi = h / group_runs;
        const int c0 = k0 + 32 * h + 8 * t;
#pragma unroll
        for (int rp = 0; rp < 2; ++rp) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(rec) + (h * 2 + rp) * 32 + lane);
            const uint2 s = __ldg(reinterpret_cast<const uint2*>(rec + kCodeBytes + gi * 128 + g * 16 + rp * 8));
            uint32_t z = 0;
            if (has_zeros) z = __ldg(reinterpret_cast<const uint32_t*>(rec + kCodeBytes + groups * 128 + gi * 64 + g * 8 + rp * 4));
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const float2 sc = scale_pair(q ? s.y : s.x, scale_bf16);
                const uint32_t w0 = q ? w.z : w.x, w1 = q ? w.w : w.y;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int64_t row = tile * kTileRows + 32 * rp + 16 * q + 8 * half + g;
                    if (row >= n) continue;
                    const float scale = half ? sc.y : sc.x;
                    const int zero = static_cast<int8_t>(z >> (16 * q + 8 * half));
                    __align__(16) T v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t word = i < 4 ? w0 : w1;
                        const int s_at = i & 3, byte = s_at == 1 ? 2 : s_at == 2 ? 1 : s_at;
                        const int code = static_cast<int>(((word >> (8 * byte + 4 * half)) & 15u) ^ 8u) - 8;
                        v[i] = from_float<T>(static_cast<float>(code - zero) * scale);
                    }
                    T* dst = out + row * out_stride + c0;
                    if (runs && c0 + 8 <= k) {
#pragma unroll
                        for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
                            reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(v)[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (c0 + i < k) dst[i] = v[i];
                    }
                }
            }
        }
    }
}

}  // namespace mvq
