// Products with 4-bit weights: y = (x W^T) * x_scale + bias + residual for a
// few rows of x (mma.sync tiles, split over the columns of W), and W itself
// written out. The weight's record layout is in include/mvquant.h.
//
// Mathematics. W[n, k] = (code - zero) * scale per row n and group of k. The
// kernel never forms the scaled weight: within a group it sums x * (code -
// zero) -- code - zero is a small integer, exact in bf16, fp16 and int8 -- and
// then adds scale * sum to the row's fp32 accumulator. So products are exact and
// weights are never rounded; what is rounded before the result are the fp32
// additions (within a group, of scaled groups, of the columns' parts) and the
// product with each group's scale.
//
// What bounds it: the codes are read once, half a byte per weight, and each
// weight costs about 1.4 instructions to become a bf16 (shift, mask-xor,
// subtract on pairs), 1.1 an fp16, 0.4 an int8, against about 2.8 issue slots
// per weight at the copy bandwidth. Yet no pipe is at its limit over a launch (one
// row through 3584 -> 28672 in bf16: ALU 43 %, issue slots 48 %, DRAM 32 %): what
// is left is the latency of the chain from a record's words over their conversion
// to the multiplication, which three warps per scheduler do not hide. The records
// hold the codes in the order of the A operand of mma.sync (16 weight rows x 16 or
// 32 columns), so a lane's 16 bytes become four operand registers by masks and
// shifts alone, and both the 16-bit and the 8-bit instruction read the same records.
#pragma once

#include <cuda_fp8.h>

#include <type_traits>

#include "mv_device.cuh"

namespace mvq {

using mv::from_float;
using mv::to_float;

constexpr int kTileRows = 64;
constexpr int kChunk = 128;
constexpr int kCodeBytes = kTileRows * kChunk / 2;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTokens = 8;  // per pass over the records: the columns of one mma.sync tile
// Row stride of the partial sums [token][64 weight rows] in shared memory, in
// floats: 68 keeps the eight rows and four token pairs that a warp stores at
// once in different banks.
constexpr int kPartStride = 68;

__host__ __device__ constexpr int record_size(int group, bool zeros) { return kCodeBytes + kChunk / group * (zeros ? 192 : 128); }

struct LinearParams {
    const void* x;
    int64_t x_stride;
    const float* x_scale;
    const uint8_t* records;
    int n, k, m;
    int chunks;        // ceil(k / 128)
    int tiles;         // ceil(n / 64)
    int scale_bf16;
    int x_dtype;
    int x_runs;        // x may be read 8 elements at a time: aligned rows, k a multiple of 8
    int x_units;       // x's rows may be copied by TMA
    int cluster;       // CTAs that share a tile's columns, each with a run of chunks
    int ksplit;        // warps of a CTA that share a tile's columns: its kWarps / ksplit tiles
    int stages;        // records in flight per warp: 2 or 3
    int x_chunks;      // chunks of x staged at a time (a multiple of ksplit)
    int ring_bytes;    // shared memory of a warp: its records, later its partial sums
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

// Operand arithmetic of each kind of product: kPlanes operand numbers make up
// one x, kRunBytes hold eight of them for the B operand, and weights() makes
// the A registers of a word of codes (rows g and g + 8 of 16 rows, four columns).
template <int KIND>
struct Act;

struct ActHalf {
    static constexpr int kPlanes = 1;
    static constexpr int kRunBytes = 16;
};

template <>
struct Act<kBF16> : ActHalf {
    // (code - zero) / 2^11 from 128 + code (bf16 numbers from 128 to 255 have a
    // step of one): (128 + code) / 2^11 - (128 + zero) / 2^11, exact. The power
    // of two (kScale) comes back after the sum; with it a group's sum of 128 products of
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
    // c = a b, without a register to be cleared first.
    __device__ __forceinline__ static void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
            "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    }
};

// fp32 x as the exact sum of three bf16 numbers (8 + 8 + 8 bits of its 24).
template <>
struct Act<kF32> : Act<kBF16> {
    static constexpr int kPlanes = 3;
};

template <>
struct Act<kF16> : ActHalf {
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
    __device__ __forceinline__ static void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
            "{%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    }
};

template <>
struct Act<kI8> {
    static constexpr int kPlanes = 1;
    static constexpr int kRunBytes = 8;
    // A nibble (code - 8 in two's complement) in a byte's high half is 16 (code - 8).
    static constexpr float kScale = 1.0f / 16.0f;
};

// The four columns of a word as int8 (code - zero), rows g and g + 8. Bytes 128 +
// code minus bytes zero borrow nothing from one another; then 128 is taken off.
__device__ __forceinline__ uint32_t bytes_minus(uint32_t w, uint32_t zero4) {
    return (and_xor(w, 0x0f0f0f0fu, 0x88888888u) - zero4) ^ 0x80808080u;
}

__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, "
        "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four e4m3 numbers as fp16, exactly.
__device__ __forceinline__ uint2 e4m3_to_half(uint32_t v) {
    const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v & 0xffffu), __NV_E4M3);
    const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v >> 16), __NV_E4M3);
    return make_uint2(lo.x | (static_cast<uint32_t>(lo.y) << 16), hi.x | (static_cast<uint32_t>(hi.y) << 16));
}

// Eight consecutive elements of a row of x, columns k..k+7 (zeros at and beyond
// `limit`), as operand numbers of kind KIND: r[plane][...] holds them in order,
// two to a register (int8: four). e4m3 numbers are exact in fp16.
template <int KIND>
__device__ __forceinline__ void load_run(const LinearParams& p, const void* row, int k, int limit,
                                         uint32_t (&r)[Act<KIND>::kPlanes][Act<KIND>::kRunBytes / 4]) {
    if constexpr (KIND == kF32) {
        const float* e = static_cast<const float*>(row);
        float f[8];
        if (p.x_runs && k < limit) {
            const float4 lo = *reinterpret_cast<const float4*>(e + k);
            const float4 hi = *reinterpret_cast<const float4*>(e + k + 4);
            f[0] = lo.x, f[1] = lo.y, f[2] = lo.z, f[3] = lo.w, f[4] = hi.x, f[5] = hi.y, f[6] = hi.z, f[7] = hi.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = k + i < limit ? e[k + i] : 0.0f;
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
        for (int pl = 0; pl < 3; ++pl)
#pragma unroll
            for (int i = 0; i < 4; ++i) r[pl][i] = (b[pl][2 * i] >> 16) | b[pl][2 * i + 1];
    } else if (KIND != kI8 && p.x_dtype != kE4M3) {
        uint4 v = make_uint4(0, 0, 0, 0);
        const uint16_t* e = static_cast<const uint16_t*>(row);
        if (p.x_runs) {
            if (k < limit) v = *reinterpret_cast<const uint4*>(e + k);
        } else {
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = k + i < limit ? e[k + i] : 0u;
            v = make_uint4(h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16));
        }
        r[0][0] = v.x, r[0][1] = v.y;
        if constexpr (Act<KIND>::kRunBytes == 16) r[0][2] = v.z, r[0][3] = v.w;
    } else {
        uint2 v = make_uint2(0, 0);
        const uint8_t* e = static_cast<const uint8_t*>(row);
        if (p.x_runs) {
            if (k < limit) v = *reinterpret_cast<const uint2*>(e + k);
        } else {
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = k + i < limit ? e[k + i] : 0u;
            v = make_uint2(h[0] | (h[1] << 8) | (h[2] << 16) | (h[3] << 24),
                           h[4] | (h[5] << 8) | (h[6] << 16) | (h[7] << 24));
        }
        if constexpr (KIND == kI8) {
            r[0][0] = v.x, r[0][1] = v.y;
        } else {
            const uint2 lo = e4m3_to_half(v.x), hi = e4m3_to_half(v.y);
            r[0][0] = lo.x, r[0][1] = lo.y, r[0][2] = hi.x, r[0][3] = hi.y;
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

// A CTA's four warps take 4 / ksplit tiles of 64 weight rows and, with the other
// CTAs of their cluster, up to eight tokens. The columns' chunks go to the
// cluster's CTAs as runs, within a CTA to the tile's ksplit warps in turn. x's
// part of the run is staged in shared memory once, as operand numbers; each warp
// streams its records through a ring of its own (cp.async and no barrier: a warp
// reads what its own lanes copied) and sums all 64 rows for all tokens; the
// partial sums meet in (distributed) shared memory and are added in a fixed order.
template <int KIND, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kThreads, 4) w4_linear_kernel(const LinearParams p) {
    using A = Act<KIND>;
    constexpr int kGroupRuns = GROUP / 32;    // 32-column runs per group
    constexpr int kGroups = kChunk / GROUP;   // groups per chunk
    constexpr int kRecord = record_size(GROUP, ZEROS);
    constexpr int kPlanes = A::kPlanes, kRunBytes = A::kRunBytes;
    extern __shared__ __align__(128) uint8_t smem[];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int rank = p.cluster > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int64_t tile0 = static_cast<int64_t>(blockIdx.x) / p.cluster * (kWarps / p.ksplit);
    const int64_t tile = tile0 + warp / p.ksplit;
    const int token0 = blockIdx.y * kTokens;
    const int tokens = min(kTokens, p.m - token0);
    // This CTA's run of chunks, and this warp's among them: begin + kpart, + ksplit, ...
    const int begin = static_cast<int>(static_cast<int64_t>(p.chunks) * rank / p.cluster);
    const int end = static_cast<int>(static_cast<int64_t>(p.chunks) * (rank + 1) / p.cluster);
    const int kpart = warp % p.ksplit;
    const int mine = tile < p.tiles && end - begin > kpart ? (end - begin - kpart + p.ksplit - 1) / p.ksplit : 0;
    const uint8_t* base = p.records + (tile * p.chunks + begin + kpart) * static_cast<int64_t>(kRecord);
    const int64_t base_step = static_cast<int64_t>(p.ksplit) * kRecord;
    const uint32_t ring = mv::smem_addr(smem) + warp * p.ring_bytes;
    uint8_t* const xs = smem + kWarps * p.ring_bytes;

    // The weights' first records come into L2 while the grid before drains. Its
    // writes are not visible yet, so nothing is read.
    for (int i = 0; i < p.stages && i < mine; ++i)
        for (int b = lane * 128; b < kRecord; b += 32 * 128)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(base + i * base_step + b));
    mv::wait_for_prior_grid();
    mv::allow_next_grid();

    int fill = 0;  // stage that the next record goes to
    const auto issue = [&](int i) {
        if (i < mine) {
            const uint8_t* rec = base + i * base_step + lane * 16;
            const uint32_t dst = ring + fill * kRecord + lane * 16;
#pragma unroll
            for (int b = 0; b < kRecord; b += 512)
                if (b + 512 <= kRecord || b + lane * 16 < kRecord) cp_async_16(dst + b, rec + b);
        }
        cp_async_commit();
        fill = fill + 1 == p.stages ? 0 : fill + 1;
    };
    for (int i = 0; i < p.stages; ++i) issue(i);

    // x: [chunk][h][plane][t][token] two quads, the columns 16 e + 4 t of h, for x_chunks chunks from `from`.
    const int plane_bytes = 4 * tokens * kRunBytes;
    const int x_size = p.x_dtype == kF32 ? 4 : p.x_dtype >= kI8 ? 1 : 2;
    const auto stage = [&](auto count, int from, int runs) {
        constexpr int kTogether = decltype(count)::value;
        for (int first_token = 0; first_token < tokens; first_token += kTogether) {
            for (int run = threadIdx.x; run < runs; run += kThreads) {
                uint32_t r[kTogether][kPlanes][kRunBytes / 4];
#pragma unroll
                for (int i = 0; i < kTogether; ++i) {
                    const int token = min(first_token + i, tokens - 1);
                    const uint8_t* row = static_cast<const uint8_t*>(p.x) + (token0 + token) * p.x_stride * x_size;
                    load_run<KIND>(p, row, (begin + from) * kChunk + run * 8, p.k, r[i]);
                }
                // The run's two quads go to lanes t = 2 (run & 1) and the next, as their columns 16 e + 4 t..
#pragma unroll
                for (int i = 0; i < kTogether; ++i) {
                    const int token = min(first_token + i, tokens - 1);
                    uint8_t* dst = xs + (run >> 2) * (kPlanes * plane_bytes) +
                                   ((run & 1) * 2 * tokens + token) * kRunBytes + (run >> 1 & 1) * (kRunBytes / 2);
#pragma unroll
                    for (int pl = 0; pl < kPlanes; ++pl) {
                        uint8_t* d = dst + pl * plane_bytes;
                        if constexpr (KIND == kI8) {  // the codes' byte order: 0, 2, 1, 3
                            *reinterpret_cast<uint32_t*>(d) = __byte_perm(r[i][0][0], 0, 0x3120);
                            *reinterpret_cast<uint32_t*>(d + tokens * kRunBytes) = __byte_perm(r[i][0][1], 0, 0x3120);
                        } else {
                            *reinterpret_cast<uint2*>(d) = make_uint2(r[i][pl][0], r[i][pl][1]);
                            *reinterpret_cast<uint2*>(d + tokens * kRunBytes) = make_uint2(r[i][pl][2], r[i][pl][3]);
                        }
                    }
                }
            }
        }
    };
    const auto stage_x = [&](int from) {
        const int runs = min(p.x_chunks, end - begin - from) * 16;  // runs of eight of a token: chunk, h, t
        // The loads of all tokens (of four, for fp32) are under way before the first is stored.
        if (tokens == 1) stage(std::integral_constant<int, 1>(), from, runs);
        else if (tokens == 2) stage(std::integral_constant<int, 2>(), from, runs);
        else if (tokens <= 4 || kPlanes == 3) stage(std::integral_constant<int, 4>(), from, runs);
        else stage(std::integral_constant<int, 8>(), from, runs);
    };

    float acc[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][e] = 0.0f;

    // A lane of a token beyond the last reads the last: its column of the product is never stored.
    const uint32_t x_lane = mv::smem_addr(xs) + (t * tokens + min(g, tokens - 1)) * kRunBytes;
    int drain = 0;  // stage of the record that is read next
    for (int from = 0; from < end - begin; from += p.x_chunks) {
    if (from) __syncthreads();  // every warp is done with the chunks of x before
    stage_x(from);
    __syncthreads();
    const int last = min(mine, (from + p.x_chunks) / p.ksplit);
    for (int i = from / p.ksplit; i < last; ++i) {
        if (p.stages == 2) cp_async_wait<1>();
        else cp_async_wait<2>();
        __syncwarp();
        const uint32_t rec = ring + drain * kRecord;
        drain = drain + 1 == p.stages ? 0 : drain + 1;
        const uint32_t scales = rec + kCodeBytes + g * 16;
        const uint32_t zeros = rec + kCodeBytes + kGroups * 128 + g * 8;
        const uint32_t x_chunk = x_lane + (i * p.ksplit + kpart - from) * (4 * kPlanes * plane_bytes);
#pragma unroll
        for (int rp = 0; rp < 2; ++rp) {  // 32 rows at a time
            if constexpr (KIND == kI8) {
                // Sums start at 1.5 2^23 as a float's bits: their float value is then one subtraction away,
                // as they stay below 2^22 (16 * 8 * 128 * 128, or 15 * 128 * 128 with zero points).
                constexpr int kBias = 0x4b400000;
                int c[2][4];
                uint32_t zl[2], zh[2];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    if (h % kGroupRuns == 0) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) c[0][e] = c[1][e] = kBias;
                        if constexpr (ZEROS) {
                            // zero - 8 as a byte, plus 8, in all four bytes of an operand.
                            const uint32_t z = lds32(zeros + (h / kGroupRuns) * 64 + rp * 4) ^ 0x88888888u;
                            const uint32_t u = (z & 0x0f0f0f0fu);
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                zl[q] = __byte_perm(u, 0, q ? 0x2222 : 0x0000);
                                zh[q] = __byte_perm(u, 0, q ? 0x3333 : 0x1111);
                            }
                        }
                    }
                    const uint4 w = lds128(rec + ((h * 2 + rp) * 32 + lane) * 16);
                    uint32_t a0[4], a1[4];
                    if constexpr (ZEROS) {
                        a0[0] = bytes_minus(w.x, zl[0]), a0[1] = bytes_minus(w.x >> 4, zh[0]);
                        a0[2] = bytes_minus(w.y, zl[0]), a0[3] = bytes_minus(w.y >> 4, zh[0]);
                        a1[0] = bytes_minus(w.z, zl[1]), a1[1] = bytes_minus(w.z >> 4, zh[1]);
                        a1[2] = bytes_minus(w.w, zl[1]), a1[3] = bytes_minus(w.w >> 4, zh[1]);
                    } else {
                        a0[0] = (w.x << 4) & 0xf0f0f0f0u, a0[1] = w.x & 0xf0f0f0f0u;
                        a0[2] = (w.y << 4) & 0xf0f0f0f0u, a0[3] = w.y & 0xf0f0f0f0u;
                        a1[0] = (w.z << 4) & 0xf0f0f0f0u, a1[1] = w.z & 0xf0f0f0f0u;
                        a1[2] = (w.w << 4) & 0xf0f0f0f0u, a1[3] = w.w & 0xf0f0f0f0u;
                    }
                    const uint2 xv = lds64(x_chunk + h * plane_bytes);
                    mma_s8(c[0], a0, xv.x, xv.y);
                    mma_s8(c[1], a1, xv.x, xv.y);
                    if (h % kGroupRuns == kGroupRuns - 1) {
                        const uint2 s = lds64(scales + (h / kGroupRuns) * 128 + rp * 8);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const float2 sc = scale_pair(q ? s.y : s.x, p.scale_bf16);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                acc[2 * rp + q][e] = fmaf(e < 2 ? sc.x : sc.y, __int_as_float(c[q][e]) - 12582912.0f,
                                                          acc[2 * rp + q][e]);
                        }
                    }
                }
            } else {
                float c[2][4];
                uint32_t zl[2], zh[2];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    if (h % kGroupRuns == 0) {
                        uint32_t z = 0;
                        if (ZEROS) z = lds32(zeros + (h / kGroupRuns) * 64 + rp * 4);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            zl[q] = A::zero_low(8 + static_cast<int8_t>(z >> (16 * q)));
                            zh[q] = A::zero_high(8 + static_cast<int8_t>(z >> (16 * q + 8)));
                        }
                    }
                    uint4 xv[kPlanes];
#pragma unroll
                    for (int pl = 0; pl < kPlanes; ++pl) xv[pl] = lds128(x_chunk + (h * kPlanes + pl) * plane_bytes);
                    const uint4 w = lds128(rec + ((h * 2 + rp) * 32 + lane) * 16);
                    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t a[4];
                        A::weights(words[j], zl[j >> 1], zh[j >> 1], a);
#pragma unroll
                        for (int pl = 0; pl < kPlanes; ++pl) {
                            const uint32_t b0 = j & 1 ? xv[pl].z : xv[pl].x, b1 = j & 1 ? xv[pl].w : xv[pl].y;
                            if (h % kGroupRuns == 0 && (j & 1) == 0 && pl == 0) A::mma_first(c[j >> 1], a, b0, b1);
                            else A::mma(c[j >> 1], a, b0, b1);
                        }
                    }
                    if (h % kGroupRuns == kGroupRuns - 1) {
                        const uint2 s = lds64(scales + (h / kGroupRuns) * 128 + rp * 8);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const float2 sc = scale_pair(q ? s.y : s.x, p.scale_bf16);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                acc[2 * rp + q][e] = fmaf(e < 2 ? sc.x : sc.y, c[q][e], acc[2 * rp + q][e]);
                        }
                    }
                }
            }
        }
        __syncwarp();  // every lane has read the record before its stage is filled again
        issue(i + p.stages);
    }
    }
    cp_async_wait<0>();
    __syncwarp();

    // Partial sums [token][row] of each warp over its own ring.
    {
        float* part = reinterpret_cast<float*>(smem + warp * p.ring_bytes);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float* at = part + 2 * t * kPartStride + 16 * r + g;
            at[0] = acc[r][0];
            at[kPartStride] = acc[r][1];
            at[8] = acc[r][2];
            at[kPartStride + 8] = acc[r][3];
        }
    }
    __syncthreads();
    const int tiles_here = kWarps / p.ksplit;
    const int outputs = tokens * tiles_here * kTileRows;
    const auto own_sum = [&](int e, uint32_t* at) {  // of this CTA's ksplit warps
        const int token = e / (tiles_here * kTileRows), row = e % (tiles_here * kTileRows);
        *at = mv::smem_addr(smem) + row / kTileRows * p.ksplit * p.ring_bytes +
              (token * kPartStride + row % kTileRows) * 4;
        float v = __uint_as_float(lds32(*at));
        for (int w = 1; w < p.ksplit; ++w) v += __uint_as_float(lds32(*at + w * p.ring_bytes));
        return v;
    };
    if (p.cluster > 1) {
        if (p.ksplit > 1)
            for (int e = threadIdx.x; e < outputs; e += kThreads) {
                uint32_t at;
                const float v = own_sum(e, &at);
                asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
            }
        cluster_barrier();
    }
    const int64_t row0 = tile0 * kTileRows;
    for (int e = rank * kThreads + threadIdx.x; e < outputs; e += kThreads * p.cluster) {
        const int token = e / (tiles_here * kTileRows), row = e % (tiles_here * kTileRows);
        if (row0 + row >= p.n) continue;
        float v = 0.0f;
        if (p.cluster > 1) {
            const uint32_t at = mv::smem_addr(smem) + row / kTileRows * p.ksplit * p.ring_bytes +
                                (token * kPartStride + row % kTileRows) * 4;
            for (int c = 0; c < p.cluster; ++c) v += ld_cluster(at, c);
        } else {
            uint32_t at;
            v = own_sum(e, &at);
        }
        const int64_t out_row = token0 + token;
        v *= ZEROS && KIND == kI8 ? 1.0f : A::kScale;
        if (p.x_scale) v *= p.x_scale[out_row];
        if (p.bias) v += load_as_float(p.bias, row0 + row, p.out_dtype);
        if (p.residual) v += load_as_float(p.residual, out_row * p.residual_stride + row0 + row, p.out_dtype);
        store_from_float(p.out, out_row * p.out_stride + row0 + row, p.out_dtype, v);
    }
    if (p.cluster > 1) cluster_barrier();  // no CTA leaves while another reads its shared memory
}

// W written out, rounded once: a warp per 32 columns of a record, the smallest
// piece that holds whole words (a record each took a small weight 5.9 us instead of
// 2.3 for 896 x 1152, for one warp's chain of steps, and 3584 x 28672 45.0 instead of
// 40.5). Bound by the output's bytes.
// A code's distance from its zero point is exact in 16 bits, and its product
// with a scale has at most 4 + 11 bits, so that a 16-bit product with a scale of
// the output's type (`same`) rounds exactly as the fp32 product does. The distance
// is taken as it is: with the products' power of two (Act<kBF16>) a scale from
// 2^117 on would have to become an infinity.
struct DistanceBF16 {
    __device__ __forceinline__ static uint32_t zero_low(int z) { return (0xc300u + z) * 0x10001u; }  // -(128 + z)
    __device__ __forceinline__ static uint32_t zero_high(int z) { return zero_low(z); }
    __device__ __forceinline__ static uint32_t distance(uint32_t w, uint32_t z) {
        const uint32_t v = and_xor(w, 0x000f000fu, 0x43084308u);  // 128 + code
        const __nv_bfloat162 d =
            __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&z));
        return *reinterpret_cast<const uint32_t*>(&d);
    }
    __device__ __forceinline__ static void weights(uint32_t w, uint32_t zl, uint32_t zh, uint32_t (&a)[4]) {
        a[0] = distance(w, zl);
        a[1] = distance(w >> 4, zh);
        a[2] = distance(w >> 8, zl);
        a[3] = distance(w >> 12, zh);
    }
};
template <typename T>
struct PairOf;
template <>
struct PairOf<__half> {
    using Kind = Act<kF16>;
    using Pair = __half2;
};
template <>
struct PairOf<__nv_bfloat16> {
    using Kind = DistanceBF16;
    using Pair = __nv_bfloat162;
};
template <>
struct PairOf<float> : PairOf<__nv_bfloat16> {};

constexpr int kDequantizeWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kDequantizeWarps * 32)
w4_dequantize_kernel(const uint8_t* records, int64_t total, int chunks, int record_bytes, int group, int has_zeros,
                     int scale_bf16, int n, int k, T* out, int64_t out_stride, int runs) {
    using Kind = typename PairOf<T>::Kind;
    using Pair = typename PairOf<T>::Pair;
    constexpr bool kBf16 = std::is_same<Kind, DistanceBF16>::value;
    mv::wait_for_prior_grid();
    mv::allow_next_grid();
    const int64_t piece = static_cast<int64_t>(blockIdx.x) * kDequantizeWarps + (threadIdx.x >> 5);
    const int64_t id = piece >> 2;
    const int h = static_cast<int>(piece & 3);
    if (id >= total) return;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t tile = id / chunks;
    const int k0 = static_cast<int>(id - tile * chunks) * kChunk;
    const uint8_t* rec = records + id * record_bytes;
    const int group_runs = group / 32, groups = kChunk / group;
    const bool same = sizeof(T) == 2 && (scale_bf16 != 0) == kBf16;
    // Rows that are not aligned go out through shared memory, so that a warp
    // stores 32 columns of one row at a time; written as 32-bit words.
    __shared__ __align__(16) T rows_out[sizeof(T) == 2 ? kDequantizeWarps : 1][sizeof(T) == 2 ? 64 * 34 : 1];
    // Plain loads: the kernel before may have written the records while this one was launched, which the read-only
    // path does not allow for.
    uint4 codes[2];
#pragma unroll
    for (int rp = 0; rp < 2; ++rp) codes[rp] = reinterpret_cast<const uint4*>(rec)[(h * 2 + rp) * 32 + lane];
    {
        const int gi = h / group_runs;
        // 16 bits: two lanes trade words, so that each holds eight columns in a row,
        // 16 bytes: the even one both quads of the first half of h, the odd one of the
        // second. fp32: a quad is 16 bytes as it is.
        constexpr bool kTrade = sizeof(T) == 2;
        const int c0 = k0 + 32 * h + (kTrade ? 16 * (t & 1) + 4 * (t & 2) : 4 * t);
#pragma unroll
        for (int rp = 0; rp < 2; ++rp) {
            uint4 w = codes[rp];
            if constexpr (kTrade) {
                const uint32_t got0 = __shfl_xor_sync(0xffffffffu, t & 1 ? w.x : w.y, 1);
                const uint32_t got1 = __shfl_xor_sync(0xffffffffu, t & 1 ? w.z : w.w, 1);
                if (t & 1) w.x = got0, w.z = got1;
                else w.y = got0, w.w = got1;
            }
            const uint2 s = *reinterpret_cast<const uint2*>(rec + kCodeBytes + gi * 128 + g * 16 + rp * 8);
            uint32_t z = 0;
            if (has_zeros) z = *reinterpret_cast<const uint32_t*>(rec + kCodeBytes + groups * 128 + gi * 64 + g * 8 + rp * 4);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const uint32_t scales = q ? s.y : s.x;
                const uint32_t zl = Kind::zero_low(8 + static_cast<int8_t>(z >> (16 * q)));
                const uint32_t zh = Kind::zero_high(8 + static_cast<int8_t>(z >> (16 * q + 8)));
                uint32_t a[2][4];  // per quad: columns 0 1 of row g, of row g + 8, columns 2 3 of row g, of row g + 8
                Kind::weights(q ? w.z : w.x, zl, zh, a[0]);
                Kind::weights(q ? w.w : w.y, zl, zh, a[1]);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int64_t row = tile * kTileRows + 32 * rp + 16 * q + 8 * half + g;
                    if (runs && row >= n) continue;
                    float f[8];
                    uint32_t v[4];
                    if (same) {
                        const uint32_t bits = __byte_perm(scales, 0, half ? 0x3232 : 0x1010);
                        const Pair sc = *reinterpret_cast<const Pair*>(&bits);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            Pair d = *reinterpret_cast<const Pair*>(&a[i >> 1][half + 2 * (i & 1)]);
                            d = __hmul2(d, sc);
                            v[i] = *reinterpret_cast<const uint32_t*>(&d);
                        }
                    } else {
                        const float2 both = scale_pair(scales, scale_bf16);
                        const float scale = half ? both.y : both.x;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t pair = a[i >> 1][half + 2 * (i & 1)];
                            const float2 d = scale_pair(pair, kBf16);
                            f[2 * i] = d.x * scale, f[2 * i + 1] = d.y * scale;
                        }
                        if constexpr (sizeof(T) == 2) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[i] = mv::MmaOp<T>::pack(f[2 * i], f[2 * i + 1]);
                        }
                    }
                    T* dst = out + row * out_stride + c0;
                    if constexpr (sizeof(T) == 4) {
#pragma unroll
                        for (int quad = 0; quad < 2; ++quad) {
                            const int c = c0 + 16 * quad;
                            if (row >= n) break;
                            if (runs && c + 4 <= k) {
                                *reinterpret_cast<float4*>(dst + 16 * quad) =
                                    make_float4(f[4 * quad], f[4 * quad + 1], f[4 * quad + 2], f[4 * quad + 3]);
                            } else {
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    if (c + i < k) dst[16 * quad + i] = f[4 * quad + i];
                            }
                        }
                    } else if (runs && c0 + 8 <= k) {
                        *reinterpret_cast<uint4*>(dst) = make_uint4(v[0], v[1], v[2], v[3]);
                    } else if (runs) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const uint16_t bits = static_cast<uint16_t>(v[i >> 1] >> (16 * (i & 1)));
                            if (c0 + i < k) dst[i] = *reinterpret_cast<const T*>(&bits);
                        }
                    } else {
                        uint32_t* at = reinterpret_cast<uint32_t*>(
                            &rows_out[threadIdx.x >> 5][(32 * rp + 16 * q + 8 * half + g) * 34 + 16 * (t & 1) + 4 * (t & 2)]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) at[i] = v[i];
                    }
                }
            }
        }
        if constexpr (sizeof(T) == 2) {
            if (!runs) {
                __syncwarp();
                const int column = k0 + 32 * h + lane;
                T* dst = out + tile * kTileRows * out_stride + column;
                const int rows_here = min(kTileRows, static_cast<int>(n - tile * kTileRows));
                if (column < k)
                    for (int row = 0; row < rows_here; ++row) dst[row * out_stride] = rows_out[threadIdx.x >> 5][row * 34 + lane];
                __syncwarp();
            }
        }
    }
}

}  // namespace mvq
