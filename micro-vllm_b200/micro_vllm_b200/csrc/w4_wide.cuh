// Products with 4-bit weights for more tokens than a few: 128 weight rows by NT
// tokens per CTA on the 5th-generation tensor cores (tcgen05.mma).
//
//   D[128, NT] = A[128, group] . X[NT, group]^T    for each group of columns
//   acc[row, :] += scale[row, group] * D[row, :]
//
// A holds code - zero (small integers, exact in 16 bits or int8) in tensor
// memory: four warps turn the records' words into operand registers by masks,
// as the mma.sync kernel does, and tcgen05.st.16x256b (int8: 16x128b) puts a
// lane's registers, rows g and g + 8 and columns 16 e + 4 t + s, in place without
// passing shared memory. X lies in shared memory (K-major, 128-byte swizzle).
// Each group's D is its own accumulation, in one of two to eight TMEM buffers; other
// warps add it, scaled, to fp32 sums in registers, a thread per weight row.
//
// What bounds it: as in the mma.sync kernel the codes' conversion, about 22
// cycles per 256 weights and scheduler at the copy bandwidth, of which bf16
// takes 14 of the ALU; the tensor work does not show up to 128 tokens. Weights
// in TMEM leave shared memory to X alone (A there would be written and read at
// twice the bandwidth that is left).
//
// Warps: 0-7 convert, two sets of four taking chunks in turn (warp w fills lanes
// 32 (w % 4).. of A); then sets of four that drain 32 columns of D each; one that
// issues the MMAs; one that issues X's TMA loads. A wait that finds its barrier
// complete still costs some 200 cycles, as does a commit, so there is one barrier
// for all that a chunk's MMAs need and one for their end, and two sets convert so
// that one's waits hide behind the other. Every wait is bounded (2 s): one that
// gives up sets the device status, and the CTA's results are NaN.
#pragma once

#include "w4_linear.cuh"

namespace mvq {

constexpr int kWideRows = 128;
constexpr int kWidePartStride = 132;  // floats per token of the partial sums [token][128 rows]

template <int KIND, int NT, int GROUP, bool ZEROS>
struct WideShape {
    static constexpr int kGroups = kChunk / GROUP;
    static constexpr int kCols = NT < 32 ? NT : 32;        // columns of D that a set drains
    static constexpr int kSets = NT / kCols;
    static constexpr int kTurns = NT == 64 ? 2 : 1;        // groups of sets that take chunks in turn (NT 128 leaves no threads for it)
    static constexpr int kThreads = (8 + 4 * kSets * kTurns + 2) * 32;
    static constexpr int kCtas = NT <= 32 ? 2 : 1;         // per SM
    // Fourteen warps fall on the four schedulers as 4 4 3 3, so that two CTAs fit as
    // sixteen each would, at 64 registers. 32 tokens would spill for that.
    static constexpr int kBoundThreads = NT == 16 ? 512 : kThreads;
    static constexpr int kStages = NT == 64 ? 5 : 3;       // records in flight per converting warp
    static constexpr int kACols = KIND == kI8 ? 32 : 64;   // TMEM columns of a chunk of A
    static constexpr int kBuffers = NT <= 32 && KIND != kI8 ? 3 : 4;  // chunks of A and of X
    static constexpr int kTmemCols = NT <= 32 ? 256 : 512;
    // Buffers of D: those of two whole chunks where they fit, so that a chunk's arrival
    // says that its D is free; else two, each group waiting for its own (d_empty).
    static constexpr bool kWholeChunks = kBuffers * kACols + 2 * kGroups * NT <= kTmemCols;
    static constexpr int kDBuffers = kWholeChunks ? 2 * kGroups : 2;
    static_assert(kBuffers * kACols + kDBuffers * NT <= kTmemCols, "TMEM columns");
    static constexpr int kXBytes = NT * (KIND == kI8 ? 128 : 256);
    static constexpr int kStageBytes = kCodeBytes / 2 + (ZEROS ? kGroups * 64 : 0);
    static constexpr int kRings = 8 * kStages * kStageBytes;
    static constexpr int kRawBytes = KIND == kE4M3 ? NT * 128 : 0;  // a chunk of e4m3 rows, before it is fp16
    static constexpr int kUsed = kBuffers * kXBytes + kRings + 2 * kRawBytes;
    static constexpr int kPart = kTurns * NT * kWidePartStride * 4;
    static constexpr int kSmem = (kUsed > kPart ? kUsed : kPart) + 1024;
};

__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr) {
    return static_cast<uint64_t>((addr >> 4) & 0x3FFF) | (static_cast<uint64_t>(1) << 16) |
           (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
           (static_cast<uint64_t>(2) << 61);
}

__device__ __forceinline__ uint32_t elect_one() {
    uint32_t leader;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(leader));
    return leader;
}

// D fp32 (1) or s32 (2); A and B fp16 (0), bf16 (1) or s8 (1); both K-major.
template <int KIND, int NT>
__host__ __device__ constexpr uint32_t wide_idesc() {
    constexpr uint32_t kHalf = KIND == kF16 || KIND == kE4M3 ? 0u : 1u;
    return ((KIND == kI8 ? 2u : 1u) << 4) | (kHalf << 7) | (kHalf << 10) |
           (static_cast<uint32_t>(NT >> 3) << 17) | (static_cast<uint32_t>(kWideRows >> 4) << 24);
}

// Issued by the lane with `leader` set, in code that the whole warp runs: the
// operands then stay in uniform registers. (In a branch of one lane each MMA took
// some 60 cycles to issue, for moving them there.)
template <int KIND>
__device__ __forceinline__ void wide_mma(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    if constexpr (KIND == kI8)
        asm volatile(
            "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
            " @q tcgen05.mma.cta_group::1.kind::i8 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
            "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(leader));
    else
        asm volatile(
            "{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
            " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
            "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(leader));
}

__device__ __forceinline__ void wide_commit(uint32_t leader, uint32_t bar) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar),
        "r"(leader)
        : "memory");
}

// As mv::mbar_wait_bounded, with each try suspended for up to 20 us: many warps
// wait here, and tries that come back at once take issue slots from those that
// convert.
__device__ __forceinline__ bool wide_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity), "r"(20000)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ bool wide_wait_lane(uint32_t bar, uint32_t parity, unsigned long long limit_ns) {
    if (wide_try(bar, parity)) return true;
    const unsigned long long start = mv::global_timer_ns();
    while (true) {
#pragma unroll 1
        for (int i = 0; i < 16; ++i)
            if (wide_try(bar, parity)) return true;
        if (mv::global_timer_ns() - start > limit_ns) return false;
    }
}
// A whole warp's wait. One that gives up sets `failed` and the device status.
__device__ __forceinline__ bool wide_wait(uint64_t* bar, uint32_t parity, volatile int* failed,
                                          unsigned long long limit_ns = mv::kWaitLimitNs) {
    const bool ok = __all_sync(0xffffffffu, wide_wait_lane(mv::smem_addr(bar), parity, limit_ns));
    if (!ok) {
        *failed = 1;
        if ((threadIdx.x & 31) == 0) atomicOr(&mv::g_device_status, mv::kStatusWaitTimeout);
    }
    return ok;
}
__device__ __forceinline__ void wide_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 16 rows x 16 32-bit columns: lane (g, t) holds columns 8 j + 2 t, + 1 of row g (r[4 j], r[4 j + 1]) and of row g + 8.
__device__ __forceinline__ void tmem_st_16x16(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// 16 rows x 8 columns: lane (g, t) holds columns t (r[0]) and 4 + t (r[2]) of row g, r[1] and r[3] of row g + 8.
__device__ __forceinline__ void tmem_st_16x8(uint32_t taddr, const uint32_t (&r)[4]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// `xmap`: X as [m, k] in boxes of NT rows of 128 bytes, where p.x_units says that it can be copied as it is.
template <int KIND, int NT, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(WideShape<KIND, NT, GROUP, ZEROS>::kBoundThreads, WideShape<KIND, NT, GROUP, ZEROS>::kCtas)
w4_wide_kernel(const LinearParams p, const __grid_constant__ CUtensorMap xmap) {
    constexpr int kOperand = KIND == kE4M3 ? kF16 : KIND;  // e4m3 rows become fp16
    using A = Act<kOperand>;
    using Shape = WideShape<KIND, NT, GROUP, ZEROS>;
    constexpr int kGroups = Shape::kGroups;
    constexpr int kRecord = record_size(GROUP, ZEROS);
    constexpr int kStages = Shape::kStages, kAB = Shape::kBuffers, kSets = Shape::kSets;
    constexpr int kTurns = Shape::kTurns, kMmaWarp = 8 + 4 * kSets * kTurns, kLoadWarp = kMmaWarp + 1;
    extern __shared__ uint8_t smem_raw[];
    // full: a chunk's A and X are in place and D of the chunk two before is
    // drained. done: its last group is multiplied, which frees A and X and hands
    // over D. part_done, for the other groups of chunks of several, has a
    // barrier for each buffer of D, or, where groups wait for their buffers, two for
    // each turn: no waiter may skip a phase, and no barrier run two phases ahead.
    __shared__ __align__(8) uint64_t full[kAB], done[kAB], part_done[2][kGroups > 2 ? kGroups : 2], d_empty[2], raw_full[2], drained;
    __shared__ uint32_t s_tmem;
    __shared__ float s_scale[NT], s_bias[kWideRows];
    __shared__ volatile int s_failed;

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = p.cluster > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int64_t block = static_cast<int64_t>(blockIdx.x) / p.cluster;  // of 128 weight rows
    const int token0 = blockIdx.y * NT;
    const int tokens = min(NT, p.m - token0);
    const int begin = static_cast<int>(static_cast<int64_t>(p.chunks) * rank / p.cluster);
    const int n = static_cast<int>(static_cast<int64_t>(p.chunks) * (rank + 1) / p.cluster) - begin;

    uint8_t* const smem =
        reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t xs = mv::smem_addr(smem);
    const uint32_t rings = xs + kAB * Shape::kXBytes;
    const uint32_t raws = rings + Shape::kRings;
    const bool raw = KIND == kE4M3 && p.x_units;  // x comes by TMA, but is not fp16 yet

    // A converting or draining warp w has rows 32 (w % 4).. of the 128: half p = w & 1
    // of tile (w % 4) >> 1. A second tile beyond the weight's last reads the
    // last one; its rows are never stored.
    const int quarter = warp & 3;
    const int64_t tile = min(2 * block + (quarter >> 1), static_cast<int64_t>(p.tiles) - 1);
    const uint8_t* const records = p.records + (tile * p.chunks + begin) * static_cast<int64_t>(kRecord);
    const uint8_t* const codes = records + (quarter & 1) * 512 + lane * 16;
    const uint32_t ring = rings + (warp & 7) * kStages * Shape::kStageBytes;
    const int set = warp < 8 ? warp >> 2 : ((warp - 8) >> 2) % kSets;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kAB; ++i) {
            mv::mbar_init(mv::smem_addr(&full[i]), 4 + 4 * kSets + 1);  // a converting set, the sets that drain a chunk, the loader
            mv::mbar_init(mv::smem_addr(&done[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            for (int j = 0; j < (kGroups > 2 ? kGroups : 2); ++j) mv::mbar_init(mv::smem_addr(&part_done[i][j]), 1);
            mv::mbar_init(mv::smem_addr(&d_empty[i]), 4 * kSets);
            mv::mbar_init(mv::smem_addr(&raw_full[i]), 1);
        }
        mv::mbar_init(mv::smem_addr(&drained), 1);
        s_failed = 0;
        mv::fence_mbar_init();
    }
    if (warp < 8)  // into L2 only: what the grid before wrote is not visible yet
        for (int i = set; i < 2 * kStages && i < n; i += 2)
            if (lane * 128 < kRecord)
                asm volatile("prefetch.global.L2 [%0];" ::"l"(records + static_cast<int64_t>(i) * kRecord + lane * 128));
    mv::wait_for_prior_grid();
    mv::allow_next_grid();

    int fill = 0;  // stage of the ring that the next record goes to
    const auto issue_codes = [&](int i) {
        if (i < n) {
            const uint8_t* rec = codes + static_cast<int64_t>(i) * kRecord;
            const uint32_t dst = ring + fill * Shape::kStageBytes + lane * 16;
#pragma unroll
            for (int h = 0; h < 4; ++h) cp_async_16(dst + h * 512, rec + h * 1024);
            if (ZEROS && lane < kGroups * 4)
                cp_async_16(dst + kCodeBytes / 2, records + static_cast<int64_t>(i) * kRecord + kCodeBytes +
                                                      kGroups * 128 + lane * 16);
        }
        cp_async_commit();
        fill = fill + 1 == kStages ? 0 : fill + 1;
    };
    if (warp < 8)
        for (int i = 0; i < kStages; ++i) issue_codes(set + 2 * i);
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(mv::smem_addr(&s_tmem)),
                     "r"(Shape::kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);  // the same in every lane, for the compiler too
    const uint32_t d_col = tmem + kAB * Shape::kACols;
    const auto wait = [&](uint64_t* bar, int parity) { return wide_wait(bar, parity & 1, &s_failed); };

    if (warp < 8) {
        const int g = lane >> 2;
        int drain = 0;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
        for (int i = set; i < n; i += 2) {
            cp_async_wait<kStages - 1>();
            if (ZEROS) __syncwarp();
            const uint32_t rec = ring + drain * Shape::kStageBytes;
            drain = drain + 1 == kStages ? 0 : drain + 1;
            if (i >= kAB && !wait(&done[i % kAB], i / kAB - 1)) break;
            fence_after();
            const uint32_t a_col = lanes + (i % kAB) * Shape::kACols;
            uint32_t zl[2], zh[2];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                if (h % (GROUP / 32) == 0) {
                    uint32_t z = 0;
                    if (ZEROS) z = lds32(rec + kCodeBytes / 2 + (h / (GROUP / 32)) * 64 + g * 8 + (quarter & 1) * 4);
                    if constexpr (KIND == kI8) {
                        const uint32_t u = (z ^ 0x88888888u) & 0x0f0f0f0fu;
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            zl[q] = __byte_perm(u, 0, q ? 0x2222 : 0x0000);
                            zh[q] = __byte_perm(u, 0, q ? 0x3333 : 0x1111);
                        }
                    } else {
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            zl[q] = A::zero_low(8 + static_cast<int8_t>(z >> (16 * q)));
                            zh[q] = A::zero_high(8 + static_cast<int8_t>(z >> (16 * q + 8)));
                        }
                    }
                }
                const uint4 w = lds128(rec + h * 512 + lane * 16);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const uint32_t w0 = q ? w.z : w.x, w1 = q ? w.w : w.y;
                    const uint32_t at = a_col + (static_cast<uint32_t>(q * 16) << 16);
                    if constexpr (KIND == kI8) {
                        // 32 columns of h: bytes in the columns' order (the codes' is 0, 2, 1, 3).
                        uint32_t r[4];
                        if (ZEROS) {
                            r[0] = bytes_minus(w0, zl[q]), r[1] = bytes_minus(w0 >> 4, zh[q]);
                            r[2] = bytes_minus(w1, zl[q]), r[3] = bytes_minus(w1 >> 4, zh[q]);
                        } else {
                            r[0] = (w0 << 4) & 0xf0f0f0f0u, r[1] = w0 & 0xf0f0f0f0u;
                            r[2] = (w1 << 4) & 0xf0f0f0f0u, r[3] = w1 & 0xf0f0f0f0u;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) r[e] = __byte_perm(r[e], 0, 0x3120);
                        tmem_st_16x8(at + h * 8, r);
                    } else {
                        uint32_t a0[4], a1[4];
                        A::weights(w0, zl[q], zh[q], a0);
                        A::weights(w1, zl[q], zh[q], a1);
                        const uint32_t r[8] = {a0[0], a0[2], a0[1], a0[3], a1[0], a1[2], a1[1], a1[3]};
                        tmem_st_16x16(at + h * 16, r);
                    }
                }
            }
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) wide_arrive(mv::smem_addr(&full[i % kAB]));
            issue_codes(i + 2 * kStages);
        }
        cp_async_wait<0>();
    } else if (warp == kMmaWarp) {
        constexpr int kSteps = KIND == kI8 ? GROUP / 32 : GROUP / 16;  // MMAs per group
        const uint32_t leader = elect_one();
        bool ok = true;
        for (int i = 0; i < n; ++i) {
            ok = wait(&full[i % kAB], i / kAB);
#pragma unroll
            for (int gi = 0; gi < kGroups; ++gi) {
                const int u = i * kGroups + gi;
                if (!Shape::kWholeChunks && u >= 2) ok = ok && wait(&d_empty[u & 1], (u >> 1) - 1);
                if (!ok) break;
                fence_after();
                const uint32_t a_at = tmem + (i % kAB) * Shape::kACols + gi * kSteps * 8;
                const uint32_t x_at = xs + (i % kAB) * Shape::kXBytes;
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    const int step = gi * kSteps + s;
                    const uint32_t b = KIND == kI8 ? x_at + step * 32 : x_at + (step >> 2) * (NT * 128) + (step & 3) * 32;
                    wide_mma<KIND>(leader, d_col + (u % Shape::kDBuffers) * NT, a_at + s * 8, sw128_desc(b), wide_idesc<KIND, NT>(), s > 0);
                }
                const int v = i / kTurns * (kGroups - 1) + gi;
                wide_commit(leader, mv::smem_addr(gi == kGroups - 1        ? &done[i % kAB]
                                                  : Shape::kWholeChunks ? &part_done[i & 1][gi]
                                                                        : &part_done[i % kTurns][v & 1]));
            }
            if (!ok) break;
        }
        // Everything issued completes before TMEM is freed.
        wide_commit(leader, mv::smem_addr(&drained));
        wait(&drained, 0);
    } else if (warp == kLoadWarp) {
        const uint32_t leader = elect_one();
        bool ok = true;
        for (int i = 0; i < n && ok; ++i) {
            if (i >= kAB) ok = wait(&done[i % kAB], i / kAB - 1);
            if (raw && i >= 2) ok = ok && wait(&full[(i - 2) % kAB], (i - 2) / kAB);  // its raw rows are read
            if (leader && ok) {
                const uint32_t bar = mv::smem_addr(&full[i % kAB]);
                if (raw) {
                    const uint32_t raw_bar = mv::smem_addr(&raw_full[i & 1]);
                    mv::mbar_arrive_expect_tx(raw_bar, Shape::kRawBytes);
                    tma_load_2d(raws + (i & 1) * Shape::kRawBytes, &xmap, (begin + i) * kChunk, token0, raw_bar);
                    wide_arrive(bar);
                } else if (p.x_units) {
                    mv::mbar_arrive_expect_tx(bar, Shape::kXBytes);
                    const uint32_t dst = xs + (i % kAB) * Shape::kXBytes;
                    const int k = (begin + i) * kChunk;
                    tma_load_2d(dst, &xmap, k, token0, bar);
                    if (KIND != kI8) tma_load_2d(dst + NT * 128, &xmap, k + 64, token0, bar);
                } else {
                    wide_arrive(bar);  // the draining warps store X themselves
                }
            }
            __syncwarp();
        }
        // What the epilogue needs of every token and row.
        for (int t = lane; t < NT; t += 32)
            s_scale[t] = (ZEROS && KIND == kI8 ? 1.0f : A::kScale) * (p.x_scale && t < tokens ? p.x_scale[token0 + t] : 1.0f);
        for (int r = lane; r < kWideRows; r += 32) {
            const int64_t column = block * kWideRows + r;
            s_bias[r] = p.bias && column < p.n ? load_as_float(p.bias, column, p.out_dtype) : 0.0f;
        }
        // A wait gave up: no barrier tells any more when the copies under way land, so give them their time.
        if (!ok)
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    } else {
        constexpr int kDrainers = 128 * kSets;
        const int turn = (warp - 8) / (4 * kSets);
        const int lt = threadIdx.x - 256 - turn * kDrainers;
        // This thread's scale: row `lane` of the quarter, its pair of rows g and g + 8 in a word.
        const uint8_t* const scale = records + kCodeBytes + ((lane & 7) * 8 + (quarter & 1) * 4 + (lane >> 4) * 2) * 2;
        const auto load_scales = [&](int i, uint32_t (&w)[kGroups]) {
#pragma unroll
            for (int gi = 0; gi < kGroups; ++gi)
                if (i < n)
                    w[gi] = *reinterpret_cast<const uint32_t*>(scale + static_cast<int64_t>(i) * kRecord + gi * 128);
        };
        // X that TMA cannot copy as it is: these warps store it, element by element at
        // worst (rows off a 16-byte boundary). e4m3 numbers that become fp16 come by TMA
        // into a buffer of their own first (3584 x 28672: 27 us at 16 rows and 53 at 64;
        // loaded here from global memory, 33 and 78; fp16 rows take 20 and 36).
        constexpr int kUnits = KIND == kI8 ? 8 : 16;  // 16-byte units of a token's chunk
        const auto place = [&](uint32_t dst, int token, int unit, const uint4& v) {
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(
                             dst + (unit >> 3) * (NT * 128) + token * 128 + (((unit & 7) ^ (token & 7)) << 4)),
                         "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                         : "memory");
        };
        const auto store_x = [&](int i) {
            const int x_size = p.x_dtype >= kI8 ? 1 : 2;
            const uint32_t dst = xs + (i % kAB) * Shape::kXBytes;
            if (raw) {
                if (!wait(&raw_full[i & 1], i >> 1)) return false;
#pragma unroll 2
                for (int u = lt; u < NT * kUnits; u += kDrainers) {
                    uint32_t a, b;
                    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                                 : "=r"(a), "=r"(b)
                                 : "r"(raws + (i & 1) * Shape::kRawBytes + u * 8));
                    const uint2 lo = e4m3_to_half(a), hi = e4m3_to_half(b);
                    place(dst, u / kUnits, u % kUnits, make_uint4(lo.x, lo.y, hi.x, hi.y));
                }
                mv::fence_proxy_async_smem();
                return true;
            }
#pragma unroll 1
            for (int u = lt; u < NT * kUnits; u += kDrainers) {
                const int token = u / kUnits, unit = u % kUnits;
                const int limit = token < tokens ? p.k : 0;
                const int k = (begin + i) * kChunk + unit * (KIND == kI8 ? 16 : 8);
                const uint8_t* row = static_cast<const uint8_t*>(p.x) + (token0 + token) * p.x_stride * x_size;
                uint32_t r[1][A::kRunBytes / 4];
                uint4 v;
                load_run<kOperand>(p, row, k, limit, r);
                if constexpr (KIND == kI8) {
                    v.x = r[0][0], v.y = r[0][1];
                    load_run<kOperand>(p, row, k + 8, limit, r);
                    v.z = r[0][0], v.w = r[0][1];
                } else {
                    v = make_uint4(r[0][0], r[0][1], r[0][2], r[0][3]);
                }
                place(dst, token, unit, v);
            }
            mv::fence_proxy_async_smem();
            return true;
        };
        float acc[Shape::kCols];
#pragma unroll
        for (int e = 0; e < Shape::kCols; ++e) acc[e] = 0.0f;
        const uint32_t lanes = d_col + set * Shape::kCols + (static_cast<uint32_t>(quarter * 32) << 16);
        const auto publish = [&](int i) {  // chunk i may be multiplied, as far as these warps go
            if (i >= n) return true;
            if ((raw || !p.x_units) && !store_x(i)) return false;
            fence_before();
            __syncwarp();
            if (lane == 0) wide_arrive(mv::smem_addr(&full[i % kAB]));
            return true;
        };
        uint32_t scales[kGroups] = {}, scales1[kGroups] = {}, scales2[kGroups] = {};
        load_scales(turn, scales);
        load_scales(turn + kTurns, scales1);
        bool ok = publish(turn);
        if (kTurns == 1) ok = ok && publish(1);
        for (int i = turn; i < n && ok; i += kTurns) {
            load_scales(i + 2 * kTurns, scales2);
            if (lane < kGroups && i + 6 < n)  // the scales come from memory: into L2 well before
                asm volatile("prefetch.global.L2 [%0];" ::"l"(records + static_cast<int64_t>(i + 6) * kRecord + kCodeBytes +
                                                             lane * 128));
#pragma unroll
            for (int gi = 0; gi < kGroups; ++gi) {
                const int u = i * kGroups + gi, v = i / kTurns * (kGroups - 1) + gi;
                const float2 both = scale_pair(scales[gi], p.scale_bf16);
                const float sc = lane & 8 ? both.y : both.x;
                ok = ok && (gi == kGroups - 1 ? wait(&done[i % kAB], i / kAB)
                                              : (Shape::kWholeChunks ? wait(&part_done[i & 1][gi], i >> 1) : wait(&part_done[turn][v & 1], v >> 1)));
                if (!ok) break;
                fence_after();
                const uint32_t from = lanes + (u % Shape::kDBuffers) * NT;
#pragma unroll
                for (int c = 0; c < Shape::kCols; c += 16) {
                    uint32_t r[16];
                    tmem_ld_16(from + c, r);
                    wait_ld();
                    if (!Shape::kWholeChunks && c + 16 == Shape::kCols) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) wide_arrive(mv::smem_addr(&d_empty[u & 1]));
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        // s32 to fp32: 1.5 2^23's bits plus the sum (below 2^22) are the float 1.5 2^23 + sum.
                        const float f = KIND == kI8 ? __uint_as_float(r[e] + 0x4b400000u) - 12582912.0f
                                                    : __uint_as_float(r[e]);
                        acc[c + e] = fmaf(sc, f, acc[c + e]);
                    }
                }
            }
            if (!ok) break;
            ok = publish(i + 2);  // D of chunk i is in registers
#pragma unroll
            for (int gi = 0; gi < kGroups; ++gi) scales[gi] = scales1[gi], scales1[gi] = scales2[gi];
        }
        // The last chunk is multiplied, so no MMA reads X and no warp converts any
        // more: the partial sums go over them.
        if (kTurns > 1 && n > 0 && ok) ok = wait(&done[(n - 1) % kAB], (n - 1) / kAB);
        float* part = reinterpret_cast<float*>(smem) + (turn * NT + set * Shape::kCols) * kWidePartStride + quarter * 32 + lane;
        const float poison = ok && !s_failed ? 0.0f : __int_as_float(0x7fffffff);
#pragma unroll
        for (int e = 0; e < Shape::kCols; ++e) part[e * kWidePartStride] = acc[e] + poison;
    }
    fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {  // before any wait for another CTA: none may wait for this one's columns meanwhile
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Shape::kTmemCols));
    }
    if (p.cluster > 1) cluster_barrier();
    // A thread keeps to one row and has eight tokens' residuals under way, as raw
    // bits: one at a time, their latencies were a third of a call.
    constexpr int kLines = Shape::kThreads / kWideRows, kPer = 8;
    const int row = threadIdx.x % kWideRows;
    const int64_t column = block * kWideRows + row;
    if (threadIdx.x < kLines * kWideRows && column < p.n) {
        const int step = kLines * p.cluster;
        const bool wide = p.out_dtype == kF32;
        for (int t0 = rank * kLines + threadIdx.x / kWideRows; t0 < tokens; t0 += kPer * step) {
            uint32_t bits[kPer] = {};
            if (p.residual) {
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    const int64_t at = (token0 + t0 + j * step) * p.residual_stride + column;
                    if (t0 + j * step < tokens)
                        bits[j] = wide ? static_cast<const uint32_t*>(p.residual)[at] : static_cast<const uint16_t*>(p.residual)[at];
                }
            }
#pragma unroll 1
            for (int j = 0; j < kPer; ++j) {
                const int token = t0 + j * step;
                if (token >= tokens) break;
                const uint32_t at = xs + (token * kWidePartStride + row) * 4;
                float v = 0.0f;
                for (int c = 0; c < p.cluster; ++c)
#pragma unroll
                    for (int turn = 0; turn < kTurns; ++turn) {
                        const uint32_t from = at + turn * NT * kWidePartStride * 4;
                        v += p.cluster > 1 ? ld_cluster(from, c) : __uint_as_float(lds32(from));
                    }
                uint32_t b = bits[0];
#pragma unroll
                for (int i = 0; i + 1 < kPer; ++i) bits[i] = bits[i + 1];
                const float residual = wide ? __uint_as_float(b)
                                       : p.out_dtype == kBF16 ? __uint_as_float(b << 16)
                                                              : __half2float(__ushort_as_half(static_cast<uint16_t>(b)));
                store_from_float(p.out, (token0 + token) * p.out_stride + column, p.out_dtype,
                                 fmaf(v, s_scale[token], s_bias[row]) + residual);
            }
        }
    }
    if (p.cluster > 1) cluster_barrier();  // no CTA leaves while another reads its shared memory
}

// The kernel's wait on a barrier that nothing completes, with a limit of its own.
__global__ void wait_timeout_selftest_kernel(unsigned long long limit_ns) {
    __shared__ __align__(8) uint64_t bar;
    __shared__ volatile int failed;
    if (threadIdx.x == 0) {
        mv::mbar_init(mv::smem_addr(&bar), 1);
        mv::fence_mbar_init();
    }
    __syncwarp();
    wide_wait(&bar, 0, &failed, limit_ns);
}

}  // namespace mvq
