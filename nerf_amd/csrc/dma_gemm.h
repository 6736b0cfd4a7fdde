// A workgroup's product of two 16-bit operands whose k is contiguous, fed by LDS-DMA: C[b][a] += sum_k B[b][k] A[a][k].
//
// TA x TB outputs, WA x WB wavefronts, k in steps of KS, P planes per operand (P = 2: each value is hi + lo and the products
// hi.hi + hi.lo + lo.hi are kept).  A step's rows reach LDS by global_load_lds_dwordx4 (64 lanes x 16 B from per-lane
// addresses to 1 KiB of LDS, no registers), ST - 1 steps ahead of their use, one barrier and one counted vmcnt per step.
// A row of a step is KS / 8 slots of 16 B; slot s of row r holds the row's octet s ^ f(r), so that the sixteen rows a
// fragment read touches fall into sixteen different 16 B columns of the 256 B bank row.
// The DMA is issued from inline asm: the compiler orders every ds_read behind all LDS-DMA it knows of (vmcnt(0)), which would
// serialise the ring.  It has no register outputs, and every step is waited for by its own counted vmcnt + barrier below.
#pragma once
#include "nrf_common.h"

namespace {

typedef unsigned u32x4_g __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8_g __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_g __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char* lds_ptr_g;

__device__ __forceinline__ void dma16(const void* src, unsigned lds_dst) {
    asm volatile(
        "s_mov_b32 m0, %1\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %0, off"
        :
        : "v"(src), "s"(lds_dst)
        : "memory");
}
__device__ __forceinline__ unsigned lds_addr(const void* p) {
    return unsigned(reinterpret_cast<uintptr_t>((lds_ptr_g)p));
}

template <bool BF16, int TA, int TB, int WA, int WB, int P, int KS, int ST>
struct DmaGemm {
    static constexpr int kWaves = WA * WB, kThreads = 64 * kWaves;
    static constexpr int kMA = TA / WA / 16, kMB = TB / WB / 16;             // 16 x 16 accumulators of a wavefront
    static constexpr int kSlots = KS / 8, kRowsPerPiece = 64 / kSlots;       // a piece = 1 KiB = one DMA instruction
    static constexpr int kPlaneA = TA * KS * 2, kPlaneB = TB * KS * 2;
    static constexpr int kStage = P * (kPlaneA + kPlaneB), kLds = ST * kStage;
    static constexpr int kPieces = kStage / 1024 / kWaves;                   // per wavefront and step
    static_assert(KS == 32 || KS == 64, "slots");
    static_assert(kStage % (1024 * kWaves) == 0 && kPlaneA % 1024 == 0 && kPlaneB % 1024 == 0, "whole pieces per wavefront");

    static __device__ __forceinline__ int swizzle(int row) { return KS == 64 ? (row >> 1) & 7 : (row >> 2) & 3; }

    const char* src[kPieces];    // this lane's 16 B of its pieces, advanced by a step each time
    unsigned lds0;
    int wave, lane;

    // row_ptr(is_b, plane, row): the address of that row's element 0 of k.  Every row must have k_steps * KS elements.
    template <class F>
    __device__ __forceinline__ void start(char* smem, F row_ptr) {
        lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        lds0 = __builtin_amdgcn_readfirstlane(lds_addr(smem) + unsigned(wave) * (kPieces * 1024));
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const int byte = (wave * kPieces + j) * 1024;
            const bool is_b = byte >= P * kPlaneA;
            const int in = is_b ? byte - P * kPlaneA : byte, size = is_b ? kPlaneB : kPlaneA;
            const int plane = in / size, row = (in % size) / (KS * 2) + lane / kSlots, slot = lane % kSlots;
            src[j] = reinterpret_cast<const char*>(row_ptr(is_b, plane, row)) + (slot ^ swizzle(row)) * 16;
        }
    }
    __device__ __forceinline__ void issue(int stage) {
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            dma16(src[j], __builtin_amdgcn_readfirstlane(lds0 + unsigned(stage) * kStage + j * 1024));
            src[j] += KS * 2;
        }
    }

    __device__ __forceinline__ f32x4 mfma(const u32x4_g& a, const u32x4_g& b, const f32x4& c) {
        if constexpr (BF16)
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_g, a), __builtin_bit_cast(bf16x8_g, b), c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_g, a), __builtin_bit_cast(f16x8_g, b), c, 0, 0, 0);
    }

    // lane (c = lane & 15, q = lane >> 4): acc[ma][mb][r] = C[b = wb + 16 mb + c][a = wa + 16 ma + 4 q + r]
    __device__ __forceinline__ int wave_a() const { return (wave % WA) * (TA / WA); }
    __device__ __forceinline__ int wave_b() const { return (wave / WA) * (TB / WB); }

    __device__ __forceinline__ void run(const char* smem, int k_steps, f32x4 (&acc)[kMA][kMB]) {
        const int c = lane & 15, q = lane >> 4, f = swizzle(c);
        const int ra = (wave_a() + c) * (KS * 2), rb = P * kPlaneA + (wave_b() + c) * (KS * 2);
#pragma unroll
        for (int s = 0; s < ST - 1; ++s)
            if (s < k_steps) issue(s);
        int slot = 0, fill = ST - 1;
        for (int k = 0; k < k_steps; ++k) {
            // steps k + 1 .. k + ST - 2 may stay in flight; near the end fewer are
            if (ST > 2 && k + ST - 2 < k_steps) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kPieces * (ST - 2)) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            if (k + ST - 1 < k_steps) issue(fill);
            const char* st = smem + slot * kStage;
#pragma unroll
            for (int kk = 0; kk < KS / 32; ++kk) {
                const int at = ((4 * kk + q) ^ f) * 16;
                u32x4_g fa[kMA][P], fb[kMB][P];
#pragma unroll
                for (int p = 0; p < P; ++p) {
#pragma unroll
                    for (int m = 0; m < kMB; ++m) fb[m][p] = *reinterpret_cast<const u32x4_g*>(st + rb + p * kPlaneB + m * (16 * KS * 2) + at);
#pragma unroll
                    for (int m = 0; m < kMA; ++m) fa[m][p] = *reinterpret_cast<const u32x4_g*>(st + ra + p * kPlaneA + m * (16 * KS * 2) + at);
                }
#pragma unroll
                for (int ma = 0; ma < kMA; ++ma)
#pragma unroll
                    for (int mb = 0; mb < kMB; ++mb) {
                        if constexpr (P == 2) {
                            acc[ma][mb] = mfma(fa[ma][0], fb[mb][1], acc[ma][mb]);
                            acc[ma][mb] = mfma(fa[ma][1], fb[mb][0], acc[ma][mb]);
                        }
                        acc[ma][mb] = mfma(fa[ma][0], fb[mb][0], acc[ma][mb]);
                    }
            }
            slot = slot + 1 == ST ? 0 : slot + 1;
            fill = fill + 1 == ST ? 0 : fill + 1;
        }
    }
};

}  // namespace
