// A workgroup's product of two 16-bit operands fed by LDS-DMA: C[b][a] += sum_k B[b][k] A[a][k].
//
// TA x TB outputs, WA x WB wavefronts, k in steps of KS, P planes per operand (P = 2: each value is hi + lo and the products
// hi.hi + hi.lo + lo.hi are kept).  A step's data reach LDS by global_load_lds_dwordx4 (64 lanes x 16 B from per-lane
// addresses to 1 KiB of LDS, no registers), up to ST steps ahead of their use, one barrier and one counted vmcnt per step.
// An operand lies in memory either with k contiguous (kRows: LDS holds [row][k], a fragment is one 16 B read) or with its row
// index contiguous (kCols: LDS holds [k][row], a fragment is two ds_read_b64_tr_b16, which turn 4 x 16 blocks on their way
// out); kGather is kCols with the address of every k looked up in a list in LDS.  Octets of 16 B are stored at slot
// octet ^ f(row or k), so that one read's lanes fall into different 16 B columns of the 256 B bank row.
// The DMA is issued from inline asm: the compiler orders every ds_read behind all LDS-DMA it knows of (vmcnt(0)), which would
// serialise the ring.  It has no register outputs, and every step is waited for by its own counted vmcnt + barrier below.
#pragma once
#include "nrf_common.h"

namespace {

typedef unsigned u32x4_g __attribute__((ext_vector_type(4)));
typedef short s16x4_g __attribute__((ext_vector_type(4)));
typedef short s16x8_g __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_g __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_g __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char* lds_ptr_g;

__device__ __forceinline__ void dma16(const char* base, unsigned offset, unsigned lds_dst) {   // base, lds_dst: uniform
    asm volatile(
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %1"
        :
        : "v"(offset), "s"(base), "s"(lds_dst)
        : "memory");
}
__device__ __forceinline__ unsigned lds_addr(const void* p) {
    return unsigned(reinterpret_cast<uintptr_t>((lds_ptr_g)p));
}

enum DmaMode { kRows, kCols, kGather };

// One operand's part of a step: R rows (outputs), wavefront `wave` of WAVES moves kPieces pieces of 1 KiB.
template <int MODE, int R, int KS, int P, int WAVES>
struct DmaSide {
    static constexpr int kPlane = R * KS * 2, kBytes = P * kPlane, kPieces = kBytes / 1024 / WAVES;
    static constexpr int kSlots = MODE == kRows ? KS / 8 : R / 8;        // octets of an LDS row
    static_assert(kBytes % (1024 * WAVES) == 0 && kPlane % 1024 == 0, "whole pieces per wavefront");
    static_assert(64 % kSlots == 0 && (MODE == kRows ? KS == 64 : P == 1), "layout");

    static __device__ __forceinline__ int swizzle(int row) {
        if (MODE == kRows) return (row >> 1) & 7;
        if (R == 64) return ((row >> 1) & 1) * 2 + ((row >> 3) & 1) * 4;
        return (row & 3) * 2 + ((row >> 3) & 1) * 8;
    }

    const char* base;         // uniform: element 0 of the operand at step 0
    unsigned src[kPieces];    // this lane's octet of each piece, in bytes from there (an operand stays under 4 GiB)

    // row / k row and octet of this lane in piece j of its wavefront
    static __device__ __forceinline__ int line(int j, int wave, int lane) {
        return ((wave * kPieces + j) % (kPlane / 1024)) * (64 / kSlots) + lane / kSlots;
    }
    static __device__ __forceinline__ int octet(int j, int wave, int lane) { return (lane % kSlots) ^ swizzle(line(j, wave, lane)); }

    // row_offset(row): bytes from `base` to k = 0 of that row; plane_bytes: from one plane to the next, which is another
    // wavefront's, so that only a plane's rows have to lie within 4 GiB
    template <class F>
    __device__ __forceinline__ void start_rows(int wave, int lane, const void* base_, int64_t plane_bytes, F row_offset) {
        static_assert(WAVES % P == 0, "a wavefront moves pieces of one plane");
        base = static_cast<const char*>(base_) + (wave * kPieces) / (kPlane / 1024) * plane_bytes;
#pragma unroll
        for (int j = 0; j < kPieces; ++j) src[j] = row_offset(line(j, wave, lane)) + octet(j, wave, lane) * 16;
    }
    // base: k = 0 of row 0; pitch: bytes from one k to the next (kGather: of one list entry); `octets` whole octets are in a row
    __device__ __forceinline__ void start_cols(int wave, int lane, const void* base_, unsigned pitch, int octets) {
        base = static_cast<const char*>(base_);
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
            const int o = octet(j, wave, lane);
            src[j] = (o < octets ? o : 0) * 16 + (MODE == kCols ? line(j, wave, lane) * pitch : 0);
        }
    }
    // piece j of a step `offset` bytes from step 0, `left` elements of k from the end: lanes past it read what is there
    // before it (their k is masked out of the fragments)
    __device__ __forceinline__ void issue(int j, int wave, int lane, unsigned lds, int left, int64_t offset, const int* list, unsigned pitch) const {
        unsigned o = src[j];
        if constexpr (MODE == kGather) {
            const int k = line(j, wave, lane);
            o += unsigned(list[k < left ? k : 0]) * pitch;
            dma16(base, o, __builtin_amdgcn_readfirstlane(lds + j * 1024));
        } else {
            if (left < KS) {
                if (MODE == kRows && octet(j, wave, lane) * 8 >= left) o -= octet(j, wave, lane) * 16;
                if (MODE == kCols && line(j, wave, lane) >= left) o -= line(j, wave, lane) * pitch;
            }
            dma16(base + offset, o, __builtin_amdgcn_readfirstlane(lds + j * 1024));
        }
    }

    // fragment m (16 rows from `first`) of k octets kk: lane (c, q) gets row first + 16 m + c, k = 32 kk + 8 q .. + 7
    static __device__ __forceinline__ u32x4_g frag(const char* plane, int first, int m, int kk, int c, int q) {
        if constexpr (MODE == kRows) {
            return *reinterpret_cast<const u32x4_g*>(plane + (first + c) * (KS * 2) + m * (16 * KS * 2) + ((4 * kk + q) ^ swizzle(c)) * 16);
        } else {
            s16x4_g part[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int k = 32 * kk + 8 * q + 4 * u + (c >> 2);
                const int octet = ((first + 16 * m) / 8 + ((c & 3) >> 1)) ^ swizzle(k);
                part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4_g*)(plane + k * (R * 2) + octet * 16 + (c & 1) * 8));
            }
            return __builtin_bit_cast(u32x4_g, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

template <bool BF16>
__device__ __forceinline__ f32x4 mfma_dma(const u32x4_g& a, const u32x4_g& b, const f32x4& c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_g, a), __builtin_bit_cast(bf16x8_g, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_g, a), __builtin_bit_cast(f16x8_g, b), c, 0, 0, 0);
}

template <bool BF16, int MODE_A, int MODE_B, int TA, int TB, int WA, int WB, int P, int ST, bool SUM_B = false>
struct DmaGemm {
    static constexpr int KS = 64, kWaves = WA * WB, kThreads = 64 * kWaves;
    static constexpr int kMA = TA / WA / 16, kMB = TB / WB / 16;             // 16 x 16 accumulators of a wavefront
    typedef DmaSide<MODE_A, TA, KS, P, kWaves> A;
    typedef DmaSide<MODE_B, TB, KS, P, kWaves> B;
    static constexpr int kStage = A::kBytes + B::kBytes, kLds = ST * kStage, kPieces = A::kPieces + B::kPieces;

    A a;
    B b;
    int64_t step_a, step_b;     // bytes from one step to the next (kRows, kCols)
    unsigned pitch_a, pitch_b;  // bytes from one k to the next (kCols), of one list entry (kGather)
    int wave, lane;
    bool idle = false;   // nothing of this wavefront's part is wanted: it moves data and keeps the barriers, but multiplies nothing

    __device__ __forceinline__ DmaGemm() : step_a(KS * 2), step_b(KS * 2), pitch_a(0), pitch_b(0), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), lane(threadIdx.x & 63) {}

    // lane (c = lane & 15, q = lane >> 4): acc[ma][mb][r] = C[b = wave_b() + 16 mb + c][a = wave_a() + 16 ma + 4 q + r]
    __device__ __forceinline__ int wave_a() const { return (wave % WA) * (TA / WA); }
    __device__ __forceinline__ int wave_b() const { return (wave / WA) * (TB / WB); }

    // piece j of step k, to the slot at lds
    __device__ __forceinline__ void issue(int j, unsigned lds, int k, int k_count, const int* list) const {
        if (j < A::kPieces)
            a.issue(j, wave, lane, lds + wave * (A::kPieces * 1024), k_count - k * KS, k * step_a, list + k * KS, pitch_a);
        else
            b.issue(j - A::kPieces, wave, lane, lds + A::kBytes + wave * (B::kPieces * 1024), k_count - k * KS, k * step_b, list + k * KS, pitch_b);
    }

    struct Frags {
        u32x4_g a[kMA][P], b[kMB][P];
    };
    static constexpr int kReads = P * (kMA + kMB);
    __device__ __forceinline__ void read(int i, Frags& f, const char* stage, int kk) const {   // fragment i of the 32 k
        const int c = lane & 15, q = lane >> 4, p = i / (kMA + kMB), m = i % (kMA + kMB);
        if (m < kMB) f.b[m][p] = B::frag(stage + A::kBytes + p * B::kPlane, wave_b(), m, kk, c, q);
        else f.a[m - kMB][p] = A::frag(stage + p * A::kPlane, wave_a(), m - kMB, kk, c, q);
    }
    __device__ __forceinline__ void read(Frags& f, const char* stage, int kk) const {
#pragma unroll
        for (int i = 0; i < kReads; ++i) read(i, f, stage, kk);
    }
    // the k of a last, partial step that lie past the end
    __device__ __forceinline__ void mask(Frags& f, int left) const {
        const int valid = left - 8 * (lane >> 4);
        u32x4_g m;
#pragma unroll
        for (int i = 0; i < 4; ++i) m[i] = valid >= 2 * i + 2 ? ~0u : valid == 2 * i + 1 ? 0xffffu : 0u;
#pragma unroll
        for (int p = 0; p < P; ++p) {
#pragma unroll
            for (int i = 0; i < kMB; ++i) f.b[i][p] &= m;
#pragma unroll
            for (int i = 0; i < kMA; ++i) f.a[i][p] &= m;
        }
    }
    __device__ __forceinline__ void multiply(int ma, const Frags& f, f32x4 (&acc)[kMA][kMB]) const {
#pragma unroll
        for (int mb = 0; mb < kMB; ++mb) {
            if constexpr (P == 2) {
                acc[ma][mb] = mfma_dma<BF16>(f.a[ma][0], f.b[mb][1], acc[ma][mb]);
                acc[ma][mb] = mfma_dma<BF16>(f.a[ma][1], f.b[mb][0], acc[ma][mb]);
            }
            acc[ma][mb] = mfma_dma<BF16>(f.a[ma][0], f.b[mb][0], acc[ma][mb]);
        }
    }
    __device__ __forceinline__ void sum_up(const Frags& f, f32x4 (*sum)[kMB], bool with_sum) const {
        if constexpr (SUM_B)
            if (with_sum) {
                const unsigned one = BF16 ? 0x3f803f80u : 0x3c003c00u;
#pragma unroll
                for (int mb = 0; mb < kMB; ++mb) (*sum)[mb] = mfma_dma<BF16>((u32x4_g){one, one, one, one}, f.b[mb][0], (*sum)[mb]);
            }
    }

    // `list`: the rows of k for kGather sides (in LDS, complete before the call).  with_sum: sum[mb][0] += sum over k of B.
    // A step is two halves of 32 k.  The second half's fragments are read while the first half is multiplied; once every
    // wavefront holds them (first barrier) the step's slot is refilled with step k + ST, the DMA issued between the rest of the
    // first half's MFMAs.  Once the next step has landed (counted vmcnt, second barrier) its first half is read between the
    // second half's MFMAs.
    __device__ __forceinline__ void run(const char* smem, int k_count, f32x4 (&acc)[kMA][kMB], const int* list = nullptr,
                                        f32x4 (*sum)[kMB] = nullptr, bool with_sum = false) {
        if (__builtin_amdgcn_readfirstlane(idle)) walk<false>(smem, k_count, acc, list, sum, false);
        else walk<true>(smem, k_count, acc, list, sum, with_sum);
    }
    template <bool WORK>
    __device__ __forceinline__ void walk(const char* smem, int k_count, f32x4 (&acc)[kMA][kMB], const int* list, f32x4 (*sum)[kMB],
                                         bool with_sum) {
        const unsigned lds = lds_addr(smem);
        const int k_steps = (k_count + KS - 1) / KS;
        if (k_steps == 0) return;
#pragma unroll
        for (int s = 0; s < ST; ++s)
            if (s < k_steps)
#pragma unroll
                for (int j = 0; j < kPieces; ++j) issue(j, lds + s * kStage, s, k_count, list);
        if (k_steps >= ST) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kPieces * (ST - 1)) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        Frags f0, f1;
        if (WORK) read(f0, smem, 0);
        int slot = 0, k = 0;
        // steps that refill their slot; steps without a step ST on; the last
        for (; k + ST < k_steps; ++k) step<WORK, true, true>(smem, lds, k, k_count, slot, f0, f1, acc, list, sum, with_sum);
        for (; k + 1 < k_steps; ++k) step<WORK, false, true>(smem, lds, k, k_count, slot, f0, f1, acc, list, sum, with_sum);
        step<WORK, false, false>(smem, lds, k, k_count, slot, f0, f1, acc, list, sum, with_sum);
    }
    template <bool WORK, bool FILL, bool NEXT>
    __device__ __forceinline__ void step(const char* smem, unsigned lds, int k, int k_count, int& slot, Frags& f0, Frags& f1,
                                         f32x4 (&acc)[kMA][kMB], const int* list, f32x4 (*sum)[kMB], bool with_sum) const {
        const int next = slot + 1 == ST ? 0 : slot + 1;
        constexpr int kHalf = kMA / 2, D = (kPieces + kMA - kHalf - 1) / (kMA - kHalf), R = (kReads + kMA - 1) / kMA;
        if (WORK) {
            read(f1, smem + slot * kStage, 1);
            __builtin_amdgcn_sched_barrier(0);
            if (!NEXT && k_count - k * KS < KS) mask(f0, k_count - k * KS), mask(f1, k_count - k * KS - 32);
#pragma unroll
            for (int ma = 0; ma < kHalf; ++ma) multiply(ma, f0, acc);
        }
        if (FILL) {     // every wavefront holds all of this step
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
        }
#pragma unroll
        for (int ma = kHalf; ma < kMA; ++ma) {
            if (WORK) multiply(ma, f0, acc);
#pragma unroll
            for (int j = 0; j < kPieces; ++j)
                if (FILL && j / D == ma - kHalf) issue(j, lds + slot * kStage, k + ST, k_count, list);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (WORK) sum_up(f0, sum, with_sum);
        if (NEXT) {     // the next step has landed; near the end fewer are in flight, and all are waited for
            if (FILL) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kPieces * (ST - 1)) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
        }
#pragma unroll
        for (int ma = 0; ma < kMA; ++ma) {
            if (WORK) multiply(ma, f1, acc);
#pragma unroll
            for (int i = 0; i < kReads; ++i)
                if (WORK && NEXT && i / R == ma) read(i, f0, smem + next * kStage, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (WORK) sum_up(f1, sum, with_sum);
        slot = next;
    }
};

}  // namespace
