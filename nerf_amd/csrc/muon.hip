// Orthogonalising a matrix by Newton-Schulz products, and the Muon update built on it.
//
//   X = G / max(|G|_F, eps);  `steps` times X <- (a I + b A + c A^2) X with A = X X^T   (X the wide orientation of G)
//
// A step maps every singular value s to a s + b s^3 + c s^5 and leaves the singular vectors: all of them are driven towards 1.
//
// Arithmetic.  Small singular values grow by a in every step (3.4445^5 = 485 with the usual coefficients) and rounding
// errors with them, so 8 significand bits per operand end 1.6e-2 off (256 x 256).  Every operand here is two fp16 terms of
// its value times 2^12, hi + lo (22 significand bits), every product hi.hi + hi.lo + lo.hi with fp32 sums: 1.8e-6 off
// float64 at 256 x 256, where the same iteration in fp32 is 1.7e-6 off.  X, A and Q = a I + b A + c A^2 are kept as those
// two terms between the products: the next product reads nothing finer, and with a I inside Q there is no other reader.
// The scale keeps lo a normal fp16 number for every entry above 2^-15 and the largest entry possible (|X| <= 1.3,
// |A| <= 1.6, |Q| <= 8 for the coefficients the entry points admit) below fp16's 65504.  |G|_F is summed in float64.
//
// Four paths, by the shorter side M and the longer side N:
//   M <= 32, N <= 128                       one wavefront per matrix, everything in registers (schulz_small_kernel);
//   M <= 64, N <= 544 and M <= 128, N <= 160  one workgroup per matrix, everything in LDS (schulz_block_kernel);
//   M <= 64, N <= 640 and M <= 128, N <= 320  the matrices' terms in the workspace, a launch per step (schulz_step_kernel), up to
//                                           256 pieces of 64 columns in all;
//   otherwise                               the same, three launches per step (schulz_product_kernel).
#include "dma_gemm.h"
#include "launch.h"
#include "split2h.h"

namespace {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr float kScale = 4096.f, kUnscale = 1.f / 4096.f;
constexpr int kMaxTensors = 32, kMaxSteps = 16;

struct Out32 {};
struct OutBf16 {};
struct OutFp16 {};
struct OutMuon {};   // g = the gradient (fp32), the parameters and the momentum updated in place
template <class T> struct Elem { typedef float type; };
template <> struct Elem<OutBf16> { typedef __bf16 type; };
template <> struct Elem<OutFp16> { typedef _Float16 type; };

struct SchulzArgs {
    const void* g[kMaxTensors];   // each (per, rows, cols)
    void* out[kMaxTensors];       // the orthogonalised matrices, or the parameters
    float* mom[kMaxTensors];
    int64_t batch;
    int per, rows, cols, steps, nesterov;
    float a, b, c, eps;
    float grad_scale, clip, mu, decay, rate;   // Muon: p <- decay p - rate O
};

__device__ __forceinline__ float clamp_grad(float g, const SchulzArgs& s) {
    g *= s.grad_scale;
    return g > s.clip ? s.clip : g < -s.clip ? -s.clip : g;   // NaN stays
}
// the matrix to orthogonalise, at element base + i of tensor t; Muon: from the gradient and the momentum before (NEW: after)
// its update.  With a uniform base and 32 bits of i an address costs one register.
template <class T, bool NEW>
__device__ __forceinline__ float element(const SchulzArgs& s, int t, int64_t base, unsigned i, float* momentum) {
    if constexpr (__is_same(T, OutMuon)) {
        const float g = clamp_grad((static_cast<const float*>(s.g[t]) + base)[i], s);
        const float old = (s.mom[t] + base)[i];
        const float m = NEW ? old : __fmaf_rn(s.mu, old, g);
        if (momentum) *momentum = m;
        return s.nesterov ? __fmaf_rn(s.mu, m, g) : m;
    } else {
        return float((static_cast<const typename Elem<T>::type*>(s.g[t]) + base)[i]);
    }
}
template <class T>
__device__ __forceinline__ void emit(const SchulzArgs& s, int t, int64_t base, unsigned i, float v, float old) {   // old: before<T>() of the element
    if constexpr (__is_same(T, OutMuon)) {
        (static_cast<float*>(s.out[t]) + base)[i] = __fmaf_rn(-s.rate, v, s.decay * old);
    } else {
        (static_cast<typename Elem<T>::type*>(s.out[t]) + base)[i] = (typename Elem<T>::type)v;
    }
}
template <class T>
__device__ __forceinline__ float before(const SchulzArgs& s, int t, int64_t base, unsigned i) {   // Muon: the parameter
    if constexpr (__is_same(T, OutMuon)) return (static_cast<const float*>(s.out[t]) + base)[i];
    else return 0.f;
}
// four consecutive elements, all of them there; rows may start anywhere
template <class T>
__device__ __forceinline__ void emit4(const SchulzArgs& s, int t, int64_t base, unsigned i, const f32x4& v) {
    typedef typename Elem<T>::type elem;
    typedef elem vec __attribute__((ext_vector_type(4), aligned(sizeof(elem))));
    vec* to = reinterpret_cast<vec*>(static_cast<elem*>(s.out[t]) + base + i);
    vec o;
    if constexpr (__is_same(T, OutMuon)) o = *to;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = __is_same(T, OutMuon) ? (elem)__fmaf_rn(-s.rate, v[r], s.decay * float(o[r])) : (elem)v[r];
    *to = o;
}
// 4096 / max(norm, eps); NaN for a norm that is not finite
__device__ __forceinline__ float start_scale(double sum, float eps) {
    double norm = sqrt(sum);
    if (norm < double(eps)) norm = double(eps);
    if (norm == double(INFINITY)) norm = double(NAN);
    return float(4096.0 / norm);
}

// a, b -> the packed pairs of their terms hi and lo (a, b already scaled).  The residual is taken from the packed word itself:
// written as a - float((_Float16)a), the compiler converts twice, once with the scaling folded in, and where the two round a tie
// apart lo belongs to another hi (2^-11 off, one entry in some thousands).  The residuals' asm may read an MFMA's result, for
// which the compiler adds no wait inside asm: it needs `hi`, and the conversion that makes it, the compiler's own, reads a and b
// first and waits.  So no asm in here may read a or b without `hi`.
__device__ __forceinline__ void split_pair_h2(float a, float b, unsigned& hi, unsigned& lo) {
    hi = pk_f16(a, b);
    lo = pk_f16(f16_residual_lo(a, hi), f16_residual_hi(b, hi));
}
__device__ __forceinline__ float pair_lo(unsigned w) { return float(__builtin_bit_cast(f16x2, w)[0]); }
__device__ __forceinline__ float pair_hi(unsigned w) { return float(__builtin_bit_cast(f16x2, w)[1]); }

// ---- one wavefront per matrix ------------------------------------------------------------------------------------------
// A 32 x 32 block V is held as an MFMA accumulator holds it: register t of lane (c, h) is V[acc_row(t, h)][c].  Its sixteen
// registers as two fragments of eight are, as either operand of v_mfma_f32_32x32x16_f16, the matrix P[r][k] = V[k][r] with k
// running through acc_row (both operands run through it alike).  So a symmetric V multiplies as it lies, and with X kept in
// both orientations (X_j: columns 32 j.. of X, Y_j = X_j^T) every product of a step is made from registers:
//   A = sum_j X_j X_j^T: operands Y_j, Y_j     A^2: A, A     X_j' = Q X_j: Q, X_j   (a tall matrix: Y_j' = Y_j Q: X_j, Q)
// The other orientation of the new X is turned through LDS (36-word rows: 16 single-word writes, 4 vector reads, no bank
// conflicts), not multiplied again: orientations that round apart would no longer damp each other's errors.
// 4096 of 32 x 63 take 33 us (66 MB: 13.5 us of HBM; MFMA 10 us; 300 conversions, permutes and sums per step of 36 MFMAs 10 us or more:
// the four matrices of a SIMD are in phase).
struct Frag {
    u32x4 hi[2], lo[2];
};
__device__ __forceinline__ Frag split_block(const f32x16& v) {
    Frag f;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unsigned hi, lo;
            split_pair_h2(v[8 * s + 2 * i], v[8 * s + 2 * i + 1], hi, lo);
            f.hi[s][i] = hi, f.lo[s][i] = lo;
        }
    return f;
}
__device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_g, a), __builtin_bit_cast(f16x8_g, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 product(const Frag& a, const Frag& b, f32x16 c) {
#pragma unroll
    for (int s = 0; s < 2; ++s) c = mfma32(a.hi[s], b.lo[s], c), c = mfma32(a.lo[s], b.hi[s], c);
#pragma unroll
    for (int s = 0; s < 2; ++s) c = mfma32(a.hi[s], b.hi[s], c);
    return c;
}
// A A with what the two terms of A leave out: rest = A - hi - lo as a third term, lo lo, hi rest and rest hi.  A is where
// rounding starts to be multiplied by b and c; with 22 bits in A's square a batch of 32 x 63 matrices was 1.1e-6 off float64,
// with these products it is as far off as the iteration in fp32.
__device__ __forceinline__ f32x16 square(const f32x16& v, const Frag& f) {
    u32x4 rest[2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = f16_residual_lo(f16_residual_lo(v[8 * s + 2 * i], f.hi[s][i]), f.lo[s][i]);
            const float b = f16_residual_hi(f16_residual_hi(v[8 * s + 2 * i + 1], f.hi[s][i]), f.lo[s][i]);
            rest[s][i] = pk_f16(a, b);
        }
    f32x16 c = {};
#pragma unroll
    for (int s = 0; s < 2; ++s) c = mfma32(f.hi[s], rest[s], c), c = mfma32(rest[s], f.hi[s], c), c = mfma32(f.lo[s], f.lo[s], c);
    return product(f, f, c);
}

constexpr int kTurnPitch = 36;
// the fragments of V^T from those of V: element pairs {hi, lo} as words through this wavefront's piece of LDS
__device__ __forceinline__ Frag turn_block(const Frag& f, unsigned* s_turn, int c, int h) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = 8 * s + 2 * i;
            s_turn[nrf::acc_row(t, h) * kTurnPitch + c] = __builtin_amdgcn_perm(f.lo[s][i], f.hi[s][i], 0x05040100u);
            s_turn[nrf::acc_row(t + 1, h) * kTurnPitch + c] = __builtin_amdgcn_perm(f.lo[s][i], f.hi[s][i], 0x07060302u);
        }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");   // one wavefront, LDS in order
    __builtin_amdgcn_wave_barrier();
    Frag o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {   // registers 4 j .. 4 j + 3: V[c][8 j + 4 h ..]
        const u32x4 w = *reinterpret_cast<const u32x4*>(s_turn + c * kTurnPitch + 8 * j + 4 * h);
        o.hi[j >> 1][2 * (j & 1)] = __builtin_amdgcn_perm(w[1], w[0], 0x05040100u);
        o.hi[j >> 1][2 * (j & 1) + 1] = __builtin_amdgcn_perm(w[3], w[2], 0x05040100u);
        o.lo[j >> 1][2 * (j & 1)] = __builtin_amdgcn_perm(w[1], w[0], 0x07060302u);
        o.lo[j >> 1][2 * (j & 1) + 1] = __builtin_amdgcn_perm(w[3], w[2], 0x07060302u);
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return o;
}

template <class T, int NB, bool TALL>
__global__ __launch_bounds__(256, NB == 1 ? 4 : (NB == 2 ? 4 : 3) - __is_same(T, OutMuon)) void schulz_small_kernel(SchulzArgs s) {
    __shared__ __align__(16) unsigned s_all[4][32 * kTurnPitch];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t m = int64_t(blockIdx.x) * 4 + wave;
    if (m >= s.batch) return;                      // no barrier below: every wavefront works alone
    unsigned* s_turn = s_all[wave];
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    const int t0 = int(m / s.per);
    const int64_t base = (m % s.per) * int64_t(s.rows) * s.cols;

    // G in blocks along its longer side, lanes along its rows: X_j of a wide matrix, Y_j of a tall one (X = G^T).  Every load
    // is made, at the nearest element there is: a load under a condition of its lanes would wait for the one before it
    f32x16 v[NB];
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const int r = (TALL ? 32 * j : 0) + nrf::acc_row(t, h), q = TALL ? c : 32 * j + c;
            const int rc = r < s.rows ? r : s.rows - 1, qc = q < s.cols ? q : s.cols - 1;
            float mom = 0.f;
            v[j][t] = element<T, false>(s, t0, base, rc * s.cols + qc, &mom);
            if (r != rc || q != qc) v[j][t] = 0.f;
            else if constexpr (__is_same(T, OutMuon)) (s.mom[t0] + base)[unsigned(r * s.cols + q)] = mom;
        }
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int t = 0; t < 16; ++t) sum = __builtin_fma(double(v[j][t]), double(v[j][t]), sum);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off);
    const float scale = start_scale(sum, s.eps);

    auto write = [&](int j, const f32x16& o) {     // the block's values, still at the scale
        int cols = s.cols;
        asm volatile("" : "+s"(cols) : : "memory");   // the offsets are computed again, not kept since the loads (Muon: 91 spills)
        const bool whole = TALL ? cols == 32 : s.rows == 32;   // every lane (row) of the shorter side is there
        float old[16];
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const int r = (TALL ? 32 * j : 0) + nrf::acc_row(t, h), q = TALL ? c : 32 * j + c;
            old[t] = before<T>(s, t0, base, (r < s.rows ? r : s.rows - 1) * cols + (q < cols ? q : cols - 1));
        }
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const int r = (TALL ? 32 * j : 0) + nrf::acc_row(t, h), q = TALL ? c : 32 * j + c;
            if ((whole || (TALL ? q < cols : r < s.rows)) && (TALL ? r < s.rows : q < cols))
                emit<T>(s, t0, base, r * cols + q, o[t] * kUnscale, old[t]);
        }
    };
    Frag here[NB];                                 // of X_j for a wide matrix, of Y_j for a tall one: all that a step keeps
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        if (s.steps == 0) write(j, v[j] * scale);
        else here[j] = split_block(v[j] * scale);
    }
    auto apply = [&](int j, const Frag& fq) {
        return TALL ? product(turn_block(here[j], s_turn, c, h), fq, (f32x16){}) : product(fq, here[j], (f32x16){});
    };
    for (int k = 1; k <= s.steps; ++k) {
        f32x16 acc = {};
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const Frag f = TALL ? here[j] : turn_block(here[j], s_turn, c, h);
            acc = product(f, f, acc);
        }
        const f32x16 gram = acc * kUnscale;
        acc = square(gram, split_block(gram));
        // Q without the scale (the matrix cores read subnormal terms: 2^-25 off at most), so that Q X has X's
        f32x16 poly = (s.b * kUnscale) * gram + (s.c * kUnscale * kUnscale) * acc;
#pragma unroll
        for (int t = 0; t < 16; ++t) poly[t] += nrf::acc_row(t, h) == c ? s.a : 0.f;
        const Frag fq = split_block(poly);
        if (k < s.steps) {
#pragma unroll
            for (int j = 0; j < NB; ++j) here[j] = split_block(apply(j, fq));
        } else {
#pragma unroll
            for (int j = 0; j < NB; ++j) write(j, apply(j, fq));
        }
    }
}

// The workspace of a matrix, in fp16 elements, M and N padded with zeros (which every product keeps) to the tile: X [2 terms]
// [M][N] and X^T [2][N][M], both twice (a step reads one and writes the other), A and Q [2][M][M].
struct LargeShape {
    int M, N, Mp, Np, tile, chunks, chunk;   // chunks: of the norm's sum, `chunk` elements each
    __host__ __device__ int64_t x_size() const { return int64_t(2) * Mp * Np; }
    __host__ __device__ int64_t s_size() const { return int64_t(2) * Mp * Mp; }
    __host__ __device__ int64_t per_matrix() const { return 4 * x_size() + 2 * s_size(); }
    __host__ __device__ int64_t x_at(int which) const { return which * 2 * x_size(); }
    __host__ __device__ int64_t xt_at(int which) const { return which * 2 * x_size() + x_size(); }
    __host__ __device__ int64_t gram_at() const { return 4 * x_size(); }
    __device__ float* parts(_Float16* w, int which) const { return reinterpret_cast<float*>(w + x_at(which ^ 1)); }
    __host__ __device__ int64_t poly_at() const { return 4 * x_size() + s_size(); }
};

// ---- one workgroup per matrix -------------------------------------------------------------------------------------------
// X, A and Q stay in LDS as their terms, rows padded by 16 B: X [2][16 MB][Np] and one square [2][16 MB][16 MB], A and then Q.  Only
// X itself is kept: A = X X^T reads its rows (k along them), X' = Q X its columns, turned on the way by ds_read_b64_tr_b16.  Eight
// wavefronts; a tile of A and of A^2 is one wavefront's, which so adds up Q from its own sums; a wavefront writes X' over the
// 16 columns that it alone read.  The LDS bounds a step (64 x 544: 1.5 MB of fragment reads, 5.3 of 7.4 us); 17 launches through the
// tiles below are worse at every size: 33 x 48 60 -> 16 us, 92 x 112 66 -> 47, 64 x 300 65 -> 35, 64 x 544 74 -> 53; 2000 of
// 64 x 64 305 -> 83, 1000 of 128 x 160 862 -> 245.
constexpr int kBlockWaves = 8, kLdsBytes = 160 * 1024;
struct BlockShape {
    int Np, pitch, square, bytes;                  // pitch of X's rows, of the square's, LDS in all; in bytes
    __host__ __device__ BlockShape(int N, int MB) : Np((N + 31) / 32 * 32), pitch(0), square(MB * 32 + 16), bytes(0) {
        pitch = Np * 2 + 16;
        bytes = 2 * 16 * MB * (pitch + square);
    }
};
__device__ __forceinline__ u32x4 block_rows(const char* plane, int pitch, int row, int k) {   // lane (c, q): row + c, k + 8 q ..
    const int c = threadIdx.x & 15, q = (threadIdx.x >> 4) & 3;
    return *reinterpret_cast<const u32x4*>(plane + (row + c) * pitch + (k + 8 * q) * 2);
}
__device__ __forceinline__ u32x4 block_cols(const char* plane, int pitch, int col, int k) {   // lane (c, q): col + c, k + 8 q ..
    const int c = threadIdx.x & 15, q = (threadIdx.x >> 4) & 3;
    s16x4_g part[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
        part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4_g*)(plane + (k + 8 * q + 4 * u + (c >> 2)) * pitch + col * 2 + (c & 3) * 8));
    return __builtin_bit_cast(u32x4, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
}
__device__ __forceinline__ f32x4 product16(const u32x4 (&a)[2], const u32x4 (&b)[2], f32x4 c) {
    c = mfma_dma<false>(a[0], b[1], c);
    c = mfma_dma<false>(a[1], b[0], c);
    return mfma_dma<false>(a[0], b[0], c);
}
__device__ __forceinline__ void block_store(char* at, int64_t plane, const f32x4& v) {
    unsigned h0, l0, h1, l1;
    split_pair_h2(v[0], v[1], h0, l0);
    split_pair_h2(v[2], v[3], h1, l1);
    *reinterpret_cast<u32x2*>(at) = (u32x2){h0, h1};
    *reinterpret_cast<u32x2*>(at + plane) = (u32x2){l0, l1};
}

// X'[row][col ..] to the output, what of it is there
template <class T>
__device__ __forceinline__ void block_emit(const SchulzArgs& s, int t, int64_t base, bool tall, int M, int N, int row, int col, const f32x4& v) {
    if (!tall && row < M && col + 3 < N) {
        emit4<T>(s, t, base, unsigned(row) * s.cols + col, v);       // (four stores of 4 B take 10 us more at 64 x 544)
        return;
    }
    unsigned at[4];
    float old[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const unsigned y = row < M ? row : M - 1, x = col + r < N ? col + r : N - 1;
        at[r] = tall ? x * s.cols + y : y * s.cols + x;
        old[r] = before<T>(s, t, base, at[r]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (row < M && col + r < N) emit<T>(s, t, base, at[r], v[r], old[r]);
}

template <class T, int MB>
__global__ __launch_bounds__(512) void schulz_block_kernel(SchulzArgs s, BlockShape L, unsigned by_cols) {
    extern __shared__ __align__(16) char smem[];
    constexpr int kJ = MB / 4, kI = MB * MB / kBlockWaves / kJ, kAhead = 8;   // kI x kJ tiles of A are a wavefront's (kI columns)
    const int64_t m = nrf::grid_block();
    if (m >= s.batch) return;
    const int t = int(m / s.per), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = threadIdx.x & 15, q = (threadIdx.x >> 4) & 3;
    const int count = s.rows * s.cols;
    const int64_t base = (m % s.per) * int64_t(count);
    const bool tall = s.rows > s.cols;
    const int M = tall ? s.cols : s.rows, N = tall ? s.rows : s.cols;
    const int plane_x = 16 * MB * L.pitch, plane_s = 16 * MB * L.square;
    char *xs = smem, *sq = smem + 2 * plane_x;

    for (int i = threadIdx.x * 16; i < 2 * plane_x; i += 512 * 16) *reinterpret_cast<u32x4*>(xs + i) = (u32x4){0, 0, 0, 0};
    double sum = 0.0;
    for (int i0 = threadIdx.x; i0 < count; i0 += 512 * kAhead) {
        float v[kAhead], mom[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + 512 * u;
            v[u] = element<T, false>(s, t, base, i < count ? i : count - 1, mom + u);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (i0 + 512 * u < count) {
                if constexpr (__is_same(T, OutMuon)) (s.mom[t] + base)[unsigned(i0 + 512 * u)] = mom[u];
                sum = __builtin_fma(double(v[u]), double(v[u]), sum);
            }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off);
    double* s_sum = reinterpret_cast<double*>(sq);
    if ((threadIdx.x & 63) == 0) s_sum[wave] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < kBlockWaves; ++w) sum += s_sum[w];
    const float scale = start_scale(sum, s.eps);
    // a second time (from the L2; a thread's own elements, as it left the momentum)
    for (int i0 = threadIdx.x; i0 < count; i0 += 512 * kAhead) {
        float v[kAhead], old[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + 512 * u < count ? i0 + 512 * u : count - 1;
            v[u] = element<T, true>(s, t, base, i, nullptr) * scale;
            old[u] = s.steps == 0 ? before<T>(s, t, base, i) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int i = i0 + 512 * u;
            if (i >= count) continue;
            const int r = by_cols ? int(__umulhi(i, by_cols)) : i, col = i - r * s.cols;
            unsigned hi, lo;
            split_pair_h2(v[u], 0.f, hi, lo);
            char* at = xs + (tall ? col : r) * L.pitch + (tall ? r : col) * 2;
            *reinterpret_cast<unsigned short*>(at) = (unsigned short)hi;
            *reinterpret_cast<unsigned short*>(at + plane_x) = (unsigned short)lo;
            if (s.steps == 0) emit<T>(s, t, base, i, v[u] * kUnscale, old[u]);
        }
    }
    const int j0 = wave / (MB / kI) * kJ, i0 = wave % (MB / kI) * kI;   // rows 16 j0 .. of A, columns 16 i0 ..
    // sums over 32 k of the wavefront's tiles of V V^T, V's rows at `from`
    auto square = [&](f32x4 (&sum)[kJ][kI], const char* from, int plane, int pitch, int n) {
        u32x4 b[kJ][2];
#pragma unroll
        for (int j = 0; j < kJ; ++j)
#pragma unroll
            for (int p = 0; p < 2; ++p) b[j][p] = block_rows(from + p * plane, pitch, 16 * (j0 + j), n);
#pragma unroll
        for (int i = 0; i < kI; ++i) {
            const u32x4 a[2] = {block_rows(from, pitch, 16 * (i0 + i), n), block_rows(from + plane, pitch, 16 * (i0 + i), n)};
#pragma unroll
            for (int j = 0; j < kJ; ++j) sum[j][i] = product16(a, b[j], sum[j][i]);
        }
    };
    char* mine = sq + (16 * j0 + c) * L.square + (16 * i0 + 4 * q) * 2;
    for (int k = 1; k <= s.steps; ++k) {
        __syncthreads();
        f32x4 gram[kJ][kI] = {}, v[kJ][kI] = {};
        for (int n = 0; n < L.Np; n += 32) square(gram, xs, plane_x, L.pitch, n);
#pragma unroll
        for (int j = 0; j < kJ; ++j)
#pragma unroll
            for (int i = 0; i < kI; ++i) {
                gram[j][i] = gram[j][i] * kUnscale;
                block_store(mine + 16 * j * L.square + 32 * i, plane_s, gram[j][i]);
            }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < 16 * MB; n += 32) square(v, sq, plane_s, L.square, n);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kJ; ++j)
#pragma unroll
            for (int i = 0; i < kI; ++i) {                         // Q without the scale, as in schulz_small_kernel
                f32x4 poly = (s.b * kUnscale) * gram[j][i] + (s.c * kUnscale * kUnscale) * v[j][i];
#pragma unroll
                for (int r = 0; r < 4; ++r) poly[r] += 16 * (i0 + i) + 4 * q + r == 16 * (j0 + j) + c ? s.a : 0.f;
                block_store(mine + 16 * j * L.square + 32 * i, plane_s, poly);
            }
        __syncthreads();
        for (int n = 16 * wave; n < N; n += 16 * kBlockWaves) {
            u32x4 x[MB / 2][2];
#pragma unroll
            for (int kk = 0; kk < MB / 2; ++kk)
#pragma unroll
                for (int p = 0; p < 2; ++p) x[kk][p] = block_cols(xs + p * plane_x, L.pitch, n, 32 * kk);
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                f32x4 o = {};
#pragma unroll
                for (int kk = 0; kk < MB / 2; ++kk) {
                    const u32x4 b[2] = {block_rows(sq, L.square, 16 * i, 32 * kk), block_rows(sq + plane_s, L.square, 16 * i, 32 * kk)};
                    o = product16(x[kk], b, o);
                }
                const int row = 16 * i + c, col = n + 4 * q;       // X'[row][col ..]
                if (k < s.steps) {
                    block_store(xs + row * L.pitch + col * 2, plane_x, o);
                } else {
                    block_emit<T>(s, t, base, tall, M, N, row, col, o * kUnscale);
                }
            }
        }
    }
}

// A whole step in one launch, for matrices of up to 128 rows that the kernel above has no LDS for: a workgroup per 64 columns of X.
// Each sums all of A = X X^T itself (X's 64-column pieces pass through a ring in LDS, its own piece stays), squares it, and
// multiplies its own columns: one launch per step for three, at the price of A's sums once per workgroup (0.7 us per piece at 128
// rows).  One round of workgroups, up to 10 pieces at 64 rows and 5 at 128: 64 x 600 80 -> 45 us, 128 x 200 73 -> 64, 2 of 128 x 283
// 75 -> 70, 50 of 128 x 300 106 -> 91.  At 128 rows one or two matrices are even with the tiles below at 384 columns (75 us both) and
// slower from 448 on (80 for 78; 640: 96 for 85), twenty are faster up to 640 (107 for 110); at 64 rows this way would win up to 1024
// columns where the pieces are one round (58 us for 90), even where they are two.
template <int MB> struct StepShape {
    typedef DmaSide<kRows, 16 * MB, 64, 2, kBlockWaves> Side;
    static constexpr int kSquare = MB * 32 + 16, kSquareBytes = 2 * 16 * MB * kSquare;
    static constexpr int kLds = Side::kBytes + (2 * Side::kBytes > kSquareBytes ? 2 * Side::kBytes : kSquareBytes);   // own piece; ring, then the square
};
template <class T, int MB, bool LAST>
__global__ __launch_bounds__(512) void schulz_step_kernel(SchulzArgs s, LargeShape L, _Float16* __restrict__ work, int which, int share) {
    typedef StepShape<MB> Shape;
    typedef typename Shape::Side Side;
    extern __shared__ __align__(16) char smem[];
    constexpr int kJ = MB / 4, kI = MB * MB / kBlockWaves / kJ, kSquare = Shape::kSquare, kPlaneS = 16 * MB * kSquare;
    const int pieces = L.Np / 64, unit = int(blockIdx.x & 7) * share + int(blockIdx.x >> 3);
    if (unit >= int(s.batch) * pieces) return;
    const int64_t m = unit / pieces;
    const int own = unit % pieces;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
    _Float16* w = work + m * L.per_matrix();
    const int64_t plane_x = int64_t(L.Mp) * L.Np;
    char *ring = smem + Side::kBytes, *sq = ring;
    const unsigned lds = lds_addr(smem) + wave * (Side::kPieces * 1024);
    Side side;
    side.start_rows(wave, lane, w + L.x_at(which), plane_x * 2, [&](int row) { return unsigned(row * L.Np) * 2u; });
    // piece i of the walk: its own first, then the others in their order through the two slots of the ring
    auto issue = [&](int i) {
        const int piece = i == 0 ? own : i <= own ? i - 1 : i;
        const unsigned to = lds + (i == 0 ? 0 : Side::kBytes * (1 + ((i - 1) & 1)));
#pragma unroll
        for (int j = 0; j < Side::kPieces; ++j) side.issue(j, wave, lane, to, 64, int64_t(piece) * 128, nullptr, 0u);
    };
    for (int i = 0; i < 3 && i < pieces; ++i) issue(i);
    const int j0 = wave / (MB / kI) * kJ, i0 = wave % (MB / kI) * kI;   // rows 16 j0 .. of A, columns 16 i0 ..
    f32x4 gram[kJ][kI] = {}, v[kJ][kI] = {};
    for (int i = 0; i < pieces; ++i) {
        // piece i has landed: one more may be in flight, two behind the first
        if (i == 0 && pieces >= 3) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * Side::kPieces) : "memory");
        else if (i + 1 < pieces) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(Side::kPieces) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        const char* from = i == 0 ? smem : ring + ((i - 1) & 1) * Side::kBytes;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            u32x4 b[kJ][2];
#pragma unroll
            for (int j = 0; j < kJ; ++j)
#pragma unroll
                for (int p = 0; p < 2; ++p) b[j][p] = Side::frag(from + p * Side::kPlane, 16 * j0, j, kk, c, q);
#pragma unroll
            for (int a_i = 0; a_i < kI; ++a_i) {
                const u32x4 a[2] = {Side::frag(from, 16 * i0, a_i, kk, c, q), Side::frag(from + Side::kPlane, 16 * i0, a_i, kk, c, q)};
#pragma unroll
                for (int j = 0; j < kJ; ++j) gram[j][a_i] = product16(a, b[j], gram[j][a_i]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();                                   // every wavefront holds what it read of this slot
        if (i >= 1 && i + 2 < pieces) issue(i + 2);
    }
    char* mine = sq + (16 * j0 + c) * kSquare + (16 * i0 + 4 * q) * 2;
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int i = 0; i < kI; ++i) {
            gram[j][i] = gram[j][i] * kUnscale;
            block_store(mine + 16 * j * kSquare + 32 * i, kPlaneS, gram[j][i]);
        }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < 16 * MB; n += 32) {
        u32x4 b[kJ][2];
#pragma unroll
        for (int j = 0; j < kJ; ++j)
#pragma unroll
            for (int p = 0; p < 2; ++p) b[j][p] = block_rows(sq + p * kPlaneS, kSquare, 16 * (j0 + j), n);
#pragma unroll
        for (int i = 0; i < kI; ++i) {
            const u32x4 a[2] = {block_rows(sq, kSquare, 16 * (i0 + i), n), block_rows(sq + kPlaneS, kSquare, 16 * (i0 + i), n)};
#pragma unroll
            for (int j = 0; j < kJ; ++j) v[j][i] = product16(a, b[j], v[j][i]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int i = 0; i < kI; ++i) {                                  // Q without the scale, as in schulz_small_kernel
            f32x4 poly = (s.b * kUnscale) * gram[j][i] + (s.c * kUnscale * kUnscale) * v[j][i];
#pragma unroll
            for (int r = 0; r < 4; ++r) poly[r] += 16 * (i0 + i) + 4 * q + r == 16 * (j0 + j) + c ? s.a : 0.f;
            block_store(mine + 16 * j * kSquare + 32 * i, kPlaneS, poly);
        }
    __syncthreads();
    // 16 columns and half of the rows per wavefront
    const int n = wave % 4 * 16, first = wave / 4 * (MB / 2);
    u32x4 x[MB / 2][2];
#pragma unroll
    for (int kk = 0; kk < MB / 2; ++kk)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            s16x4_g part[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int row = 32 * kk + 8 * q + 4 * u + (c >> 2), octet = (n / 8 + ((c & 3) >> 1)) ^ Side::swizzle(row);
                part[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s16x4_g*)(smem + p * Side::kPlane + row * 128 + octet * 16 + (c & 1) * 8));
            }
            x[kk][p] = __builtin_bit_cast(u32x4, __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
    const int t = int(m / s.per), col = own * 64 + n + 4 * q;
    const int64_t base = (m % s.per) * int64_t(s.rows) * s.cols;
    const bool tall = s.rows > s.cols;
#pragma unroll
    for (int i = 0; i < MB / 2; ++i) {
        f32x4 o = {};
#pragma unroll
        for (int kk = 0; kk < MB / 2; ++kk) {
            const u32x4 b[2] = {block_rows(sq, kSquare, 16 * (first + i), 32 * kk), block_rows(sq + kPlaneS, kSquare, 16 * (first + i), 32 * kk)};
            o = product16(x[kk], b, o);
        }
        const int row = 16 * (first + i) + c;                           // X'[row][col ..]
        if constexpr (!LAST) {
            block_store(reinterpret_cast<char*>(w + L.x_at(which ^ 1) + int64_t(row) * L.Np + col), plane_x * 2, o);
        } else {
            block_emit<T>(s, t, base, tall, L.M, L.N, row, col, o * kUnscale);
        }
    }
}

// ---- larger matrices ----------------------------------------------------------------------------------------------------
constexpr int kNormBatch = 8;       // elements of a thread at a time, all loaded before the first is used

// |G|_F^2 in L.chunks parts; Muon: the momentum's update.  2 of 1024 x 4096 in bf16: 6 us, 2.8 TB/s.
template <class T>
__global__ __launch_bounds__(256) void schulz_norm_kernel(SchulzArgs s, LargeShape L, double* __restrict__ parts) {
    const int64_t m = blockIdx.y, count = int64_t(s.rows) * s.cols;
    const int t = int(m / s.per);
    const int64_t base = (m % s.per) * count;
    const int64_t begin = int64_t(blockIdx.x) * L.chunk, end = begin + L.chunk < count ? begin + L.chunk : count;
    double sum = 0.0;
    for (int64_t i0 = begin; i0 < end; i0 += 256 * kNormBatch) {
        const unsigned left = unsigned(end - i0 < 256 * kNormBatch ? end - i0 : 256 * kNormBatch);
        float v[kNormBatch], mom[kNormBatch];
#pragma unroll
        for (int u = 0; u < kNormBatch; ++u) {
            const unsigned i = 256 * u + threadIdx.x;
            v[u] = element<T, false>(s, t, base + i0, i < left ? i : left - 1, mom + u);
        }
#pragma unroll
        for (int u = 0; u < kNormBatch; ++u) {
            const unsigned i = 256 * u + threadIdx.x;
            if (i >= left) continue;
            if constexpr (__is_same(T, OutMuon)) (s.mom[t] + base + i0)[i] = mom[u];
            sum = __builtin_fma(double(v[u]), double(v[u]), sum);
        }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off);
    __shared__ double s_sum[4];
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) parts[m * L.chunks + blockIdx.x] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
}

// X and X^T from G: one 64 x 64 tile of G's padded (rows, cols) per workgroup.  HBM bounds it: 2 of 1024 x 4096 (84 MB) 16 us, 5.2 TB/s.
template <class T>
__global__ __launch_bounds__(256) void schulz_start_kernel(SchulzArgs s, LargeShape L, const double* __restrict__ parts,
                                                           _Float16* __restrict__ work) {
    __shared__ float s_tile[64][65];
    const int64_t m = blockIdx.z, count = int64_t(s.rows) * s.cols;
    const bool tall = s.rows > s.cols;
    const int t = int(m / s.per), r0 = blockIdx.y * 64, q0 = blockIdx.x * 64;
    const int64_t base = (m % s.per) * count + int64_t(r0 < s.rows ? r0 : 0) * s.cols;
    const int lane = threadIdx.x & 63;
    double sum = 0.0;                                                // every wavefront for itself
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int i = 64 * u + lane;
        const double part = parts[m * L.chunks + (i < L.chunks ? i : 0)];
        sum += i < L.chunks ? part : 0.0;
    }
    const int q = (threadIdx.x & 31) * 2;                            // a pair of columns
    float v[8][2];
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = r0 + (threadIdx.x >> 5) + 8 * u, col = q0 + q + i;
            const bool in = r < s.rows && col < s.cols;
            const float x = element<T, true>(s, t, base, in ? unsigned(r - r0) * s.cols + col : 0u, nullptr);
            v[u][i] = in ? x : 0.f;
        }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off);
    const float scale = start_scale(sum, s.eps);
    const int rp = tall ? L.Np : L.Mp, cp = tall ? L.Mp : L.Np;      // padded rows and columns of G
    _Float16* w = work + m * L.per_matrix();
    _Float16* straight = w + (tall ? L.xt_at(0) : L.x_at(0));        // [rp][cp]
    _Float16* turned = w + (tall ? L.x_at(0) : L.xt_at(0));          // [cp][rp]
    unsigned *straight32 = reinterpret_cast<unsigned*>(straight), *turned32 = reinterpret_cast<unsigned*>(turned);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int r = (threadIdx.x >> 5) + 8 * u;
        v[u][0] *= scale, v[u][1] *= scale;
        s_tile[r][q] = v[u][0], s_tile[r][q + 1] = v[u][1];
        unsigned hi, lo;
        split_pair_h2(v[u][0], v[u][1], hi, lo);
        const int64_t at = int64_t(r0 + r) * cp + q0 + q;
        straight32[at >> 1] = hi, straight32[(int64_t(rp) * cp + at) >> 1] = lo;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int r = (threadIdx.x >> 5) + 8 * u;
        unsigned hi, lo;
        split_pair_h2(s_tile[q][r], s_tile[q + 1][r], hi, lo);
        const int64_t at = int64_t(q0 + r) * rp + r0 + q;
        turned32[at >> 1] = hi, turned32[(int64_t(rp) * cp + at) >> 1] = lo;
    }
}

enum Product { kGram, kPoly, kApply, kLast, kGramPart };

// 64 x 64 or 128 x 128 outputs by four wavefronts
template <int TT> using SchulzGemm = DmaGemm<false, kRows, kRows, TT, TT, 2, 2, 2, 2>;

// words[i] = {hi, lo} of eight consecutive elements -> 16 B of each plane
__device__ __forceinline__ void store_octet(_Float16* dst, int64_t plane, const unsigned (&w)[8]) {
    u32x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        hi[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05040100u);
        lo[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07060302u);
    }
    *reinterpret_cast<u32x4*>(dst) = hi;
    *reinterpret_cast<u32x4*>(dst + plane) = lo;
}

// A TT x TT tile of words {hi, lo} in LDS ([a][b], rows of TT + 1) to rows `row0 ..` and columns `col0 ..` of a matrix of
// `pitch`: its rows b (TURN) or its rows a, 16 B per lane and plane
template <int TT, bool TURN>
__device__ __forceinline__ void write_terms(const unsigned* s_out, _Float16* dst, int64_t plane, int pitch, int row0, int col0) {
#pragma unroll 4
    for (int i = threadIdx.x; i < TT * TT / 8; i += 256) {
        const int row = i / (TT / 8), col = i % (TT / 8) * 8;
        unsigned v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = s_out[TURN ? (col + j) * (TT + 1) + row : row * (TT + 1) + col + j];
        store_octet(dst + int64_t(row0 + row) * pitch + col0 + col, plane, v);
    }
}

// One product of a step: A = X X^T and Q = a I + b A + c A A (symmetric: the tiles on and over the diagonal, each written to
// both places), X' = Q X (to X' and X'^T; the last step: to the output).  Workgroups are dealt out to the XCDs in turn, so each
// XCD takes consecutive tiles, which share their operands' rows in its L2.  A finished tile goes through LDS (rows of TT + 1
// words), so that both orientations are written 16 B per lane: as the accumulators lie, a lane has 4 elements of one
// orientation and 1 of the other.
// 2 of 1024 x 4096: Q X 62 us (51.5 GFLOP of fp16 terms, 830 TFLOP/s; the 67 MB of X' and X'^T are a quarter of it), X X^T in three parts
// 37 us (700 TFLOP/s), Q 18 us; 14 of 256 x 256: 5.6, 6.4 and 6.6 us, launch and four steps.
template <class T, int WHAT, int TT>
__global__ __launch_bounds__(256) void schulz_product_kernel(SchulzArgs s, LargeShape L, _Float16* __restrict__ work, int which, int tiles, int share, int splits) {
    typedef SchulzGemm<TT> Gemm;
    constexpr bool kSym = WHAT == kGram || WHAT == kGramPart || WHAT == kPoly, kX = WHAT == kGram || WHAT == kGramPart;   // A or Q; of X X^T
    extern __shared__ __align__(16) char smem[];
    int unit = int(blockIdx.x & 7) * share + int(blockIdx.x >> 3);
    if (unit >= int(s.batch) * tiles * splits) return;
    const int split = unit / tiles % splits;          // of kGramPart: an XCD's units share a stretch of k
    const int64_t m = unit / (tiles * splits);
    _Float16* w = work + m * L.per_matrix();
    const int tiles_m = L.Mp / TT;
    int ta, tb;
    if (kSym) {   // tile pairs (ta <= tb), tb-th row has tb + 1
        int left = unit % tiles;
        for (tb = 0; left > tb; ++tb) left -= tb + 1;
        ta = left;
    } else {
        ta = unit % tiles % tiles_m, tb = unit % tiles / tiles_m;
    }
    const int a0 = ta * TT, b0 = tb * TT;
    const int K = kX ? L.Np : L.Mp;
    const int per = ((K / 64 + splits - 1) / splits) * 64, k0 = split * per < K ? split * per : K, count = K - k0 < per ? K - k0 : per;
    const _Float16* pa = w + (kX ? L.x_at(which) : WHAT == kPoly ? L.gram_at() : L.poly_at()) + k0;
    const _Float16* pb = w + (kX ? L.x_at(which) : WHAT == kPoly ? L.gram_at() : L.xt_at(which)) + k0;
    const int64_t plane_a = int64_t(L.Mp) * K, plane_b = int64_t(kSym ? L.Mp : L.Np) * K;
    Gemm gemm;
    // offsets inside a tile: at most 128 rows of 65536 terms
    gemm.a.start_rows(gemm.wave, gemm.lane, pa + int64_t(a0) * K, plane_a * 2, [&](int row) { return unsigned(row * K) * 2u; });
    gemm.b.start_rows(gemm.wave, gemm.lane, pb + int64_t(b0) * K, plane_b * 2, [&](int row) { return unsigned(row * K) * 2u; });
    f32x4 acc[Gemm::kMA][Gemm::kMB] = {};
    gemm.run(smem, count, acc);

    constexpr int kPitch = TT + 1;
    static_assert(TT * kPitch * 4 <= Gemm::kLds, "the tile in LDS");
    unsigned* s_out = reinterpret_cast<unsigned*>(smem);              // [a][b]
    const int c = gemm.lane & 15, q = gemm.lane >> 4, t = int(m / s.per);
    const int64_t plane = int64_t(L.Mp) * (kSym ? L.Mp : L.Np);
    if constexpr (WHAT == kGramPart) {   // a tile [b][a], in place of the next X (see gram_splits)
        float* part = L.parts(w, which) + (int64_t(split) * tiles + unit % tiles) * (TT * TT);
#pragma unroll
        for (int ma = 0; ma < Gemm::kMA; ++ma)
#pragma unroll
            for (int mb = 0; mb < Gemm::kMB; ++mb)
                *reinterpret_cast<f32x4*>(part + (gemm.wave_b() + 16 * mb + c) * TT + gemm.wave_a() + 16 * ma + 4 * q) = acc[ma][mb];
        return;
    }
    __syncthreads();
#pragma unroll
    for (int ma = 0; ma < Gemm::kMA; ++ma)
#pragma unroll
        for (int mb = 0; mb < Gemm::kMB; ++mb) {
            const int a = gemm.wave_a() + 16 * ma + 4 * q, b = gemm.wave_b() + 16 * mb + c;
            f32x4 v = acc[ma][mb] * kUnscale;
            if (WHAT == kPoly) {
                const int64_t at = int64_t(b0 + b) * L.Mp + a0 + a;
                const u32x2 hi = *reinterpret_cast<const u32x2*>(w + L.gram_at() + at);
                const u32x2 lo = *reinterpret_cast<const u32x2*>(w + L.gram_at() + plane + at);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float g = r & 1 ? pair_hi(hi[r >> 1]) + pair_hi(lo[r >> 1]) : pair_lo(hi[r >> 1]) + pair_lo(lo[r >> 1]);
                    v[r] = s.b * g + s.c * v[r] + (a0 + a + r == b0 + b ? s.a * kScale : 0.f);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                unsigned w0, w1;
                if (WHAT == kLast) {
                    w0 = __builtin_bit_cast(unsigned, v[r] * kUnscale), w1 = __builtin_bit_cast(unsigned, v[r + 1] * kUnscale);
                } else {
                    unsigned hi, lo;
                    split_pair_h2(v[r], v[r + 1], hi, lo);
                    w0 = __builtin_amdgcn_perm(lo, hi, 0x05040100u), w1 = __builtin_amdgcn_perm(lo, hi, 0x07060302u);
                }
                s_out[(a + r) * kPitch + b] = w0, s_out[(a + r + 1) * kPitch + b] = w1;
            }
        }
    __syncthreads();
    if constexpr (WHAT == kLast) {
        // lanes along the output's rows; a Muon step's parameters are loaded sixteen ahead, under no condition
        const bool tall = s.rows > s.cols;
        const int64_t base = (m % s.per) * int64_t(s.rows) * s.cols;
        const int r0 = tall ? b0 : a0, q0 = tall ? a0 : b0;
        constexpr int kAhead = 16;
        for (int i0 = 0; i0 < TT * TT; i0 += 256 * kAhead) {
            float old[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int i = i0 + 256 * u + int(threadIdx.x), r = r0 + i / TT, col = q0 + i % TT;
                old[u] = before<T>(s, t, base, unsigned(r < s.rows ? r : s.rows - 1) * s.cols + (col < s.cols ? col : s.cols - 1));
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int i = i0 + 256 * u + int(threadIdx.x), r = i / TT, col = i % TT;
                const float v = __builtin_bit_cast(float, s_out[tall ? col * kPitch + r : r * kPitch + col]);
                if (r0 + r < s.rows && q0 + col < s.cols) emit<T>(s, t, base, unsigned(r0 + r) * s.cols + q0 + col, v, old[u]);
            }
        }
    } else {
        _Float16* straight = w + (WHAT == kGram ? L.gram_at() : WHAT == kPoly ? L.poly_at() : L.xt_at(which ^ 1));   // rows b
        _Float16* turned = WHAT == kApply ? w + L.x_at(which ^ 1) : straight;                                        // rows a
        const int pitch_turned = WHAT == kApply ? L.Np : L.Mp;
        write_terms<TT, true>(s_out, straight, plane, L.Mp, b0, a0);
        if (WHAT == kApply || ta != tb) write_terms<TT, false>(s_out, turned, plane, pitch_turned, a0, b0);
    }
}

// A from its parts: one 64 x 64 block of a tile per workgroup (2 of 1024 x 1024 from 3 parts: 5.7 us, 3.9 TB/s)
template <int TT>
__global__ __launch_bounds__(256) void schulz_join_kernel(int64_t batch, LargeShape L, _Float16* __restrict__ work, int which, int tiles, int splits) {
    constexpr int kBlocks = TT / 64 * (TT / 64), kPitch = 65;
    __shared__ unsigned s_out[64 * kPitch];
    const int tile = blockIdx.x / kBlocks % tiles, block = blockIdx.x % kBlocks;
    const int64_t m = blockIdx.x / kBlocks / tiles;
    _Float16* w = work + m * L.per_matrix();
    int tb = 0, ta = tile;
    for (; ta > tb; ++tb) ta -= tb + 1;
    const int a_in = block % (TT / 64) * 64, b_in = block / (TT / 64) * 64, a = a_in + int(threadIdx.x & 15) * 4, row = threadIdx.x >> 4;
    const float* part = L.parts(w, which) + int64_t(tile) * (TT * TT) + a;
    f32x4 v[4] = {};
    for (int i = 0; i < splits; ++i, part += int64_t(tiles) * (TT * TT))
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] += *reinterpret_cast<const f32x4*>(part + (b_in + row + 16 * u) * TT);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        v[u] = v[u] * kUnscale;
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
            unsigned hi, lo;
            split_pair_h2(v[u][r], v[u][r + 1], hi, lo);
            unsigned* to = s_out + (a - a_in + r) * kPitch + row + 16 * u;
            to[0] = __builtin_amdgcn_perm(lo, hi, 0x05040100u), to[kPitch] = __builtin_amdgcn_perm(lo, hi, 0x07060302u);
        }
    }
    __syncthreads();
    write_terms<64, true>(s_out, w + L.gram_at(), int64_t(L.Mp) * L.Mp, L.Mp, tb * TT + b_in, ta * TT + a_in);
    if (ta != tb) write_terms<64, false>(s_out, w + L.gram_at(), int64_t(L.Mp) * L.Mp, L.Mp, ta * TT + a_in, tb * TT + b_in);
}

// no step at all: the scaled matrix itself
template <class T>
__global__ __launch_bounds__(256) void schulz_copy_kernel(SchulzArgs s, LargeShape L, const double* __restrict__ parts) {
    const int64_t m = blockIdx.y, count = int64_t(s.rows) * s.cols;
    double sum = 0.0;
    for (int i = 0; i < L.chunks; ++i) sum += parts[m * L.chunks + i];
    const float scale = start_scale(sum, s.eps);     // 1 / norm itself would be subnormal from norms of 8.5e37 on
    const int t = int(m / s.per);
    const int64_t base = (m % s.per) * count;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < count; i += int64_t(gridDim.x) * 256)
        emit<T>(s, t, base + i, 0, element<T, true>(s, t, base + i, 0, nullptr) * scale * kUnscale, before<T>(s, t, base + i, 0));
}

bool small_path(int rows, int cols) {
    const int lo = rows < cols ? rows : cols, hi = rows < cols ? cols : rows;
    return lo <= 32 && hi <= 128;
}

// the row blocks of the one-workgroup kernel that takes a matrix, 0 for none
int block_path(int rows, int cols) {
    const int lo = rows < cols ? rows : cols, hi = rows < cols ? cols : rows;
    for (int MB = 4; MB <= 8; MB += 4)
        if (lo <= 16 * MB && hi <= 1024 && BlockShape(hi, MB).bytes <= kLdsBytes) return MB;
    return 0;
}

LargeShape large_shape(int rows, int cols) {
    LargeShape L;
    L.M = rows < cols ? rows : cols, L.N = rows < cols ? cols : rows;
    L.tile = L.M > 512 ? 128 : 64;
    L.Mp = (L.M + L.tile - 1) / L.tile * L.tile, L.Np = (L.N + L.tile - 1) / L.tile * L.tile;
    // at most 512 parts, which every workgroup of schulz_start_kernel adds up again
    const int64_t count = int64_t(rows) * cols, least = 256 * kNormBatch;
    const int64_t times = (count + 512 * least - 1) / (512 * least);
    L.chunk = int(times * least);
    L.chunks = int((count + L.chunk - 1) / L.chunk);
    return L;
}

template <class T, bool TALL>
void launch_small(const SchulzArgs& s, hipStream_t stream) {
    const int longer = s.rows < s.cols ? s.cols : s.rows;
    const dim3 grid(unsigned((s.batch + 3) / 4));
    if (longer <= 32) schulz_small_kernel<T, 1, TALL><<<grid, 256, 0, stream>>>(s);
    else if (longer <= 64) schulz_small_kernel<T, 2, TALL><<<grid, 256, 0, stream>>>(s);
    else schulz_small_kernel<T, 4, TALL><<<grid, 256, 0, stream>>>(s);
}

template <class T, int MB>
int launch_block(const SchulzArgs& s, hipStream_t stream) {
    const BlockShape L(s.rows < s.cols ? s.cols : s.rows, MB);
    auto kernel = &schulz_block_kernel<T, MB>;
    if (L.bytes > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                               kLdsBytes) != hipSuccess)
        return NRF_ERR_LAUNCH;
    // i / cols = i * by_cols >> 32 for i < 2^32 / cols (an element's index is below 2^16); 0 for a single column
    kernel<<<nrf::grid_rows(s.batch), 512, L.bytes, stream>>>(s, L, s.cols == 1 ? 0u : unsigned((int64_t(1) << 32) / s.cols + 1));
    return NRF_OK;
}

template <class T, int WHAT, int TT>
int launch_tiles(const SchulzArgs& s, const LargeShape& L, _Float16* work, int which, hipStream_t stream, int splits = 1) {
    typedef SchulzGemm<TT> Gemm;
    const int m = L.Mp / TT, n = L.Np / TT;
    const int tiles = WHAT == kGram || WHAT == kGramPart || WHAT == kPoly ? m * (m + 1) / 2 : m * n;
    auto kernel = &schulz_product_kernel<T, WHAT, TT>;
    if (Gemm::kLds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                                  Gemm::kLds) != hipSuccess)
        return NRF_ERR_LAUNCH;
    // tiles of an XCD: whole matrices, the same for every product, while its 32 CUs have one tile each at most
    const int64_t whole = (s.batch + 7) / 8 * tiles;
    const int share = whole <= 32 && splits == 1 ? int(whole) : (int(s.batch) * tiles * splits + 7) / 8;
    kernel<<<8 * share, 256, Gemm::kLds, stream>>>(s, L, work, which, tiles, share, splits);
    return NRF_OK;
}

// Tiles of 128 x 128 read half as much as tiles of 64 x 64, but one of them holds a CU by itself (128 KiB of LDS): they are
// for products that have enough of them.
template <class T, int WHAT>
int launch_product(const SchulzArgs& s, const LargeShape& L, _Float16* work, int which, hipStream_t stream) {
    const int64_t m = L.Mp / 128, n = L.Np / 128;
    const int64_t tiles = (WHAT == kPoly ? m * (m + 1) / 2 : m * n) * s.batch;
    return L.tile == 128 && tiles >= 192 ? launch_tiles<T, WHAT, 128>(s, L, work, which, stream) : launch_tiles<T, WHAT, 64>(s, L, work, which, stream);
}
// A long k with few tiles is split, in shares of at least eight steps, until the tiles fill the chip.  The parts lie where the
// step's new X will: splits m (m + 1) / 2 tiles of fp32 within 8 Mp Np bytes.
int gram_splits(const SchulzArgs& s, const LargeShape& L) {
    const int64_t m = L.Mp / L.tile, tiles = m * (m + 1) / 2;
    int64_t splits = 256 / (tiles * s.batch);
    if (splits > L.Np / 512) splits = L.Np / 512;
    const int64_t room = 8 * int64_t(L.Mp) * L.Np / (tiles * L.tile * L.tile * 4);
    if (splits > room) splits = room;
    return splits < 2 ? 1 : int(splits);
}
template <int TT>
int launch_gram_parts(const SchulzArgs& s, const LargeShape& L, _Float16* work, int which, int splits, hipStream_t stream) {
    const int st = launch_tiles<Out32, kGramPart, TT>(s, L, work, which, stream, splits);
    if (st != NRF_OK) return st;
    const int tiles = L.Mp / TT * (L.Mp / TT + 1) / 2;
    schulz_join_kernel<TT><<<unsigned(s.batch * tiles * (TT / 64) * (TT / 64)), 256, 0, stream>>>(s.batch, L, work, which, tiles, splits);
    return NRF_OK;
}
int launch_gram(const SchulzArgs& s, const LargeShape& L, _Float16* work, int which, hipStream_t stream) {
    const int splits = gram_splits(s, L);
    const int64_t m = L.Mp / 128;
    if (splits > 1) return L.tile == 128 ? launch_gram_parts<128>(s, L, work, which, splits, stream) : launch_gram_parts<64>(s, L, work, which, splits, stream);
    return L.tile == 128 && m * (m + 1) / 2 * s.batch >= 192 ? launch_tiles<Out32, kGram, 128>(s, L, work, which, stream)
                                                             : launch_tiles<Out32, kGram, 64>(s, L, work, which, stream);
}

bool step_path(const SchulzArgs& s, const LargeShape& L) {
    return L.Mp <= 128 && L.Np <= (L.Mp == 64 ? 640 : 320) && s.batch * (L.Np / 64) <= 256;
}
template <class T, int MB, bool LAST>
int launch_step(const SchulzArgs& s, const LargeShape& L, _Float16* work, int which, hipStream_t stream) {
    auto kernel = &schulz_step_kernel<T, MB, LAST>;
    constexpr int lds = StepShape<MB>::kLds;
    if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds) != hipSuccess)
        return NRF_ERR_LAUNCH;
    const int pieces = L.Np / 64, whole = int((s.batch + 7) / 8) * pieces;   // whole matrices per XCD while they fit its CUs
    const int share = whole <= 32 ? whole : (int(s.batch) * pieces + 7) / 8;
    kernel<<<8 * share, 512, lds, stream>>>(s, L, work, which, share);
    return NRF_OK;
}
template <class T, int MB>
int run_steps(const SchulzArgs& s, const LargeShape& L, _Float16* work, hipStream_t stream) {
    for (int k = 0; k < s.steps; ++k) {
        const int st = k + 1 < s.steps ? launch_step<Out32, MB, false>(s, L, work, k & 1, stream) : launch_step<T, MB, true>(s, L, work, k & 1, stream);
        if (st != NRF_OK) return st;
    }
    return NRF_OK;
}
template <class T>
int run_large(const SchulzArgs& s, const LargeShape& L, double* parts, _Float16* work, hipStream_t stream) {
    const dim3 cover(unsigned((s.rows > s.cols ? L.Mp : L.Np) / 64), unsigned((s.rows > s.cols ? L.Np : L.Mp) / 64), unsigned(s.batch));
    schulz_norm_kernel<T><<<dim3(unsigned(L.chunks), unsigned(s.batch)), 256, 0, stream>>>(s, L, parts);
    if (s.steps == 0) {
        schulz_copy_kernel<T><<<dim3(unsigned(L.chunks), unsigned(s.batch)), 256, 0, stream>>>(s, L, parts);
        return NRF_OK;
    }
    schulz_start_kernel<T><<<cover, 256, 0, stream>>>(s, L, parts, work);
    if (step_path(s, L)) return L.Mp == 64 ? run_steps<T, 4>(s, L, work, stream) : run_steps<T, 8>(s, L, work, stream);
    for (int k = 0; k < s.steps; ++k) {
        int st = launch_gram(s, L, work, k & 1, stream);   // the output's type matters to kLast alone
        if (st == NRF_OK) st = launch_product<Out32, kPoly>(s, L, work, k & 1, stream);
        if (st == NRF_OK)
            st = k + 1 < s.steps ? launch_product<Out32, kApply>(s, L, work, k & 1, stream)
                                 : launch_product<T, kLast>(s, L, work, k & 1, stream);
        if (st != NRF_OK) return st;
    }
    return NRF_OK;
}

template <class T>
int run(const SchulzArgs& s, void* workspace, hipStream_t stream) {
    nrf_launch_begin();
    if (small_path(s.rows, s.cols)) {
        if (s.rows > s.cols) launch_small<T, true>(s, stream);
        else launch_small<T, false>(s, stream);
        return nrf_launch_status();
    }
    if (const int MB = block_path(s.rows, s.cols)) {
        const int st = MB == 4 ? launch_block<T, 4>(s, stream) : launch_block<T, 8>(s, stream);
        return st != NRF_OK ? st : nrf_launch_status();
    }
    const LargeShape L = large_shape(s.rows, s.cols);
    double* parts = static_cast<double*>(workspace);
    _Float16* work = reinterpret_cast<_Float16*>(parts + ((s.batch * L.chunks + 31) & ~int64_t(31)));
    const int st = run_large<T>(s, L, parts, work, stream);
    return st != NRF_OK ? st : nrf_launch_status();
}

bool schulz_shape_ok(int64_t batch, int rows, int cols) {
    if (batch < 0 || rows < 1 || cols < 1 || rows > 65536 || cols > 65536) return false;
    if (small_path(rows, cols) || block_path(rows, cols)) return batch <= int64_t(1) << 24;
    const LargeShape L = large_shape(rows, cols);       // (2^24 tiles are 1 TB of workspace: no launch comes near 2^32 work-items)
    return batch <= 65535 && batch * (int64_t(L.Mp / 64) * (L.Np / 64)) <= int64_t(1) << 24;
}
// the iteration on the singular values, which start in [0, 1]: entries of X, A and Q must stay inside fp16 at scale 2^12
bool coefficients_ok(int steps, float a, float b, float c) {
    if (steps < 0 || steps > kMaxSteps) return false;
    for (int i = 0; i <= 256; ++i) {
        double v = i / 256.0;
        for (int k = 0; k < steps; ++k) {
            const double q = a + (b + c * v * v) * v * v;
            v *= q;
            if (!(v >= -1.5 && v <= 1.5) || !(q >= -12.0 && q <= 12.0)) return false;
        }
    }
    return true;
}

}  // namespace

NRF_EXPORT int64_t nrf_newton_schulz_workspace_bytes(int64_t batch, int rows, int cols) {
    if (!schulz_shape_ok(batch, rows, cols)) return -1;
    if (small_path(rows, cols) || block_path(rows, cols)) return 0;
    const LargeShape L = large_shape(rows, cols);
    return ((batch * L.chunks + 31) & ~int64_t(31)) * 8 + batch * L.per_matrix() * 2;
}

NRF_EXPORT int nrf_newton_schulz(const void* g, void* out, int64_t batch, int rows, int cols, int dtype, int steps, float a,
                                 float b, float c, float eps, void* workspace, int64_t workspace_bytes, nrf_stream_t stream_) {
    const int64_t need = nrf_newton_schulz_workspace_bytes(batch, rows, cols);
    if (need < 0 || dtype < NRF_DTYPE_FP32 || dtype > NRF_DTYPE_FP16 || !(eps >= 1e-30f) || !coefficients_ok(steps, a, b, c))
        return NRF_ERR_SHAPE;
    if (batch == 0) return NRF_OK;
    if (!g || !out || (need > 0 && !workspace)) return NRF_ERR_NULL;
    if (workspace_bytes < need) return NRF_ERR_WORKSPACE;
    const uintptr_t low = dtype == NRF_DTYPE_FP32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(out)) & low || (need > 0 && !nrf_aligned16(workspace)))
        return NRF_ERR_ALIGN;
    const int64_t bytes = batch * rows * cols * (dtype == NRF_DTYPE_FP32 ? 4 : 2);
    if (g != out && nrf::overlap(g, bytes, out, bytes)) return NRF_ERR_SHAPE;   // one matrix' result over another's input
    SchulzArgs s{};
    s.g[0] = g, s.out[0] = out, s.batch = batch, s.per = int(batch), s.rows = rows, s.cols = cols, s.steps = steps;
    s.a = a, s.b = b, s.c = c, s.eps = eps;
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    if (dtype == NRF_DTYPE_FP32) return run<Out32>(s, workspace, stream);
    if (dtype == NRF_DTYPE_BF16) return run<OutBf16>(s, workspace, stream);
    return run<OutFp16>(s, workspace, stream);
}

NRF_EXPORT int nrf_muon_update(float* const* params, const float* const* grads, float* const* momentum, int n_tensors, int64_t batch,
                               int rows, int cols, float grad_scale, float clip_value, float mu, int nesterov, float lr,
                               float weight_decay, int steps, float a, float b, float c, float eps, void* workspace,
                               int64_t workspace_bytes, nrf_stream_t stream) {
    if (n_tensors < 0 || n_tensors > kMaxTensors || batch < 0 || batch > (int64_t(1) << 24)) return NRF_ERR_SHAPE;
    const int64_t need = nrf_newton_schulz_workspace_bytes(batch * n_tensors, rows, cols);
    if (need < 0 || !(eps >= 1e-30f) || !(clip_value > 0.f) || !(mu >= 0.f && mu < 1.f) || !coefficients_ok(steps, a, b, c)) return NRF_ERR_SHAPE;
    if (batch == 0 || n_tensors == 0) return NRF_OK;
    if (!params || !grads || !momentum || (need > 0 && !workspace)) return NRF_ERR_NULL;
    if (workspace_bytes < need) return NRF_ERR_WORKSPACE;
    if (need > 0 && !nrf_aligned16(workspace)) return NRF_ERR_ALIGN;
    SchulzArgs s{};
    for (int i = 0; i < n_tensors; ++i) {
        if (!params[i] || !grads[i] || !momentum[i]) return NRF_ERR_NULL;
        if ((reinterpret_cast<uintptr_t>(params[i]) | reinterpret_cast<uintptr_t>(grads[i]) | reinterpret_cast<uintptr_t>(momentum[i])) & 3)
            return NRF_ERR_ALIGN;
        s.g[i] = grads[i], s.out[i] = params[i], s.mom[i] = momentum[i];
    }
    const int64_t bytes = batch * rows * cols * 4;
    const auto shared = [bytes](const float* x, const float* y) { return nrf::overlap(x, bytes, y, bytes); };
    for (int i = 0; i < n_tensors; ++i)      // a tensor twice, or as gradient and momentum, or in parts: read while it is written
        for (int j = 0; j < n_tensors; ++j)
            if (shared(params[i], momentum[j]) || shared(params[i], grads[j]) || shared(momentum[i], grads[j]) ||
                (i != j && (shared(params[i], params[j]) || shared(momentum[i], momentum[j]))))
                return NRF_ERR_SHAPE;
    s.batch = batch * n_tensors, s.per = int(batch), s.rows = rows, s.cols = cols, s.steps = steps, s.nesterov = nesterov != 0;
    s.a = a, s.b = b, s.c = c, s.eps = eps, s.grad_scale = grad_scale, s.clip = clip_value, s.mu = mu;
    s.decay = float(1.0 - double(lr) * double(weight_decay));
    s.rate = float(double(lr) * sqrt(rows > cols ? double(rows) / cols : 1.0));
    return run<OutMuon>(s, workspace, static_cast<hipStream_t>(stream));
}
