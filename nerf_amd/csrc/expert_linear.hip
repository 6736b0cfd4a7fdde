// The experts' matrix products (experts.h: rows grouped by expert) and their gradients.
//
//   y[i] = act(W[e_i] x[i] + b[e_i])      dz[i] = dy[i] (y[i] > 0)      dx[i] = W[e_i]^T dz[i]
//   dW[e] = sum_{i of e} dz[i] x[i]^T     db[e] = sum_{i of e} dz[i]
//
// One kernel shape serves the three products: C[b][a] = sum_k B[b][k] A[a][k], A the side whose index is contiguous in the
// output (so a lane's four accumulator rows are one vector store), both operands staged in LDS as [row][k]:
//   forward   a = output feature (W rows)             b = batch row (x rows, gathered)       k = input
//   dx        a = input feature (W columns)           b = batch row (dz rows, gathered)      k = output
//   dW        a = input feature (x columns, gathered) b = output feature (dz columns)        k = the expert's batch rows
// bf16 / fp16 operands go to the matrix cores as they are, so do those of fp32 layers up to 64 x 64.  Other fp32 operands are split
// into three bf16 terms on their way into LDS (split3.h: 24 significand bits, six products, fp32 sums): one that is not finite
// gives NaN.  Sums are fp32; an output is rounded to its type once, after bias and relu.
#include "dma_gemm.h"
#include "experts.h"
#include "launch.h"
#include "split3.h"

namespace {

using nrf::PlanLayout;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
enum Form { kForward, kDx, kDw };

struct Bf16 {};
struct Fp16 {};
struct Fp32 {};
template <class T> struct Traits;
template <> struct Traits<Bf16> { typedef unsigned short elem; static constexpr int planes = 1; };
template <> struct Traits<Fp16> { typedef unsigned short elem; static constexpr int planes = 1; };
template <> struct Traits<Fp32> { typedef float elem; static constexpr int planes = 3; };

// eight consecutive elements; rows may start at any multiple of the element size (the hardware takes unaligned vectors)
typedef unsigned u32x4_u2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f32x4_u4 __attribute__((ext_vector_type(4), aligned(4)));
template <class T> struct Oct;
template <> struct Oct<Fp32> {
    f32x4 lo, hi;
    // the eight elements from p on, those before `end` (the tensor's) at least
    __device__ __forceinline__ void load(const float* p, const float* end) {
        if (p + 8 <= end) {
            lo = *reinterpret_cast<const f32x4_u4*>(p), hi = *reinterpret_cast<const f32x4_u4*>(p + 4);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) lo[j] = p + j < end ? p[j] : 0.f, hi[j] = p + 4 + j < end ? p[4 + j] : 0.f;
        }
    }
    __device__ __forceinline__ void limit(int valid) {   // zeros from element `valid` on
#pragma unroll
        for (int j = 0; j < 4; ++j) lo[j] = j < valid ? lo[j] : 0.f, hi[j] = 4 + j < valid ? hi[j] : 0.f;
    }
    __device__ __forceinline__ void keep_positive(const Oct& y) {
#pragma unroll
        for (int j = 0; j < 4; ++j) lo[j] = y.lo[j] > 0.f ? lo[j] : 0.f, hi[j] = y.hi[j] > 0.f ? hi[j] : 0.f;
    }
    // -> the eight elements of each bf16 term.  Elements that belong to different outputs (`apart`) are split each for itself, four more
    // instructions per pair: dot2 multiplies the pair's other element by zero, and one that is not finite would make NaN of both
    __device__ __forceinline__ void terms(const SplitSel& sel, bool apart, u32x4 (&out)[3]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = j < 2 ? lo[2 * j] : hi[2 * j - 4], b = j < 2 ? lo[2 * j + 1] : hi[2 * j - 3];
            unsigned p0, p1, p2;
            if (apart) split_pair(a, b, p0, p1, p2);
            else split_pair_dot2(sel, a, b, p0, p1, p2);
            out[0][j] = p0, out[1][j] = p1, out[2][j] = p2;
        }
    }
};
template <class T, unsigned INF> struct Oct16 {
    u32x4 v;
    __device__ __forceinline__ void load(const unsigned short* p, const unsigned short* end) {
        if (p + 8 <= end) {
            v = *reinterpret_cast<const u32x4_u2*>(p);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = (p + 2 * j < end ? unsigned(p[2 * j]) : 0u) | (p + 2 * j + 1 < end ? unsigned(p[2 * j + 1]) << 16 : 0u);
        }
    }
    __device__ __forceinline__ void limit(int valid) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] &= (2 * j < valid ? 0xffffu : 0u) | (2 * j + 1 < valid ? 0xffff0000u : 0u);
    }
    __device__ __forceinline__ void keep_positive(const Oct16& y) {   // positive: bits in 1 .. INF (NaN lies above)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned lo = y.v[j] & 0xffffu, hi = y.v[j] >> 16;
            v[j] &= (lo - 1u < INF ? 0xffffu : 0u) | (hi - 1u < INF ? 0xffff0000u : 0u);
        }
    }
    __device__ __forceinline__ void terms(const SplitSel&, bool, u32x4 (&out)[1]) const { out[0] = v; }
};
template <> struct Oct<Bf16> : Oct16<Bf16, 0x7f80u> {};
template <> struct Oct<Fp16> : Oct16<Fp16, 0x7c00u> {};

template <class T>
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
    if constexpr (__is_same(T, Fp16))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// the products of an operand pair's terms, small ones first
template <class T>
__device__ __forceinline__ f32x4 mfma_terms(const u32x4* a, const u32x4* b, f32x4 c) {
    if constexpr (Traits<T>::planes == 3) {
        c = mfma16<T>(a[0], b[2], c), c = mfma16<T>(a[1], b[1], c), c = mfma16<T>(a[2], b[0], c);
        c = mfma16<T>(a[0], b[1], c), c = mfma16<T>(a[1], b[0], c);
    }
    return mfma16<T>(a[0], b[0], c);
}

__device__ __forceinline__ float to_float(float v, Fp32) { return v; }
__device__ __forceinline__ float to_float(unsigned short v, Bf16) { return __uint_as_float(unsigned(v) << 16); }
__device__ __forceinline__ float to_float(unsigned short v, Fp16) { return float(__builtin_bit_cast(_Float16, v)); }
__device__ __forceinline__ float from_float(float v, Fp32) { return v; }
__device__ __forceinline__ unsigned short from_float(float v, Bf16) { return __builtin_bit_cast(unsigned short, (__bf16)v); }
__device__ __forceinline__ unsigned short from_float(float v, Fp16) { return __builtin_bit_cast(unsigned short, (_Float16)v); }

// four consecutive outputs, `valid` of them inside the row
template <class T>
__device__ __forceinline__ void store4(typename Traits<T>::elem* p, const f32x4& v, int valid) {
    typedef typename Traits<T>::elem elem;
    typedef elem vec __attribute__((ext_vector_type(4), aligned(sizeof(elem))));
    if (valid >= 4) {
        vec o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = from_float(v[j], T{});
        *reinterpret_cast<vec*>(p) = o;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < valid) p[j] = from_float(v[j], T{});
    }
}

// dW and db in parts (fp32, db behind dW): either of runs of at most kPartRows rows -- part (first place >> 8) + expert, no two
// runs share one; experts of a single run are written at once -- or `splits` equal shares of every expert's rows, part
// share * E + expert.  expert_sum_kernel adds an expert's parts in their order.
constexpr int kPartRows = 256, kPartTable = 3;
__host__ __device__ constexpr int64_t part_size(int n_in, int n_out) { return int64_t(n_out) * (n_in + 1); }

struct ExpertArgs {
    const void *x, *w, *bias, *y, *g;     // y: the saved outputs whose sign is the relu's mask, or NULL
    const int* plan;
    void *out, *db;                       // the product's output; db: dW only, may be NULL
    float* partial;                       // dW's parts
    int64_t n;
    int E, n_in, n_out, relu, splits;     // splits: 0 for parts by runs
};

// four consecutive outputs of a product, after bias and relu
template <class T>
__device__ __forceinline__ void finish_row(typename Traits<T>::elem* out, f32x4 v, int valid, const typename Traits<T>::elem* bias, int relu) {
    if (bias)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < valid) v[j] += to_float(bias[j], T{});
    if (relu)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = v[j] < 0.f ? 0.f : v[j];   // NaN stays
    store4<T>(out, v, valid);
}

// Consecutive workgroups go to different XCDs: each XCD takes a contiguous eighth of the long row runs and of the short
// ones (an expert's runs share its weights in that XCD's L2).  -> the `local`-th run of this one, -1 past its last.
__device__ __forceinline__ int xcd_run(const int* runs, int xcd, int local) {
    const int longs = runs[0], shorts = runs[1] - longs;
    int begin = int(int64_t(longs) * xcd / 8), end = int(int64_t(longs) * (xcd + 1) / 8);
    if (local < end - begin) return begin + local;
    local -= end - begin;
    begin = int(int64_t(shorts) * xcd / 8), end = int(int64_t(shorts) * (xcd + 1) / 8);
    return local < end - begin ? longs + begin + local : -1;
}
constexpr int64_t xcd_blocks(int64_t runs, int a_tiles) { return (runs / 8 + 2) * 8 * a_tiles; }

// The expert with the `rank`-th most rows (of at most 64; equal ones by number).  A tile of dW takes as long as its expert has
// rows, and the longest tiles have to begin first: begun by number, the CUs of 16 uneven experts were busy 67% of the time.
__device__ __forceinline__ int expert_of_rank(const int* counts, int E, int rank) {
    const int lane = threadIdx.x & 63, mine = lane < E ? counts[lane] : -1;
    int above = 0;
    for (int e = 0; e < E; ++e) {
        const int other = __builtin_amdgcn_readlane(mine, e);
        above += other > mine || (other == mine && e < lane);
    }
    return __ffsll((long long)__ballot(lane < E && above == rank)) - 1;
}

// dW's unit of this workgroup: which expert, which of its `tiles`.  Every XCD takes a contiguous eighth of each expert's tiles
// (whole experts per XCD leave the XCD of the two most popular of sixteen with twice the average: 172 us where this takes
// 99); fewer than eight go round.
__device__ __forceinline__ bool dw_unit(const int* counts, int E, int tiles, int block, int& expert, int& at) {
    const int local = block / 8, xcd = block % 8;
    if (tiles >= 8) {
        const int per = (tiles + 7) / 8;
        expert = local / per, at = int(int64_t(tiles) * xcd / 8) + local % per;
        if (at >= int(int64_t(tiles) * (xcd + 1) / 8)) return false;
    } else {
        expert = (local * 8 + xcd) / tiles, at = (local * 8 + xcd) % tiles;
    }
    if (expert >= E) return false;
    if (E <= 64) expert = expert_of_rank(counts, E, expert);
    return true;
}
int64_t dw_blocks(int64_t tiles, int E) { return tiles >= 8 ? E * ((tiles + 7) / 8) * 8 : (E * tiles + 7) / 8 * 8; }

// The general tile: TT x TT outputs (64 or 128), k in steps of 32 D, four wavefronts of a quarter each, the next step's loads in
// registers while this step is multiplied (D = 2 for 16-bit operands, whose 32 k are multiplied sooner than loaded).  Any size, any alignment.  The larger tile splits fp32 operands half as often per
// product (splitting 32 elements per thread and step takes about half as long as the step's 96 MFMAs; at 64 x 64 as long as its
// 24); the smaller one fills the chip with small problems.
constexpr int kK = 32, kPitch = kK + 8;   // LDS row pitch: 80 B, so that 16 rows' 16 B reads spread over the banks

template <class T, int FORM, int TT>
__global__ __launch_bounds__(256) void expert_tile_kernel(ExpertArgs g, int a_tiles, int b_tiles) {
    typedef typename Traits<T>::elem elem;
    constexpr int P = Traits<T>::planes, D = P == 1 ? 2 : 1, kSets = TT == 64 ? 2 : 1, kTable = TT == 64 ? 1 : 2, M = TT / 32;   // 16-row blocks per wave
    constexpr bool a_cols = FORM != kForward, b_cols = FORM == kDw;
    typedef DmaSide<kCols, TT, kK, 1, 4> Cols;
    constexpr int kPlaneA = TT * (a_cols ? kK : kPitch), kPlaneB = TT * (b_cols ? kK : kPitch), kStep = D * kK;
    __shared__ __align__(16) unsigned short s_a[D][P][kPlaneA], s_b[D][P][kPlaneB];
    __shared__ int s_rows[TT];            // forward / dx: the tile's batch rows
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, c = lane & 15, q = lane >> 4;
    const int wa = (wave & 1) * (TT / 2), wb = (wave >> 1) * (TT / 2);
    const PlanLayout L(g.n, g.E);
    const int* order = g.plan + L.order;

    int expert, a0, b0 = 0, b_count, k_begin = 0, k_end;   // a0: first A row = first output column
    const int n_a = FORM == kForward ? g.n_out : g.n_in;
    int64_t part = 0;                     // dW in parts: which
    bool in_parts = false;
    if (FORM == kDw && g.splits != 0) {
        int at;
        if (!dw_unit(g.plan, g.E, a_tiles * b_tiles * g.splits, nrf::grid_block(), expert, at)) return;
        const int split = at / (a_tiles * b_tiles), tile = at % (a_tiles * b_tiles);
        const int first = g.plan[L.offsets + expert], rows = g.plan[expert];
        const int per = (((rows + g.splits - 1) / g.splits) + kK - 1) / kK * kK;   // whole k steps
        k_begin = first + (split * per < rows ? split * per : rows);
        k_end = first + (split * per + per < rows ? split * per + per : rows);
        part = int64_t(split) * g.E + expert, in_parts = g.splits > 1;
        a0 = tile % a_tiles * TT, b0 = tile / a_tiles * TT;
    } else {                              // a run of rows, all of whose tiles are the same XCD's
        constexpr int table = FORM == kDw ? kPartTable : kTable;
        const int tiles = a_tiles * b_tiles, block = nrf::grid_block(), local = block / 8, tile = local % tiles;
        const int at = xcd_run(g.plan + L.runs + 2 * table, block % 8, local / tiles);
        if (at < 0) return;
        const int2 run = reinterpret_cast<const int2*>(g.plan + L.tiles[table])[at];
        b_count = run.y >> 16, expert = run.y & 0xffff;
        a0 = tile % a_tiles * TT, b0 = tile / a_tiles * TT;
        if (FORM == kDw) {
            if (expert == g.E) return;
            k_begin = run.x, k_end = run.x + b_count;
            part = (run.x >> 8) + expert, in_parts = g.plan[expert] > kPartRows;
        } else {
            if (t < TT) s_rows[t] = t < b_count ? order[run.x + t] : -1;
            __syncthreads();
            k_end = FORM == kForward ? g.n_in : g.n_out;
        }
    }
    if (FORM == kDw) b_count = g.n_out - b0 < TT ? g.n_out - b0 : TT;
    const bool none = FORM != kDw && expert == g.E;   // rows of no expert: zeros
    const int64_t w_off = int64_t(none ? 0 : expert) * g.n_out * g.n_in;
    const elem* w = static_cast<const elem*>(g.w) + w_off;
    const elem* x = static_cast<const elem*>(g.x);
    const elem* dy = static_cast<const elem*>(g.g);
    const elem* ys = static_cast<const elem*>(g.y);
    const SplitSel sel = SplitSel::make();

    // This thread's eight elements of a step and operand, kOcts times: along k for an operand whose k is contiguous, along the
    // tile's rows otherwise.  (16-bit: 64 k, eight lanes and 128 B of one row; rows that are 4 B aligned move 118 B/ns per CU so,
    // 67 with four lanes of 64 B.)  Rows past the operand's last one read a row that is there (their outputs are not stored),
    // octets may run on into the next row, and what lies past the end of k is zeroed on its way into LDS: no load stands under
    // a condition but at the very end of a tensor.
    const elem *w_end = w + int64_t(g.n_out) * g.n_in, *x_end = x + g.n * g.n_in, *dy_end = dy + g.n * g.n_out, *ys_end = ys + g.n * g.n_out;
    constexpr int kLanes = kStep / 8, kOcts = TT * kLanes / 256, kDown = 256 / kLanes, kAlong = TT / 8, kNext = 256 / kAlong;
    int my_row[kOcts], k_row[kOcts];
    const int kr = t / kLanes, kc = t % kLanes * 8;   // [TT rows][kLanes octets of k]: rows kr + kDown j
    const int ck = t / kAlong, cr = t % kAlong * 8;   // [kStep k][kAlong octets of rows]: k = ck + kNext j
#pragma unroll
    for (int j = 0; j < kOcts; ++j) {
        my_row[j] = FORM == kDw ? 0 : s_rows[kr + kDown * j] < 0 ? s_rows[0] : s_rows[kr + kDown * j];
        k_row[j] = 0;
    }
    // dW: the batch rows of a step, looked up a step before its loads
    auto look_up = [&](int k0) {
        if (FORM == kDw)
#pragma unroll
            for (int j = 0; j < kOcts; ++j) k_row[j] = order[k0 + ck + kNext * j < k_end ? k0 + ck + kNext * j : k_end - 1];
    };
    auto load_a = [&](Oct<T>& v, int j, int k0) {
        const int row = a0 + kr + kDown * j, k = k0 + ck + kNext * j, col = a0 + cr < n_a ? a0 + cr : 0;
        if (FORM == kForward) v.load(w + int64_t(row < n_a ? row : n_a - 1) * g.n_in + (k0 + kc < k_end ? k0 + kc : 0), w_end);
        else if (FORM == kDx) v.load(w + int64_t(k < k_end ? k : 0) * g.n_in + col, w_end);
        else v.load(x + int64_t(k_row[j]) * g.n_in + col, x_end);
    };
    auto load_b = [&](Oct<T>& v, Oct<T>& s, int j, int k0) {
        if (FORM == kForward) {
            v.load(x + int64_t(my_row[j]) * g.n_in + (k0 + kc < k_end ? k0 + kc : 0), x_end);
            return;
        }
        const int64_t at = FORM == kDx ? int64_t(my_row[j]) * g.n_out + (k0 + kc < k_end ? k0 + kc : 0)
                                       : int64_t(k_row[j]) * g.n_out + (cr < b_count ? b0 + cr : 0);
        v.load(dy + at, dy_end);
        if (g.relu) s.load(ys + at, ys_end);
    };
    // LDS holds, per 32 k, [row][k] (pitch kPitch) of an operand whose k is contiguous, [k][row] of the others, read back transposed
    auto stage = [&](unsigned short* s, int plane, Oct<T> v, int j, int k0, bool cols) {
        const int k = cols ? ck + kNext * j : kc, row = cols ? cr : kr + kDown * j;
        if (k0 + kStep > k_end) v.limit(cols ? (k0 + k < k_end ? 8 : 0) : k_end - k0 - k);
        u32x4 p[P];
        v.terms(sel, cols, p);
        unsigned short* to = s + k / kK * (P * plane) + (cols ? k % kK * TT + ((row / 8) ^ Cols::swizzle(k % kK)) * 8 : row * kPitch + k % kK);
#pragma unroll
        for (int i = 0; i < P; ++i) *reinterpret_cast<u32x4*>(to + i * plane) = p[i];
    };
    auto fragment = [&](const unsigned short* s, int first, int m, bool cols) {
        return cols ? __builtin_bit_cast(u32x4, Cols::frag(reinterpret_cast<const char*>(s), first, m, 0, c, q))
                    : *reinterpret_cast<const u32x4*>(&s[(first + 16 * m + c) * kPitch + 8 * q]);
    };

    f32x4 acc[M][M] = {};
    f32x4 sum[M] = {};                                // dW: db of this wavefront's outputs
    const bool with_db = FORM == kDw && g.db && a0 == 0 && wa == 0;
    const unsigned one = __is_same(T, Fp16) ? 0x3c003c00u : 0x3f803f80u;
    const u32x4 ones = {one, one, one, one};
    if (!none && k_begin < k_end) {
        struct Step {                                 // a step's octets, on their way
            Oct<T> a[kOcts], b[kOcts], s[kOcts];
        };
        auto load = [&](Step& r, int k0) {
#pragma unroll
            for (int j = 0; j < kOcts; ++j) load_a(r.a[j], j, k0), load_b(r.b[j], r.s[j], j, k0);
        };
        auto walk = [&](Step& r, int k0) {
#pragma unroll
            for (int j = 0; j < kOcts; ++j) {
                stage(s_a[0][0], kPlaneA, r.a[j], j, k0, a_cols);
                if (FORM != kForward && g.relu) r.b[j].keep_positive(r.s[j]);
                stage(s_b[0][0], kPlaneB, r.b[j], j, k0, b_cols);
            }
            __syncthreads();
            if (k0 + kSets * kStep < k_end) {
                load(r, k0 + kSets * kStep);
                look_up(k0 + (kSets + 1) * kStep);
            }
#pragma unroll
            for (int d = 0; d < D; ++d) {
                if (d > 0 && k0 + d * kK >= k_end) break;
                u32x4 fb[M][P];
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int i = 0; i < P; ++i) fb[m][i] = fragment(s_b[d][i], wb, m, b_cols);
#pragma unroll
                for (int ma = 0; ma < M; ++ma) {
                    u32x4 fa[P];
#pragma unroll
                    for (int i = 0; i < P; ++i) fa[i] = fragment(s_a[d][i], wa, ma, a_cols);
#pragma unroll
                    for (int mb = 0; mb < M; ++mb) {
                        // fp32: a step's six products among themselves, then one rounding at the size of the whole sum, not six
                        // (200 rows of 1000 -> 300: 1.2e-7 off float64 for 4.8e-7; dW's tile of 128 has no registers left for it)
                        if constexpr (P == 3 && (FORM != kDw || TT == 64)) acc[ma][mb] = acc[ma][mb] + mfma_terms<T>(fa, fb[mb], (f32x4){});
                        else acc[ma][mb] = mfma_terms<T>(fa, fb[mb], acc[ma][mb]);
                    }
                }
                if (with_db)
#pragma unroll
                    for (int mb = 0; mb < M; ++mb)
#pragma unroll
                        for (int i = P - 1; i >= 0; --i) sum[mb] = mfma16<T>(ones, fb[mb][i], sum[mb]);
            }
            __syncthreads();
        };
        Step r[kSets];
        look_up(k_begin);
#pragma unroll
        for (int u = 0; u < kSets; ++u) {
            load(r[u], k_begin + u * kStep);
            look_up(k_begin + (u + 1) * kStep);
        }
        for (int k0 = k_begin; k0 < k_end; k0 += kSets * kStep)
#pragma unroll
            for (int u = 0; u < kSets; ++u)
                if (u == 0 || k0 + u * kStep < k_end) walk(r[u], k0 + u * kStep);
    }

    // lane (c, q) holds outputs a0 + wa + 16 ma + 4 q .. + 3 of b row wb + 16 mb + c
#pragma unroll
    for (int mb = 0; mb < M; ++mb) {
        const int br = wb + 16 * mb + c;
        if (br >= b_count) continue;
#pragma unroll
        for (int ma = 0; ma < M; ++ma) {
            const int a = a0 + wa + 16 * ma + 4 * q, valid = n_a - a;
            if (valid <= 0) continue;
            if (FORM == kDw) {
                const int64_t at = int64_t(b0 + br) * g.n_in + a, size = int64_t(g.n_out) * g.n_in;
                if (in_parts) store4<Fp32>(g.partial + part * (size + g.n_out) + at, acc[ma][mb], valid);
                else store4<T>(static_cast<elem*>(g.out) + expert * size + at, acc[ma][mb], valid);
            } else {
                const elem* bias = FORM == kForward && g.bias && !none ? static_cast<const elem*>(g.bias) + int64_t(expert) * g.n_out + a : nullptr;
                finish_row<T>(static_cast<elem*>(g.out) + int64_t(s_rows[br]) * n_a + a, acc[ma][mb], valid, bias, FORM == kForward ? g.relu : 0);
            }
        }
        if (with_db && q == 0) {
            const int64_t size = int64_t(g.n_out) * g.n_in;
            if (in_parts) g.partial[part * (size + g.n_out) + size + b0 + br] = sum[mb][0];
            else static_cast<elem*>(g.db)[int64_t(expert) * g.n_out + b0 + br] = from_float(sum[mb][0], T{});
        }
    }
}

// ---- bf16 / fp16, wide layers ----------------------------------------------------------------------------------------------
// Forward and dx: 256 output columns by a run of batch rows, eight wavefronts.  Runs of more than 128 rows: 256 x 256, 128 x 64
// per wavefront (12 KiB of LDS reads to 32 MFMAs), two steps of 64 k in LDS (128 KiB).  Shorter runs wait for data, not for the
// matrix cores: 256 x 128 with three steps in LDS, 256 x 64 with four, so that more of the weights is on its way (a run of 64
// rows through the 256 x 256 form takes three quarters of a whole run's time).  dx reads the weights' columns (DmaGemm: kCols),
// whose transposing reads need registers that the 256 x 256 form has not left: its runs are of 128 rows; so are the forward's
// where 256 would leave the chip less than two workgroups per CU (dx of 16 k rows, 16 experts, 1536 -> 1024: 92 us, 116 in runs
// of 256).  g.g holds dz.
constexpr int kWideA = 256;
template <class T, int FORM, int ROWS> struct WideRows {
    static constexpr int kWA = ROWS == 256 ? 2 : 4, kST = ROWS == 256 ? 2 : ROWS == 128 ? 3 : 4;
    typedef DmaGemm<__is_same(T, Bf16), FORM == kForward ? kRows : kCols, kRows, kWideA, ROWS, kWA, 8 / kWA, 1, kST> Gemm;
};
constexpr int kWideLds = 4 * (256 + 64) * 128;   // of the 256 x 64 form, the largest

template <class T, int FORM, int ROWS>
__device__ __forceinline__ void wide_rows_tile(const ExpertArgs& g, char* smem, int a0, int b_count, int expert, const int* order) {
    typedef typename WideRows<T, FORM, ROWS>::Gemm Gemm;
    typedef unsigned short elem;
    static_assert(Gemm::kLds <= kWideLds && Gemm::kThreads == 512, "one launch for all forms");
    const bool none = expert == g.E;
    const int n_a = FORM == kForward ? g.n_out : g.n_in, n_k = FORM == kForward ? g.n_in : g.n_out;
    const elem* w = static_cast<const elem*>(g.w) + int64_t(none ? 0 : expert) * g.n_out * g.n_in;
    Gemm gemm;
    f32x4 acc[Gemm::kMA][Gemm::kMB] = {};
    if (!none) {
        const unsigned pitch = unsigned(n_k) * 2u;
        if constexpr (FORM == kForward) {
            gemm.a.start_rows(gemm.wave, gemm.lane, w, 0, [&](int row) { return unsigned(a0 + row < n_a ? a0 + row : n_a - 1) * pitch; });
        } else {
            gemm.pitch_a = unsigned(n_a) * 2u, gemm.step_a = int64_t(n_a) * 128;
            gemm.a.start_cols(gemm.wave, gemm.lane, w + a0, gemm.pitch_a, (n_a - a0) / 8);
        }
        gemm.b.start_rows(gemm.wave, gemm.lane, FORM == kForward ? g.x : g.g, 0, [&](int row) { return unsigned(order[row < b_count ? row : 0]) * pitch; });
        gemm.idle = gemm.wave_b() >= b_count || a0 + gemm.wave_a() >= n_a;
        gemm.run(smem, n_k, acc);
    }
    const int c = gemm.lane & 15, q = gemm.lane >> 4;
#pragma unroll
    for (int mb = 0; mb < Gemm::kMB; ++mb) {
        const int br = gemm.wave_b() + 16 * mb + c;
        if (br >= b_count) continue;
        elem* out = static_cast<elem*>(g.out) + int64_t(order[br]) * n_a;
#pragma unroll
        for (int ma = 0; ma < Gemm::kMA; ++ma) {
            const int a = a0 + gemm.wave_a() + 16 * ma + 4 * q, valid = n_a - a;
            if (valid <= 0) continue;
            const elem* bias = FORM == kForward && g.bias && !none ? static_cast<const elem*>(g.bias) + int64_t(expert) * g.n_out + a : nullptr;
            finish_row<T>(out + a, acc[ma][mb], valid, bias, FORM == kForward ? g.relu : 0);
        }
    }
}
template <class T, int FORM, int ROWS>   // runs of at most ROWS rows
__global__ __launch_bounds__(512) void expert_wide_rows_kernel(ExpertArgs g, int a_tiles) {
    extern __shared__ __align__(16) char smem[];
    constexpr int table = ROWS == 256 ? 3 : 2;
    const PlanLayout L(g.n, g.E);
    const int local = blockIdx.x / 8, at = xcd_run(g.plan + L.runs + 2 * table, blockIdx.x % 8, local / a_tiles);
    if (at < 0) return;
    const int2 tile = reinterpret_cast<const int2*>(g.plan + L.tiles[table])[at];
    const int b_count = tile.y >> 16, expert = tile.y & 0xffff, a0 = local % a_tiles * kWideA;
    const int* order = g.plan + L.order + tile.x;
    if (ROWS == 256 && b_count > 128) wide_rows_tile<T, FORM, ROWS>(g, smem, a0, b_count, expert, order);
    else if (b_count > 64) wide_rows_tile<T, FORM, 128>(g, smem, a0, b_count, expert, order);
    else wide_rows_tile<T, FORM, 64>(g, smem, a0, b_count, expert, order);
}

// dW: 256 input columns x 128 output columns, k the expert's rows through the list of them in LDS, kListRows at a time.
constexpr int kListRows = 4096;
template <class T> struct WideDw {
    static constexpr int kA = 256, kB = 128;
    typedef DmaGemm<__is_same(T, Bf16), kGather, kGather, kA, kB, 4, 2, 1, 2, true> Gemm;
    static constexpr int kLds = Gemm::kLds + kListRows * 4;
};
template <class T>
__global__ __launch_bounds__(512) void expert_wide_dw_kernel(ExpertArgs g, int a_tiles, int b_tiles) {
    typedef WideDw<T> W;
    typedef typename W::Gemm Gemm;
    typedef unsigned short elem;
    extern __shared__ __align__(16) char smem[];
    int* s_list = reinterpret_cast<int*>(smem + Gemm::kLds);
    const PlanLayout L(g.n, g.E);
    int expert, at;
    if (!dw_unit(g.plan, g.E, a_tiles * b_tiles * g.splits, blockIdx.x, expert, at)) return;
    const int split = at / (a_tiles * b_tiles), tile = at % (a_tiles * b_tiles);
    const int a0 = tile % a_tiles * W::kA, b0 = tile / a_tiles * W::kB;
    const int rows = g.plan[expert], per = ((rows + g.splits - 1) / g.splits + 63) / 64 * 64;
    const int begin = split * per < rows ? split * per : rows, end = begin + per < rows ? begin + per : rows;
    const int* order = g.plan + L.order + g.plan[L.offsets + expert];
    Gemm gemm;
    f32x4 acc[Gemm::kMA][Gemm::kMB] = {}, sum[Gemm::kMB] = {};
    gemm.pitch_a = unsigned(g.n_in) * 2u, gemm.pitch_b = unsigned(g.n_out) * 2u;
    gemm.a.start_cols(gemm.wave, gemm.lane, static_cast<const elem*>(g.x) + a0, 0, (g.n_in - a0) / 8);
    gemm.b.start_cols(gemm.wave, gemm.lane, static_cast<const elem*>(g.g) + b0, 0, (g.n_out - b0) / 8);
    gemm.idle = b0 + gemm.wave_b() >= g.n_out || a0 + gemm.wave_a() >= g.n_in;
    const bool with_db = g.db && a0 == 0 && gemm.wave_a() == 0;
    for (int r0 = begin; r0 < end; r0 += kListRows) {
        const int count = end - r0 < kListRows ? end - r0 : kListRows;
        __syncthreads();
        for (int i = threadIdx.x; i < count; i += 512) s_list[i] = order[r0 + i];
        __syncthreads();
        gemm.run(smem, count, acc, s_list, &sum, with_db);
    }
    const int c = gemm.lane & 15, q = gemm.lane >> 4;
    const int64_t size = int64_t(g.n_out) * g.n_in;
    float* part = g.partial + (int64_t(split) * g.E + expert) * part_size(g.n_in, g.n_out);
#pragma unroll
    for (int mb = 0; mb < Gemm::kMB; ++mb) {
        const int br = b0 + gemm.wave_b() + 16 * mb + c;
        if (br >= g.n_out) continue;
#pragma unroll
        for (int ma = 0; ma < Gemm::kMA; ++ma) {
            const int a = a0 + gemm.wave_a() + 16 * ma + 4 * q, valid = g.n_in - a;
            if (valid <= 0) continue;
            const int64_t at = int64_t(br) * g.n_in + a;
            if (g.splits > 1) store4<Fp32>(part + at, acc[ma][mb], valid);
            else store4<T>(static_cast<elem*>(g.out) + expert * size + at, acc[ma][mb], valid);
        }
        if (with_db && q == 0) {
            if (g.splits > 1) part[size + br] = sum[mb][0];
            else static_cast<elem*>(g.db)[int64_t(expert) * g.n_out + br] = from_float(sum[mb][0], T{});
        }
    }
}

// dz = dy where y > 0: read twice by the products, which move their operands without looking at them.  HBM bounds it: 16 k rows of
// 1536 in fp16 (151 MB) take 25 us, 6.0 TB/s.
template <class T>
__global__ __launch_bounds__(256) void expert_mask_kernel(const u32x4* __restrict__ dy, const u32x4* __restrict__ y, int64_t octets,
                                                          u32x4* __restrict__ dz) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < octets; i += int64_t(gridDim.x) * 256) {
        Oct<T> v, s;
        v.v = dy[i], s.v = y[i];
        v.keep_positive(s);
        dz[i] = v.v;
    }
}

int allow_lds(const void* kernel, int bytes) {
    return bytes <= 65536 || hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess ? NRF_OK : NRF_ERR_LAUNCH;
}

template <class T, int FORM, int ROWS>
int launch_wide_rows(const ExpertArgs& g, hipStream_t stream) {
    const int a_tiles = ((FORM == kForward ? g.n_out : g.n_in) + kWideA - 1) / kWideA;
    auto kernel = &expert_wide_rows_kernel<T, FORM, ROWS>;
    const int st = allow_lds(reinterpret_cast<const void*>(kernel), kWideLds);
    if (st != NRF_OK) return st;
    const int64_t blocks = xcd_blocks(PlanLayout::most_runs(g.n, g.E, ROWS == 256 ? 3 : 2), a_tiles);   // under 2^23 (wide)
    kernel<<<dim3(unsigned(blocks)), 512, kWideLds, stream>>>(g, a_tiles);
    return NRF_OK;
}
template <class T>
int launch_wide_forward(const ExpertArgs& g, hipStream_t stream) {
    const int64_t tiles = (g.n / 256 + (g.E < g.n ? g.E : g.n) / 2) * ((g.n_out + kWideA - 1) / kWideA);
    return tiles < 512 ? launch_wide_rows<T, kForward, 128>(g, stream) : launch_wide_rows<T, kForward, 256>(g, stream);
}
template <class T>
int launch_wide_dw(const ExpertArgs& g, hipStream_t stream) {
    typedef WideDw<T> W;
    const int a_tiles = (g.n_in + W::kA - 1) / W::kA, b_tiles = (g.n_out + W::kB - 1) / W::kB;
    auto kernel = &expert_wide_dw_kernel<T>;
    const int st = allow_lds(reinterpret_cast<const void*>(kernel), W::kLds);
    if (st != NRF_OK) return st;
    const int64_t blocks = dw_blocks(int64_t(a_tiles) * b_tiles * g.splits, g.E);
    kernel<<<dim3(unsigned(blocks)), 512, W::kLds, stream>>>(g, a_tiles, b_tiles);
    return NRF_OK;
}

// Whether the wide kernels take a product: octets that do not straddle rows (of x and w alone for the forward, which stores its
// outputs at any alignment), operands under 4 GiB and at least half a tile's columns.  Any number of rows: single tokens through 32 experts of 1024 -> 2048
// take 17 us (7.3 TB/s of weights), the general tile 25.  A launch of 512 threads stays under 2^23 workgroups: rows times columns
// under 2^31 leave 2^18 whole tiles, 16384 experts 2^22 short runs' tiles, and dW's tiles hold 2^14 weights each (2^37 fill the memory).
bool wide(int64_t n, int E, int n_in, int n_out, int dtype, bool forward = false) {
    return dtype != NRF_DTYPE_FP32 && n_in % 8 == 0 && (forward || n_out % 8 == 0) && n_in >= 128 && n_out >= 128 &&
           n * (n_in > n_out ? n_in : n_out) < int64_t(1) << 31 && int64_t(n_out) * n_in < int64_t(1) << 31;
}

// ---- fp32, thousands of tiny layers (at most 64 x 64) -----------------------------------------------------------------------
// v_mfma_f32_32x32x2_f32 on 32 rows per wavefront: memory bounds these (a 63 -> 32 layer moves 380 B and multiplies 2016 times
// per row; the fp32 matrix pipe needs half of that time).  Rows of any length and alignment are loaded lanes along the row,
// 4 B each (fragments straight from memory, 16 B per lane at row pitch, occupy the address unit for longer than the rest
// takes: 47 us for 262 k rows, 63 -> 32; rows by 4 B LDS-DMA 59 us), and turned through LDS at an odd pitch.
#define NRF_MFMA_F32(a, b, c) __builtin_amdgcn_mfma_f32_32x32x2f32((a), (b), (c), 0, 0, 0)

// COUNT rows (row i at base + row_of(i) * width, uniform), one load of 64 lanes x 4 B each; zeros past the row's end.  Lanes past
// it read its last element: loads under no condition are in flight together.
template <int COUNT, class F>
__device__ __forceinline__ void load_rows(float (&v)[COUNT], const float* base, int width, int lane, F row_of) {
    const int at = lane < width ? lane : width - 1;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] = (base + int64_t(__builtin_amdgcn_readfirstlane(row_of(i))) * width)[at];
#pragma unroll
    for (int i = 0; i < COUNT; ++i) v[i] = lane < width ? v[i] : 0.f;
}
// a wavefront's own LDS: in order in the hardware, the compiler kept from moving accesses across
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
template <int COUNT>
__device__ __forceinline__ void keep_rows(const float (&v)[COUNT], int padded, float* s_rows, int pitch, int lane) {
    if (lane < padded)
#pragma unroll
        for (int i = 0; i < COUNT; ++i) s_rows[i * pitch + lane] = v[i];
}

// A workgroup takes a run of at most 128 rows of one expert, a wavefront 32 of them; the weights are shared.
constexpr int kCellRows = 128, kCellRowsTable = 2;
template <int NI, int NO>
__global__ __launch_bounds__(256) void expert_cell_forward_kernel(ExpertArgs g) {
    constexpr int kPitch = 32 * NI + 1;
    __shared__ float s_w[NO * 32 * kPitch], s_all[4][32 * 33];
    const PlanLayout L(g.n, g.E);
    const int2 tile = reinterpret_cast<const int2*>(g.plan + L.tiles[kCellRowsTable])[blockIdx.x];   // inside the table's room
    if (int(blockIdx.x) >= g.plan[L.runs + 2 * kCellRowsTable + 1]) return;
    const int expert = tile.y & 0xffff, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane & 31, h = lane >> 5;
    const int left = (tile.y >> 16) - wave * 32, rows = left < 0 ? 0 : left < 32 ? left : 32;
    const bool none = expert == g.E;
    float* s_x = s_all[wave];
    const int mine = c < rows ? g.plan[L.order + tile.x + wave * 32 + c] : 0;
    f32x16 acc[NO] = {};
    if (!none) {
        const float* w = static_cast<const float*>(g.w) + int64_t(expert) * g.n_out * g.n_in;
        const int f0 = wave * 8 * NO;
        float wv[8 * NO], xv[32];
        load_rows<8 * NO>(wv, w, g.n_in, lane, [&](int i) { return f0 + i < g.n_out ? f0 + i : g.n_out - 1; });
        load_rows<32>(xv, static_cast<const float*>(g.x), g.n_in, lane, [&](int i) { return __builtin_amdgcn_readlane(mine, i); });
        if (g.bias) {
            const float* b = static_cast<const float*>(g.bias) + int64_t(expert) * g.n_out;
#pragma unroll
            for (int o = 0; o < NO; ++o)
#pragma unroll
                for (int t = 0; t < 16; ++t) {
                    const int f = 32 * o + nrf::acc_row(t, h);
                    acc[o][t] = f < g.n_out ? b[f] : 0.f;
                }
        }
        keep_rows(wv, 32 * NI, s_w + f0 * kPitch, kPitch, lane);
        __syncthreads();
        const float *px = s_x + c * 33 + h, *pw = s_w + c * kPitch + h;
#pragma unroll
        for (int half = 0; half < NI; ++half) {        // 32 inputs at a time through the wavefront's own piece of LDS
            if (half) wave_order();
            if (NI == 1 ? lane < 32 : lane >> 5 == half)
#pragma unroll
                for (int i = 0; i < 32; ++i) s_x[i * 33 + c] = xv[i];
            wave_order();
#pragma unroll
            for (int k = 0; k < 32; k += 2)
#pragma unroll
                for (int o = 0; o < NO; ++o) acc[o] = NRF_MFMA_F32(pw[32 * o * kPitch + 32 * half + k], px[k], acc[o]);
        }
    }
    if (c >= rows) return;
    float* y = static_cast<float*>(g.out) + int64_t(mine) * g.n_out;
#pragma unroll
    for (int o = 0; o < NO; ++o)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int f = 32 * o + 8 * j + 4 * h;
            f32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = acc[o][4 * j + i];
                if (g.relu) v[i] = v[i] < 0.f ? 0.f : v[i];
            }
            if (f < g.n_out) store4<Fp32>(y + f, v, g.n_out - f);
        }
}

// Backward: a workgroup takes a run of at most 256 rows of one expert, each wavefront every fourth 32 of them: dx of those rows
// and their part of dW and db, summed over the wavefronts in LDS (parts by runs: see ExpertArgs).
template <int NI, int NO>
__global__ __launch_bounds__(256) void expert_cell_backward_kernel(ExpertArgs g, float* dx_out) {
    __shared__ float s_turn[4][32 * 33], s_db[4][NO * 32];
    const PlanLayout L(g.n, g.E);
    const int2 tile = reinterpret_cast<const int2*>(g.plan + L.tiles[kPartTable])[blockIdx.x];   // inside the table's room
    if (int(blockIdx.x) >= g.plan[L.runs + 2 * kPartTable + 1]) return;
    const int rows = tile.y >> 16, expert = tile.y & 0xffff, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 31, h = lane >> 5;
    const int* order = g.plan + L.order + tile.x;
    const float *x = static_cast<const float*>(g.x), *dy = static_cast<const float*>(g.g), *ys = static_cast<const float*>(g.y);
    if (expert == g.E) {                               // rows of no expert
        if (dx_out)
            for (int i = threadIdx.x; i < rows * g.n_in; i += 256) dx_out[int64_t(order[i / g.n_in]) * g.n_in + i % g.n_in] = 0.f;
        return;
    }
    const bool with_w = g.out != nullptr;
    float* s_dz = s_turn[wave];
    const float* w = static_cast<const float*>(g.w) + int64_t(expert) * g.n_out * g.n_in;
    constexpr bool kHoldW = NI * NO <= 2;              // the weights, lanes along a row: in registers where they fit beside the rest
    float wv[kHoldW ? 16 * NO : 1][NI] = {};           // (a feature past the last repeats it: its dz is zero, its dx not stored)
    if (kHoldW && dx_out)
#pragma unroll
        for (int i = 0; i < 16 * NO; ++i)
#pragma unroll
            for (int b = 0; b < NI; ++b) {
                const int f = 2 * i + h < g.n_out ? 2 * i + h : g.n_out - 1, j = 32 * b + c < g.n_in ? 32 * b + c : g.n_in - 1;
                wv[kHoldW ? i : 0][b] = w[int64_t(f) * g.n_in + j];
            }
    f32x16 dw[NO][NI] = {};
    float db[NO] = {};
    for (int r0 = wave * 32; r0 < rows; r0 += 128) {
        const int count = rows - r0 < 32 ? rows - r0 : 32;
        const int mine = order[r0 + (c < count ? c : 0)];
        // two rows per load, lanes along the row: row 2 p + h (a row past the end is the first one again, its dz and x zeroed)
        float xv[16][NI], dz[16][NO], yv[16][NO];
        int64_t row[16];
#pragma unroll
        for (int p = 0; p < 16; ++p) {
            row[p] = __shfl(mine, 2 * p + h);
#pragma unroll
            for (int o = 0; o < NO; ++o) dz[p][o] = dy[row[p] * g.n_out + (32 * o + c < g.n_out ? 32 * o + c : g.n_out - 1)];
        }
        if (g.relu)
#pragma unroll
            for (int p = 0; p < 16; ++p)
#pragma unroll
                for (int o = 0; o < NO; ++o) yv[p][o] = ys[row[p] * g.n_out + (32 * o + c < g.n_out ? 32 * o + c : g.n_out - 1)];
        if (with_w)
#pragma unroll
            for (int p = 0; p < 16; ++p)
#pragma unroll
                for (int b = 0; b < NI; ++b) xv[p][b] = x[row[p] * g.n_in + (32 * b + c < g.n_in ? 32 * b + c : g.n_in - 1)];
#pragma unroll
        for (int p = 0; p < 16; ++p) {
            const bool there = 2 * p + h < count;
#pragma unroll
            for (int o = 0; o < NO; ++o) {
                const bool keep = there && 32 * o + c < g.n_out && (!g.relu || yv[p][o] > 0.f);
                dz[p][o] = keep ? dz[p][o] : 0.f;
            }
#pragma unroll
            for (int b = 0; b < NI; ++b) xv[p][b] = there ? xv[p][b] : 0.f;
        }
        if (dx_out) {
            f32x16 acc[NI] = {};
#pragma unroll
            for (int o = 0; o < NO; ++o) {             // dz turned through the wavefront's own piece of LDS: lanes down the rows
                wave_order();
#pragma unroll
                for (int p = 0; p < 16; ++p) s_dz[(2 * p + h) * 33 + c] = dz[p][o];
                wave_order();
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const int f = 32 * o + k + h;
                    const float d = s_dz[c * 33 + k + h];
#pragma unroll
                    for (int b = 0; b < NI; ++b) {
                        const int j = 32 * b + c;
                        const float wk = kHoldW ? wv[kHoldW ? 16 * o + k / 2 : 0][b] : f < g.n_out && j < g.n_in ? w[int64_t(f) * g.n_in + j] : 0.f;
                        acc[b] = NRF_MFMA_F32(wk, d, acc[b]);
                    }
                }
            }
            if (c < count)
#pragma unroll
                for (int b = 0; b < NI; ++b)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int at = 32 * b + 8 * j + 4 * h;
                        if (at < g.n_in)
                            store4<Fp32>(dx_out + int64_t(mine) * g.n_in + at,
                                         (f32x4){acc[b][4 * j], acc[b][4 * j + 1], acc[b][4 * j + 2], acc[b][4 * j + 3]}, g.n_in - at);
                    }
        }
        if (with_w)
#pragma unroll
            for (int p = 0; p < 16; ++p)
#pragma unroll
                for (int o = 0; o < NO; ++o) {
                    db[o] += dz[p][o];
#pragma unroll
                    for (int b = 0; b < NI; ++b) dw[o][b] = NRF_MFMA_F32(xv[p][b], dz[p][o], dw[o][b]);
                }
    }
    if (!with_w) return;
    const bool whole = g.plan[expert] <= kPartRows;
    float* to_w = whole ? static_cast<float*>(g.out) + int64_t(expert) * g.n_out * g.n_in
                        : g.partial + ((tile.x >> 8) + expert) * part_size(g.n_in, g.n_out);
    float* to_b = !whole ? to_w + int64_t(g.n_out) * g.n_in : g.db ? static_cast<float*>(g.db) + int64_t(expert) * g.n_out : nullptr;
    // the wavefronts' parts of each 32 x 32 block, summed in their order.  Lane (c, h) register t: dW[32 o + c][32 b + acc_row(t, h)]
#pragma unroll
    for (int o = 0; o < NO; ++o) {
        const float both = nrf_add_halves(db[o]);
        if (h == 0) s_db[wave][32 * o + c] = both;
#pragma unroll
        for (int b = 0; b < NI; ++b) {
            if (o + b) __syncthreads();
            else wave_order();
#pragma unroll
            for (int t = 0; t < 16; ++t) s_dz[c * 33 + nrf::acc_row(t, h)] = dw[o][b][t];
            __syncthreads();
            const int j = 32 * b + (threadIdx.x & 31);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int f = 32 * o + 8 * r + (threadIdx.x >> 5), at = (f & 31) * 33 + (threadIdx.x & 31);
                if (f < g.n_out && j < g.n_in) to_w[int64_t(f) * g.n_in + j] = ((s_turn[0][at] + s_turn[1][at]) + s_turn[2][at]) + s_turn[3][at];
            }
        }
    }
    if (to_b && int(threadIdx.x) < g.n_out) {
        const int f = threadIdx.x;
        to_b[f] = ((s_db[0][f] + s_db[1][f]) + s_db[2][f]) + s_db[3][f];
    }
}
int launch_cell_forward(const ExpertArgs& g, hipStream_t stream) {
    const bool i2 = g.n_in > 32, o2 = g.n_out > 32;
    const dim3 grid(unsigned(PlanLayout::most_runs(g.n, g.E, kCellRowsTable)));
    if (i2 && o2) expert_cell_forward_kernel<2, 2><<<grid, 256, 0, stream>>>(g);
    else if (i2) expert_cell_forward_kernel<2, 1><<<grid, 256, 0, stream>>>(g);
    else if (o2) expert_cell_forward_kernel<1, 2><<<grid, 256, 0, stream>>>(g);
    else expert_cell_forward_kernel<1, 1><<<grid, 256, 0, stream>>>(g);
    return NRF_OK;
}
template <int NI, int NO>
int launch_cell_backward(const ExpertArgs& g, float* dx, hipStream_t stream) {
    expert_cell_backward_kernel<NI, NO><<<dim3(unsigned(PlanLayout::most_runs(g.n, g.E, kPartTable))), 256, 0, stream>>>(g, dx);
    return NRF_OK;
}
int launch_cell_backward(const ExpertArgs& g, float* dx, hipStream_t stream) {
    const bool i2 = g.n_in > 32, o2 = g.n_out > 32;
    return i2 && o2 ? launch_cell_backward<2, 2>(g, dx, stream) : i2 ? launch_cell_backward<2, 1>(g, dx, stream)
         : o2       ? launch_cell_backward<1, 2>(g, dx, stream) : launch_cell_backward<1, 1>(g, dx, stream);
}
bool cells(int n_in, int n_out, int dtype) { return dtype == NRF_DTYPE_FP32 && n_in <= 64 && n_out <= 64; }

// An expert's parts, added in their order; zeros for an expert without rows.  256 outputs at a time; where there are FEW experts, an
// expert's many parts are dealt to the four wavefronts, 64 outputs at a time, and their sums joined in order (for every number of
// experts in one kernel: 13 us for 4096 cells of 32 x 32 and 131 k rows, this way 7 - 9).  7 us for 8 experts of 319 x 256 and 20 k rows: launch
// and one chain of loads.
constexpr int kManyParts = 32;
template <class T, bool FEW>
__global__ __launch_bounds__(256) void expert_sum_kernel(ExpertArgs g) {
    typedef typename Traits<T>::elem elem;
    __shared__ double s_sum[FEW ? 4 : 1][64];
    const PlanLayout L(g.n, g.E);
    const int expert = blockIdx.y, rows = g.plan[expert], wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const bool by_runs = g.splits == 0;
    if (by_runs && rows > 0 && rows <= kPartRows) return;              // written at once
    const int64_t size = part_size(g.n_in, g.n_out), weights = int64_t(g.n_out) * g.n_in;
    const int64_t first = by_runs ? (g.plan[L.offsets + expert] >> 8) + expert : expert, step = by_runs ? 1 : g.E;
    const int parts = by_runs ? (rows + kPartRows - 1) / kPartRows : g.splits;
    const bool dealt = FEW && parts >= kManyParts;
    const int wide = dealt ? 64 : 256, begin = dealt ? int(int64_t(parts) * wave / 4) : 0, end = dealt ? int(int64_t(parts) * (wave + 1) / 4) : parts;
    for (int64_t base = int64_t(blockIdx.x) * wide; base < size; base += int64_t(gridDim.x) * wide) {
        const int64_t i = base + (dealt ? lane : int(threadIdx.x));
        const float* p = g.partial + first * size + (i < size ? i : size - 1);
        double sum = 0.0;          // 2^26 rows are 2^18 parts: a running sum of 32 bits no longer takes in a part's last bits (0.4 % off)
        if (dealt) {
#pragma unroll 16
            for (int r = begin; r < end; ++r) sum += double(p[r * step * size]);
            s_sum[wave][lane] = sum;
            __syncthreads();
            sum = ((s_sum[0][lane] + s_sum[1][lane]) + s_sum[2][lane]) + s_sum[3][lane];
            __syncthreads();
            if (wave != 0) continue;
        } else {
#pragma unroll 4
            for (int r = begin; r < end; ++r) sum += double(p[r * step * size]);
        }
        if (i >= size) continue;
        const float v = float(sum);
        if (i < weights) static_cast<elem*>(g.out)[expert * weights + i] = from_float(v, T{});
        else if (g.db) static_cast<elem*>(g.db)[int64_t(expert) * g.n_out + i - weights] = from_float(v, T{});
    }
}

// The general tile's size for a product: 128 where that leaves at least one and a half workgroups per CU.
int64_t tile_count(int form, int64_t n, int E, int n_in, int n_out, int tile) {
    const int64_t in = (n_in + tile - 1) / tile, out = (n_out + tile - 1) / tile, rows = n / tile + (E < n ? E : n) / 2;
    return form == kForward ? rows * out : form == kDx ? rows * in : in * out * E;
}
// Two tiles of 128 fit a CU: they are taken where they fill one round (20 k rows, 319 -> 256 fp32: 495 tiles, backward 80 us, with
// tiles of 64 89) or several, and dW's shares of uneven experts only in several (16 k rows, 1001 -> 1001 fp16: 512 tiles,
// backward 306 us, with tiles of 64 256; 16 k rows, 500 -> 500 fp32: 540 tiles, forward 100 us, 90; 1032 of 1001 -> 1001: 94, 112).
int tile_size(int form, int64_t n, int E, int n_in, int n_out, int splits) {
    if (n / E <= 64 || n_in <= 64 || n_out <= 64) return 64;
    const bool by_runs = form == kDw && splits == 0;
    const int64_t tiles = tile_count(form, n, E, n_in, n_out, 128) * (by_runs ? n / E / kPartRows : splits);
    return (tiles >= 384 && tiles <= 512 && (form != kDw || by_runs)) || tiles >= 960 ? 128 : 64;
}
// How dW's sum over an expert's rows is cut (see ExpertArgs): not at all where the outputs alone give 512 workgroups; else by
// runs, which balances uneven experts, while the parts stay under 1 GiB; else into equal shares.  Wide kernels: equal shares of
// at least 512 rows of the average expert, enough for a workgroup per CU.  (The tiny fp32 layers' kernel always cuts by runs: its parts,
// (n_in + 1) n_out words per 256 rows and per expert, are at most a quarter of what x, dy and the weights hold.)
int dw_splits(int64_t n, int E, int n_in, int n_out, bool is_wide) {
    int64_t want, most;
    if (is_wide) {
        typedef WideDw<Bf16> W;
        const int64_t tiles = int64_t(E) * ((n_in + W::kA - 1) / W::kA) * ((n_out + W::kB - 1) / W::kB);
        want = (256 + tiles - 1) / tiles, most = n / E / 512;
    } else {
        const int64_t tiles = tile_count(kDw, n, E, n_in, n_out, n_in > 64 && n_out > 64 ? 128 : 64);
        if (tiles >= 512 || n / E < 2 * kPartRows) return 1;
        if (PlanLayout::slots(n, E, kPartTable) * part_size(n_in, n_out) * 4 <= int64_t(1) << 30) return 0;
        want = (512 + tiles - 1) / tiles, most = n / E / 256;
    }
    const int64_t s = want < most ? want : most;
    return s < 1 ? 1 : s > 64 ? 64 : int(s);
}
int64_t part_bytes(int64_t n, int E, int n_in, int n_out, int splits) {
    const int64_t parts = splits == 0 ? PlanLayout::slots(n, E, kPartTable) : splits > 1 ? int64_t(splits) * E : 0;
    return parts * part_size(n_in, n_out) * 4;
}

template <int FORM, int TT>
void launch_tile(int dtype, const ExpertArgs& g, hipStream_t stream) {
    const int a_tiles = ((FORM == kForward ? g.n_out : g.n_in) + TT - 1) / TT, b_tiles = FORM == kDw ? (g.n_out + TT - 1) / TT : 1;
    const int table = FORM == kDw ? kPartTable : TT == 64 ? 1 : 2;
    const int64_t blocks = FORM == kDw && g.splits != 0 ? dw_blocks(int64_t(g.splits) * a_tiles * b_tiles, g.E)
                                                        : xcd_blocks(PlanLayout::most_runs(g.n, g.E, table), a_tiles * b_tiles);
    const dim3 grid = nrf::grid_rows(blocks);
    if (dtype == NRF_DTYPE_FP32) expert_tile_kernel<Fp32, FORM, TT><<<grid, 256, 0, stream>>>(g, a_tiles, b_tiles);
    else if (dtype == NRF_DTYPE_BF16) expert_tile_kernel<Bf16, FORM, TT><<<grid, 256, 0, stream>>>(g, a_tiles, b_tiles);
    else expert_tile_kernel<Fp16, FORM, TT><<<grid, 256, 0, stream>>>(g, a_tiles, b_tiles);
}
template <int FORM>
void launch_tile(int dtype, const ExpertArgs& g, hipStream_t stream) {
    if (tile_size(FORM, g.n, g.E, g.n_in, g.n_out, g.splits) == 128) launch_tile<FORM, 128>(dtype, g, stream);
    else launch_tile<FORM, 64>(dtype, g, stream);
}

void launch_sum(int dtype, const ExpertArgs& g, hipStream_t stream) {
    // of tiny layers' outputs, few workgroups per expert where there are many experts, else about 1024 in all (262 k rows of 64 x 64: one
    // expert 645 -> 235 us, 8 experts 261 -> 209, 2 M rows of one expert 6.6 -> 2.1 ms; 4096 cells of 32 x 32 keep one each)
    const int64_t size = part_size(g.n_in, g.n_out), least = size > 8192 ? (size + 255) / 256 : (size + 2047) / 2048, most = (size + 63) / 64;
    const int64_t want = (1024 + g.E - 1) / g.E, blocks = want < least ? least : want < most ? want : most;
    const bool few = want > least;
    const dim3 grid(unsigned(blocks < 1024 ? blocks : 1024), unsigned(g.E));
    if (dtype == NRF_DTYPE_FP32) few ? expert_sum_kernel<Fp32, true><<<grid, 256, 0, stream>>>(g) : expert_sum_kernel<Fp32, false><<<grid, 256, 0, stream>>>(g);
    else if (dtype == NRF_DTYPE_BF16) few ? expert_sum_kernel<Bf16, true><<<grid, 256, 0, stream>>>(g) : expert_sum_kernel<Bf16, false><<<grid, 256, 0, stream>>>(g);
    else few ? expert_sum_kernel<Fp16, true><<<grid, 256, 0, stream>>>(g) : expert_sum_kernel<Fp16, false><<<grid, 256, 0, stream>>>(g);
}

bool shapes_ok(int64_t n, int E, int n_in, int n_out, int dtype, int act) {
    return n >= 0 && n <= nrf::kMaxExpertRows && E >= 1 && E <= nrf::kMaxExperts && n_in >= 1 && n_in <= 65536 && n_out >= 1 &&
           n_out <= 65536 && dtype >= NRF_DTYPE_FP32 && dtype <= NRF_DTYPE_FP16 && (act == NRF_ACT_NONE || act == NRF_ACT_RELU);
}

int elem_bytes(int dtype) { return dtype == NRF_DTYPE_FP32 ? 4 : 2; }
bool elem_aligned(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & unsigned(elem_bytes(dtype) - 1)) == 0; }

}  // namespace

NRF_EXPORT int nrf_expert_linear(const void* x, const void* weight, const void* bias, const void* plan, int64_t n_rows,
                                 int num_experts, int n_in, int n_out, int dtype, int act, void* y, nrf_stream_t stream) {
    if (!shapes_ok(n_rows, num_experts, n_in, n_out, dtype, act)) return NRF_ERR_SHAPE;
    if (n_rows == 0) return NRF_OK;
    if (!x || !weight || !plan || !y) return NRF_ERR_NULL;
    if (!elem_aligned(x, dtype) || !elem_aligned(weight, dtype) || !elem_aligned(bias, dtype) || !elem_aligned(y, dtype) ||
        !nrf_aligned16(plan))
        return NRF_ERR_ALIGN;
    const int64_t size = elem_bytes(dtype), y_bytes = n_rows * n_out * size;
    if (nrf::overlap(y, y_bytes, x, n_rows * n_in * size) || nrf::overlap(y, y_bytes, weight, int64_t(num_experts) * n_out * n_in * size) ||
        nrf::overlap(y, y_bytes, bias, int64_t(num_experts) * n_out * size))
        return NRF_ERR_SHAPE;
    ExpertArgs g{};
    g.x = x, g.w = weight, g.bias = bias, g.plan = static_cast<const int*>(plan), g.out = y;
    g.n = n_rows, g.E = num_experts, g.n_in = n_in, g.n_out = n_out, g.relu = act == NRF_ACT_RELU, g.splits = 1;
    nrf_launch_begin();
    if (wide(n_rows, num_experts, n_in, n_out, dtype, true) && nrf_aligned16(x) && nrf_aligned16(weight)) {
        const int st = dtype == NRF_DTYPE_BF16 ? launch_wide_forward<Bf16>(g, static_cast<hipStream_t>(stream))
                                               : launch_wide_forward<Fp16>(g, static_cast<hipStream_t>(stream));
        return st != NRF_OK ? st : nrf_launch_status();
    }
    if (cells(n_in, n_out, dtype)) {
        const int st = launch_cell_forward(g, static_cast<hipStream_t>(stream));
        return st != NRF_OK ? st : nrf_launch_status();
    }
    launch_tile<kForward>(dtype, g, static_cast<hipStream_t>(stream));
    return nrf_launch_status();
}

namespace {
// the backward's workspace: the masked gradient (wide kernels behind a relu), then the partial sums of dW and db
struct BackwardWork {
    int64_t dz, partial;
    BackwardWork(int64_t n, int E, int n_in, int n_out, int dtype) {
        const bool is_wide = wide(n, E, n_in, n_out, dtype);
        dz = is_wide ? (n * n_out * 2 + 255) & ~int64_t(255) : 0;
        partial = part_bytes(n, E, n_in, n_out, cells(n_in, n_out, dtype) ? 0 : dw_splits(n, E, n_in, n_out, false));
        if (is_wide) {   // either kernel may run: alignment is known at the call
            const int64_t p = part_bytes(n, E, n_in, n_out, dw_splits(n, E, n_in, n_out, true));
            if (p > partial) partial = p;
        }
    }
};
}  // namespace

NRF_EXPORT int64_t nrf_expert_linear_backward_workspace_bytes(int64_t n_rows, int num_experts, int n_in, int n_out, int dtype) {
    if (!shapes_ok(n_rows, num_experts, n_in, n_out, dtype, NRF_ACT_NONE)) return -1;
    const BackwardWork work(n_rows, num_experts, n_in, n_out, dtype);
    return work.dz + work.partial;
}

NRF_EXPORT int nrf_expert_linear_backward(const void* grad_y, const void* x, const void* weight, const void* y, const void* plan,
                                          int64_t n_rows, int num_experts, int n_in, int n_out, int dtype, int act, void* grad_x,
                                          void* grad_weight, void* grad_bias, void* workspace, int64_t workspace_bytes,
                                          nrf_stream_t stream_) {
    if (!shapes_ok(n_rows, num_experts, n_in, n_out, dtype, act)) return NRF_ERR_SHAPE;
    if (!grad_x && !grad_weight && !grad_bias) return NRF_OK;
    if (!plan || (n_rows > 0 && (!grad_y || !x || !weight || (act == NRF_ACT_RELU && !y)))) return NRF_ERR_NULL;
    if (grad_bias && !grad_weight) return NRF_ERR_NULL;   // the bias sums ride in the weight product
    const void* elems[] = {grad_y, x, weight, y, grad_x, grad_weight, grad_bias};
    for (const void* p : elems)
        if (!elem_aligned(p, dtype)) return NRF_ERR_ALIGN;
    if (!nrf_aligned16(plan) || !nrf_aligned16(workspace)) return NRF_ERR_ALIGN;
    const BackwardWork work(n_rows, num_experts, n_in, n_out, dtype);
    if (work.dz + work.partial > 0 && (!workspace || workspace_bytes < work.dz + work.partial)) return NRF_ERR_WORKSPACE;
    const int64_t size = elem_bytes(dtype), x_bytes = n_rows * n_in * size, y_bytes = n_rows * n_out * size,
                  w_bytes = int64_t(num_experts) * n_out * n_in * size, b_bytes = int64_t(num_experts) * n_out * size;
    const struct { const void* p; int64_t bytes; } parts[] = {{grad_x, x_bytes}, {grad_weight, w_bytes}, {grad_bias, b_bytes},
                                                              {grad_y, y_bytes}, {x, x_bytes}, {weight, w_bytes}, {act == NRF_ACT_RELU ? y : nullptr, y_bytes}};
    for (int i = 0; i < 3; ++i)              // an output with another, or with an operand that is read again after it was written
        for (int j = i + 1; j < 7; ++j)
            if (nrf::overlap(parts[i].p, parts[i].bytes, parts[j].p, parts[j].bytes)) return NRF_ERR_SHAPE;
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    ExpertArgs g{};
    g.x = x, g.w = weight, g.y = y, g.g = grad_y, g.plan = static_cast<const int*>(plan);
    g.n = n_rows, g.E = num_experts, g.n_in = n_in, g.n_out = n_out, g.relu = act == NRF_ACT_RELU;
    g.partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + work.dz);
    const bool is_wide = work.dz > 0 && n_rows > 0 && nrf_aligned16(grad_y) && nrf_aligned16(x) && nrf_aligned16(weight) &&
                         nrf_aligned16(y);
    int st = NRF_OK;
    nrf_launch_begin();
    if (cells(n_in, n_out, dtype) && n_rows > 0) {
        g.out = grad_weight, g.db = grad_bias;
        g.splits = 0;
        st = launch_cell_backward(g, static_cast<float*>(grad_x), stream);
        if (st == NRF_OK && grad_weight) launch_sum(dtype, g, stream);
        return st != NRF_OK ? st : nrf_launch_status();
    }
    if (is_wide && g.relu) {
        const int64_t octets = n_rows * n_out / 8, blocks = (octets + 255) / 256;
        const dim3 grid(unsigned(blocks < 8192 ? blocks : 8192));
        const u32x4 *dy = static_cast<const u32x4*>(grad_y), *ys = static_cast<const u32x4*>(y);
        u32x4* dz = static_cast<u32x4*>(workspace);
        if (dtype == NRF_DTYPE_BF16) expert_mask_kernel<Bf16><<<grid, 256, 0, stream>>>(dy, ys, octets, dz);
        else expert_mask_kernel<Fp16><<<grid, 256, 0, stream>>>(dy, ys, octets, dz);
        g.g = dz, g.relu = 0;
    }
    if (grad_x && n_rows > 0) {
        g.out = grad_x, g.splits = 1;
        if (!is_wide) launch_tile<kDx>(dtype, g, stream);
        else st = dtype == NRF_DTYPE_BF16 ? launch_wide_rows<Bf16, kDx, 128>(g, stream) : launch_wide_rows<Fp16, kDx, 128>(g, stream);
    }
    if (grad_weight && st == NRF_OK) {
        g.splits = dw_splits(n_rows, num_experts, n_in, n_out, is_wide);
        g.out = grad_weight, g.db = grad_bias;
        if (!is_wide) launch_tile<kDw>(dtype, g, stream);
        else st = dtype == NRF_DTYPE_BF16 ? launch_wide_dw<Bf16>(g, stream) : launch_wide_dw<Fp16>(g, stream);
        if (g.splits != 1 && st == NRF_OK) launch_sum(dtype, g, stream);
    }
    return st != NRF_OK ? st : nrf_launch_status();
}
