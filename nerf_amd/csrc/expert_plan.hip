// The plan of a batch whose rows are dealt to experts (experts.h): a stable counting sort of the rows by expert.
//
// Every wavefront owns a contiguous run of rows and a private 16-bit counter per expert in LDS.  It counts its rows; the
// counters become exclusive sums over the wavefronts before it; then it walks its rows again, 64 at a time, and a row's place
// is the counter of its expert plus the number of lower lanes with the same expert (found with one ballot per bit of the
// expert's number, no atomics), so equal keys keep their order and the result is the same on every run.
// Up to kSingleRows rows are one workgroup and one launch.  Beyond, the rows are cut into chunks, one workgroup each: chunk
// histograms (launch 1), an exclusive sum over the chunks per expert (launch 2), the walk and beside it the run tables (launch 3).
#include "experts.h"

namespace {

using nrf::PlanLayout;

constexpr int64_t kSingleRows = 8192;

__device__ __forceinline__ int wave_scan_int(int v) {   // inclusive, within the registers: rows of 16 lanes, then over the rows
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);   // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);   // lane 15 of rows 0 and 2 to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);   // lane 31 to rows 2 and 3
    return v;
}

// The keys of rows first, first + stride, ... (kAhead of them, their loads in flight together), -1 past `end`
constexpr int kAhead = 8;
__device__ __forceinline__ void load_keys(const int* __restrict__ index, int64_t first, int stride, int64_t end, int E, int (&key)[kAhead]) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) key[i] = first + i * stride < end ? index[first + i * stride] : 0;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const int k = (unsigned)key[i] < (unsigned)E ? key[i] : E;
        key[i] = first + i * stride < end ? k : -1;
    }
}

// A key's rows as runs of 2^s: the long ones, and whether half a run or less is left
__device__ __forceinline__ int long_runs(int rows, int s) { return int((unsigned(rows) + (1u << (s - 1)) - 1u) >> s); }
__device__ __forceinline__ int short_run(int rows, int s) { return rows > long_runs(rows, s) << s; }

// Exclusive sums over the keys' rows (and over their long and short runs of (Q - 1) / 2 run lengths from table0 on): thread i owns the
// keys [i per, (i + 1) per).  before[]: the sums over all keys before this thread's; total[]: over all.  `part`: Q per wavefront.
template <int WAVES, int Q, class F>
__device__ __forceinline__ void key_sums(int keys, int* part, F rows_of, int (&before)[Q], int (&total)[Q], int table0 = 0) {
    const int per = (keys + WAVES * 64 - 1) / (WAVES * 64), at = threadIdx.x * per, wave = threadIdx.x >> 6;
    int sum[Q] = {};
    for (int k = at; k < at + per && k < keys; ++k) {
        const int c = rows_of(k);
        sum[0] += c;
#pragma unroll
        for (int t = 0; t < (Q - 1) / 2; ++t) {
            const int s = nrf::kTileShift0 + table0 + t;
            sum[1 + 2 * t] += long_runs(c, s), sum[2 + 2 * t] += short_run(c, s);
        }
    }
#pragma unroll
    for (int i = 0; i < Q; ++i) {
        const int incl = wave_scan_int(sum[i]);
        before[i] = incl - sum[i];
        if ((threadIdx.x & 63) == 63) part[wave * Q + i] = incl;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Q; ++i) {
        total[i] = 0;
        for (int w = 0; w < WAVES; ++w) {
            if (w == wave) before[i] += total[i];
            total[i] += part[w * Q + i];
        }
    }
    __syncthreads();
}

// Key k's runs of 2^s rows in table `out` (long ones from `first`, a short one at `last`), where `mine`: the first runs and the
// short one by the key's own lane, further ones by the wavefront; of a key of more than kShared runs, where it is not alone,
// share `share` of `shares`.  All 64 lanes call it; rows = 0 has none.
__device__ __forceinline__ int2 run_of(int s, int k, int off, int rows, int r) {
    const int left = rows - (r << s);
    return make_int2(off + (r << s), (left < 1 << s ? left : 1 << s) << 16 | k);
}
constexpr int kShared = 1024;
__device__ __forceinline__ void fill_runs(int2* out, int s, int k, int off, int rows, int first, int last, bool mine, int share, int shares) {
    const int runs = long_runs(rows, s), direct = !mine ? 0 : runs < 16 ? runs : 16;
    for (int r = 0; r < direct; ++r) out[first + r] = run_of(s, k, off, rows, r);
    for (unsigned long long many = __ballot(runs > 16 && (mine || runs > kShared)); many; many &= many - 1) {
        const int l = __ffsll((long long)many) - 1;
        const int w = __builtin_amdgcn_readlane(runs, l), f = __builtin_amdgcn_readlane(first, l), c = __builtin_amdgcn_readlane(rows, l),
                  o = __builtin_amdgcn_readlane(off, l), key = __builtin_amdgcn_readlane(k, l);
        const int from = w > kShared ? share : 0, step = w > kShared ? shares : 1;
        for (int r = 16 + 64 * from + int(threadIdx.x & 63); r < w; r += 64 * step) out[f + r] = run_of(s, key, o, c, r);
    }
    if (mine && short_run(rows, s)) out[last] = run_of(s, k, off, rows, runs);
}
constexpr int kSums = 1 + 2 * nrf::kTileTables;
// counts, offsets and the run tables' lengths; at: this thread's sums before its key k, total: over all keys
__device__ __forceinline__ void write_key(const PlanLayout& L, int* plan, int E, int k, int rows, int off) {
    plan[L.offsets + k] = off;
    if (k < E) plan[k] = rows;
}
__device__ __forceinline__ void write_lengths(const PlanLayout& L, int* plan, const int (&total)[kSums]) {
#pragma unroll
    for (int t = 0; t < nrf::kTileTables; ++t)
        plan[L.runs + 2 * t] = total[1 + 2 * t], plan[L.runs + 2 * t + 1] = total[1 + 2 * t] + total[2 + 2 * t];
}
__device__ __forceinline__ void pass_key(int rows, int (&at)[kSums]) {
    at[0] += rows;
#pragma unroll
    for (int t = 0; t < nrf::kTileTables; ++t) {
        const int s = nrf::kTileShift0 + t;
        at[1 + 2 * t] += long_runs(rows, s), at[2 + 2 * t] += short_run(rows, s);
    }
}

// Rows of every key in a chunk: 2 M rows, 4096 experts 8 us (1 TB/s of keys; half of it LDS atomics on the cells' runs of equal keys)
__global__ __launch_bounds__(512) void plan_hist_kernel(const int* __restrict__ index, int64_t n, int E, int64_t chunk,
                                                        int* __restrict__ hist) {
    extern __shared__ int s_count[];
    for (int k = threadIdx.x; k <= E; k += 512) s_count[k] = 0;
    __syncthreads();
    const int64_t begin = blockIdx.x * chunk, end = begin + chunk < n ? begin + chunk : n;
    for (int64_t r = begin + threadIdx.x; r < end; r += 512 * kAhead) {
        int key[kAhead];
        load_keys(index, r, 512, end, E, key);
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (key[i] >= 0) atomicAdd(&s_count[key[i]], 1);
    }
    __syncthreads();
    for (int k = threadIdx.x; k <= E; k += 512) hist[int64_t(blockIdx.x) * (E + 1) + k] = s_count[k];
}

// hist[chunk][key] -> exclusive sums over the chunks, totals[key].  64 keys per workgroup, the chunks dealt to 16 wavefronts.
// 248 chunks of 4097 keys: 6 us, 8 MB through the L2.
__global__ __launch_bounds__(1024) void plan_chunks_kernel(int* __restrict__ hist, int chunks, int E, int* __restrict__ totals) {
    __shared__ int s_sum[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, key = blockIdx.x * 64 + lane;
    const int per = (chunks + 15) / 16, c0 = wave * per, c1 = c0 + per < chunks ? c0 + per : chunks;
    int sum = 0;
    if (key <= E)
#pragma unroll 16
        for (int c = c0; c < c1; ++c) sum += hist[int64_t(c) * (E + 1) + key];
    s_sum[wave][lane] = sum;
    __syncthreads();
    int run = 0;
    for (int w = 0; w < wave; ++w) run += s_sum[w][lane];
    if (key > E) return;
    if (wave == 15) totals[key] = run + sum;
#pragma unroll 16
    for (int c = c0; c < c1; ++c) {
        int* p = hist + int64_t(c) * (E + 1) + key;
        const int v = *p;
        *p = run;
        run += v;
    }
}

// The walk of 2 M rows over 4096 experts takes 21 us: 3 launch, 3.5 counting again, 3 sums and places, 10 ranks (15 ballots per 64
// rows, 8 up to 255 experts, a chain through the counters), the rest scattered 4 B stores; the tables beside it 5.  2048 rows in one workgroup: 5 us.
// Workgroups 0 .. kTableBlocks - 1: the run tables, kTableShares for each table; table 0's also write counts and offsets.  Those
// behind them: the walk.  SINGLE: one workgroup does it all.
constexpr int kTableShares = 2, kTableBlocks = nrf::kTileTables * kTableShares;
template <int WAVES, bool SINGLE>
__global__ __launch_bounds__(WAVES * 64) void plan_place_kernel(const int* __restrict__ index, int64_t n, int E, int64_t chunk,
                                                                const int* __restrict__ hist, const int* __restrict__ totals,
                                                                int* __restrict__ plan) {
    constexpr int THREADS = WAVES * 64;
    extern __shared__ int s_mem[];
    __shared__ int s_part[WAVES * kSums];
    const PlanLayout L(n, E);
    const int keys = E + 1, stride = (keys + 1) & ~1;      // 16-bit counters, an even number per wavefront
    const int each = (keys + THREADS - 1) / THREADS;
    int* s_off = s_mem;                                    // [keys], rounded up to a pair: the keys' rows, then their places
    if (!SINGLE) {
#pragma unroll 8
        for (int k = threadIdx.x; k < keys; k += THREADS) s_off[k] = totals[k];
        if (blockIdx.x < kTableBlocks) {
            const int t = blockIdx.x / kTableShares, share = blockIdx.x % kTableShares, s = nrf::kTileShift0 + t;
            int2* out = reinterpret_cast<int2*>(plan + L.tiles[0] + (t > 0 ? L.tiles[1] - L.tiles[0] : 0) + (t > 1 ? L.tiles[2] - L.tiles[1] : 0) +
                                                (t > 2 ? L.tiles[3] - L.tiles[2] : 0));
            __syncthreads();
            int at[3], total[3];
            key_sums<WAVES, 3>(keys, s_part, [&](int k) { return s_off[k]; }, at, total, t);
            for (int i = 0; i < each; ++i) {
                const int k = threadIdx.x * each + i, rows = k < keys ? s_off[k] : 0;
                const bool mine = i % kTableShares == share;
                if (t == 0 && mine && k < keys) write_key(L, plan, E, k, rows, at[0]);
                fill_runs(out, s, k, at[0], rows, at[1], total[1] + at[2], mine, share, kTableShares);
                at[0] += rows, at[1] += long_runs(rows, s), at[2] += short_run(rows, s);
            }
            if (share == 0 && threadIdx.x == 0) plan[L.runs + 2 * t] = total[1], plan[L.runs + 2 * t + 1] = total[1] + total[2];
            return;
        }
    }
    const int64_t block = SINGLE ? 0 : blockIdx.x - kTableBlocks;
    unsigned* s_cnt32 = reinterpret_cast<unsigned*>(s_mem + stride);
    unsigned short* s_cnt = reinterpret_cast<unsigned short*>(s_cnt32);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

    for (int i = threadIdx.x; i < WAVES * stride / 2; i += THREADS) s_cnt32[i] = 0;
    __syncthreads();

    const int64_t begin = block * chunk, end = begin + chunk < n ? begin + chunk : n;
    const int64_t per = ((end - begin + THREADS - 1) / THREADS) * 64;   // rows of a wavefront, whole 64s
    const int64_t w0 = begin + wave * per, w1 = w0 + per < end ? w0 + per : end;
    unsigned short* mine = s_cnt + wave * stride;
    for (int64_t r = w0 + lane; r < w1; r += 64 * kAhead) {
        int key[kAhead];
        load_keys(index, r, 64, w1, E, key);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int slot = wave * stride + key[i];
            if (key[i] >= 0) atomicAdd(&s_cnt32[slot >> 1], (slot & 1) ? 0x10000u : 1u);
        }
    }
    __syncthreads();
    for (int p = threadIdx.x; p < stride / 2; p += THREADS) {   // two keys at a time: a chunk's counts stay under 2^16
        unsigned run = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const unsigned v = s_cnt32[w * (stride / 2) + p];
            s_cnt32[w * (stride / 2) + p] = run;
            run += v;
        }
        if (SINGLE) s_off[2 * p] = int(run & 0xffffu), s_off[2 * p + 1] = int(run >> 16);
    }
    __syncthreads();
    // where this chunk's rows of each key begin
    if (SINGLE) {
        int at[kSums], total[kSums];
        key_sums<WAVES, kSums>(keys, s_part, [&](int k) { return s_off[k]; }, at, total);
        for (int i = 0; i < each; ++i) {
            const int k = threadIdx.x * each + i, rows = k < keys ? s_off[k] : 0;
            if (k < keys) write_key(L, plan, E, k, rows, at[0]), s_off[k] = at[0];
#pragma unroll
            for (int t = 0; t < nrf::kTileTables; ++t)
                fill_runs(reinterpret_cast<int2*>(plan + L.tiles[t]), nrf::kTileShift0 + t, k, at[0], rows, at[1 + 2 * t],
                          total[1 + 2 * t] + at[2 + 2 * t], true, 0, 1);
            pass_key(rows, at);
        }
        if (threadIdx.x == 0) write_lengths(L, plan, total);
    } else {
        int at[1], total[1];
        key_sums<WAVES, 1>(keys, s_part, [&](int k) { return s_off[k]; }, at, total);
        for (int k = threadIdx.x * each; k < int(threadIdx.x + 1) * each && k < keys; ++k) {
            const int rows = s_off[k];
            s_off[k] = at[0];
            at[0] += rows;
        }
        __syncthreads();
#pragma unroll 8
        for (int k = threadIdx.x; k < keys; k += THREADS) s_off[k] += hist[block * keys + k];
    }
    __syncthreads();

    int* order = plan + L.order;
    const int bits = 32 - __clz(E);                        // keys 0 .. E
    const unsigned long long below = (1ull << lane) - 1;
    for (int64_t r0 = w0; r0 < w1; r0 += 64 * kAhead) {
        int keys_ahead[kAhead];
        load_keys(index, r0 + lane, 64, w1, E, keys_ahead);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int key = keys_ahead[i];
            if (r0 + 64 * i >= w1) break;
            const unsigned long long there = __ballot(key >= 0);
            unsigned lo = unsigned(there), hi = unsigned(there >> 32);   // the lanes with this one's key
#pragma unroll
            for (int b = 0; b < 15; ++b) {                               // bits that no key has change nothing
                if (b >= 8 && bits <= 8) continue;
                const int one = (key << (31 - b)) >> 31;                 // all ones where bit b is set
                const unsigned long long m = __ballot(one != 0);
                lo &= ~(unsigned(m) ^ unsigned(one)), hi &= ~(unsigned(m >> 32) ^ unsigned(one));
            }
            const unsigned long long same = (unsigned long long)hi << 32 | lo;
            if (key >= 0) {
                const int start = mine[key];
                order[s_off[key] + start + __popcll(same & below)] = int(r0) + 64 * i + lane;
                if ((same >> lane) == 1) mine[key] = (unsigned short)(start + __popcll(same));   // the highest lane of the key
            }
            // the next 64 rows' lanes read what these lanes wrote: same wavefront, LDS in order, the compiler kept from moving it
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
}

int64_t plan_chunk(int64_t n) {
    int64_t chunk = (n + 247) / 248;          // with the tables' 8, one workgroup per CU; a counter of a chunk has 16 bits
    if (chunk < 2048) chunk = 2048;
    return chunk > 32768 ? 32768 : chunk;
}
bool plan_single(int64_t n) { return n <= kSingleRows; }

size_t place_lds(int E, int waves) {
    return size_t((E + 2) & ~1) * 4 + size_t(waves) * ((E + 2) & ~1) * 2;
}

template <int WAVES, bool SINGLE>
int launch_place(const int* index, int64_t n, int E, int64_t chunk, int64_t chunks, const int* hist, const int* totals, int* plan,
                 hipStream_t stream) {
    if (place_lds(E, WAVES) > 65536 - 1024 &&
        hipFuncSetAttribute(reinterpret_cast<const void*>(&plan_place_kernel<WAVES, SINGLE>), hipFuncAttributeMaxDynamicSharedMemorySize,
                            int(place_lds(E, WAVES))) != hipSuccess)
        return NRF_ERR_LAUNCH;
    const unsigned grid = unsigned(chunks) + (SINGLE ? 0 : kTableBlocks);
    plan_place_kernel<WAVES, SINGLE><<<dim3(grid), WAVES * 64, place_lds(E, WAVES), stream>>>(index, n, E, chunk, hist, totals, plan);
    return NRF_OK;
}

}  // namespace

NRF_EXPORT int64_t nrf_expert_plan_bytes(int64_t n_rows, int num_experts) {
    if (n_rows < 0 || n_rows > nrf::kMaxExpertRows || num_experts < 1 || num_experts > nrf::kMaxExperts) return -1;
    return PlanLayout(n_rows, num_experts).total * 4;
}

NRF_EXPORT int64_t nrf_expert_plan_workspace_bytes(int64_t n_rows, int num_experts) {
    if (n_rows < 0 || n_rows > nrf::kMaxExpertRows || num_experts < 1 || num_experts > nrf::kMaxExperts) return -1;
    if (plan_single(n_rows)) return 0;
    const int64_t chunk = plan_chunk(n_rows), chunks = (n_rows + chunk - 1) / chunk;
    return (chunks + 1) * int64_t(num_experts + 1) * 4;
}

NRF_EXPORT int nrf_expert_plan(const int32_t* index, int64_t n_rows, int num_experts, void* plan, int64_t plan_bytes,
                               void* workspace, int64_t workspace_bytes, nrf_stream_t stream_) {
    const int64_t need = nrf_expert_plan_bytes(n_rows, num_experts);
    if (need < 0) return NRF_ERR_SHAPE;
    const int64_t work = nrf_expert_plan_workspace_bytes(n_rows, num_experts);
    if (!plan || (n_rows > 0 && !index) || (work > 0 && !workspace)) return NRF_ERR_NULL;
    if (plan_bytes < need || workspace_bytes < work) return NRF_ERR_WORKSPACE;
    if (!nrf_aligned16(plan) || (work > 0 && !nrf_aligned16(workspace))) return NRF_ERR_ALIGN;
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    const int E = num_experts;
    const bool wide = E > 4096;               // eight wavefronts' counters fit in LDS up to 4096 experts, two's beyond
    int* out = static_cast<int*>(plan);
    nrf_launch_begin();
    if (plan_single(n_rows)) {
        const int64_t chunk = n_rows > 0 ? n_rows : 1;
        const int st = wide ? launch_place<2, true>(index, n_rows, E, chunk, 1, nullptr, nullptr, out, stream)
                            : launch_place<8, true>(index, n_rows, E, chunk, 1, nullptr, nullptr, out, stream);
        return st != NRF_OK ? st : nrf_launch_status();
    }
    const int64_t chunk = plan_chunk(n_rows), chunks = (n_rows + chunk - 1) / chunk;
    int* hist = static_cast<int*>(workspace);
    int* totals = hist + chunks * (E + 1);
    const size_t hist_lds = size_t(E + 1) * 4;
    if (hist_lds > 65536 - 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(&plan_hist_kernel),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, int(hist_lds)) != hipSuccess)
        return NRF_ERR_LAUNCH;
    plan_hist_kernel<<<dim3(unsigned(chunks)), 512, hist_lds, stream>>>(index, n_rows, E, chunk, hist);
    plan_chunks_kernel<<<dim3(unsigned(E / 64 + 1)), 1024, 0, stream>>>(hist, int(chunks), E, totals);
    // sixteen wavefronts hide more of a long chunk's latency than their counters cost (2 M rows in runs of one expert, 4096 of them:
    // 22.7 us for 24.5; 262 k rows: 12.7 for 10.4).  Rows of any order: the whole call takes 35 us for 44 with 1024 experts, 55 for 52
    // with 4096 and 61 for 56 with 64; between the two lengths neither wins everywhere
    const int st = wide            ? launch_place<2, false>(index, n_rows, E, chunk, chunks, hist, totals, out, stream)
                   : chunk >= 6000 ? launch_place<16, false>(index, n_rows, E, chunk, chunks, hist, totals, out, stream)
                                   : launch_place<8, false>(index, n_rows, E, chunk, chunks, hist, totals, out, stream);
    return st != NRF_OK ? st : nrf_launch_status();
}
