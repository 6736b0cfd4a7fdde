// The plan of a batch whose rows are dealt to experts (experts.h): a stable counting sort of the rows by expert.
//
// Every wavefront owns a contiguous run of rows and a private 16-bit counter per expert in LDS.  It counts its rows; the
// counters become exclusive sums over the wavefronts before it; then it walks its rows again, 64 at a time, and a row's place
// is the counter of its expert plus the number of lower lanes with the same expert (found with one ballot per bit of the
// expert's number, no atomics), so equal keys keep their order and the result is the same on every run.
// Up to kSingleRows rows are one workgroup and one launch.  Beyond, the rows are cut into chunks, one workgroup each: chunk
// histograms (launch 1), an exclusive sum over the chunks per expert (launch 2), the walk (launch 3).
#include "experts.h"

namespace {

using nrf::PlanLayout;

constexpr int64_t kSingleRows = 8192;

__device__ __forceinline__ int wave_scan_int(int v) {   // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int u = __shfl_up(v, off);
        if (lane >= off) v += u;
    }
    return v;
}

__device__ __forceinline__ int key_of(const int* __restrict__ index, int64_t row, int E) {
    const int e = index[row];
    return (unsigned)e < (unsigned)E ? e : E;
}

// In place: s[0 .. count) -> exclusive sums, s[count] = total.  All THREADS threads; `part` has THREADS / 64 ints.
template <int THREADS>
__device__ void block_exclusive(int* s, int count, int* part) {
    const int per = (count + THREADS - 1) / THREADS, at = threadIdx.x * per;
    int sum = 0;
    for (int i = 0; i < per; ++i)
        if (at + i < count) sum += s[at + i];
    const int incl = wave_scan_int(sum);
    if ((threadIdx.x & 63) == 63) part[threadIdx.x >> 6] = incl;
    __syncthreads();
    int run = incl - sum;
    for (int w = 0; w < int(threadIdx.x >> 6); ++w) run += part[w];
    for (int i = 0; i < per; ++i)
        if (at + i < count) {
            const int v = s[at + i];
            s[at + i] = run;
            run += v;
        }
    if (threadIdx.x == THREADS - 1) s[count] = run;   // its range is the last one (empty ranges carry the sum on)
    __syncthreads();
}

__global__ __launch_bounds__(512) void plan_hist_kernel(const int* __restrict__ index, int64_t n, int E, int64_t chunk,
                                                        int* __restrict__ hist) {
    extern __shared__ int s_count[];
    for (int k = threadIdx.x; k <= E; k += 512) s_count[k] = 0;
    __syncthreads();
    const int64_t begin = blockIdx.x * chunk, end = begin + chunk < n ? begin + chunk : n;
    for (int64_t r = begin + threadIdx.x; r < end; r += 512) atomicAdd(&s_count[key_of(index, r, E)], 1);
    __syncthreads();
    for (int k = threadIdx.x; k <= E; k += 512) hist[int64_t(blockIdx.x) * (E + 1) + k] = s_count[k];
}

// hist[chunk][key] -> exclusive sums over the chunks, totals[key].  64 keys per workgroup, the chunks dealt to 16 wavefronts.
__global__ __launch_bounds__(1024) void plan_chunks_kernel(int* __restrict__ hist, int chunks, int E, int* __restrict__ totals) {
    __shared__ int s_sum[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, key = blockIdx.x * 64 + lane;
    const int per = (chunks + 15) / 16, c0 = wave * per, c1 = c0 + per < chunks ? c0 + per : chunks;
    int sum = 0;
    if (key <= E)
#pragma unroll 8
        for (int c = c0; c < c1; ++c) sum += hist[int64_t(c) * (E + 1) + key];
    s_sum[wave][lane] = sum;
    __syncthreads();
    int run = 0;
    for (int w = 0; w < wave; ++w) run += s_sum[w][lane];
    if (key > E) return;
#pragma unroll 8
    for (int c = c0; c < c1; ++c) {
        int* p = hist + int64_t(c) * (E + 1) + key;
        const int v = *p;
        *p = run;
        run += v;
    }
    if (wave == 15) totals[key] = run;
}

// The walk.  SINGLE: the one workgroup of a small batch, which also makes the totals.
template <int WAVES, bool SINGLE>
__global__ __launch_bounds__(WAVES * 64) void plan_place_kernel(const int* __restrict__ index, int64_t n, int E, int64_t chunk,
                                                                const int* __restrict__ hist, const int* __restrict__ totals,
                                                                int* __restrict__ plan) {
    constexpr int THREADS = WAVES * 64;
    extern __shared__ int s_mem[];
    __shared__ int s_part[WAVES];
    const int keys = E + 1, stride = (keys + 1) & ~1;      // 16-bit counters, an even number per wavefront
    int* s_off = s_mem;                                    // [keys + 1]
    int* s_run = s_mem + ((keys + 2) & ~1);                // [keys + 1]
    unsigned* s_cnt32 = reinterpret_cast<unsigned*>(s_mem + 2 * ((keys + 2) & ~1));
    unsigned short* s_cnt = reinterpret_cast<unsigned short*>(s_cnt32);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

    for (int i = threadIdx.x; i < WAVES * stride / 2; i += THREADS) s_cnt32[i] = 0;
    if (!SINGLE)
        for (int k = threadIdx.x; k < keys; k += THREADS) s_off[k] = totals[k];
    __syncthreads();

    const int64_t begin = blockIdx.x * chunk, end = begin + chunk < n ? begin + chunk : n;
    const int64_t per = ((end - begin + THREADS - 1) / THREADS) * 64;   // rows of a wavefront, whole 64s
    const int64_t w0 = begin + wave * per, w1 = w0 + per < end ? w0 + per : end;
    unsigned short* mine = s_cnt + wave * stride;
    for (int64_t r = w0 + lane; r < w1; r += 64) {
        const int slot = wave * stride + key_of(index, r, E);
        atomicAdd(&s_cnt32[slot >> 1], (slot & 1) ? 0x10000u : 1u);
    }
    __syncthreads();
    for (int k = threadIdx.x; k < keys; k += THREADS) {
        int run = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const int v = s_cnt[w * stride + k];
            s_cnt[w * stride + k] = (unsigned short)run;
            run += v;
        }
        if (SINGLE) s_off[k] = run;
    }
    __syncthreads();
    block_exclusive<THREADS>(s_off, keys, s_part);

    const PlanLayout L(n, E);
    for (int k = blockIdx.x * THREADS + threadIdx.x; k < keys; k += gridDim.x * THREADS) {
        plan[L.offsets + k] = s_off[k];
        if (k < E) plan[k] = s_off[k + 1] - s_off[k];
    }
    // the tables: whole runs look their key up in the keys' sums, then every key with a rest has one run more
    for (int t = 0; t < nrf::kTileTables; ++t) {
        const int s = nrf::kTileShift0 + t;
        int2* out = reinterpret_cast<int2*>(plan + L.tiles[t]);
        for (int k = threadIdx.x; k < keys; k += THREADS) s_run[k] = (s_off[k + 1] - s_off[k]) >> s;
        __syncthreads();
        block_exclusive<THREADS>(s_run, keys, s_part);
        const int whole = s_run[keys];
        for (int run = blockIdx.x * THREADS + threadIdx.x; run < whole; run += gridDim.x * THREADS) {
            int lo = 0, hi = E;   // the last key whose first run is not past this one: it has a run
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (s_run[mid] <= run) lo = mid;
                else hi = mid - 1;
            }
            out[run] = make_int2(s_off[lo] + ((run - s_run[lo]) << s), 1 << (16 + s) | lo);
        }
        __syncthreads();
        for (int k = threadIdx.x; k < keys; k += THREADS) s_run[k] = ((s_off[k + 1] - s_off[k]) & ((1 << s) - 1)) != 0;
        __syncthreads();
        block_exclusive<THREADS>(s_run, keys, s_part);
        for (int k = blockIdx.x * THREADS + threadIdx.x; k < keys; k += gridDim.x * THREADS) {
            const int rest = (s_off[k + 1] - s_off[k]) & ((1 << s) - 1);
            if (rest) out[whole + s_run[k]] = make_int2(s_off[k + 1] - rest, rest << 16 | k);
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) plan[L.runs + 2 * t] = whole, plan[L.runs + 2 * t + 1] = whole + s_run[keys];
        __syncthreads();
    }
    if (!SINGLE) {
        __syncthreads();
        for (int k = threadIdx.x; k < keys; k += THREADS) s_off[k] += hist[int64_t(blockIdx.x) * keys + k];
    }
    __syncthreads();

    int* order = plan + L.order;
    const int bits = 32 - __clz(E);                        // keys 0 .. E
    const unsigned long long below = (1ull << lane) - 1;
    for (int64_t r0 = w0; r0 < w1; r0 += 64) {
        const int64_t r = r0 + lane;
        const bool there = r < w1;
        const int key = there ? key_of(index, r, E) : 0;
        unsigned long long same = __ballot(there);
        for (int b = 0; b < bits; ++b) {
            const bool one = (key >> b) & 1;
            const unsigned long long m = __ballot(one);
            same &= one ? m : ~m;
        }
        if (there) {
            const int start = mine[key];
            order[s_off[key] + start + __popcll(same & below)] = int(r);
            if ((same >> lane) == 1) mine[key] = (unsigned short)(start + __popcll(same));   // the highest lane of the key
        }
        // the next 64 rows' lanes read what these lanes wrote: same wavefront, LDS in order, the compiler kept from moving it
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

int64_t plan_chunk(int64_t n) {
    int64_t chunk = (n + 255) / 256;          // one workgroup per CU; a counter of a chunk has 16 bits
    if (chunk < 2048) chunk = 2048;
    return chunk > 32768 ? 32768 : chunk;
}
bool plan_single(int64_t n) { return n <= kSingleRows; }

size_t place_lds(int E, int waves) {
    return size_t((E + 3) & ~1) * 8 + size_t(waves) * ((E + 2) & ~1) * 2;
}

template <int WAVES, bool SINGLE>
int launch_place(const int* index, int64_t n, int E, int64_t chunk, int64_t chunks, const int* hist, const int* totals, int* plan,
                 hipStream_t stream) {
    if (place_lds(E, WAVES) > 65536 - 1024 &&
        hipFuncSetAttribute(reinterpret_cast<const void*>(&plan_place_kernel<WAVES, SINGLE>), hipFuncAttributeMaxDynamicSharedMemorySize,
                            int(place_lds(E, WAVES))) != hipSuccess)
        return NRF_ERR_LAUNCH;
    plan_place_kernel<WAVES, SINGLE><<<dim3(unsigned(chunks)), WAVES * 64, place_lds(E, WAVES), stream>>>(index, n, E, chunk, hist,
                                                                                                         totals, plan);
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
    const bool wide = E > 4096;               // eight wavefronts' counters fit in LDS up to 4096 experts, one's beyond
    int* out = static_cast<int*>(plan);
    nrf_launch_begin();
    if (plan_single(n_rows)) {
        const int64_t chunk = n_rows > 0 ? n_rows : 1;
        const int st = wide ? launch_place<1, true>(index, n_rows, E, chunk, 1, nullptr, nullptr, out, stream)
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
    const int st = wide ? launch_place<1, false>(index, n_rows, E, chunk, chunks, hist, totals, out, stream)
                        : launch_place<8, false>(index, n_rows, E, chunk, chunks, hist, totals, out, stream);
    return st != NRF_OK ? st : nrf_launch_status();
}
