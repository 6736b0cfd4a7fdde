// Rows grouped by expert: the plan that nrf_expert_plan (expert_plan.hip) leaves for the grouped products
// (expert_linear.hip).  All of it is int32, in one buffer:
//   counts   [E]                 rows of expert e
//   offsets  [E + 1]             first grouped place of expert e; offsets[E] = rows that have an expert
//   order    [n]                 the row at each grouped place: expert 0's rows ascending, expert 1's, ..., then the rows
//                                of no expert (index outside [0, E)) ascending
//   runs     [4][2]              for each of the tables below: how many long runs it holds, and how many in all
//   tiles    for 32, 64, 128 and 256 rows: {first grouped place, rows << 16 | expert} of the runs of at most that many rows of
//            one expert ("expert" E: the rows of no expert): first, in grouped order, the long runs (all but those of half
//            the length and less: as costly as whole ones, next to the runs that share their weights), then the short rests
//            (a product's last workgroups are then its shortest; 32 k rows, 32 experts of 2048 x 2048, five routings: 375 -
//            398 us, with every rest at the end 397 - 406, with none there 381 - 396)
// A table of runs of 2^s rows has at most (n >> s) + E + 1 entries, and no more than rows: the host sizes the products' grids
// with that and never reads a count back; workgroups past the table's count leave at once.
#pragma once
#include "nrf_common.h"

namespace nrf {

constexpr int kMaxExperts = 16384;            // 15 bits of a tile word; the keys' counters of a workgroup fit in LDS
constexpr int64_t kMaxExpertRows = 1ll << 28;
constexpr int kTileShift0 = 5, kTileTables = 4;   // 32, 64, 128, 256 rows

struct PlanLayout {
    int64_t offsets, order, runs, tiles[kTileTables], total;   // in int32 words; counts at 0
    __host__ __device__ static constexpr int64_t up4(int64_t v) { return (v + 3) & ~int64_t(3); }
    __host__ __device__ static constexpr int64_t slots(int64_t n, int E, int table) { return (n >> (kTileShift0 + table)) + E + 1; }
    static constexpr int64_t most_runs(int64_t n, int E, int table) { return slots(n, E, table) < n ? slots(n, E, table) : n; }
    __host__ __device__ constexpr PlanLayout(int64_t n, int E) : offsets(up4(E)), order(0), runs(0), tiles{0, 0, 0, 0}, total(0) {
        order = offsets + up4(E + 1);
        runs = order + up4(n);
        int64_t at = runs + 2 * kTileTables;
        for (int t = 0; t < kTileTables; ++t) {
            tiles[t] = at;
            at += up4(2 * slots(n, E, t));
        }
        total = at;
    }
};

}  // namespace nrf
