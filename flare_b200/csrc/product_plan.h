// product_plan.h -- how a 4-bit product's K is shared among the blocks of a cluster (plain C++, no CUDA needed).
#pragma once

#ifdef __CUDACC__
#define FLARE_BOTH __host__ __device__
#else
#define FLARE_BOTH
#endif

namespace flare {

constexpr int MOST_PARTS = 8;  // the largest cluster that every device allows

// stages of K per block of a cluster: an even number, as scales are read two stages at a time
FLARE_BOTH constexpr int part_of_k(int all, int S) { return S == 1 ? all : ((all + S - 1) / S + 1) / 2 * 2; }

// Clusters of S blocks, one a multiprocessor, that a B200 runs at once (as the runtime's occupancy count has it): its 148
// multiprocessors lie in groups that a cluster does not leave.  16 clusters of 8 take two turns (24 x 2048 x 8192: 12.2 us,
// 6 parts 7.8).
constexpr int clusters_at_once(int S) {
    constexpr int n[MOST_PARTS + 1] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
    return n[S];
}

// Blocks that share a tile of `all` stages, of whose columns `columns` are stored: the number that takes the least time.  A stage
// takes 0.38 us (0.6 where a block quantises rows on the way); a cluster's barriers 0.75; a column of the sum 0.165, and
// the blocks share the columns, so one without stages of its own may still help.  One B200, us, by 1 2 4 8 parts:
//    64 x 1024 x 1024 (4 stages)  5.9 10.9  8.1 6.9     64 x 1024 x 8192  16.7 16.4 10.7 7.9
//     4 x 1024 x 1024, quantised  4.9  5.3  5.1 5.0      4 x 4096 x 4096, plain rows  14.7 11.5 8.2 -
inline int parts_of_k(int all, long long tiles, int columns, bool plain_rows) {
    int best = 1;
    float least = 0.0f;
    for (int S = 1; S <= MOST_PARTS; ++S) {
        if (S > 1 && tiles > clusters_at_once(S)) continue;
        const float sum = S == 1 ? 0.0f : 0.75f + 0.165f * (float)((columns + S - 1) / S);
        const float time = (plain_rows ? 0.6f : 0.38f) * (float)part_of_k(all, S) + sum;
        if (S > 1 && time >= least) continue;
        least = time;
        best = S;
    }
    return best;
}

}  // namespace flare
