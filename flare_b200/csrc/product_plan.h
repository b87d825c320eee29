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
// multiprocessors lie in groups that a cluster does not leave.
constexpr int clusters_at_once(int S) {
    constexpr int n[MOST_PARTS + 1] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
    return n[S];
}

// How a tile's rows of 128 leave: as columns of the output, as its rows by 16 bytes, or as its rows element by element.
enum class Store { columns, rows_of_16, rows };

// The time in us of a product whose blocks have `all` stages of K, shared by clusters of S; negative where S is not possible.  A
// stage takes 0.38 us, 0.6 where a block quantises rows on the way.  Clusters take 0.75 for their barriers and a time for
// each column of the sum, which their blocks share, so one without stages of its own may still help.  Blocks of two stages
// are small enough for a second one a multiprocessor, which takes 0.7 longer than a machine of its own; 16 clusters of 8 larger
// ones take two turns (24 x 2048 x 8192: 13.6 us, by 6 parts 8.7).  Element by element, a tile's rows take longer than they do
// from a cluster, which spreads them.
inline float product_time(int S, int all, long long tiles, int columns, bool plain_rows, Store store) {
    const int per = part_of_k(all, S);
    const float stages = (plain_rows ? 0.6f : 0.38f) * (float)per;
    if (S == 1) return stages + (store == Store::rows && columns > 12 ? 0.165f * (float)(columns - 12) : 0.0f);
    const bool second = tiles > clusters_at_once(S);
    if (second && (plain_rows || per > 2 || tiles * S > clusters_at_once(1))) return -1.0f;
    const float column = store == Store::columns ? 0.165f : 0.27f;
    return stages + 0.75f + (second ? 0.7f : 0.0f) + column * (float)((columns + S - 1) / S);
}

// Blocks that share a tile of `all` stages, of whose columns `columns` are stored: what takes the least time.  One B200, us, the
// larger matrix not in L2, by 1 2 4 8 parts:
//    64 x 1024 x 1024   6.5 11.3  8.5 7.3     64 x 1024 x 8192  17.5 17.0 11.2 8.5
//     4 x 1024 x 2048   7.3  6.7  5.7 5.6      4 x 4096 x 4096, plain rows  15.4 12.2 9.1 -
//   1024 x 61 x 2048   15.1 14.7 10.1 8.3   2048 x 64 x 2048     7.6 16.2 10.7 10.3
// Over 277 such sizes the time taken is 0.4 % above the best number's.
inline int parts_of_k(int all, long long tiles, int columns, bool plain_rows, Store store) {
    int best = 1;
    float least = product_time(1, all, tiles, columns, plain_rows, store);
    for (int S = 2; S <= MOST_PARTS; ++S) {
        const float time = product_time(S, all, tiles, columns, plain_rows, store);
        if (time < 0.0f || time >= least) continue;
        least = time;
        best = S;
    }
    return best;
}

}  // namespace flare
