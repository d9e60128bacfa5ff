// Dealing out the tiles of a backward pass (gemm_grad.cu) to the workers of a persistent kernel (host + device).
//
// There are two kinds of tile, kind 0 with the longer contraction.  Kind 0 goes round-robin; a worker that got one
// tile fewer than others first takes `extra` tiles of kind 1; the rest of kind 1 goes round-robin.  `extra` is the
// number that ends the busiest worker soonest.  Every role of the kernel enumerates the same list, so the roles agree
// without talking.
#pragma once

#ifndef __CUDACC__
#define I4L_GRAD_HD inline
#else
#define I4L_GRAD_HD __host__ __device__ __forceinline__
#endif

namespace i4l {

struct Deal {
    int tiles[2] = {0, 0};
    int extra = 0;

    // The i-th tile of a worker: its kind and index; false when there is none.
    I4L_GRAD_HD bool tile_of(int worker, int workers, int i, int& kind, int& tile) const
    {
        const int mine = worker < tiles[0] ? (tiles[0] - worker + workers - 1) / workers : 0;
        if (i < mine) { kind = 0; tile = worker + i * workers; return true; }
        kind = 1;
        i -= mine;
        const int full = tiles[0] % workers;  // workers [full, workers) have one tile of kind 0 fewer
        const int few = workers - full;
        const long long wanted = static_cast<long long>(few) * extra;
        const int dealt = wanted < tiles[1] ? static_cast<int>(wanted) : tiles[1];
        if (worker >= full) {
            const int at = worker - full, own = at < dealt ? (dealt - at + few - 1) / few : 0;
            if (i < own) { tile = at + i * few; return true; }
            i -= own;
        }
        const long long t = dealt + worker + static_cast<long long>(i) * workers;
        tile = static_cast<int>(t);
        return t < tiles[1];
    }
};

// cost0 >= cost1: time of a tile of either kind, in any unit.
inline Deal deal_tiles(int tiles0, int tiles1, int cost0, int cost1, int workers)
{
    Deal d;
    d.tiles[0] = tiles0;
    d.tiles[1] = tiles1;
    const int full = tiles0 % workers;
    if (full == 0) return d;
    const long long few = workers - full, rounds0 = tiles0 / workers;
    long long best = -1;
    for (long long extra = 0; extra <= cost0 / cost1 + 1; ++extra) {
        const long long dealt = few * extra < tiles1 ? few * extra : tiles1, rest = tiles1 - dealt;
        // The rest goes to workers 0, 1, ..., so those with one tile more of kind 0 (they come first) get the odd ones.
        const long long hi = (rounds0 + 1) * cost0 + (rest + workers - 1) / workers * cost1;
        const long long odd = rest % workers > full ? 1 : 0;
        const long long lo = rounds0 * cost0 + ((dealt + few - 1) / few + rest / workers + odd) * cost1;
        const long long end = hi > lo ? hi : lo;
        if (best < 0 || end < best) {
            best = end;
            d.extra = static_cast<int>(extra);
        }
    }
    return d;
}

}  // namespace i4l
