// Dealing out the tiles of a backward pass (gemm_grad.cu) to the workers of a persistent kernel (host + device).
//
// There are two kinds of tile, kind 0 with the longer contraction.  Kind 0 goes round-robin; a worker that got one
// tile fewer than others first takes `extra` tiles of kind 1, about as long as one of kind 0 together; the rest of
// kind 1 goes round-robin.  Every role of the kernel enumerates the same list, so the roles agree without talking.
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

// steps0 >= steps1: lengths of the two kinds' contractions.
inline Deal deal_tiles(int tiles0, int tiles1, int steps0, int steps1, int workers)
{
    Deal d;
    d.tiles[0] = tiles0;
    d.tiles[1] = tiles1;
    d.extra = tiles0 % workers == 0 ? 0 : (steps0 + steps1 / 2) / steps1;
    return d;
}

}  // namespace i4l
