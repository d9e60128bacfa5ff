// CPU check of how the tiles of a backward pass are dealt out (int4linear_b200/csrc/grad_schedule.cuh): for many
// combinations every tile of both kinds belongs to exactly one worker, each worker's list ends, and the busiest worker
// has at most the mean load and one longest tile.  Prints "DEAL_OK <cases>".
#include <algorithm>
#include <cstdio>
#include <vector>

#include "../int4linear_b200/csrc/grad_schedule.cuh"

using namespace i4l;

static int check(int t0, int t1, int s0, int s1, int max_workers)
{
    const int workers = std::min(t0 + t1, max_workers);
    const Deal d = deal_tiles(t0, t1, s0, s1, workers);
    std::vector<int> seen[2] = {std::vector<int>(t0, 0), std::vector<int>(t1, 0)};
    long long busiest = 0;
    for (int w = 0; w < workers; ++w) {
        long long load = 0;
        int kind = -1, tile = -1, i = 0;
        for (; d.tile_of(w, workers, i, kind, tile); ++i) {
            if (kind < 0 || kind > 1 || tile < 0 || tile >= (kind ? t1 : t0)) return 1;
            ++seen[kind][tile];
            load += kind ? s1 : s0;
            if (i > t0 + t1) return 2;
        }
        busiest = std::max(busiest, load);
    }
    for (const auto& v : seen)
        for (int c : v)
            if (c != 1) return 3;
    const double mean = (static_cast<double>(t0) * s0 + static_cast<double>(t1) * s1) / workers;
    if (busiest > mean + 1.5 * s0 + s1) return 4;
    return 0;
}

int main()
{
    const int counts[] = {0, 1, 2, 5, 16, 34, 73, 74, 75, 148, 255, 256, 896, 1792};
    const int lengths[] = {1, 2, 3, 16, 17, 64, 86, 448};
    int cases = 0;
    for (int t0 : counts)
        for (int t1 : counts)
            for (int s0 : lengths)
                for (int s1 : lengths)
                    for (int workers : {1, 2, 7, 66, 74}) {
                        if (t0 + t1 == 0 || s1 > s0) continue;
                        if (const int rc = check(t0, t1, s0, s1, workers)) {
                            std::printf("FAIL %d: %d %d tiles, %d %d steps, %d workers\n", rc, t0, t1, s0, s1, workers);
                            return 1;
                        }
                        ++cases;
                    }
    std::printf("DEAL_OK %d\n", cases);
    return 0;
}
