// What a backward pass of microscaled matrices (gemm_grad.cu) does, from its sizes alone: which operands are expanded by a launch
// of their own, whether the gate's gradients are carried in one term or two, into how many parts contractions are cut,
// and the workspace.  Host only; a test runs it on the CPU.
#pragma once

#include <cmath>

namespace i4l {

constexpr int kBN = 256, kStepK = 64;  // columns of a tile, contraction of a step

// One kind of tile: dx (its A operand is K-major), or a weight gradient (`matrices` of them, A MN-major).  A contraction
// is `segments` runs of `seg_steps` steps, each over operands of its own, cut into `parts`.
struct Kind {
    int weight, matrices;
    int rows, cols;         // of one result
    int tiles_m, tiles_n;   // of one result
    int segments, seg_steps, parts;
};
// Everything that follows from the sizes alone: kinds, parts, and the workspace's pieces, each on a 256-byte boundary.
struct Plan {
    Kind dx, dw;
    bool fine = false;
    bool unpack = false;  // the products expand w and x themselves
    long long tiles_dx = 0, tiles_dw = 0;
    long long d[4] = {}, w[2] = {}, x = 0, partial[3] = {}, bytes = 0, ld = 0;
};
constexpr int kPlanWorkers = 74;  // CTA pairs of a B200
constexpr int kTileSteps = 6;     // a tile's epilogue, in steps: it runs beside the next tile's steps, and is longer than few of them
constexpr int kMinPart = 8;       // steps of a part: less would be the time of a tile's start and end
constexpr int kMaxParts = 74;
constexpr double kSumSteps = 12;       // the third launch, in steps (0.28 us each)
constexpr double kStepBytes = 1.8e6;   // that pass through HBM in a step's time

// terms of dg and du: 1, 2, or 0 for the rule below.
inline Plan plan(long long m, long long n, long long k, bool gated, bool want_dx, bool want_dw, int terms = 0)
{
    Plan p;
    const int matrices = gated ? 2 : 1;
    const int steps_n = static_cast<int>((n + kStepK - 1) / kStepK), steps_m = static_cast<int>((m + kStepK - 1) / kStepK);
    const int tn = static_cast<int>((k + kBN - 1) / kBN);
    p.dx = Kind{0, 1, static_cast<int>(m), static_cast<int>(k), static_cast<int>((m + 255) / 256), tn, matrices, steps_n, 1};
    p.dw = Kind{1, matrices, static_cast<int>(n), static_cast<int>(k), static_cast<int>((n + 255) / 256), tn, 1, steps_m, 1};
    // What is decided here does not depend on which gradients are wanted, so their bits do not either.
    const double tiles_dx = static_cast<double>(p.dx.tiles_m) * tn, tiles_dw = static_cast<double>(matrices) * p.dw.tiles_m * tn;
    const double load = (tiles_dx * matrices * steps_n + tiles_dw * steps_m) / kPlanWorkers;  // steps of a worker
    // Expanded operands go to memory and come back: four times their bytes, twice, which few tokens do not repay, and
    // it is a launch of its own.  The in-kernel expansion holds the products below 1.4 PFLOP/s.  Measured, in-kernel
    // against expanded, back to back in a graph: mxfp4 64 x 8192 x 4096 45 us and 54 (dx alone 27 and 36), 256 rows 55 and 64, 512 rows
    // 82 and 89, 1024 rows 131 and 127, gated 512 rows 164 and 177; nvfp4 1024 rows 129 and 132, 4096 x 4096 x 8192 444
    // and 424.  A small layer gains by the launch it saves, called from a program (128 x 1024 x 1024 14.2 us and 16.4, 1021 rows
    // 14.3 and 16.5), and loses as much in a graph, where launches are cheap; 600 x 3000 x 1024 19.8 and 20.7.
    p.unpack = m <= 512 || load <= 24.0;
    // Two terms for dg and du where twice the steps are a few microseconds, or where there are so few values of them
    // that the time goes into the weights.
    p.fine = gated && (terms == 2 || (terms == 0 && (2.0 * load <= 24.0 || m * n <= 65536)));
    if (p.fine) {
        p.dx.segments *= 2;
        p.dw.segments *= 2;
    }
    // Parts.  A gradient alone takes the rounds of the busiest worker; both together the mean load or the longest tile, since
    // the shorter tiles fill the gaps of the longer.  Either way the parts' sums are written and read back, and that
    // costs a third launch.  One number of parts serves all calls: it is the one with the least product of both times,
    // each against that of whole contractions.  (Weighing the rounds alone cut gated 2048 x 8192 x 4096 in four: 505 us
    // against 462 whole, and 306 against 274 for dx alone.  512 x 8192 x 4096 shows what is weighed: cut in two
    // dx alone takes 43 us instead of 61, both together 83 instead of 78.)
    const double tiles[2] = {tiles_dx, tiles_dw};
    auto part_steps = [](const Kind& kind, int parts) { return (kind.segments * kind.seg_steps + parts - 1) / parts; };
    auto tile_time = [](int steps) { return static_cast<double>(steps > kTileSteps ? steps : kTileSteps); };
    auto cut = [&](Kind& kind, const Kind& other) {
        const double own = tiles[kind.weight], others = tiles[other.weight];
        if (own >= 4.0 * kPlanWorkers) return;
        const int steps = kind.segments * kind.seg_steps, others_steps = part_steps(other, other.parts);
        const double others_load = others * other.parts * tile_time(others_steps);
        auto product = [&](int parts) {
            const int part = part_steps(kind, parts);
            const double sums = parts > 1 ? kSumSteps + 8.0 * parts * kind.matrices * kind.rows * kind.cols / kStepBytes : 0.0;
            const double alone = std::ceil(own * parts / kPlanWorkers) * (part + kTileSteps) + sums;
            const double mean = (own * parts * tile_time(part) + others_load) / kPlanWorkers;
            return alone * (std::fmax(mean, std::fmax(part, others_steps)) + sums);
        };
        double best = 0.95 * product(1);
        for (int parts = 2; parts <= kMaxParts && steps / parts >= kMinPart; ++parts) {
            const double time = product(parts);
            if (time < best) { best = time; kind.parts = parts; }
        }
    };
    cut(p.dx, p.dw);
    cut(p.dw, p.dx);
    p.tiles_dx = want_dx ? static_cast<long long>(tiles_dx) * p.dx.parts : 0;
    p.tiles_dw = want_dw ? static_cast<long long>(tiles_dw) * p.dw.parts : 0;

    p.ld = (n + 7) / 8 * 8;
    auto piece = [&](long long bytes) { const long long at = p.bytes; p.bytes += (bytes + 255) / 256 * 256; return at; };
    if (gated || n % 8 != 0) p.d[0] = piece(m * p.ld * 2);  // (else dy is read as it is)
    if (gated) p.d[1] = piece(m * p.ld * 2);
    if (p.fine) { p.d[2] = piece(m * p.ld * 2); p.d[3] = piece(m * p.ld * 2); }
    if (want_dx && !p.unpack) { p.w[0] = piece(n * k * 2); if (gated) p.w[1] = piece(n * k * 2); }
    if (want_dw && !p.unpack) p.x = piece(m * k * 2);
    if (want_dx && p.dx.parts > 1) p.partial[0] = piece(p.dx.parts * m * k * 4);
    if (want_dw && p.dw.parts > 1) for (int i = 0; i < matrices; ++i) p.partial[1 + i] = piece(p.dw.parts * n * k * 4);
    return p;
}

}  // namespace i4l
