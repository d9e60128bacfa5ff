// When the few-rows kernel of the microscaled products (gemm_fp4_fewrows.cu) is taken, and its launch: plain arithmetic on
// the sizes.
#pragma once

namespace i4l {

constexpr int kFewRowsTile = 128;                           // rows of w per tile, and of x per group
constexpr int kFewRowsStepBytes = 128, kFewRowsStepK = 256;  // of a row, per step
constexpr int kFewRowsMaxStages = 3;
constexpr int kSmShared = 228 * 1024;  // of an SM; each CTA takes 1 KB more than it asks for
constexpr int kSharedPerCol = 448;     // least shared memory per tensor-memory column
static_assert(kSmShared / kSharedPerCol < 512 + 128, "no mixture of CTAs may exceed the 512 columns");

// Layout of a stage: w codes, scales (w, x), then the x codes (rounded up: a stage starts on 1024 bytes).
template <bool kBlock16, bool kGated>
struct FewRowsGeo {
    static constexpr int kTilesK = kBlock16 ? 4 : 2;
    static constexpr int kW = kGated ? 2 : 1;                 // weight matrices
    static constexpr int kScaleBytes = kTilesK * 512;
    static constexpr int kScaleCols = 4 * kTilesK * (kW + 1);  // tensor-memory columns of a stage's scales
    static constexpr int kCodesW = kFewRowsTile * kFewRowsStepBytes;
    static constexpr int kOffScales = kW * kCodesW;
    static constexpr int kOffX = kOffScales + (kW + 1) * kScaleBytes;
    static_assert(kOffX % 1024 == 0, "x tile must keep the swizzle alignment");
};

struct FewRowsPlan {
    int n_pad;    // rows of x in the UMMA, a multiple of 16
    int tiles;    // of 128 rows of w
    int groups;   // of 128 rows of x
    int split;    // CTAs per cluster, each with a part of k
    int stages, stage_bytes, cols;
    int smem;
};

// Up to 64 rows this kernel is the faster one everywhere (64 x 14336 x 4096: 11.5 us against 11.9; 1 x 4096 x 4096: 6.1
// against 8.2), from there on only where the tiles of gemm_fp4.cu leave most SMs idle for a long k: 128 x 1024 x 8192
// 8.9 us against 13.9, 256 x 1024 x 8192 10.1 against 14.8, but 128 x 1024 x 1024 7.1 against 5.2 and 256 x 4096 x 4096
// 10.8 against 9.9.  A gated tile has twice the partial sums to exchange and does not profit.
inline bool fewrows_preferred(int m, int n, int k, bool gated, int sm_count)
{
    if (m <= 64) return true;
    if (gated || m > 256 || k <= 6144) return false;
    const int tiles = (n + kFewRowsTile - 1) / kFewRowsTile * ((m + 127) / 128);
    return tiles <= sm_count / 4;
}

template <bool kBlock16, bool kGated>
inline FewRowsPlan fewrows_plan(int m, int n, int k, int sm_count)
{
    using G = FewRowsGeo<kBlock16, kGated>;
    FewRowsPlan p = {};
    p.n_pad = m >= 128 ? 128 : (m + 15) / 16 * 16;
    p.groups = (m + 127) / 128;
    p.tiles = (n + kFewRowsTile - 1) / kFewRowsTile;
    const int steps = (k + kFewRowsStepK - 1) / kFewRowsStepK;
    // About two CTAs per SM.  More rows of x make the reduction the larger part: a CTA then takes at least 4 steps
    // (64 x 4096 x 4096 mxfp4: 7.9 us with 4 CTAs to a tile, 8.7 with 8; 16 rows: 6.3 and 6.2).
    int split = 2 * sm_count / (p.tiles * p.groups);
    if (p.n_pad > 32 && split > steps / 4) split = steps / 4;
    split = split < 1 ? 1 : (split > 8 ? 8 : split);
    if (split > steps) split = steps;
    p.split = split;
    const int steps_cta = (steps + split - 1) / split;
    p.stage_bytes = (G::kOffX + p.n_pad * kFewRowsStepBytes + 1023) / 1024 * 1024;
    // As many stages as half an SM's shared memory takes, fewer where their scales do not fit half its tensor memory (at
    // least two either way: the rule above sends at most 128 columns of accumulators and 46 KB a stage here).
    const int acc = G::kW * p.n_pad;
    const int room = kSmShared / 2 - 1024 - 2048;  // less alignment and static part
    int stages = room / p.stage_bytes < (256 - acc) / G::kScaleCols ? room / p.stage_bytes : (256 - acc) / G::kScaleCols;
    if (stages > kFewRowsMaxStages) stages = kFewRowsMaxStages;
    if (stages > steps_cta) stages = steps_cta;
    p.stages = stages;
    const int cols = acc + stages * G::kScaleCols;
    p.cols = cols <= 128 ? 128 : 256;
    p.smem = 1024 + stages * p.stage_bytes;
    const int partials = split > 1 ? 1024 + G::kW * p.n_pad * kFewRowsTile * 4 : 0;
    if (p.smem < partials) p.smem = partials;
    const int share = p.cols * kSharedPerCol - 1024;
    if (p.smem < share) p.smem = share;
    return p;
}

}  // namespace i4l
