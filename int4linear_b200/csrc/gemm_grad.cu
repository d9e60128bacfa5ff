// Backward pass of the products of microscaled matrices (fp4.cuh, gemm_fp4.cu):
//
//     y = x w^T             dx = dy w                  dw = dy^T x
//     h = act(g) u          dg = dh u act'(g),  du = dh act(g)
//                           dx = dg wg + du wu         dwg = dg^T x,  dwu = du^T x
//
// with respect to the values the operands stand for.  The contraction runs over n or m, across the blocks that
// share a scale, so the block-scaled instruction does not apply: the operands are expanded to bf16 first.  That
// loses nothing (a code times its e8m0 or e4m3 scale has at most 6 significant bits).  Only dg and du are rounded, to
// bf16 as the gradients of a bf16 network are: with the rounding of the result that is 1.4 times the error of one
// rounding (2.4e-3 in the mean square against 1.7e-3).  Where it costs next to nothing (plan() says when), or where the caller
// asks for it, they are carried as the sum of two bf16 values instead, 16 bits, as contractions of twice the length.
//
// Up to three launches.  The first prepares: dg and du (or dy with a row pitch that TMA takes), and the expansions.  The second
// is all products in one persistent kernel, a CTA pair per 256 x 256 tile (tcgen05.mma kind::f16, cta_group::2), two
// accumulators in tensor memory so that the epilogue overlaps the next tile:
//     warp 0      TMA, steps of 64 along the contraction, into 128-byte-swizzled slots
//     warp 1      UMMA issue (CTA 0 for both)
//     warps 2-5   epilogue: scale, round to bf16, staged TMA stores
// For few tokens the second launch expands w and x itself: three groups of four warps take turns at turning a step's codes
// and scales, loaded into a ring of their own, into the bf16 tile that the UMMA reads.
//
// No operand is ever transposed: where the contraction runs down the rows of a matrix (w and x always, dy for
// dw), its tile is read as it lies and the UMMA takes it MN-major.
//
// Where the tiles are too few to occupy the GPU for their length (few tokens, so that dx is a handful of tiles of a
// contraction over all columns), contractions are cut into parts; the parts' fp32 sums go to the workspace, and a third
// launch adds them in order, so that the result does not depend on timing.
//
// The tensor scales are kept out of the expanded matrices.  dx = dg wg + du wu is one contraction over both, so dg and
// du are multiplied by their weight's tensor scale before they are rounded, and the weight gradients take it out again.
//
// dx and dw tiles have contractions of different length (n or 2 n, and m), and with separate launches each product
// leaves a partly filled last wave.  Together they are dealt out in advance: the longer kind round-robin, the shorter
// kind first to the workers that got one fewer, then round-robin (grad_schedule.cuh; gated 4096 x 14336 x 4096 on 74
// pairs, in tile times of the weight gradients: 28 + 13 + 13 apart, 49 together, 48.4 the mean).
//
// Measured, a single call on an idle GPU and, under the power limit, call after call: 4096 x 4096 x 8192 nvfp4 352 and 430 us (1.56 and 1.28
// PFLOP/s, tensor pipe 91 % busy at the 1.5 GHz the limit leaves), gated 4096 x 14336 x 4096 mxfp4 1.35 and 1.60 ms, of which
// the preparation takes 0.14 (it writes 0.7 GB); dx alone 237 and 226 us, 1.02 and 0.93 ms.
#include "epilogue.cuh"
#include "fp4_expand.cuh"
#include "gate.cuh"
#include "grad_plan.cuh"
#include "grad_schedule.cuh"
#include "ptx.cuh"

namespace i4l {

namespace {

// ------------------------------------------------------------- preparation

// dg = dh u act'(g) f_g, du = dh act(g) f_u with a row pitch of ld; without `gate` a copy of dh.
struct GateJob {
    const __nv_bfloat16* dh; const __nv_bfloat16* gate; const __nv_bfloat16* up;
    __nv_bfloat16* dg; __nv_bfloat16* du;
    __nv_bfloat16* dg_lo; __nv_bfloat16* du_lo;  // what the rounding left, rounded again; or null
    const float* f_g; const float* f_u;
    int m, n, act, vec;
    long long ld;
};
struct ExpandJob {
    const uint8_t* codes; const uint8_t* scales; const float* tensor_scale;
    __nv_bfloat16* dst;
    int rows, k;
};
// Blocks [0, first[0]) belong to the gate, [first[i], first[i + 1]) to expansion i.
struct PrepArgs {
    GateJob gate;
    ExpandJob expand[3];
    uint32_t first[4];
};

template <int kAct>
__device__ __forceinline__ void gate_grad(float dh, float g, float u, float fg, float fu, float& dg, float& du)
{
    float act, slope;
    gate_act_slope<kAct>(g, act, slope);
    dg = dh * u * slope * fg;
    du = dh * act * fu;
}

// What rounding v to `first` left (nothing to add to an infinity).
__device__ __forceinline__ __nv_bfloat16 second_term(float v, __nv_bfloat16 first)
{
    const float f = __bfloat162float(first);
    return __float2bfloat16_rn(isinf(f) ? 0.0f : v - f);
}

// A warp's unit: 256 columns of one row, eight per lane (consecutive where 16-byte accesses are possible, else 32
// apart).  Bound by HBM: 10 bytes per element.
template <int kAct>
__device__ __forceinline__ void gate_block(const GateJob& j, uint32_t block)
{
    const uint32_t u = block * (kUnitThreads / 32) + threadIdx.x / 32, chunks = (j.n + 255u) / 256u;
    const uint32_t row = u / chunks;
    if (row >= static_cast<uint32_t>(j.m)) return;
    const int lane = threadIdx.x & 31, col0 = (u - row * chunks) * 256;
    const size_t src = static_cast<size_t>(row) * j.n, dst = static_cast<size_t>(row) * j.ld;
    float fg = j.f_g != nullptr ? __ldg(j.f_g) : 1.0f, fu = j.f_u != nullptr ? __ldg(j.f_u) : 1.0f;
    if (fg == 0.0f) fg = 1.0f;
    if (fu == 0.0f) fu = 1.0f;
    __align__(16) __nv_bfloat16 h[8] = {}, g[8] = {}, up[8] = {}, og[8], ou[8], lg[8], lu[8];
    auto one = [&](int e) {
        float a, b;
        gate_grad<kAct>(__bfloat162float(h[e]), __bfloat162float(g[e]), __bfloat162float(up[e]), fg, fu, a, b);
        og[e] = __float2bfloat16_rn(a);
        ou[e] = __float2bfloat16_rn(b);
        lg[e] = second_term(a, og[e]);
        lu[e] = second_term(b, ou[e]);
    };
    if (j.vec) {
        const int col = col0 + lane * 8;
        if (col >= j.n) return;
        auto load = [&](const __nv_bfloat16* p) { return __ldg(reinterpret_cast<const uint4*>(p + src + col)); };
        auto store = [&](__nv_bfloat16* p, const __nv_bfloat16 (&v)[8]) { *reinterpret_cast<uint4*>(p + dst + col) = *reinterpret_cast<const uint4*>(v); };
        *reinterpret_cast<uint4*>(h) = load(j.dh);
        *reinterpret_cast<uint4*>(g) = load(j.gate);
        *reinterpret_cast<uint4*>(up) = load(j.up);
#pragma unroll
        for (int e = 0; e < 8; ++e) one(e);
        store(j.dg, og);
        store(j.du, ou);
        if (j.dg_lo != nullptr) { store(j.dg_lo, lg); store(j.du_lo, lu); }
    } else {
        const int col = col0 + lane;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (col + 32 * e < j.n) { h[e] = j.dh[src + col + 32 * e]; g[e] = j.gate[src + col + 32 * e]; up[e] = j.up[src + col + 32 * e]; }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (col + 32 * e >= j.n) break;
            one(e);
            const size_t at = dst + col + 32 * e;
            j.dg[at] = og[e];
            j.du[at] = ou[e];
            if (j.dg_lo != nullptr) { j.dg_lo[at] = lg[e]; j.du_lo[at] = lu[e]; }
        }
    }
}

__device__ __forceinline__ void copy_block(const GateJob& j, uint32_t block)
{
    const uint32_t u = block * (kUnitThreads / 32) + threadIdx.x / 32, chunks = (j.n + 255u) / 256u;
    const uint32_t row = u / chunks;
    if (row >= static_cast<uint32_t>(j.m)) return;
    const int col = (u - row * chunks) * 256 + (threadIdx.x & 31);
    const size_t src = static_cast<size_t>(row) * j.n, dst = static_cast<size_t>(row) * j.ld;
    __nv_bfloat16 v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (col + 32 * e < j.n) v[e] = j.dh[src + col + 32 * e];
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (col + 32 * e < j.n) j.dg[dst + col + 32 * e] = v[e];
}

template <bool kBlock16>
__global__ void __launch_bounds__(kUnitThreads)
backward_prepare_kernel(const __grid_constant__ PrepArgs a)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t b = blockIdx.x;
    if (b < a.first[0]) {
        if (a.gate.gate == nullptr) copy_block(a.gate, b);
        else if (a.gate.act == kActSilu) gate_block<kActSilu>(a.gate, b);
        else if (a.gate.act == kActGelu) gate_block<kActGelu>(a.gate, b);
        else gate_block<kActGeluTanh>(a.gate, b);
    } else {
        const int i = b < a.first[1] ? 0 : (b < a.first[2] ? 1 : 2);
        const ExpandJob& j = a.expand[i];
        fp4_expand_block<INT4L_TYPE_BF16, kBlock16>(b - a.first[i], j.codes, j.scales, j.tensor_scale, false, j.dst, j.rows, j.k);
    }
}

// ---------------------------------------------------------------- products

constexpr int kBM = 128;
constexpr int kStage = 2 * 128 * 128;          // A and B tile of one CTA, 16 KB each
constexpr int kChunk = kStepK * 128;           // a box: 64 columns x 64 rows
constexpr int kStoreStage = 4096;              // per warp and buffer
constexpr int kPackedStages = 6;
constexpr int kGroups = 3;                     // expansion groups of 4 warps, taking turns (2: a tenth slower)
// (every use of a packed stage by the same group: a wait names a phase by its parity only)
static_assert(kPackedStages % kGroups == 0, "ring depth and groups");
constexpr int kPackedCodes = kStepK * 64;      // 64 rows x 128 codes
constexpr int kPackedStage = kPackedCodes + 1024;  // and the scale tiles of those columns: one (mxfp4) or two (nvfp4)

// kUnpack: the B operand is expanded inside the kernel.
template <bool kUnpack>
struct Geo {
    static constexpr int kThreads = 32 * (kUnpack ? 7 + 4 * kGroups : 6);
    static constexpr int kStages = kUnpack ? 5 : 6;
    static constexpr int kPacked = kUnpack ? kPackedStages : 0;
    static constexpr int kNumBarriers = 2 * kStages + 4 + 2 * kPacked;
    static constexpr int kSmemBytes = 1024 + kStages * kStage + kPacked * kPackedStage + 4 * 2 * kStoreStage + kNumBarriers * 8 + 16;
    static_assert(kSmemBytes <= 232448, "shared memory budget");
};

struct GradArgs {
    Kind kind[2];           // the one with the longer contraction first; kind[1] may have no tiles
    Deal deal;
    int fine;               // d[2], d[3]: second terms of d[0], d[1]
    float* partial[3];      // dx, dw, dw_up: the parts' sums, [part][row][col], where parts > 1
    const float* num; const float* den[2];  // dw[i] *= num / den[i]
    const float* dx_scale;                  // dx *= this
    // In-kernel expansion: scales and (for a scale of 0) tensor scales of w, w_up, x; rows of w and of x; scale tiles along k.
    const uint8_t* scales[3]; const float* ts[3];
    int n, m, ktiles;
    int* status;
};
struct Maps {
    CUtensorMap d[4], w[2], x, dx, dw[2];  // w, x: the expanded matrices, or their codes
};

// One arrival of the warp, not before every lane's loads have returned (mbar_arrive_after, for a whole warp).
__device__ __forceinline__ void mbar_arrive_after_warp(uint32_t bar, uint32_t loaded, int lane)
{
    const uint32_t all = __reduce_xor_sync(0xFFFFFFFFu, loaded);
    if (lane == 0) mbar_arrive_after(bar, all);
}

// 64 codes of one row and their scales (a word of 4 in nvfp4, 2 bytes in mxfp4) -> 64 bf16, eight 16-byte chunks of a
// 128-byte-swizzled row.  Rows outside the matrix are 0 whatever their scale; factor is 0 under a tensor scale of 0, else 1 (a
// NaN scale stays NaN).
template <bool kBlock16>
__device__ __forceinline__ void expand_row(uint4 lo, uint4 hi, uint32_t scale_word, bool outside, float factor, uint32_t row_at, int row)
{
    const uint32_t words[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        const uint32_t byte = (scale_word >> (8 * (kBlock16 ? c / 2 : c / 4))) & 0xFFu;
        float sc = fp4_scale<kBlock16>(byte);
        if (kBlock16) sc *= factor;
        if (outside) sc = 0.0f;
        uint32_t h2[4];
        fp4_codes_to_halves(words[c], h2);
        uint32_t out[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h2[b]));
            out[b] = pack16<false>(v.x * sc, v.y * sc);  // exact
        }
        sts128(row_at + ((c ^ (row & 7)) << 4), make_uint4(out[0], out[1], out[2], out[3]));
    }
}

__device__ __forceinline__ float result_scale(const float* num, const float* den)
{
    float v = num != nullptr ? __ldg(num) : 1.0f;
    if (den != nullptr) {
        const float d = __ldg(den);
        if (d != 0.0f) v /= d;  // (0: dg was left as it is)
    }
    return v;
}

struct Tile {
    const Kind* kind;
    int weight, matrix, part, tm, tn;
    int step0, step1;  // of the contraction
};
__device__ __forceinline__ bool take_tile(const GradArgs& a, int worker, int workers, int i, Tile& t)
{
    int kind, tile;
    if (!a.deal.tile_of(worker, workers, i, kind, tile)) return false;
    const Kind& k = a.kind[kind];
    t.kind = &k;
    t.weight = k.weight;
    const int per = k.tiles_m * k.tiles_n;
    t.matrix = tile / (per * k.parts);
    tile -= t.matrix * per * k.parts;
    t.part = tile / per;
    tile -= t.part * per;
    const long long steps = static_cast<long long>(k.segments) * k.seg_steps;
    t.step0 = static_cast<int>(steps * t.part / k.parts);
    t.step1 = static_cast<int>(steps * (t.part + 1) / k.parts);
    // Raster: groups of 16 row blocks share their column panel in L2.
    constexpr int kGroupM = 16;
    const int group = tile / (kGroupM * k.tiles_n);
    const int gm = min(k.tiles_m - group * kGroupM, kGroupM);
    const int in_group = tile - group * kGroupM * k.tiles_n;
    t.tm = group * kGroupM + in_group % gm;
    t.tn = in_group / gm;
    return true;
}

template <bool kUnpack, bool kBlock16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Geo<kUnpack>::kThreads, 1)
grad_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ GradArgs a)
{
    using G = Geo<kUnpack>;
    constexpr int S = G::kStages, P = G::kPacked;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* gbase = smem_raw + (base - raw);

    const uint32_t ring = base;
    const uint32_t packed = ring + S * kStage;
    const uint32_t st_base = packed + P * kPackedStage;
    const uint32_t bar_base = st_base + 4 * 2 * kStoreStage;
    auto full     = [&](int i) { return bar_base + 8u * i; };  // (CTA 0's, for the loads of both)
    auto empty    = [&](int i) { return bar_base + 8u * (S + i); };
    auto tm_full  = [&](int i) { return bar_base + 8u * (2 * S + i); };
    auto tm_empty = [&](int i) { return bar_base + 8u * (2 * S + 2 + i); };
    auto pk_full  = [&](int i) { return bar_base + 8u * (2 * S + 4 + i); };
    auto pk_empty = [&](int i) { return bar_base + 8u * (2 * S + 4 + P + i); };
    const uint32_t misc_off = (bar_base - base) + 8u * G::kNumBarriers;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + misc_off);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + misc_off + 4);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t cta_rank = cluster_cta_rank();
    const int worker = static_cast<int>(cluster_id_x());
    const int workers = static_cast<int>(cluster_count_x());

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(full(i), kUnpack ? 1 + 2 * 4 : 1); mbar_init(empty(i), 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(tm_full(i), 1); mbar_init(tm_empty(i), 4 * 2); }
        for (int i = 0; i < P; ++i) { mbar_init(pk_full(i), 1); mbar_init(pk_empty(i), 4); }
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 1) {
        tmem_alloc<2>(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
        tmem_relinquish<2>();
    }
    tc_fence_before_sync();
    cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    if (warp == 0) {
        // ------------------------------------------------------ TMA producer
        uint32_t it = 0;
        bool alive = true;
        Tile t;
        for (int i = 0; alive && take_tile(a, worker, workers, i, t); ++i) {
            const int row = (t.tm * 2 + static_cast<int>(cta_rank)) * kBM;
            const int col = t.tn * kBN + static_cast<int>(cta_rank) * 128;
            int seg = t.step0 / t.kind->seg_steps, in_seg = t.step0 - seg * t.kind->seg_steps;
            for (int st = t.step0; st < t.step1; ++st, ++it) {
                const uint32_t s = it % S, r = it / S;
                if (!mbar_wait_warp(empty(s), (r & 1u) ^ 1u, abort_flag)) { alive = false; break; }
                if (elect_one()) {
                    // Both CTAs' loads are counted on CTA 0's barrier (which cannot complete before this announcement).
                    if (cta_rank == 0) mbar_expect_tx(full(s), kUnpack ? kStage : 2 * kStage);
                    const uint32_t bar = cluster_address(full(s), 0);
                    const uint32_t dst = ring + s * kStage;
                    // dx: d[0] w[0] (+ d[2] w[0]) + d[1] w[1] (+ d[3] w[1]); dw[i]: d[i]^T x (+ d[i + 2]^T x)
                    const int term = a.fine ? seg & 1 : 0, which = t.weight ? t.matrix : (a.fine ? seg >> 1 : seg);
                    const int k0 = in_seg * kStepK;
                    const CUtensorMap* ta = &maps.d[which + 2 * term];
                    const CUtensorMap* tb = t.weight ? &maps.x : &maps.w[which];
                    tma_load_2d_pair(dst, ta, bar, t.weight ? row : k0, t.weight ? k0 : row);
                    tma_load_2d_pair(dst + kChunk, ta, bar, t.weight ? row + 64 : k0, t.weight ? k0 : row + 64);
                    if constexpr (!kUnpack) {
                        tma_load_2d_pair(dst + 2 * kChunk, tb, bar, col, k0);
                        tma_load_2d_pair(dst + 3 * kChunk, tb, bar, col + 64, k0);
                    }
                }
                __syncwarp();
                if (++in_seg == t.kind->seg_steps) { in_seg = 0; ++seg; }
            }
        }
    } else if (warp == 1) {
        if (cta_rank == 0) {
            // ----------------------------------------------------- UMMA issuer
            // The warp walks the ring together and one elected thread issues.
            uint32_t it = 0;
            bool alive = true;
            Tile t;
            for (int i = 0; alive && take_tile(a, worker, workers, i, t); ++i) {
                const uint32_t buf = i & 1u, br = static_cast<uint32_t>(i) >> 1;
                if (!mbar_wait_warp(tm_empty(buf), (br & 1u) ^ 1u, abort_flag)) break;
                tc_fence_after_sync();
                const uint32_t d_tmem = tmem_base + buf * kBN;
                const uint32_t idesc = umma_idesc_bf16(2 * kBM, kBN, false, true) | (t.weight ? 1u << 15 : 0u);
                // 16 elements of the contraction on: 32 bytes of a K-major row, or two 1024-byte atoms
                const uint32_t step_a = t.weight ? 2048 >> 4 : 32 >> 4, step_b = 2048 >> 4;
                for (int st = t.step0; st < t.step1; ++st, ++it) {
                    const uint32_t s = it % S, r = it / S;
                    if (!mbar_wait_warp(full(s), r & 1u, abort_flag)) { alive = false; break; }
                    tc_fence_after_sync();
                    const uint32_t a_addr = ring + s * kStage;
                    const uint64_t a_desc = t.weight ? umma_desc_mn_sw128(a_addr, kChunk) : umma_desc_sw128(a_addr);
                    const uint64_t b_desc = umma_desc_mn_sw128(a_addr + 2 * kChunk, kChunk);
                    if (elect_one()) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            umma_bf16_pair(d_tmem, a_desc + step_a * j, b_desc + step_b * j, idesc, (st > t.step0 || j > 0) ? 1u : 0u);
                        umma_commit_2cta(empty(s), 3);
                        if (st == t.step1 - 1) umma_commit_2cta(tm_full(buf), 3);
                    }
                    __syncwarp();
                }
            }
        }
        __syncwarp();
    } else if (kUnpack && warp == 6) {
        // ------------------------- TMA producer of codes and scales, a ring of its own ahead of the expansion
        uint32_t it = 0;
        bool alive = true;
        Tile t;
        for (int i = 0; alive && take_tile(a, worker, workers, i, t); ++i) {
            const int col = t.tn * kBN + static_cast<int>(cta_rank) * 128;
            int seg = t.step0 / t.kind->seg_steps, in_seg = t.step0 - seg * t.kind->seg_steps;
            const int per_step = kBlock16 ? 2 : 1;  // scale tiles of 128 columns
            const int first_tile = col / 128 * per_step;
            const int tiles = min(per_step, a.ktiles - first_tile);  // (none beyond the matrix: those columns are clipped)
            for (int st = t.step0; st < t.step1; ++st, ++it) {
                const uint32_t s = it % (P ? P : 1), r = it / (P ? P : 1);
                if (!mbar_wait_warp(pk_empty(s), (r & 1u) ^ 1u, abort_flag)) { alive = false; break; }
                if (elect_one()) {
                    const int which = t.weight ? 2 : (a.fine ? seg >> 1 : seg);
                    const int k0 = in_seg * kStepK;
                    const uint32_t dst = packed + s * kPackedStage;
                    mbar_expect_tx(pk_full(s), kPackedCodes + (tiles > 0 ? tiles * kScaleTileBytes : 0));
                    tma_load_2d(dst, t.weight ? &maps.x : &maps.w[which], pk_full(s), col / 2, k0);
                    if (tiles > 0)
                        bulk_load(dst + kPackedCodes, a.scales[which] + (static_cast<size_t>(k0 >> 7) * a.ktiles + first_tile) * kScaleTileBytes,
                                  tiles * kScaleTileBytes, pk_full(s));
                }
                __syncwarp();
                if (++in_seg == t.kind->seg_steps) { in_seg = 0; ++seg; }
            }
        }
    } else if (kUnpack && warp >= 7) {
        // ------------------- expansion: a thread takes 64 columns (half h) of one of the step's 64 rows
        const int group = (warp - 7) >> 2, h = ((warp - 7) >> 1) & 1, row = ((warp - 7) & 1) * 32 + lane;
        uint32_t it = 0;
        bool alive = true;
        Tile t;
        float ts[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) ts[i] = a.ts[i] != nullptr ? __ldg(a.ts[i]) : 1.0f;
        for (int i = 0; alive && take_tile(a, worker, workers, i, t); ++i) {
            int seg = t.step0 / t.kind->seg_steps, in_seg = t.step0 - seg * t.kind->seg_steps;
            for (int st = t.step0; st < t.step1; ++st, ++it) {
                const uint32_t ps = it % (P ? P : 1), pr = it / (P ? P : 1), s = it % S, r = it / S;
                const int which = t.weight ? 2 : (a.fine ? seg >> 1 : seg);
                const int k0 = in_seg * kStepK;
                if (++in_seg == t.kind->seg_steps) { in_seg = 0; ++seg; }
                if (static_cast<int>(it % kGroups) != group) continue;
                if (!mbar_wait_warp(pk_full(ps), pr & 1u, abort_flag)) { alive = false; break; }
                const uint32_t src = packed + ps * kPackedStage;
                // (64-byte swizzle: 16-byte chunk index XOR (row / 2) % 4)
                const uint32_t row_at = src + row * 64, x = (row >> 1) & 3;
                const uint4 lo = lds128(row_at + (((2 * h) ^ x) << 4)), hi = lds128(row_at + (((2 * h + 1) ^ x) << 4));
                const int rr = (k0 + row) & 127;
                uint32_t word;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(word) : "r"(src + kPackedCodes + (kBlock16 ? h * kScaleTileBytes : 0) + (rr & 31) * 16 + (rr >> 5) * 4));
                if (!kBlock16) word >>= 16 * h;
                mbar_arrive_after_warp(pk_empty(ps), lo.x ^ lo.y ^ lo.z ^ lo.w ^ hi.x ^ hi.y ^ hi.z ^ hi.w ^ word, lane);
                // Rows beyond the matrix have code 0 (read out of bounds) and no defined scale.
                const bool outside = k0 + row >= (t.weight ? a.m : a.n);
                if (!mbar_wait_warp(empty(s), (r & 1u) ^ 1u, abort_flag)) { alive = false; break; }
                expand_row<kBlock16>(lo, hi, word, outside, ts[which] == 0.0f ? 0.0f : 1.0f, ring + s * kStage + (2 + h) * kChunk + row * 128, row);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(full(s), 0);
            }
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------- epilogue
        const int sp = warp & 3;
        const uint32_t stage0 = st_base + (warp - 2) * 2 * kStoreStage;
        uint32_t chunk_no = 0;
        Tile t;
        for (int i = 0; take_tile(a, worker, workers, i, t); ++i) {
            const uint32_t buf = i & 1u, br = static_cast<uint32_t>(i) >> 1;
            const bool whole = t.kind->parts == 1;
            const float alpha = !whole ? 1.0f : (t.weight ? result_scale(a.num, a.den[t.matrix]) : result_scale(a.dx_scale, nullptr));
            float* partial = a.partial[t.weight ? 1 + t.matrix : 0] + (whole ? 0 : static_cast<size_t>(t.part) * t.kind->rows * t.kind->cols);
            const CUtensorMap* out = t.weight ? &maps.dw[t.matrix] : &maps.dx;
            if (!mbar_wait_warp(tm_full(buf), br & 1u, abort_flag)) break;
            tc_fence_after_sync();
            const int row0 = (t.tm * 2 + static_cast<int>(cta_rank)) * kBM + sp * 32;
            const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(sp * 32) << 16) + buf * kBN;
            const int col_first = t.tn * kBN;
            const int chunks = row0 < t.kind->rows ? min(kBN, t.kind->cols - col_first + 63) / 64 : 0;  // of 64 columns
            if (!whole) {
#pragma unroll 1
                for (int c = 0; c < chunks; ++c) {
                    uint32_t v[64];
                    load64(t_addr + 64 * c, v);
                    tmem_ld_wait();
                    const int col0 = col_first + 64 * c;
                    if (row0 + lane >= t.kind->rows) continue;
                    float* dst = partial + static_cast<size_t>(row0 + lane) * t.kind->cols + col0;
#pragma unroll
                    for (int q = 0; q < 16; ++q)  // (cols is a multiple of 32)
                        if (col0 + 4 * q < t.kind->cols) reinterpret_cast<uint4*>(dst)[q] = make_uint4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                }
            } else if (chunks > 0) {
                // 32 columns at a time, the next 32 on their way from tensor memory meanwhile.
                uint32_t v0[32], v1[32];
                auto put32 = [&](const uint32_t (&v)[32], uint32_t stg, int half) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t h[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) h[e] = pack16<false>(__uint_as_float(v[8 * q + 2 * e]) * alpha, __uint_as_float(v[8 * q + 2 * e + 1]) * alpha);
                        sts128(stg + lane * 128 + (((4 * half + q) ^ (lane & 7)) << 4), make_uint4(h[0], h[1], h[2], h[3]));
                    }
                };
                tmem_ld_32x32(t_addr, v0);
#pragma unroll 1
                for (int c = 0; c < chunks; ++c) {
                    const uint32_t stg = stage0 + (chunk_no & 1u) * kStoreStage;
                    if (lane == 0) tma_store_wait_read<1>();
                    __syncwarp();
                    tmem_ld_wait();
                    tmem_ld_32x32(t_addr + 64 * c + 32, v1);
                    put32(v0, stg, 0);
                    tmem_ld_wait();
                    if (c + 1 < chunks) tmem_ld_32x32(t_addr + 64 * c + 64, v0);
                    put32(v1, stg, 1);
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_2d(out, stg, col_first + 64 * c, row0);
                        tma_store_commit();
                    }
                    ++chunk_no;
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(tm_empty(buf), 0);
        }
        if (lane == 0) tma_store_wait_all<0>();
        __syncwarp();
    }

    // ------------------------------------------------------------- teardown
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        if (tid == 0) atomicExch(a.status, INT4L_ERR_DEVICE_TIMEOUT);
        for (int i = 0; i < 100; ++i) __nanosleep(1000);  // copies in flight land
        __syncthreads();
    }
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc<2>(tmem_base, 512);
    }
}

// ------------------------------------------------------------- adding parts

struct SumJob {
    const float* partial;
    __nv_bfloat16* out;
    const float* num; const float* den;
    long long count;  // elements, a multiple of 32
    int parts;
};
struct SumArgs {
    SumJob job[3];
    uint32_t first[4];  // blocks of job i: [first[i], first[i + 1])
};
constexpr int kSumThreads = 256, kSumElems = 4;

__global__ void __launch_bounds__(kSumThreads)
sum_parts_kernel(const __grid_constant__ SumArgs a)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t b = blockIdx.x;
    const int i = b < a.first[1] ? 0 : (b < a.first[2] ? 1 : 2);
    const SumJob& j = a.job[i];
    const long long at = (static_cast<long long>(b - a.first[i]) * kSumThreads + threadIdx.x) * kSumElems;
    if (at >= j.count) return;
    float4 sum = __ldg(reinterpret_cast<const float4*>(j.partial + at));
#pragma unroll 4
    for (int p = 1; p < j.parts; ++p) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(j.partial + p * j.count + at));
        sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
    }
    const float alpha = result_scale(j.num, j.den);
    *reinterpret_cast<uint2*>(j.out + at) = make_uint2(pack16<false>(sum.x * alpha, sum.y * alpha), pack16<false>(sum.z * alpha, sum.w * alpha));
}

// The launch may begin while the one before it in the stream ends; the kernels wait before they touch memory.
void allow_overlap(cudaLaunchConfig_t& cfg, cudaStream_t stream, cudaLaunchAttribute (&attr)[1])
{
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    count_launch();
}

bool unaligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

}  // namespace

long long fp4_backward_workspace(long long m, long long n, long long k, bool gated, bool want_dx, bool want_dw, int terms)
{
    return plan(m, n, k, gated, want_dx, want_dw, terms).bytes;
}

int setup_fp4_backward(DeviceCtx*)
{
    const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
    const bool ok = cudaFuncSetAttribute(grad_gemm_kernel<false, false>, attr, Geo<false>::kSmemBytes) == cudaSuccess &&
                    cudaFuncSetAttribute(grad_gemm_kernel<true, false>, attr, Geo<true>::kSmemBytes) == cudaSuccess &&
                    cudaFuncSetAttribute(grad_gemm_kernel<true, true>, attr, Geo<true>::kSmemBytes) == cudaSuccess;
    return ok ? INT4L_OK : INT4L_ERR_CUDA;
}

int launch_fp4_backward(DeviceCtx* ctx, const Fp4Backward& b, cudaStream_t stream)
{
    using B = __nv_bfloat16;
    const Fp4Problem& p = b.forward;
    const Plan l = plan(p.m, p.n, p.k, p.gated, b.dx != nullptr, b.dw != nullptr, b.terms);
    uint8_t* ws = b.workspace;
    const bool direct = !p.gated && p.n % 8 == 0;  // dy as it is
    auto at = [&](long long piece) { return reinterpret_cast<B*>(ws + piece); };
    const void* d[4] = {direct ? b.dy : ws + l.d[0], ws + l.d[1], ws + l.d[2], ws + l.d[3]};

    // ------------------------------------------------------------ preparation
    PrepArgs pa = {};
    long long blocks = 0;
    if (!direct) {
        pa.gate = GateJob{static_cast<const B*>(b.dy), static_cast<const B*>(b.gate), static_cast<const B*>(b.up), at(l.d[0]), at(l.d[1]),
                          l.fine ? at(l.d[2]) : nullptr, l.fine ? at(l.d[3]) : nullptr, p.w.tensor_scale, p.w_up.tensor_scale,
                          p.m, p.n, p.act, p.n % 8 == 0 && !unaligned16(b.dy) && !unaligned16(b.gate) && !unaligned16(b.up), l.ld};
        const long long units = static_cast<long long>(p.m) * ((p.n + 255) / 256);
        if (units > 0xFFFFFFFFll - 8) return INT4L_ERR_TOO_LARGE;
        blocks = (units + kUnitThreads / 32 - 1) / (kUnitThreads / 32);
    }
    int jobs = 0;
    auto expand = [&](const Fp4& q, long long piece) {
        pa.first[jobs] = static_cast<uint32_t>(blocks);
        pa.expand[jobs++] = ExpandJob{q.codes, q.scales, q.tensor_scale, at(piece), q.rows, q.k};
        blocks += fp4_expand_blocks(q.rows, q.k);
    };
    if (b.dx && !l.unpack) {
        expand(p.w, l.w[0]);
        if (p.gated) expand(p.w_up, l.w[1]);
    }
    if (b.dw && !l.unpack) expand(p.x, l.x);
    if (blocks > 0x7FFFFFFF) return INT4L_ERR_TOO_LARGE;
    for (int i = jobs; i < 4; ++i) pa.first[i] = static_cast<uint32_t>(blocks);
    cudaLaunchAttribute attr[1];
    if (blocks > 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
        cfg.blockDim = dim3(kUnitThreads, 1, 1);
        allow_overlap(cfg, stream, attr);
        if (cudaLaunchKernelEx(&cfg, p.x.block16 ? backward_prepare_kernel<true> : backward_prepare_kernel<false>, pa) != cudaSuccess) {
            cudaGetLastError();
            return INT4L_ERR_CUDA;
        }
    }

    // --------------------------------------------------------------- products
    GradArgs a = {};
    Maps maps;
    const int matrices = p.gated ? 2 : 1;
    if (l.tiles_dx + l.tiles_dw > (1 << 30)) return INT4L_ERR_TOO_LARGE;
    auto part_steps = [](const Kind& k) { return (k.segments * k.seg_steps + k.parts - 1) / k.parts; };
    auto tile_cost = [&](const Kind& k) { return part_steps(k) > kTileSteps ? part_steps(k) : kTileSteps; };
    const bool dx_first = l.tiles_dw == 0 || (l.tiles_dx > 0 && part_steps(l.dx) >= part_steps(l.dw));
    a.kind[0] = dx_first ? l.dx : l.dw;
    a.kind[1] = dx_first ? l.dw : l.dx;
    const int workers = l.tiles_dx + l.tiles_dw < ctx->max_pairs ? static_cast<int>(l.tiles_dx + l.tiles_dw) : ctx->max_pairs;
    a.deal = deal_tiles(static_cast<int>(dx_first ? l.tiles_dx : l.tiles_dw), static_cast<int>(dx_first ? l.tiles_dw : l.tiles_dx),
                        tile_cost(a.kind[0]), tile_cost(a.kind[1]), workers);
    a.fine = l.fine;
    for (int i = 0; i < 3; ++i) a.partial[i] = reinterpret_cast<float*>(ws + l.partial[i]);
    a.num = p.x.tensor_scale;
    if (p.gated) { a.den[0] = p.w.tensor_scale; a.den[1] = p.w_up.tensor_scale; }
    else a.dx_scale = p.w.tensor_scale;
    const Fp4* operands[3] = {&p.w, &p.w_up, &p.x};
    for (int i = 0; i < 3; ++i) { a.scales[i] = operands[i]->scales; a.ts[i] = operands[i]->tensor_scale; }
    a.n = p.n; a.m = p.m;
    a.ktiles = fp4_ktiles(p.k, p.x.block16);
    a.status = ctx->status_dev;
    const uint64_t d_pitch = direct ? static_cast<uint64_t>(p.n) * 2 : static_cast<uint64_t>(l.ld) * 2, k_pitch = static_cast<uint64_t>(p.k) * 2;
    int rc = INT4L_OK;
    auto map = [&](CUtensorMap* out, const void* at, int cols, int rows, uint64_t pitch, int box_rows) {
        if (rc == INT4L_OK) rc = encode_tensor_map_2d(ctx, out, at, 2, cols, rows, pitch, 64, box_rows, true);
    };
    auto codes = [&](CUtensorMap* out, const Fp4& q) {
        if (rc == INT4L_OK) rc = encode_tensor_map_2d(ctx, out, q.codes, 1, static_cast<uint64_t>(q.k) / 2, q.rows, static_cast<uint64_t>(q.k) / 2, 64, kStepK, false, true);
    };
    for (int i = 0; i < matrices; ++i) {
        map(&maps.d[i], d[i], p.n, p.m, d_pitch, 64);
        if (l.fine) map(&maps.d[2 + i], d[2 + i], p.n, p.m, d_pitch, 64);
        if (b.dx && l.unpack) codes(&maps.w[i], i ? p.w_up : p.w);
        else if (b.dx) map(&maps.w[i], ws + l.w[i], p.k, p.n, k_pitch, 64);
        if (b.dw) map(&maps.dw[i], i ? b.dw_up : b.dw, p.k, p.n, k_pitch, 32);
    }
    if (b.dw && l.unpack) codes(&maps.x, p.x);
    else if (b.dw) map(&maps.x, ws + l.x, p.k, p.m, k_pitch, 64);
    if (b.dx) map(&maps.dx, b.dx, p.k, p.m, k_pitch, 32);
    if (rc != INT4L_OK) return rc;
    cudaLaunchConfig_t cfg2 = {};
    cfg2.gridDim = dim3(workers * 2, 1, 1);
    cfg2.blockDim = dim3(l.unpack ? Geo<true>::kThreads : Geo<false>::kThreads, 1, 1);
    cfg2.dynamicSmemBytes = l.unpack ? Geo<true>::kSmemBytes : Geo<false>::kSmemBytes;
    allow_overlap(cfg2, stream, attr);
    const auto kernel = !l.unpack ? grad_gemm_kernel<false, false> : (p.x.block16 ? grad_gemm_kernel<true, true> : grad_gemm_kernel<true, false>);
    if (cudaLaunchKernelEx(&cfg2, kernel, maps, a) != cudaSuccess) { cudaGetLastError(); return INT4L_ERR_CUDA; }

    // ----------------------------------------------------------- adding parts
    SumArgs sa = {};
    blocks = 0;
    jobs = 0;
    auto add = [&](const Kind& kind, int i, void* out, const float* num, const float* den) {
        if (kind.parts == 1 || out == nullptr) return;
        const long long count = static_cast<long long>(kind.rows) * kind.cols;
        sa.first[jobs] = static_cast<uint32_t>(blocks);
        sa.job[jobs++] = SumJob{a.partial[i], static_cast<B*>(out), num, den, count, kind.parts};
        blocks += (count + kSumThreads * kSumElems - 1) / (kSumThreads * kSumElems);
    };
    add(l.dx, 0, b.dx, a.dx_scale, nullptr);
    add(l.dw, 1, b.dw, a.num, a.den[0]);
    add(l.dw, 2, b.dw_up, a.num, a.den[1]);
    if (jobs == 0) return INT4L_OK;
    if (blocks > 0x7FFFFFFF) return INT4L_ERR_TOO_LARGE;
    for (int i = jobs; i < 4; ++i) sa.first[i] = static_cast<uint32_t>(blocks);
    cudaLaunchConfig_t cfg3 = {};
    cfg3.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
    cfg3.blockDim = dim3(kSumThreads, 1, 1);
    allow_overlap(cfg3, stream, attr);
    if (cudaLaunchKernelEx(&cfg3, sum_parts_kernel, sa) != cudaSuccess) { cudaGetLastError(); return INT4L_ERR_CUDA; }
    return INT4L_OK;
}

}  // namespace i4l
