// The product of two microscaled 4-bit matrices on the tensor cores, and the gated pair of products:
//
//     y = x w^T * (ts_x ts_w) + bias                  16-bit floats, fp32 accumulation
//     h = act(x w_gate^T * a) * (x w_up^T * b)        both products, activation and multiplication in one kernel
//
// The 5th-generation tensor cores multiply e2m1 codes and apply the block scales themselves
// (tcgen05.mma kind::mxf4 / mxf4nvf4), so the operands go from HBM to the tensor core with nothing but copies:
//
//     warp 0      TMA: per step of 256 elements of k (128 bytes a row, one swizzle line) the code tiles of x and
//                 w and their scale tiles, which the format keeps contiguous (fp4.cuh)
//     warp 1      tcgen05.cp of the scale tiles into tensor memory, then 4 UMMAs of k = 64 (CTA 0 of the pair
//                 issues for both)
//     warps 2-9   epilogue
//
// Tile: a CTA pair computes 256 x 256 accumulators (cta_group::2).  A gated tile is 128 columns of the gate
// product beside the same 128 columns of the up product: CTA 0 loads its 128 rows of w from the gate matrix,
// CTA 1 from the up matrix, and the epilogue finds both factors of an output in the same lane.
//
// Tensor memory (512 columns): 256 for the accumulator and 48 (nvfp4) or 24 for the scales of each stage of the
// ring, so that a stage's scale columns are free whenever its shared memory is.  One accumulator, not two: the
// eight epilogue warps take the whole tile into registers (128 columns of 32 lanes each) and hand the columns
// over at once; the next tile's UMMAs run while the values are converted and stored.  (Two accumulators that
// share 128 columns were built first; they left two scale slots for nvfp4, and waiting for the UMMAs two steps
// back held the step at 0.95 us.)
//
// Both CTAs' loads are counted on CTA 0's barrier, whose UMMAs read them: with CTA 1 passing on its own
// barrier's completion instead, a step of the 5-stage ring took 0.41 us even without any UMMA.
//
// The issuing warp sets the pace next: a step is 10 (mxfp4) or 16 (nvfp4) instructions to the tensor pipe.  One elected
// thread of a converged warp issues them (with `if (lane == 0)` the step took 0.56 us instead of 0.36), with 32-bit
// descriptor arithmetic (nvfp4 gated 4096 x 8192 x 2048: 63 -> 57 us).
//
// Measured, a single call on an idle GPU and, under the power limit, call after call: 8192 x 8192 x 16384 mxfp4 334 and 421 us (6.6 and
// 5.2 PFLOP/s), 8192^3 nvfp4 179 and 231 us, gated gelu 4096 x 14336 x 4096 nvfp4 174 and 215 us (262 and 257 with both
// products kept); at 8192^3 the tensor pipe is 82 % busy at 1.57 GHz, the clock that the limit leaves.
#include "epilogue.cuh"
#include "fp4.cuh"
#include "gate.cuh"
#include "ptx.cuh"

namespace i4l {

namespace {

constexpr int kBM = 128;          // rows of x per CTA
constexpr int kBN = 256;          // accumulator columns of the pair's tile
constexpr int kStepBytes = 128;   // bytes of a row per step
constexpr int kStepK = 256;       // elements of a row per step
constexpr int kThreads = 32 * 10;
constexpr int kStages = 5;
constexpr int kStoreStage = 4096;  // per epilogue warp: 32 rows x 64 16-bit columns
constexpr uint32_t kScaleCol = 256;
constexpr int kNumBarriers = 2 * kStages + 2;

template <bool kBlock16>
struct Geo {
    static constexpr int kTilesK = kBlock16 ? 4 : 2;  // scale tiles per step along k
    static constexpr int kScaleBytesA = kTilesK * kScaleTileBytes;
    static constexpr int kScaleBytesB = 2 * kScaleBytesA;
    static constexpr int kCodeBytes = 2 * 128 * kStepBytes;  // x and w tile of one CTA
    static constexpr int kStage = kCodeBytes + kScaleBytesA + kScaleBytesB;
    static constexpr int kScaleCols = kTilesK * 12;  // 4 columns for x, 8 for w, per scale tile
    static constexpr int kSmemBytes = 1024 + kStages * kStage + 8 * kStoreStage + kNumBarriers * 8 + 16;
    static_assert(kStage % 1024 == 0, "stage bases must keep the swizzle alignment");
    static_assert(kScaleCol + kStages * kScaleCols <= 512, "tensor memory budget");
    static_assert(kSmemBytes <= 232448, "shared memory budget");
};

struct Args {
    const float* ts_x; const float* ts_w; const float* ts_w_up;    // tensor scales, may be null
    const float* bias;
    unsigned short* y; unsigned short* keep_gate; unsigned short* keep_up;
    int m, n, k;
    int tiles_m, tiles_n;
    int act, tma_store;
    int* status;
};

template <int kAct, bool kHalf>
__device__ __forceinline__ void gate_block(const uint32_t (&g)[64], const uint32_t (&u)[64], float alpha_g, float alpha_u, uint32_t (&h)[32])
{
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        const float a = gate_act<kAct>(__uint_as_float(g[2 * j]) * alpha_g) * (__uint_as_float(u[2 * j]) * alpha_u);
        const float b = gate_act<kAct>(__uint_as_float(g[2 * j + 1]) * alpha_g) * (__uint_as_float(u[2 * j + 1]) * alpha_u);
        h[j] = pack16<kHalf>(a, b);
    }
}

template <bool kHalf>
__device__ __forceinline__ void scale_block(const uint32_t (&v)[64], float alpha, uint32_t (&h)[32])
{
#pragma unroll
    for (int j = 0; j < 32; ++j) h[j] = pack16<kHalf>(__uint_as_float(v[2 * j]) * alpha, __uint_as_float(v[2 * j + 1]) * alpha);
}

// The same with the bias of each column: lane l fetches those of columns l and l + 32, the others get them by shuffle.
template <bool kHalf>
__device__ __forceinline__ void scale_bias_block(const uint32_t (&v)[64], float alpha, const float* bias, int col0, int n, int lane, uint32_t (&h)[32])
{
    float b[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) b[e] = __ldg(bias + min(col0 + 32 * e + lane, n - 1));
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        const float b0 = __shfl_sync(0xFFFFFFFFu, b[j >> 4], (2 * j) & 31);
        const float b1 = __shfl_sync(0xFFFFFFFFu, b[j >> 4], (2 * j + 1) & 31);
        h[j] = pack16<kHalf>(fmaf(__uint_as_float(v[2 * j]), alpha, b0), fmaf(__uint_as_float(v[2 * j + 1]), alpha, b1));
    }
}

template <bool kBlock16, bool kGated, bool kHalf>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
gemm_fp4_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                const __grid_constant__ CUtensorMap tm_w_up, const __grid_constant__ CUtensorMap tm_sx,
                const __grid_constant__ CUtensorMap tm_sw, const __grid_constant__ CUtensorMap tm_sw_up,
                const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ CUtensorMap tm_keep_gate,
                const __grid_constant__ CUtensorMap tm_keep_up, const __grid_constant__ Args a)
{
    using G = Geo<kBlock16>;
    constexpr int S = kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* gbase = smem_raw + (base - raw);

    const uint32_t ring = base;
    const uint32_t st_base = ring + S * G::kStage;
    const uint32_t bar_base = st_base + 8 * kStoreStage;
    auto full  = [&](int i) { return bar_base + 8u * i; };  // (CTA 0's, for the loads of both)
    auto empty = [&](int i) { return bar_base + 8u * (S + i); };
    const uint32_t acc_full = bar_base + 8u * (2 * S);
    const uint32_t acc_free = bar_base + 8u * (2 * S + 1);
    const uint32_t misc_off = (bar_base - base) + 8u * kNumBarriers;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + misc_off);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + misc_off + 4);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t cta_rank = cluster_cta_rank();
    const int worker = static_cast<int>(cluster_id_x());
    const int workers = static_cast<int>(cluster_count_x());

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(full(i), 1); mbar_init(empty(i), 1); }
        mbar_init(acc_full, 1);
        mbar_init(acc_free, 8 * 2);
        *abort_flag = 0;
        mbar_init_fence();
        tma_prefetch_desc(&tm_x);
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_sx);
        tma_prefetch_desc(&tm_sw);
    }
    if (warp == 1) {
        tmem_alloc<2>(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
        tmem_relinquish<2>();
    }
    tc_fence_before_sync();
    cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    // Everything above may run while the launch before this one in the stream ends.
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const int num_tiles = a.tiles_m * a.tiles_n;
    const int steps = (a.k + kStepK - 1) / kStepK;
    // Raster: groups of 16 tiles of x rows share a panel of w in L2.
    constexpr int kGroupM = 16;
    auto tile_coord = [&](int tile, int& tm, int& tn) {
        const int group_size = kGroupM * a.tiles_n;
        const int group = tile / group_size;
        const int first_m = group * kGroupM;
        const int gm = min(a.tiles_m - first_m, kGroupM);
        const int in_group = tile - group * group_size;
        tm = first_m + in_group % gm;
        tn = in_group / gm;
    };

    if (warp == 0) {
        // ------------------------------------------------------ TMA producer
        uint32_t it = 0;
        bool alive = true;
        for (int tile = worker; alive && tile < num_tiles; tile += workers) {
            int tm, tn;
            tile_coord(tile, tm, tn);
            const int group_x = tm * 2 + static_cast<int>(cta_rank);
            const CUtensorMap* map_w = (kGated && cta_rank) ? &tm_w_up : &tm_w;
            const int group_w = kGated ? tn : tn * 2 + static_cast<int>(cta_rank);
            for (int kb = 0; kb < steps; ++kb, ++it) {
                const uint32_t s = it % S, r = it / S;
                if (!mbar_wait_warp(empty(s), (r & 1u) ^ 1u, abort_flag)) { alive = false; break; }
                if (elect_one()) {
                    // CTA 1's bytes may be counted before CTA 0 announces them: the phase cannot end before the
                    // announcement, which is its one arrival.  What lies outside a matrix is read as 0 and counted.
                    if (cta_rank == 0) mbar_expect_tx(full(s), 2 * G::kStage);
                    const uint32_t bar = cluster_address(full(s), 0);
                    const uint32_t dst = ring + s * G::kStage;
                    tma_load_2d_pair(dst, &tm_x, bar, kb * kStepBytes, group_x * 128);
                    tma_load_2d_pair(dst + 128 * kStepBytes, map_w, bar, kb * kStepBytes, group_w * 128);
                    const int sc = kb * (G::kScaleBytesA / 8);  // (8-byte elements: a box has at most 256)
                    tma_load_2d_pair(dst + G::kCodeBytes, &tm_sx, bar, sc, group_x);
                    if constexpr (kGated) {
                        tma_load_2d_pair(dst + G::kCodeBytes + G::kScaleBytesA, &tm_sw, bar, sc, tn);
                        tma_load_2d_pair(dst + G::kCodeBytes + 2 * G::kScaleBytesA, &tm_sw_up, bar, sc, tn);
                    } else {
                        tma_load_2d_pair(dst + G::kCodeBytes + G::kScaleBytesA, &tm_sw, bar, sc, tn * 2);  // two groups
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        if (cta_rank == 0) {
            // ----------------------------------------------------- UMMA issuer
            // The warp walks the ring together and one elected thread issues.
            uint32_t s = 0, phase = 0, local_tile = 0;
            bool alive = true;
            const uint32_t codes_low = umma_desc_sw128_low(ring), scales_low = scale_tile_low(ring + G::kCodeBytes);
            const uint32_t scale_cols = tmem_base + kScaleCol;
            const int last_count = (a.k - (steps - 1) * kStepK + 63) / 64;  // UMMAs of the last step
            // One step: scales, then `count` UMMAs (a constant but in the last step).
            auto issue = [&](int count, bool first) {
                const uint32_t x_low = codes_low + s * (G::kStage / 16), w_low = x_low + 128 * kStepBytes / 16;
                const uint32_t sfa_low = scales_low + s * (G::kStage / 16), sfb_low = sfa_low + G::kScaleBytesA / 16;
                const uint32_t sfa = scale_cols + s * G::kScaleCols, sfb = sfa + 4 * G::kTilesK;
#pragma unroll
                for (int t = 0; t < G::kTilesK; ++t) {
                    tmem_copy_scales<2>(sfa + 4 * t, sfa_low + t * (kScaleTileBytes / 16));
                    tmem_copy_scales<2>(sfb + 8 * t, sfb_low + t * (kScaleTileBytes / 16));
                    tmem_copy_scales<2>(sfb + 8 * t + 4, sfb_low + (G::kScaleBytesA + t * kScaleTileBytes) / 16);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j >= count) break;
                    const int t = kBlock16 ? j : j >> 1;
                    const uint32_t idesc = umma_idesc_fp4(2 * kBM, kBN, !kBlock16, kBlock16 ? 0u : 2u * (j & 1));
                    umma_fp4<2, kBlock16>(tmem_base, x_low + 2 * j, w_low + 2 * j, idesc, sfa + 4 * t, sfb + 8 * t, (j > 0 || !first) ? 1u : 0u);
                }
                umma_commit_2cta(empty(s), 3);
            };
            for (int tile = worker; alive && tile < num_tiles; tile += workers, ++local_tile) {
                if (local_tile > 0 && !mbar_wait_warp(acc_free, (local_tile - 1) & 1u, abort_flag)) break;
                for (int kb = 0; kb < steps; ++kb) {
                    if (!mbar_wait_warp(full(s), phase, abort_flag)) { alive = false; break; }
                    tc_fence_after_sync();
                    if (elect_one()) {
                        if (kb < steps - 1) {
                            issue(4, kb == 0);
                        } else {
                            issue(last_count, kb == 0);
                            umma_commit_2cta(acc_full, 3);
                        }
                    }
                    __syncwarp();
                    if (++s == S) { s = 0; phase ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------- epilogue
        const int quarter = warp & 3, half = (warp - 2) >> 2;
        const uint32_t stg = st_base + (warp - 2) * kStoreStage;
        const float ts_x = a.ts_x != nullptr ? __ldg(a.ts_x) : 1.0f;
        const float alpha = ts_x * (a.ts_w != nullptr ? __ldg(a.ts_w) : 1.0f);
        const float alpha_up = kGated ? ts_x * (a.ts_w_up != nullptr ? __ldg(a.ts_w_up) : 1.0f) : 0.0f;
        const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + half * 64;
        uint32_t local_tile = 0;
        for (int tile = worker; tile < num_tiles; tile += workers, ++local_tile) {
            int tm, tn;
            tile_coord(tile, tm, tn);
            if (!mbar_wait_warp(acc_full, local_tile & 1u, abort_flag)) break;
            tc_fence_after_sync();
            const int row0 = (tm * 2 + static_cast<int>(cta_rank)) * kBM + quarter * 32;
            // Columns [64 half, 64 half + 64) of both 128-column halves: gate and up, or twice 64 of y.
            uint32_t v[64], w[64], h[32];
            load64(t_addr, v);
            load64(t_addr + 128, w);
            tmem_ld_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc_free, 0);
            if constexpr (kGated) {
                const int col0 = tn * 128 + half * 64;
                if (a.keep_gate != nullptr) {
                    scale_block<kHalf>(v, alpha, h);
                    store_block(h, stg, &tm_keep_gate, a.keep_gate, row0, col0, a.m, a.n, a.tma_store, lane);
                    scale_block<kHalf>(w, alpha_up, h);
                    store_block(h, stg, &tm_keep_up, a.keep_up, row0, col0, a.m, a.n, a.tma_store, lane);
                }
                if (a.act == kActSilu) gate_block<kActSilu, kHalf>(v, w, alpha, alpha_up, h);
                else if (a.act == kActGelu) gate_block<kActGelu, kHalf>(v, w, alpha, alpha_up, h);
                else gate_block<kActGeluTanh, kHalf>(v, w, alpha, alpha_up, h);
                store_block(h, stg, &tm_y, a.y, row0, col0, a.m, a.n, a.tma_store, lane);
            } else {
                const int col0 = tn * kBN + half * 64, col1 = col0 + 128;
                if (a.bias != nullptr) scale_bias_block<kHalf>(v, alpha, a.bias, col0, a.n, lane, h);
                else scale_block<kHalf>(v, alpha, h);
                store_block(h, stg, &tm_y, a.y, row0, col0, a.m, a.n, a.tma_store, lane);
                if (a.bias != nullptr) scale_bias_block<kHalf>(w, alpha, a.bias, col1, a.n, lane, h);
                else scale_block<kHalf>(w, alpha, h);
                store_block(h, stg, &tm_y, a.y, row0, col1, a.m, a.n, a.tma_store, lane);
            }
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

template <bool kBlock16, bool kGated, bool kHalf>
int launch_cfg(DeviceCtx* ctx, const Fp4Problem& p, cudaStream_t stream)
{
    Args a = {};
    a.ts_x = p.x.tensor_scale; a.ts_w = p.w.tensor_scale; a.ts_w_up = p.w_up.tensor_scale;
    a.bias = p.bias;
    a.y = static_cast<unsigned short*>(p.y);
    a.keep_gate = static_cast<unsigned short*>(p.keep_gate);
    a.keep_up = static_cast<unsigned short*>(p.keep_up);
    a.m = p.m; a.n = p.n; a.k = p.k;
    a.tiles_m = (p.m + 255) / 256;
    a.tiles_n = kGated ? (p.n + 127) / 128 : (p.n + kBN - 1) / kBN;
    a.act = p.act;
    a.tma_store = p.n % 8 == 0;
    a.status = ctx->status_dev;
    const uint64_t pitch = static_cast<uint64_t>(p.k) / 2, out_pitch = static_cast<uint64_t>(p.n) * 2;
    CUtensorMap tm_x, tm_w, tm_w_up, tm_sx, tm_sw, tm_sw_up, tm_y, tm_g, tm_u;
    int rc = encode_tensor_map_2d(ctx, &tm_x, p.x.codes, 1, pitch, p.m, pitch, kStepBytes, kBM, true);
    if (rc == INT4L_OK) rc = encode_tensor_map_2d(ctx, &tm_w, p.w.codes, 1, pitch, p.n, pitch, kStepBytes, 128, true);
    if (rc == INT4L_OK) rc = fp4_scale_map(ctx, &tm_sx, p.x, Geo<kBlock16>::kScaleBytesA, 1);
    if (rc == INT4L_OK) rc = fp4_scale_map(ctx, &tm_sw, p.w, Geo<kBlock16>::kScaleBytesA, kGated ? 1 : 2);
    tm_w_up = tm_w;
    tm_sw_up = tm_sw;
    if (rc == INT4L_OK && kGated) {
        rc = encode_tensor_map_2d(ctx, &tm_w_up, p.w_up.codes, 1, pitch, p.n, pitch, kStepBytes, 128, true);
        if (rc == INT4L_OK) rc = fp4_scale_map(ctx, &tm_sw_up, p.w_up, Geo<kBlock16>::kScaleBytesA, 1);
    }
    tm_y = tm_x;
    if (rc == INT4L_OK && a.tma_store) rc = encode_tensor_map_2d(ctx, &tm_y, p.y, 2, p.n, p.m, out_pitch, 64, 32, true);
    tm_g = tm_u = tm_y;
    if (rc == INT4L_OK && a.tma_store && p.keep_gate) {
        rc = encode_tensor_map_2d(ctx, &tm_g, p.keep_gate, 2, p.n, p.m, out_pitch, 64, 32, true);
        if (rc == INT4L_OK) rc = encode_tensor_map_2d(ctx, &tm_u, p.keep_up, 2, p.n, p.m, out_pitch, 64, 32, true);
    }
    if (rc != INT4L_OK) return rc;
    const long long tiles = static_cast<long long>(a.tiles_m) * a.tiles_n;
    if (tiles > (1 << 30)) return INT4L_ERR_TOO_LARGE;
    const int pairs = tiles < ctx->max_pairs ? static_cast<int>(tiles) : ctx->max_pairs;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(pairs * 2, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = Geo<kBlock16>::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm_fp4_kernel<kBlock16, kGated, kHalf>, tm_x, tm_w, tm_w_up, tm_sx, tm_sw, tm_sw_up,
                                             tm_y, tm_g, tm_u, a);
    count_launch();
    if (e != cudaSuccess) { cudaGetLastError(); return INT4L_ERR_CUDA; }
    return INT4L_OK;
}

template <bool kBlock16, bool kGated>
bool set_attr()
{
    return cudaFuncSetAttribute(gemm_fp4_kernel<kBlock16, kGated, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<kBlock16>::kSmemBytes) == cudaSuccess &&
           cudaFuncSetAttribute(gemm_fp4_kernel<kBlock16, kGated, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<kBlock16>::kSmemBytes) == cudaSuccess;
}

template <bool kBlock16, bool kGated>
int launch_typed(DeviceCtx* ctx, const Fp4Problem& p, cudaStream_t stream)
{
    return p.fp16 ? launch_cfg<kBlock16, kGated, true>(ctx, p, stream) : launch_cfg<kBlock16, kGated, false>(ctx, p, stream);
}

}  // namespace

int setup_fp4_gemm(DeviceCtx*)
{
    return set_attr<false, false>() && set_attr<false, true>() && set_attr<true, false>() && set_attr<true, true>() ? INT4L_OK : INT4L_ERR_CUDA;
}

int launch_fp4_gemm(DeviceCtx* ctx, const Fp4Problem& p, cudaStream_t stream)
{
    if (p.x.block16) return p.gated ? launch_typed<true, true>(ctx, p, stream) : launch_typed<true, false>(ctx, p, stream);
    return p.gated ? launch_typed<false, true>(ctx, p, stream) : launch_typed<false, false>(ctx, p, stream);
}

}  // namespace i4l
