// The product of two microscaled 4-bit matrices on the tensor cores, and the gated pair of products:
//
//     y = x w^T * (ts_x ts_w) + bias                  16-bit floats, fp32 accumulation
//     h = act(x w_gate^T * a) * (x w_up^T * b)        both products, activation and multiplication in one kernel
//
// The 5th-generation tensor cores multiply e2m1 codes and apply the block scales themselves
// (tcgen05.mma kind::mxf4 / mxf4nvf4), so the operands go from HBM to the tensor core with nothing but copies:
//
//     warp 0      TMA: per step of 256 elements of k (128 bytes a row, one swizzle line) the code tiles of x and
//                 w, and by untiled bulk copies their scale tiles, which the format keeps contiguous (fp4.cuh)
//     warp 1      tcgen05.cp of the scale tiles into tensor memory, then 4 UMMAs of k = 64 (CTA 0 of the pair
//                 issues for both; in CTA 1 this warp forwards "my tiles have landed")
//     warps 2-9   epilogue
//
// Tile: a CTA pair computes 256 x 256 accumulators (cta_group::2).  A gated tile is 128 columns of the gate
// product beside the same 128 columns of the up product: CTA 0 loads its 128 rows of w from the gate matrix,
// CTA 1 from the up matrix, and the epilogue finds both factors of an output in the same lane.
//
// Tensor memory (512 columns): two accumulators of 256 columns leave no room for scales, so the two overlap:
// [0, 256) and [128, 384), scales from 384 on.  The epilogue drains the shared 128 columns first, into registers
// (8 warps: 64 columns of 32 lanes each), and hands them over at once; the next tile's UMMAs then run while the
// rest is drained.  The scale columns are a ring of their own: a slot is written again only after the UMMAs that
// read it have completed (their commit is waited for; it lies one or more steps back, so nothing stalls).
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
constexpr uint32_t kAccCol1 = 128, kScaleCol = 384;
constexpr int kNumBarriers = 3 * kStages + 2;

template <bool kBlock16>
struct Geo {
    static constexpr int kTilesK = kBlock16 ? 4 : 2;  // scale tiles per step along k
    static constexpr int kScaleBytesA = kTilesK * kScaleTileBytes;
    static constexpr int kScaleBytesB = 2 * kScaleBytesA;
    static constexpr int kCodeBytes = 2 * 128 * kStepBytes;  // x and w tile of one CTA
    static constexpr int kStage = kCodeBytes + kScaleBytesA + kScaleBytesB;
    static constexpr int kScaleCols = kTilesK * 12;  // 4 columns for x, 8 for w, per scale tile
    static constexpr int kScaleSlots = kBlock16 ? 2 : 4;
    static constexpr int kSmemBytes = 1024 + kStages * kStage + 8 * kStoreStage + kNumBarriers * 8 + 16;
    static_assert(kStage % 1024 == 0, "stage bases must keep the swizzle alignment");
    static_assert(kScaleCol + kScaleSlots * kScaleCols <= 512, "tensor memory budget");
    static_assert(kScaleSlots <= kStages, "a slot's previous reader is found in the ring of stages");
    static_assert(kSmemBytes <= 232448, "shared memory budget");
};

struct Args {
    const uint8_t* sx; const uint8_t* sw; const uint8_t* sw_up;    // scales
    const float* ts_x; const float* ts_w; const float* ts_w_up;    // tensor scales, may be null
    const float* bias;
    unsigned short* y; unsigned short* keep_gate; unsigned short* keep_up;
    int m, n, k;
    int tiles_m, tiles_n;
    int act, fp16, tma_store;
    int* status;
};

template <int kAct>
__device__ __forceinline__ void gate_block(const uint32_t (&g)[64], const uint32_t (&u)[64], float alpha_g, float alpha_u, int fp16, uint32_t (&h)[32])
{
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        const float a = gate_act<kAct>(__uint_as_float(g[2 * j]) * alpha_g) * (__uint_as_float(u[2 * j]) * alpha_u);
        const float b = gate_act<kAct>(__uint_as_float(g[2 * j + 1]) * alpha_g) * (__uint_as_float(u[2 * j + 1]) * alpha_u);
        h[j] = pack16(a, b, fp16);
    }
}

__device__ __forceinline__ void scale_block(const uint32_t (&v)[64], float alpha, int fp16, uint32_t (&h)[32])
{
#pragma unroll
    for (int j = 0; j < 32; ++j) h[j] = pack16(__uint_as_float(v[2 * j]) * alpha, __uint_as_float(v[2 * j + 1]) * alpha, fp16);
}

template <bool kBlock16, bool kGated>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
gemm_fp4_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                const __grid_constant__ CUtensorMap tm_w_up, const __grid_constant__ CUtensorMap tm_y,
                const __grid_constant__ CUtensorMap tm_keep_gate, const __grid_constant__ CUtensorMap tm_keep_up,
                const __grid_constant__ Args a)
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
    auto full      = [&](int i) { return bar_base + 8u * i; };
    auto empty     = [&](int i) { return bar_base + 8u * (S + i); };
    auto peer_full = [&](int i) { return bar_base + 8u * (2 * S + i); };
    const uint32_t acc_full = bar_base + 8u * (3 * S);
    const uint32_t acc_free = bar_base + 8u * (3 * S + 1);  // the columns both accumulators share are drained
    const uint32_t misc_off = (bar_base - base) + 8u * kNumBarriers;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + misc_off);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + misc_off + 4);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t cta_rank = cluster_cta_rank();
    const int worker = static_cast<int>(cluster_id_x());
    const int workers = static_cast<int>(cluster_count_x());

    if (tid == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(full(i), 1); mbar_init(empty(i), 1); mbar_init(peer_full(i), 1); }
        mbar_init(acc_full, 1);
        mbar_init(acc_free, 8 * 2);
        *abort_flag = 0;
        mbar_init_fence();
        tma_prefetch_desc(&tm_x);
        tma_prefetch_desc(&tm_w);
    }
    if (warp == 1) {
        tmem_alloc<2>(smem_u32(const_cast<uint32_t*>(tmem_slot)), 512);
        tmem_relinquish<2>();
    }
    tc_fence_before_sync();
    cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    const int num_tiles = a.tiles_m * a.tiles_n;
    const int steps = (a.k + kStepK - 1) / kStepK;
    const int ktiles = fp4_ktiles(a.k, kBlock16);
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
        if (lane == 0) {
            const int last_group_m = (a.m - 1) >> 7, last_group_n = (a.n - 1) >> 7;
            uint32_t it = 0;
            bool alive = true;
            for (int tile = worker; alive && tile < num_tiles; tile += workers) {
                int tm, tn;
                tile_coord(tile, tm, tn);
                const int row_x = (tm * 2 + static_cast<int>(cta_rank)) * kBM;
                // Scale tiles of 128-row groups beyond the matrix do not exist; their rows are all clipped, any
                // other group's scales will do.
                const uint8_t* sa = a.sx + static_cast<size_t>(min(row_x >> 7, last_group_m)) * ktiles * kScaleTileBytes;
                const int group_n = kGated ? tn : tn * 2;
                const uint8_t* sb0 = a.sw + static_cast<size_t>(group_n) * ktiles * kScaleTileBytes;
                const uint8_t* sb1 = kGated ? a.sw_up + static_cast<size_t>(group_n) * ktiles * kScaleTileBytes
                                            : a.sw + static_cast<size_t>(min(group_n + 1, last_group_n)) * ktiles * kScaleTileBytes;
                const CUtensorMap* map_b = (kGated && cta_rank) ? &tm_w_up : &tm_w;
                const int row_b = kGated ? tn * 128 : tn * kBN + static_cast<int>(cta_rank) * 128;
                for (int kb = 0; kb < steps; ++kb, ++it) {
                    const uint32_t s = it % S, r = it / S;
                    if (!mbar_wait(empty(s), (r & 1u) ^ 1u, abort_flag)) { alive = false; break; }
                    const uint32_t bytes = min(G::kTilesK, ktiles - kb * G::kTilesK) * kScaleTileBytes;
                    mbar_expect_tx(full(s), G::kCodeBytes + 3 * bytes);
                    const uint32_t dst = ring + s * G::kStage;
                    tma_load_2d(dst, &tm_x, full(s), kb * kStepBytes, row_x);
                    tma_load_2d(dst + 128 * kStepBytes, map_b, full(s), kb * kStepBytes, row_b);
                    const size_t off = static_cast<size_t>(kb) * G::kScaleBytesA;
                    bulk_load(dst + G::kCodeBytes, sa + off, bytes, full(s));
                    bulk_load(dst + G::kCodeBytes + G::kScaleBytesA, sb0 + off, bytes, full(s));
                    bulk_load(dst + G::kCodeBytes + 2 * G::kScaleBytesA, sb1 + off, bytes, full(s));
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0 && cta_rank == 0) {
            // ----------------------------------------------------- UMMA issuer
            uint32_t it = 0, local_tile = 0;
            bool alive = true;
            for (int tile = worker; alive && tile < num_tiles; tile += workers, ++local_tile) {
                // The previous tile's accumulator shares 128 columns with this one's (and the one before it,
                // in the same columns, was drained earlier still).
                if (local_tile > 0 && !mbar_wait(acc_free, (local_tile - 1) & 1u, abort_flag)) { alive = false; break; }
                tc_fence_after_sync();
                const uint32_t d_tmem = tmem_base + (local_tile & 1u) * kAccCol1;
                for (int kb = 0; kb < steps; ++kb, ++it) {
                    const uint32_t s = it % S, r = it / S;
                    if (!mbar_wait(full(s), r & 1u, abort_flag) || !mbar_wait(peer_full(s), r & 1u, abort_flag)) { alive = false; break; }
                    if (it >= G::kScaleSlots) {
                        const uint32_t before = it - G::kScaleSlots;  // the step whose UMMAs read this slot's scales
                        if (!mbar_wait(empty(before % S), (before / S) & 1u, abort_flag)) { alive = false; break; }
                    }
                    tc_fence_after_sync();
                    const uint32_t a_addr = ring + s * G::kStage;
                    const uint32_t sfa_smem = a_addr + G::kCodeBytes, sfb_smem = sfa_smem + G::kScaleBytesA;
                    const uint32_t sfa = tmem_base + kScaleCol + (it % G::kScaleSlots) * G::kScaleCols;
                    const uint32_t sfb = sfa + 4 * G::kTilesK;
                    const int umma_count = min(4, (a.k - kb * kStepK + 63) / 64);
                    const int scale_tiles = min(G::kTilesK, ktiles - kb * G::kTilesK);
                    for (int t = 0; t < scale_tiles; ++t) {
                        tmem_copy_scales<2>(sfa + 4 * t, scale_tile_desc(sfa_smem + t * kScaleTileBytes));
                        tmem_copy_scales<2>(sfb + 8 * t, scale_tile_desc(sfb_smem + t * kScaleTileBytes));
                        tmem_copy_scales<2>(sfb + 8 * t + 4, scale_tile_desc(sfb_smem + G::kScaleBytesA + t * kScaleTileBytes));
                    }
                    const uint64_t a_desc = umma_desc_sw128(a_addr);
                    const uint64_t b_desc = umma_desc_sw128(a_addr + 128 * kStepBytes);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (j >= umma_count) break;
                        const int t = kBlock16 ? j : j >> 1;
                        const uint32_t idesc = umma_idesc_fp4(2 * kBM, kBN, !kBlock16, kBlock16 ? 0u : 2u * (j & 1));
                        umma_fp4<2, kBlock16>(d_tmem, a_desc + 2u * j, b_desc + 2u * j, idesc, sfa + 4 * t, sfb + 8 * t, (kb | j) != 0 ? 1u : 0u);
                    }
                    umma_commit_2cta(empty(s), 3);
                }
                if (alive) umma_commit_2cta(acc_full, 3);
            }
        } else if (lane == 0) {
            // ------------- second CTA of the pair: tell CTA 0 when this CTA's tiles have landed
            uint32_t it = 0;
            bool alive = true;
            for (int tile = worker; alive && tile < num_tiles; tile += workers) {
                for (int kb = 0; kb < steps; ++kb, ++it) {
                    const uint32_t s = it % S, r = it / S;
                    if (!mbar_wait(full(s), r & 1u, abort_flag)) { alive = false; break; }
                    mbar_arrive_cluster(peer_full(s), 0);
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
        uint32_t local_tile = 0;
        for (int tile = worker; tile < num_tiles; tile += workers, ++local_tile) {
            int tm, tn;
            tile_coord(tile, tm, tn);
            if (!mbar_wait_warp(acc_full, local_tile & 1u, abort_flag)) break;
            tc_fence_after_sync();
            const uint32_t buf = local_tile & 1u;
            const int row0 = (tm * 2 + static_cast<int>(cta_rank)) * kBM + quarter * 32;
            const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * kAccCol1 + half * 64;
            const int first = buf ? 0 : 128;  // the half of the tile in the shared columns
            uint32_t v[64];
            load64(t_addr + first, v);
            tmem_ld_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc_free, 0);
            if constexpr (kGated) {
                const int col0 = tn * 128 + half * 64;
                uint32_t w[64], h[32];
                load64(t_addr + (128 - first), w);
                tmem_ld_wait();
                if (buf == 0) {  // v holds the up product then
#pragma unroll
                    for (int i = 0; i < 64; ++i) { const uint32_t t = v[i]; v[i] = w[i]; w[i] = t; }
                }
                if (a.keep_gate != nullptr) {
                    scale_block(v, alpha, a.fp16, h);
                    store_block(h, stg, &tm_keep_gate, a.keep_gate, row0, col0, a.m, a.n, a.tma_store, lane);
                    scale_block(w, alpha_up, a.fp16, h);
                    store_block(h, stg, &tm_keep_up, a.keep_up, row0, col0, a.m, a.n, a.tma_store, lane);
                }
                if (a.act == kActSilu) gate_block<kActSilu>(v, w, alpha, alpha_up, a.fp16, h);
                else if (a.act == kActGelu) gate_block<kActGelu>(v, w, alpha, alpha_up, a.fp16, h);
                else gate_block<kActGeluTanh>(v, w, alpha, alpha_up, a.fp16, h);
                store_block(h, stg, &tm_y, a.y, row0, col0, a.m, a.n, a.tma_store, lane);
            } else {
#pragma unroll 1
                for (int part = 0; part < 2; ++part) {
                    const int off = part == 0 ? first : 128 - first;
                    const int col0 = tn * kBN + off + half * 64;
                    if (part == 1) {
                        load64(t_addr + off, v);
                        tmem_ld_wait();
                    }
                    uint32_t h[32];
                    if (a.bias != nullptr) {
                        float b[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) b[e] = __ldg(a.bias + min(col0 + 32 * e + lane, a.n - 1));
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            const float b0 = __shfl_sync(0xFFFFFFFFu, b[j >> 4], (2 * j) & 31);
                            const float b1 = __shfl_sync(0xFFFFFFFFu, b[j >> 4], (2 * j + 1) & 31);
                            h[j] = pack16(fmaf(__uint_as_float(v[2 * j]), alpha, b0), fmaf(__uint_as_float(v[2 * j + 1]), alpha, b1), a.fp16);
                        }
                    } else {
                        scale_block(v, alpha, a.fp16, h);
                    }
                    store_block(h, stg, &tm_y, a.y, row0, col0, a.m, a.n, a.tma_store, lane);
                }
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

template <bool kBlock16, bool kGated>
int launch_cfg(DeviceCtx* ctx, const Fp4Problem& p, cudaStream_t stream)
{
    Args a = {};
    a.sx = p.x.scales; a.sw = p.w.scales; a.sw_up = p.w_up.scales;
    a.ts_x = p.x.tensor_scale; a.ts_w = p.w.tensor_scale; a.ts_w_up = p.w_up.tensor_scale;
    a.bias = p.bias;
    a.y = static_cast<unsigned short*>(p.y);
    a.keep_gate = static_cast<unsigned short*>(p.keep_gate);
    a.keep_up = static_cast<unsigned short*>(p.keep_up);
    a.m = p.m; a.n = p.n; a.k = p.k;
    a.tiles_m = (p.m + 255) / 256;
    a.tiles_n = kGated ? (p.n + 127) / 128 : (p.n + kBN - 1) / kBN;
    a.act = p.act; a.fp16 = p.fp16;
    a.tma_store = p.n % 8 == 0;
    a.status = ctx->status_dev;
    const uint64_t pitch = static_cast<uint64_t>(p.k) / 2, out_pitch = static_cast<uint64_t>(p.n) * 2;
    CUtensorMap tm_x, tm_w, tm_w_up, tm_y, tm_g, tm_u;
    int rc = encode_tensor_map_2d(ctx, &tm_x, p.x.codes, 1, pitch, p.m, pitch, kStepBytes, kBM, true);
    if (rc == INT4L_OK) rc = encode_tensor_map_2d(ctx, &tm_w, p.w.codes, 1, pitch, p.n, pitch, kStepBytes, 128, true);
    tm_w_up = tm_w;
    if (rc == INT4L_OK && kGated) rc = encode_tensor_map_2d(ctx, &tm_w_up, p.w_up.codes, 1, pitch, p.n, pitch, kStepBytes, 128, true);
    tm_y = tm_x;
    if (rc == INT4L_OK && a.tma_store) rc = encode_tensor_map_2d(ctx, &tm_y, p.y, 2, p.n, p.m, out_pitch, 64, 32, true);
    tm_g = tm_u = tm_y;
    if (rc == INT4L_OK && a.tma_store && p.keep_gate) {
        rc = encode_tensor_map_2d(ctx, &tm_g, p.keep_gate, 2, p.n, p.m, out_pitch, 64, 32, true);
        if (rc == INT4L_OK) rc = encode_tensor_map_2d(ctx, &tm_u, p.keep_up, 2, p.n, p.m, out_pitch, 64, 32, true);
    }
    if (rc != INT4L_OK) return rc;
    const long long tiles = static_cast<long long>(a.tiles_m) * a.tiles_n;
    if (tiles > 0x7FFFFFFF) return INT4L_ERR_TOO_LARGE;
    const int pairs = tiles < ctx->max_pairs ? static_cast<int>(tiles) : ctx->max_pairs;
    gemm_fp4_kernel<kBlock16, kGated><<<pairs * 2, kThreads, Geo<kBlock16>::kSmemBytes, stream>>>(tm_x, tm_w, tm_w_up, tm_y, tm_g, tm_u, a);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? INT4L_OK : INT4L_ERR_CUDA;
}

template <bool kBlock16, bool kGated>
bool set_attr()
{
    return cudaFuncSetAttribute(gemm_fp4_kernel<kBlock16, kGated>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<kBlock16>::kSmemBytes) == cudaSuccess;
}

}  // namespace

int setup_fp4_gemm(DeviceCtx*)
{
    return set_attr<false, false>() && set_attr<false, true>() && set_attr<true, false>() && set_attr<true, true>() ? INT4L_OK : INT4L_ERR_CUDA;
}

int launch_fp4_gemm(DeviceCtx* ctx, const Fp4Problem& p, cudaStream_t stream)
{
    if (p.x.block16) return p.gated ? launch_cfg<true, true>(ctx, p, stream) : launch_cfg<true, false>(ctx, p, stream);
    return p.gated ? launch_cfg<false, true>(ctx, p, stream) : launch_cfg<false, false>(ctx, p, stream);
}

}  // namespace i4l
