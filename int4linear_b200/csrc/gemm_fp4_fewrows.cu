// The products of gemm_fp4.cu for few rows of x (decode batches): a stream of the weights.
//
// Every byte of w is used once, so the time is that of bringing w in, and nearly all SMs have to take part from the
// start.  The operands are swapped: the UMMA's 128-row side holds rows of w, its narrow side the rows of x (padded to
// 16), the accumulator is a tile of y transposed.  128 rows of w at a time would give a projection of a few
// thousand columns far fewer tiles than there are SMs, so k is cut as well: a cluster of up to 8 CTAs shares one
// tile, each contracts its part of k, and the parts are added up through distributed shared memory, in the order of
// k, so the result does not depend on timing and no workspace exists.  A gated tile is 128 rows of the gate matrix and
// the same 128 of the up matrix, in two accumulators.
//
// Bound: HBM.  A CTA's shared memory is kept to a half or a third of an SM's, so that the loads of one CTA cover the
// start and the reduction of another.  Tensor memory is shared between the CTAs of an SM too, and its allocation
// waits while there is none.  Every launch takes at least 448 bytes of shared memory per column, which keeps any
// mixture of resident CTAs of this kernel within the 512 columns (228 KB / 448 = 521, and allocations are multiples of
// 128), so none of its allocations waits for another.
//     warp 0      TMA (as in gemm_fp4.cu)
//     warp 1      tcgen05.cp of the scales and UMMAs
//     all 4       epilogue
//
// Measured, per launch in a graph with weights from HBM: 1 x 14336 x 4096 mxfp4 8.8 us (3.5 TB/s), 16 rows nvfp4 9.7, gated
// 16 rows mxfp4 15.1 (4.1 TB/s), 1 x 4096 x 4096 6.1, 16 x 28672 x 8192 24 (5.2 TB/s); the fixed part is 4 us.
#include "epilogue.cuh"
#include "fp4.cuh"
#include "fp4_fewrows_plan.cuh"
#include "gate.cuh"
#include "ptx.cuh"

namespace i4l {

namespace {

constexpr int kRows = kFewRowsTile;
constexpr int kStepBytes = kFewRowsStepBytes, kStepK = kFewRowsStepK;
constexpr int kThreads = 128;
constexpr int kMaxStages = kFewRowsMaxStages;

template <bool kBlock16, bool kGated>
using Geo = FewRowsGeo<kBlock16, kGated>;
static_assert(Geo<false, false>::kScaleBytes == 2 * kScaleTileBytes, "scale tile");

struct Args {
    const float* ts_x; const float* ts_w; const float* ts_w_up;
    const float* bias;
    unsigned short* y; unsigned short* keep_gate; unsigned short* keep_up;
    int m, n, k;
    int n_pad;     // rows of x in the UMMA, a multiple of 16
    int stages, stage_bytes, cols;
    int split;     // CTAs per cluster
    int tiles;     // of 128 rows of w
    int act, fp16;
    int* status;
};

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}

__device__ __forceinline__ float act_of(float g, int act)
{
    if (act == kActSilu) return gate_act<kActSilu>(g);
    if (act == kActGelu) return gate_act<kActGelu>(g);
    return gate_act<kActGeluTanh>(g);
}

template <bool kBlock16, bool kGated>
__global__ void __launch_bounds__(kThreads)
gemm_fp4_fewrows_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                        const __grid_constant__ CUtensorMap tm_w_up, const __grid_constant__ CUtensorMap tm_sx,
                        const __grid_constant__ CUtensorMap tm_sw, const __grid_constant__ CUtensorMap tm_sw_up,
                        const __grid_constant__ Args a)
{
    using G = Geo<kBlock16, kGated>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 1];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t ring = (raw + 1023u) & ~1023u;
    const uint32_t bar_base = smem_u32(bars);
    auto full  = [&](int i) { return bar_base + 8u * i; };
    auto empty = [&](int i) { return bar_base + 8u * (kMaxStages + i); };
    const uint32_t acc_full = bar_base + 8u * (2 * kMaxStages);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int split = a.split;
    const int rank = static_cast<int>(blockIdx.x) % split;
    const int item = static_cast<int>(blockIdx.x) / split;
    const int tile = item % a.tiles, group = item / a.tiles;  // 128 rows of w, 128 rows of x
    const int m = min(128, a.m - group * 128);                // (of x, here)
    const size_t out0 = static_cast<size_t>(group) * 128 * a.n;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int i = 0; i < kMaxStages; ++i) { mbar_init(full(i), 1); mbar_init(empty(i), 1); }
        mbar_init(acc_full, 1);
        *abort_flag = 0;
        mbar_init_fence();
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(&tmem_slot), a.cols);
        tmem_relinquish<1>();
    }
    if (warp == 0 && elect_one()) {
        tma_prefetch_desc(&tm_x);
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_sx);
        tma_prefetch_desc(&tm_sw);
        if (kGated) { tma_prefetch_desc(&tm_w_up); tma_prefetch_desc(&tm_sw_up); }
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_slot;
    // Everything above may run while the launch before this one in the stream still works.
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const int steps = (a.k + kStepK - 1) / kStepK;
    const int kb0 = static_cast<int>(static_cast<long long>(steps) * rank / split);
    const int kb1 = static_cast<int>(static_cast<long long>(steps) * (rank + 1) / split);

    if (warp == 0) {
        int s = 0;
        uint32_t phase = 1;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait_warp(empty(s), phase, abort_flag)) break;
            if (elect_one()) {
                mbar_expect_tx(full(s), G::kOffX + a.n_pad * kStepBytes);
                const uint32_t dst = ring + s * a.stage_bytes;
                const int sc = kb * (G::kScaleBytes / 8);
                tma_load_2d(dst, &tm_w, full(s), kb * kStepBytes, tile * kRows);
                if (kGated) tma_load_2d(dst + G::kCodesW, &tm_w_up, full(s), kb * kStepBytes, tile * kRows);
                tma_load_2d(dst + G::kOffScales, &tm_sw, full(s), sc, tile);
                if (kGated) tma_load_2d(dst + G::kOffScales + G::kScaleBytes, &tm_sw_up, full(s), sc, tile);
                tma_load_2d(dst + G::kOffScales + G::kW * G::kScaleBytes, &tm_sx, full(s), sc, group);
                tma_load_2d(dst + G::kOffX, &tm_x, full(s), kb * kStepBytes, group * 128);
            }
            __syncwarp();
            if (++s == a.stages) { s = 0; phase ^= 1u; }
        }
    } else if (warp == 1) {
        const uint32_t scale_cols = tmem_base + G::kW * a.n_pad;
        int s = 0;
        uint32_t phase = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait_warp(full(s), phase, abort_flag)) break;
            tc_fence_after_sync();
            const uint32_t at = ring + s * a.stage_bytes;
            const uint32_t sf = scale_cols + s * G::kScaleCols;
            const uint32_t sfx = sf + 4 * G::kTilesK * G::kW;
            const int umma_count = min(4, (a.k - kb * kStepK + 63) / 64);
            const uint32_t x_low = umma_desc_sw128_low(at + G::kOffX), w_low = umma_desc_sw128_low(at), scales_low = scale_tile_low(at + G::kOffScales);
            if (elect_one()) {
#pragma unroll
                for (int t = 0; t < (G::kW + 1) * G::kTilesK; ++t)
                    tmem_copy_scales<1>(sf + 4 * t, scales_low + t * (kScaleTileBytes / 16));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j >= umma_count) break;
                    const int t = kBlock16 ? j : j >> 1;
                    const uint32_t idesc = umma_idesc_fp4(kRows, 0, !kBlock16, kBlock16 ? 0u : 2u * (j & 1)) | (static_cast<uint32_t>(a.n_pad >> 3) << 17);
#pragma unroll
                    for (int i = 0; i < G::kW; ++i)
                        umma_fp4<1, kBlock16>(tmem_base + i * a.n_pad, w_low + i * (G::kCodesW / 16) + 2 * j, x_low + 2 * j, idesc,
                                              sf + 4 * (i * G::kTilesK + t), sfx + 4 * t, (kb > kb0 || j > 0) ? 1u : 0u);
                }
                umma_commit(empty(s));
                if (kb == kb1 - 1) umma_commit(acc_full);
            }
            __syncwarp();
            if (++s == a.stages) { s = 0; phase ^= 1u; }
        }
    }
    __syncwarp();

    // ---------------------------------------------------------------- epilogue
    // A bias is fetched while the products run: of the thread's column, or of the four it sums up below.
    auto bias_of = [&](int col) { return (!kGated && a.bias != nullptr && col < a.n) ? __ldg(a.bias + col) : 0.0f; };
    const int bias_col = tile * kRows + (split == 1 ? tid : 4 * lane);
    float bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = (e == 0 || split > 1) ? bias_of(bias_col + e) : 0.0f;
    const bool ok = mbar_wait_warp(acc_full, 0, abort_flag);
    tc_fence_after_sync();
    const float ts_x = a.ts_x != nullptr ? __ldg(a.ts_x) : 1.0f;
    const float alpha = ts_x * (a.ts_w != nullptr ? __ldg(a.ts_w) : 1.0f);
    const float alpha_up = kGated ? ts_x * (a.ts_w_up != nullptr ? __ldg(a.ts_w_up) : 1.0f) : 0.0f;
    auto bits = [&](float v) { return scaled_to_bits(v, a.fp16); };
    // One value of y, from its sum (or its two) and, for a product, its column's bias.
    auto put = [&](int i, int col, float acc, float acc_up, float bias) {
        const size_t at = out0 + static_cast<size_t>(i) * a.n + col;
        if constexpr (kGated) {
            const float g = acc * alpha, u = acc_up * alpha_up;
            a.y[at] = bits(act_of(g, a.act) * u);
            if (a.keep_gate != nullptr) { a.keep_gate[at] = bits(g); a.keep_up[at] = bits(u); }
        } else {
            a.y[at] = bits(fmaf(acc, alpha, bias));
        }
    };
    const uint32_t lanes = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
    // All UMMAs of this CTA are done with the ring (acc_full): it takes the partial sums, [x row][w row] floats.
    if (ok) {
        const int col = tile * kRows + tid;
#pragma unroll 1
        for (int c = 0; c < m; c += 16) {
            uint32_t v[G::kW][16];
#pragma unroll
            for (int i = 0; i < G::kW; ++i) tmem_ld_16(lanes + i * a.n_pad + c, v[i]);
            tmem_ld_wait();
            if (split == 1) {
                if (col < a.n) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (c + e < m) put(c + e, col, __uint_as_float(v[0][e]), __uint_as_float(v[G::kW - 1][e]), bias[0]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < G::kW; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sts32(ring + ((i * a.n_pad + c + e) * kRows + tid) * 4, v[i][e]);
            }
        }
    }
    // Tensor memory goes back before any wait for another CTA: whoever holds it never waits for a CTA that might wait
    // for it.
    tc_fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        if (tid == 0) atomicExch(a.status, INT4L_ERR_DEVICE_TIMEOUT);
        for (int i = 0; i < 100; ++i) __nanosleep(1000);  // copies and UMMAs in flight end
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc<1>(tmem_base, a.cols);
    }
    __syncwarp();
    if (split > 1) {
        cluster_sync_all();
        // Rows of x are dealt out to the warps of the cluster, four columns to a lane; each value is summed in the
        // order of k.
        const int col = tile * kRows + 4 * lane;
        if (ok) {
#pragma unroll 2
            for (int i = warp * split + rank; i < m; i += 4 * split) {
                float4 sum[G::kW];
#pragma unroll
                for (int w = 0; w < G::kW; ++w) {
                    const uint32_t mine = ring + ((w * a.n_pad + i) * kRows + 4 * lane) * 4;
                    float4 part[8];
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (r < split) part[r] = ld_cluster_f32x4(cluster_address(mine, r));
                    sum[w] = part[0];
#pragma unroll
                    for (int r = 1; r < 8; ++r)
                        if (r < split) { sum[w].x += part[r].x; sum[w].y += part[r].y; sum[w].z += part[r].z; sum[w].w += part[r].w; }
                }
                const float4 s0 = sum[0], s1 = sum[G::kW - 1];
                if (a.n % 4 == 0 && col < a.n) {  // (then all four columns exist, on 8 bytes)
                    const float acc[4] = {s0.x, s0.y, s0.z, s0.w}, acc_up[4] = {s1.x, s1.y, s1.z, s1.w};
                    unsigned short h[4], hg[4], hu[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (kGated) {
                            const float g = acc[e] * alpha, u = acc_up[e] * alpha_up;
                            h[e] = bits(act_of(g, a.act) * u);
                            hg[e] = bits(g);
                            hu[e] = bits(u);
                        } else {
                            h[e] = bits(fmaf(acc[e], alpha, bias[e]));
                        }
                    }
                    auto store4 = [&](unsigned short* dst, const unsigned short (&t)[4]) {
                        *reinterpret_cast<uint2*>(dst + out0 + static_cast<size_t>(i) * a.n + col) =
                            make_uint2(t[0] | (static_cast<uint32_t>(t[1]) << 16), t[2] | (static_cast<uint32_t>(t[3]) << 16));
                    };
                    store4(a.y, h);
                    if (kGated && a.keep_gate != nullptr) { store4(a.keep_gate, hg); store4(a.keep_up, hu); }
                    continue;
                }
                if (col < a.n) put(i, col, s0.x, s1.x, bias[0]);
                if (col + 1 < a.n) put(i, col + 1, s0.y, s1.y, bias[1]);
                if (col + 2 < a.n) put(i, col + 2, s0.z, s1.z, bias[2]);
                if (col + 3 < a.n) put(i, col + 3, s0.w, s1.w, bias[3]);
            }
        }
        __syncwarp();
        cluster_sync_all();  // no CTA leaves while another reads its shared memory
    }
}

template <bool kBlock16, bool kGated>
int launch_cfg(DeviceCtx* ctx, const Fp4Problem& p, cudaStream_t stream)
{
    const FewRowsPlan l = fewrows_plan<kBlock16, kGated>(p.m, p.n, p.k, ctx->sm_count);
    Args a = {};
    a.ts_x = p.x.tensor_scale; a.ts_w = p.w.tensor_scale; a.ts_w_up = p.w_up.tensor_scale;
    a.bias = p.bias;
    a.y = static_cast<unsigned short*>(p.y);
    a.keep_gate = static_cast<unsigned short*>(p.keep_gate);
    a.keep_up = static_cast<unsigned short*>(p.keep_up);
    a.m = p.m; a.n = p.n; a.k = p.k;
    a.n_pad = l.n_pad;
    a.stages = l.stages; a.stage_bytes = l.stage_bytes; a.cols = l.cols;
    a.split = l.split;
    a.tiles = l.tiles;
    a.act = p.act;
    a.fp16 = p.fp16;
    a.status = ctx->status_dev;

    const uint64_t pitch = static_cast<uint64_t>(p.k) / 2;
    CUtensorMap tm_x, tm_w, tm_w_up, tm_sx, tm_sw, tm_sw_up;
    int rc = encode_tensor_map_2d(ctx, &tm_x, p.x.codes, 1, pitch, p.m, pitch, kStepBytes, a.n_pad, true);
    if (rc == INT4L_OK) rc = encode_tensor_map_2d(ctx, &tm_w, p.w.codes, 1, pitch, p.n, pitch, kStepBytes, kRows, true);
    if (rc == INT4L_OK) rc = fp4_scale_map(ctx, &tm_sx, p.x, Geo<kBlock16, kGated>::kScaleBytes, 1);
    if (rc == INT4L_OK) rc = fp4_scale_map(ctx, &tm_sw, p.w, Geo<kBlock16, kGated>::kScaleBytes, 1);
    tm_w_up = tm_w;
    tm_sw_up = tm_sw;
    if (rc == INT4L_OK && kGated) {
        rc = encode_tensor_map_2d(ctx, &tm_w_up, p.w_up.codes, 1, pitch, p.n, pitch, kStepBytes, kRows, true);
        if (rc == INT4L_OK) rc = fp4_scale_map(ctx, &tm_sw_up, p.w_up, Geo<kBlock16, kGated>::kScaleBytes, 1);
    }
    if (rc != INT4L_OK) return rc;

    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(l.tiles * l.split * l.groups, 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = l.smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = l.split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, gemm_fp4_fewrows_kernel<kBlock16, kGated>, tm_x, tm_w, tm_w_up, tm_sx, tm_sw, tm_sw_up, a);
    count_launch();
    if (e != cudaSuccess) { cudaGetLastError(); return INT4L_ERR_CUDA; }
    return INT4L_OK;
}

template <bool kBlock16, bool kGated>
bool set_attr()
{
    return cudaFuncSetAttribute(gemm_fp4_fewrows_kernel<kBlock16, kGated>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmShared / 2) == cudaSuccess;
}

}  // namespace

int setup_fp4_fewrows(DeviceCtx*)
{
    return set_attr<false, false>() && set_attr<false, true>() && set_attr<true, false>() && set_attr<true, true>() ? INT4L_OK : INT4L_ERR_CUDA;
}

bool fp4_fewrows_preferred(const DeviceCtx* ctx, const Fp4Problem& p) { return fewrows_preferred(p.m, p.n, p.k, p.gated, ctx->sm_count); }

int launch_fp4_fewrows(DeviceCtx* ctx, const Fp4Problem& p, cudaStream_t stream)
{
    if (p.x.block16) return p.gated ? launch_cfg<true, true>(ctx, p, stream) : launch_cfg<true, false>(ctx, p, stream);
    return p.gated ? launch_cfg<false, true>(ctx, p, stream) : launch_cfg<false, false>(ctx, p, stream);
}

}  // namespace i4l
