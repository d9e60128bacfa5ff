// Backward pass of the products of microscaled matrices (fp4.cuh, gemm_fp4.cu):
//
//     y = x w^T             dx = dy w                  dw = dy^T x
//     h = act(g) u          dg = dh u act'(g),  du = dh act(g)
//                           dx = dg wg + du wu         dwg = dg^T x,  dwu = du^T x
//
// with respect to the values the operands stand for.  The contraction runs over n or m, across the blocks that
// share a scale, so the block-scaled instruction does not apply: the operands are expanded to bf16 first.  That
// loses nothing (a code times its e8m0 or e4m3 scale has at most 6 significant bits); only the incoming gradient
// is rounded, dg and du to bf16, as the gradients of a bf16 network are.
//
// The products are one persistent kernel, a CTA pair per 256 x 256 tile (tcgen05.mma kind::f16, cta_group::2),
// two accumulators in tensor memory so that the epilogue overlaps the next tile:
//     warp 0      TMA, steps of 64 along the contraction, into 128-byte-swizzled slots
//     warp 1      UMMA issue (CTA 0 for both)
//     warps 2-5   epilogue: scale, round to bf16, staged TMA stores
// No operand is ever transposed: where the contraction runs down the rows of a matrix (w and x always, dy for
// dw), its tile is read as it lies and the UMMA takes it MN-major.
#include "epilogue.cuh"
#include "fp4.cuh"
#include "gate.cuh"
#include "ptx.cuh"

namespace i4l {

namespace {

constexpr int kBM = 128, kBN = 256, kStepK = 64;
constexpr int kThreads = 32 * 6;
constexpr int kStages = 6;
constexpr int kStage = 2 * 128 * 128;          // A and B tile of one CTA, 16 KB each
constexpr int kChunk = kStepK * 128;           // MN-major: 64 columns x 64 rows
constexpr int kStoreStage = 4096;              // per warp and buffer
constexpr int kNumBarriers = 2 * kStages + 4;
constexpr int kSmemBytes = 1024 + kStages * kStage + 4 * 2 * kStoreStage + kNumBarriers * 8 + 16;
static_assert(kSmemBytes <= 232448, "shared memory budget");

struct GradArgs {
    const float* num; const float* den;
    int rows, cols;        // of the result
    int tiles_m, tiles_n;
    int steps, segments;   // steps per segment of the contraction
    int* status;
};

template <bool kWeight>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
grad_gemm_kernel(const __grid_constant__ CUtensorMap tm_a0, const __grid_constant__ CUtensorMap tm_a1,
                 const __grid_constant__ CUtensorMap tm_b0, const __grid_constant__ CUtensorMap tm_b1,
                 const __grid_constant__ CUtensorMap tm_c, const __grid_constant__ GradArgs a)
{
    constexpr int S = kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* gbase = smem_raw + (base - raw);

    const uint32_t ring = base;
    const uint32_t st_base = ring + S * kStage;
    const uint32_t bar_base = st_base + 4 * 2 * kStoreStage;
    auto full     = [&](int i) { return bar_base + 8u * i; };
    auto empty    = [&](int i) { return bar_base + 8u * (S + i); };
    auto tm_full  = [&](int i) { return bar_base + 8u * (2 * S + i); };
    auto tm_empty  = [&](int i) { return bar_base + 8u * (2 * S + 2 + i); };
    const uint32_t misc_off = (bar_base - base) + 8u * kNumBarriers;
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + misc_off);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + misc_off + 4);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t cta_rank = cluster_cta_rank();
    const int worker = static_cast<int>(cluster_id_x());
    const int workers = static_cast<int>(cluster_count_x());

    if (tid == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(full(i), 1); mbar_init(empty(i), 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(tm_full(i), 1); mbar_init(tm_empty(i), 4 * 2); }
        *abort_flag = 0;
        mbar_init_fence();
        tma_prefetch_desc(&tm_a0);
        tma_prefetch_desc(&tm_b0);
        tma_prefetch_desc(&tm_c);
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
    const int steps = a.steps * a.segments;
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
            const int row = (tm * 2 + static_cast<int>(cta_rank)) * kBM;
            const int col = tn * kBN + static_cast<int>(cta_rank) * 128;
            for (int st = 0; st < steps; ++st, ++it) {
                const uint32_t s = it % S, r = it / S;
                if (!mbar_wait_warp(empty(s), (r & 1u) ^ 1u, abort_flag)) { alive = false; break; }
                if (elect_one()) {
                    // Both CTAs' loads are counted on CTA 0's barrier (which cannot complete before this announcement).
                    if (cta_rank == 0) mbar_expect_tx(full(s), 2 * kStage);
                    const uint32_t bar = cluster_address(full(s), 0);
                    const uint32_t dst = ring + s * kStage;
                    const bool second = st >= a.steps;
                    const int k0 = (second ? st - a.steps : st) * kStepK;
                    const CUtensorMap* ta = second ? &tm_a1 : &tm_a0;
                    const CUtensorMap* tb = second ? &tm_b1 : &tm_b0;
                    if constexpr (kWeight) {
                        tma_load_2d_pair(dst, ta, bar, row, k0);
                        tma_load_2d_pair(dst + kChunk, ta, bar, row + 64, k0);
                    } else {
                        tma_load_2d_pair(dst, ta, bar, k0, row);
                    }
                    tma_load_2d_pair(dst + 2 * kChunk, tb, bar, col, k0);
                    tma_load_2d_pair(dst + 3 * kChunk, tb, bar, col + 64, k0);
                }
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        if (cta_rank == 0) {
            // ----------------------------------------------------- UMMA issuer
            // The warp walks the ring together and one elected thread issues.
            constexpr uint32_t idesc = umma_idesc_bf16(2 * kBM, kBN, kWeight, true);
            uint32_t it = 0, local_tile = 0;
            bool alive = true;
            for (int tile = worker; alive && tile < num_tiles; tile += workers, ++local_tile) {
                const uint32_t buf = local_tile & 1u, br = local_tile >> 1;
                if (!mbar_wait_warp(tm_empty(buf), (br & 1u) ^ 1u, abort_flag)) break;
                tc_fence_after_sync();
                const uint32_t d_tmem = tmem_base + buf * kBN;
                for (int st = 0; st < steps; ++st, ++it) {
                    const uint32_t s = it % S, r = it / S;
                    if (!mbar_wait_warp(full(s), r & 1u, abort_flag)) { alive = false; break; }
                    tc_fence_after_sync();
                    const uint32_t a_addr = ring + s * kStage;
                    const uint64_t a_desc = kWeight ? umma_desc_mn_sw128(a_addr, kChunk) : umma_desc_sw128(a_addr);
                    const uint64_t b_desc = umma_desc_mn_sw128(a_addr + 2 * kChunk, kChunk);
                    // 16 elements of the contraction on: 32 bytes of a K-major row, or two 1024-byte atoms
                    constexpr uint32_t kStepA = kWeight ? 2048 >> 4 : 32 >> 4, kStepB = 2048 >> 4;
                    if (elect_one()) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            umma_bf16<2>(d_tmem, a_desc + kStepA * j, b_desc + kStepB * j, idesc, (st | j) != 0 ? 1u : 0u);
                        umma_commit_2cta(empty(s), 3);
                        if (st == steps - 1) umma_commit_2cta(tm_full(buf), 3);
                    }
                    __syncwarp();
                }
            }
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------- epilogue
        const int sp = warp & 3;
        const uint32_t stage0 = st_base + (warp - 2) * 2 * kStoreStage;
        float alpha = a.num != nullptr ? __ldg(a.num) : 1.0f;
        if (a.den != nullptr) {
            const float d = __ldg(a.den);
            if (d != 0.0f) alpha /= d;
        }
        uint32_t local_tile = 0, chunk_no = 0;
        for (int tile = worker; tile < num_tiles; tile += workers, ++local_tile) {
            int tm, tn;
            tile_coord(tile, tm, tn);
            const uint32_t buf = local_tile & 1u, br = local_tile >> 1;
            if (!mbar_wait_warp(tm_full(buf), br & 1u, abort_flag)) break;
            tc_fence_after_sync();
            const int row0 = (tm * 2 + static_cast<int>(cta_rank)) * kBM + sp * 32;
            const uint32_t t_addr = tmem_base + (static_cast<uint32_t>(sp * 32) << 16) + buf * kBN;
#pragma unroll 1
            for (int c = 0; c < kBN; c += 64) {
                const int col0 = tn * kBN + c;
                if (row0 >= a.rows || col0 >= a.cols) break;
                uint32_t v[64], h[32];
                load64(t_addr + c, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) h[j] = pack16<false>(__uint_as_float(v[2 * j]) * alpha, __uint_as_float(v[2 * j + 1]) * alpha);
                const uint32_t stg = stage0 + (chunk_no & 1u) * kStoreStage;
                if (lane == 0) tma_store_wait_read<1>();
                __syncwarp();
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    sts128(stg + lane * 128 + ((q ^ (lane & 7)) << 4), make_uint4(h[4 * q], h[4 * q + 1], h[4 * q + 2], h[4 * q + 3]));
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    tma_store_2d(&tm_c, stg, col0, row0);
                    tma_store_commit();
                }
                ++chunk_no;
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

// ------------------------------------------------------------------ dg and du

constexpr int kGateThreads = 256;

template <int kAct>
__device__ __forceinline__ void gate_grad(float dh, float g, float u, float fg, float fu, float& dg, float& du)
{
    float act, slope;
    gate_act_slope<kAct>(g, act, slope);
    dg = dh * u * slope * fg;
    du = dh * act * fu;
}

// Eight columns per thread where rows are 16-byte aligned, else one.  Bound by HBM: 10 bytes per element.
template <int kAct, bool kVec>
__global__ void __launch_bounds__(kGateThreads)
gate_backward_kernel(const __nv_bfloat16* __restrict__ dh, const __nv_bfloat16* __restrict__ gate, const __nv_bfloat16* __restrict__ up,
                     __nv_bfloat16* __restrict__ dg, __nv_bfloat16* __restrict__ du, const float* __restrict__ f_g,
                     const float* __restrict__ f_u, int m, int n, long long ld)
{
    float fg = f_g != nullptr ? __ldg(f_g) : 1.0f, fu = f_u != nullptr ? __ldg(f_u) : 1.0f;
    if (fg == 0.0f) fg = 1.0f;
    if (fu == 0.0f) fu = 1.0f;
    constexpr int kE = kVec ? 8 : 1;
    const int per_row = n / kE;
    const long long total = static_cast<long long>(m) * per_row;
    const long long stride = static_cast<long long>(gridDim.x) * kGateThreads;
    for (long long i = blockIdx.x * static_cast<long long>(kGateThreads) + threadIdx.x; i < total; i += stride) {
        const long long row = i / per_row;
        const int col = static_cast<int>(i - row * per_row) * kE;
        const size_t src = static_cast<size_t>(row) * n + col, dst = static_cast<size_t>(row) * ld + col;
        __align__(16) __nv_bfloat16 e_dh[kE], e_g[kE], e_u[kE], o_g[kE], o_u[kE];
        if constexpr (kVec) {
            *reinterpret_cast<uint4*>(e_dh) = __ldg(reinterpret_cast<const uint4*>(dh + src));
            *reinterpret_cast<uint4*>(e_g) = __ldg(reinterpret_cast<const uint4*>(gate + src));
            *reinterpret_cast<uint4*>(e_u) = __ldg(reinterpret_cast<const uint4*>(up + src));
        } else {
            e_dh[0] = dh[src]; e_g[0] = gate[src]; e_u[0] = up[src];
        }
#pragma unroll
        for (int e = 0; e < kE; ++e) {
            float a, b;
            gate_grad<kAct>(__bfloat162float(e_dh[e]), __bfloat162float(e_g[e]), __bfloat162float(e_u[e]), fg, fu, a, b);
            o_g[e] = __float2bfloat16_rn(a);
            o_u[e] = __float2bfloat16_rn(b);
        }
        if constexpr (kVec) {
            *reinterpret_cast<uint4*>(dg + dst) = *reinterpret_cast<const uint4*>(o_g);
            *reinterpret_cast<uint4*>(du + dst) = *reinterpret_cast<const uint4*>(o_u);
        } else {
            dg[dst] = o_g[0]; du[dst] = o_u[0];
        }
    }
}

template <bool kWeight>
int launch_grad(DeviceCtx* ctx, const GradProduct& p, cudaStream_t stream)
{
    GradArgs a = {};
    a.num = p.num; a.den = p.den;
    a.rows = kWeight ? p.n : p.m;
    a.cols = p.k;
    a.tiles_m = (a.rows + 255) / 256;
    a.tiles_n = (p.k + kBN - 1) / kBN;
    a.steps = ((kWeight ? p.m : p.n) + kStepK - 1) / kStepK;
    a.segments = p.d1 != nullptr ? 2 : 1;
    a.status = ctx->status_dev;
    const uint64_t ld_bytes = static_cast<uint64_t>(p.ld) * 2, k_bytes = static_cast<uint64_t>(p.k) * 2;
    const int b_rows = kWeight ? p.m : p.n;
    CUtensorMap a0, a1, b0, b1, c;
    const uint32_t box_a = kWeight ? kStepK : kBM;
    int rc = encode_tensor_map_2d(ctx, &a0, p.d0, 2, p.n, p.m, ld_bytes, 64, box_a, true);
    if (rc == INT4L_OK) rc = encode_tensor_map_2d(ctx, &b0, p.b0, 2, p.k, b_rows, k_bytes, 64, kStepK, true);
    a1 = a0; b1 = b0;
    if (rc == INT4L_OK && p.d1 != nullptr) {
        rc = encode_tensor_map_2d(ctx, &a1, p.d1, 2, p.n, p.m, ld_bytes, 64, box_a, true);
        if (rc == INT4L_OK) rc = encode_tensor_map_2d(ctx, &b1, p.b1, 2, p.k, b_rows, k_bytes, 64, kStepK, true);
    }
    if (rc == INT4L_OK) rc = encode_tensor_map_2d(ctx, &c, p.out, 2, p.k, a.rows, k_bytes, 64, 32, true);
    if (rc != INT4L_OK) return rc;
    const long long tiles = static_cast<long long>(a.tiles_m) * a.tiles_n;
    const int pairs = tiles < ctx->max_pairs ? static_cast<int>(tiles) : ctx->max_pairs;
    grad_gemm_kernel<kWeight><<<pairs * 2, kThreads, kSmemBytes, stream>>>(a0, a1, b0, b1, c, a);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? INT4L_OK : INT4L_ERR_CUDA;
}

}  // namespace

int setup_grad(DeviceCtx*)
{
    const bool ok = cudaFuncSetAttribute(grad_gemm_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) == cudaSuccess &&
                    cudaFuncSetAttribute(grad_gemm_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) == cudaSuccess;
    return ok ? INT4L_OK : INT4L_ERR_CUDA;
}

int launch_grad_product(DeviceCtx* ctx, const GradProduct& p, cudaStream_t stream)
{
    return p.weight ? launch_grad<true>(ctx, p, stream) : launch_grad<false>(ctx, p, stream);
}

int launch_gate_backward(DeviceCtx* ctx, const void* dh, const void* gate, const void* up, void* dg, void* du, int act,
                         const float* f_g, const float* f_u, int m, int n, long long ld, cudaStream_t stream)
{
    using B = __nv_bfloat16;
    const bool vec = n % 8 == 0 && ((reinterpret_cast<uintptr_t>(dh) | reinterpret_cast<uintptr_t>(gate) | reinterpret_cast<uintptr_t>(up)) & 15u) == 0;
    const long long units = static_cast<long long>(m) * (vec ? n / 8 : n);
    const long long blocks = (units + kGateThreads - 1) / kGateThreads, cap = static_cast<long long>(ctx->sm_count) * 32;
    const int grid = static_cast<int>(blocks < cap ? blocks : cap);
    auto go = [&](auto kernel) {
        kernel<<<grid, kGateThreads, 0, stream>>>(static_cast<const B*>(dh), static_cast<const B*>(gate), static_cast<const B*>(up),
                                                  static_cast<B*>(dg), static_cast<B*>(du), f_g, f_u, m, n, ld);
    };
    if (act == kActSilu) vec ? go(gate_backward_kernel<kActSilu, true>) : go(gate_backward_kernel<kActSilu, false>);
    else if (act == kActGelu) vec ? go(gate_backward_kernel<kActGelu, true>) : go(gate_backward_kernel<kActGelu, false>);
    else vec ? go(gate_backward_kernel<kActGeluTanh, true>) : go(gate_backward_kernel<kActGeluTanh, false>);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? INT4L_OK : INT4L_ERR_CUDA;
}

}  // namespace i4l
