// Quantisation into, and expansion out of, microscaled 4-bit floating point (format: fp4.cuh).
//
// Quantisation, for each block with amax = max |x|:
//     mxfp4  scale 2^e, e = floor(log2 amax) - 2 (so amax / 2^e lies in [4, 8)), at least 2^-127; the rule
//            of the OCP MX specification;
//     nvfp4  the values are first multiplied by 1 / tensor_scale (one fp32 rounding); scale = amax / 6 rounded
//            to the nearest e4m3, at most 448; a scale of 0 makes every code 0;
//     codes  x / scale rounded to the nearest e2m1 value, ties to the even code, at most 6.
// All of it is exact: the power-of-two division loses nothing, the two e4m3 divisions are rounded so that
// no tie is created or missed (below), so a code or scale never depends on how the work is cut.
// A block that holds a NaN or an infinity gets the scale NaN, and so does every product with it.
//
// Bound: HBM.  Each element is read once (2 or 4 bytes) and written once (half a byte and 1/32 or 1/16).
#include "fp4.cuh"

namespace i4l {

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // row chunks in flight per warp

template <int kType> struct Src;
template <> struct Src<INT4L_TYPE_BF16> { using T = __nv_bfloat16; };
template <> struct Src<INT4L_TYPE_F16> { using T = __half; };
template <> struct Src<INT4L_TYPE_F32> { using T = float; };

__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(float v) { return v; }

// Eight elements from p (any alignment; `vec` says 16 bytes).
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&v)[8])
{
    __align__(16) T e[8];
    if (vec) {
        constexpr int kVecs = sizeof(T) * 8 / 16;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) reinterpret_cast<uint4*>(e)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_float(e[i]);
}

// Eight floats -> eight codes, element 0 in the low nibble; nearest, ties to even, saturating.
__device__ __forceinline__ uint32_t to_e2m1x8(const float (&v)[8])
{
    uint32_t r;
    asm("{\n\t"
        ".reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t"
        "}\n"
        : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// The e4m3 byte of a >= 0 (finite), nearest even, saturating at 448.
__device__ __forceinline__ uint32_t to_e4m3(float a)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(a));
    return r & 0xFFu;
}
__device__ __forceinline__ float from_e4m3(uint32_t byte)
{
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(byte)));
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h2 & 0xFFFFu)));
}

// One warp handles 256 consecutive elements of a row at a time, eight per lane: a lane's loads are 16 (or 32)
// bytes, the warp's code store 128, and a block's scale is agreed on by 4 (mxfp4) or 2 (nvfp4) lanes.  The
// words of a scale tile (4 scales) are put together by 16 or 8 lanes and stored by the first of them.
// Rows are padded to 128 and scales to whole words with zeros, so that nothing in a scale tile is undefined.
template <int kType, bool kBlock16>
__global__ void __launch_bounds__(kThreads)
fp4_quantize_kernel(const typename Src<kType>::T* __restrict__ src, long long pitch, uint8_t* __restrict__ codes,
                    uint8_t* __restrict__ scales, const float* __restrict__ tensor_scale, int rows, int k)
{
    constexpr int kLanes = kBlock16 ? 2 : 4;  // lanes of a block
    using T = typename Src<kType>::T;
    const int lane = threadIdx.x & 31;
    const int chunks = (k + 255) / 256;
    const int rows_padded = (rows + 127) / 128 * 128;
    const int ktiles = fp4_ktiles(k, kBlock16);
    const long long total = static_cast<long long>(rows_padded) * chunks;
    const long long warps = static_cast<long long>(gridDim.x) * (kThreads / 32);
    const bool vec = (reinterpret_cast<uintptr_t>(src) & 15u) == 0 && (pitch * sizeof(T)) % 16 == 0;
    float inv = 1.0f;
    if (kBlock16 && tensor_scale != nullptr) {
        const float ts = __ldg(tensor_scale);
        inv = ts != 0.0f ? 1.0f / ts : 0.0f;
    }
    for (long long u0 = (blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x) / 32; u0 < total; u0 += warps * kUnroll) {
        float v[kUnroll][8];
        int row[kUnroll], col[kUnroll];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            const long long u = u0 + i * warps;
            row[i] = u < total ? static_cast<int>(u / chunks) : rows_padded;
            col[i] = static_cast<int>(u - static_cast<long long>(u / chunks) * chunks) * 256 + lane * 8;
            if (row[i] < rows && col[i] < k) {
                load8(src + row[i] * pitch + col[i], vec, v[i]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            if (row[i] >= rows_padded) break;  // (uniform over the warp)
            const bool live = row[i] < rows && col[i] < k;
            uint32_t top = 0;  // |x| as bits: orders like the values, infinities and NaNs on top
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (kBlock16) v[i][e] *= inv;
                top = max(top, __float_as_uint(v[i][e]) & 0x7FFFFFFFu);
            }
#pragma unroll
            for (int d = 1; d < kLanes; d *= 2) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
            uint32_t byte;
            if constexpr (kBlock16) {
                // amax / 6 cut short with its last bit set when anything was lost (round to odd): 24 such bits
                // round to e4m3's 4 as the exact quotient does.
                const float a = __uint_as_float(top);
                float q = __fdiv_rz(a, 6.0f);
                if (fmaf(-q, 6.0f, a) != 0.0f) q = __uint_as_float(__float_as_uint(q) | 1u);
                byte = to_e4m3(q);
                const float s = from_e4m3(byte);
                // x / s correctly rounded from a correctly rounded reciprocal and one residual step
                // (Markstein, "Computation of elementary functions on the IBM RISC System/6000", 1990).  No
                // rounding of it lands on a tie that the exact quotient misses: a tie times s has at most 7 bits,
                // so it is itself a float, and the quotients of its neighbours are at least an ulp away.
                const float r = s > 0.0f ? __frcp_rn(s) : 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float q0 = v[i][e] * r;
                    v[i][e] = copysignf(fmaf(fmaf(-q0, s, v[i][e]), r, q0), v[i][e]);  // (the residual step loses the sign of -0)
                }
                if (top >= 0x7F800000u) byte = 0x7Fu;
            } else {
                const int e8 = max(static_cast<int>(top >> 23) - 2, 0);
                byte = static_cast<uint32_t>(e8);
                // 2^(127 - e8), from 2^127 down to 2^-125: exact, and normal wherever a value survives
                const float r = __uint_as_float(static_cast<uint32_t>(254 - e8) << 23);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[i][e] *= r;
                if (top >= 0x7F800000u) byte = 0xFFu;
            }
            if (!live) byte = 0;
            if (live) reinterpret_cast<uint32_t*>(codes)[(static_cast<size_t>(row[i]) * k + col[i]) / 8] = to_e2m1x8(v[i]);
            // Four neighbouring scales -> one word.
            uint32_t word = byte;
            word |= __shfl_down_sync(0xFFFFFFFFu, byte, kLanes) << 8;
            word |= __shfl_down_sync(0xFFFFFFFFu, byte, 2 * kLanes) << 16;
            word |= __shfl_down_sync(0xFFFFFFFFu, byte, 3 * kLanes) << 24;
            const int kt = col[i] / (4 * kLanes * 8);
            if (lane % (4 * kLanes) == 0 && kt < ktiles)
                *reinterpret_cast<uint32_t*>(scales + fp4_scale_word(row[i], kt, ktiles)) = word;
        }
    }
}

// Eight codes and their scale -> eight values per thread.
template <int kType, bool kBlock16>
__global__ void __launch_bounds__(kThreads)
fp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const float* __restrict__ tensor_scale,
                      int apply_tensor_scale, typename Src<kType>::T* __restrict__ dst, int rows, int k)
{
    using T = typename Src<kType>::T;
    const int words = k / 8;
    const int ktiles = fp4_ktiles(k, kBlock16);
    const long long total = static_cast<long long>(rows) * words;
    const long long stride = static_cast<long long>(gridDim.x) * kThreads;
    float ts = tensor_scale != nullptr ? __ldg(tensor_scale) : 1.0f;
    // Operands of the gradient products keep the tensor scale out (their epilogue applies it), but a matrix
    // whose tensor scale is 0 is 0 there too.
    if (!apply_tensor_scale) ts = ts == 0.0f ? 0.0f : 1.0f;
    for (long long i0 = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x; i0 < total; i0 += stride * kUnroll) {
        uint32_t word[kUnroll];
        uint32_t byte[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long long i = i0 + u * stride;
            if (i < total) {
                const int row = static_cast<int>(i / words), col = static_cast<int>(i - static_cast<long long>(row) * words) * 8;
                const int blk = col / (kBlock16 ? 16 : 32);
                word[u] = __ldg(reinterpret_cast<const uint32_t*>(codes) + i);
                byte[u] = __ldg(scales + fp4_scale_word(row, blk >> 2, ktiles) + (blk & 3));
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const long long i = i0 + u * stride;
            if (i >= total) break;
            float s;
            if constexpr (kBlock16) {
                s = from_e4m3(byte[u]);  // 0x7F converts to NaN
            } else {
                // 2^(b - 127); 2^-127 is subnormal
                s = byte[u] == 0xFFu ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float(byte[u] ? byte[u] << 23 : 0x00400000u);
            }
            __align__(16) T out[8];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                uint32_t h2;
                asm("{\n\t.reg .b8 c;\n\tcvt.u8.u32 c, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, c;\n\t}\n" : "=r"(h2) : "r"((word[u] >> (8 * b)) & 0xFFu));
                const float lo = __half2float(__ushort_as_half(static_cast<unsigned short>(h2 & 0xFFFFu)));
                const float hi = __half2float(__ushort_as_half(static_cast<unsigned short>(h2 >> 16)));
                if constexpr (kType == INT4L_TYPE_BF16) {
                    out[2 * b] = __float2bfloat16_rn(lo * s * ts);
                    out[2 * b + 1] = __float2bfloat16_rn(hi * s * ts);
                } else if constexpr (kType == INT4L_TYPE_F16) {
                    out[2 * b] = __float2half_rn(lo * s * ts);
                    out[2 * b + 1] = __float2half_rn(hi * s * ts);
                } else {
                    out[2 * b] = lo * s * ts;
                    out[2 * b + 1] = hi * s * ts;
                }
            }
            uint4* d = reinterpret_cast<uint4*>(dst + i * 8);
#pragma unroll
            for (int q = 0; q < static_cast<int>(sizeof(T)) / 2; ++q) d[q] = reinterpret_cast<const uint4*>(out)[q];
        }
    }
}

// Enough blocks to fill the GPU a few times over, fewer when there is less to do.
int grid_for(const DeviceCtx* ctx, long long units_per_block_pass, long long units)
{
    const long long want = (units + units_per_block_pass - 1) / units_per_block_pass;
    const long long cap = static_cast<long long>(ctx->sm_count) * 16;
    return static_cast<int>(want < 1 ? 1 : (want < cap ? want : cap));
}

template <int kType>
int quantize_typed(DeviceCtx* ctx, const void* src, long long pitch, const Fp4& d, cudaStream_t stream)
{
    using T = typename Src<kType>::T;
    const long long units = static_cast<long long>((d.rows + 127ll) / 128 * 128) * ((d.k + 255) / 256);
    const int grid = grid_for(ctx, kThreads / 32, units);
    uint8_t* codes = const_cast<uint8_t*>(d.codes);
    uint8_t* scales = const_cast<uint8_t*>(d.scales);
    if (d.block16)
        fp4_quantize_kernel<kType, true><<<grid, kThreads, 0, stream>>>(static_cast<const T*>(src), pitch, codes, scales, d.tensor_scale, d.rows, d.k);
    else
        fp4_quantize_kernel<kType, false><<<grid, kThreads, 0, stream>>>(static_cast<const T*>(src), pitch, codes, scales, d.tensor_scale, d.rows, d.k);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? INT4L_OK : INT4L_ERR_CUDA;
}

template <int kType>
int dequantize_typed(DeviceCtx* ctx, const Fp4& s, void* dst, bool apply, cudaStream_t stream)
{
    using T = typename Src<kType>::T;
    const int grid = grid_for(ctx, kThreads * kUnroll, static_cast<long long>(s.rows) * (s.k / 8));
    if (s.block16)
        fp4_dequantize_kernel<kType, true><<<grid, kThreads, 0, stream>>>(s.codes, s.scales, s.tensor_scale, apply, static_cast<T*>(dst), s.rows, s.k);
    else
        fp4_dequantize_kernel<kType, false><<<grid, kThreads, 0, stream>>>(s.codes, s.scales, s.tensor_scale, apply, static_cast<T*>(dst), s.rows, s.k);
    count_launch();
    return cudaGetLastError() == cudaSuccess ? INT4L_OK : INT4L_ERR_CUDA;
}

}  // namespace

int launch_fp4_quantize(DeviceCtx* ctx, const void* src, int src_type, long long src_pitch, const Fp4& dst, cudaStream_t stream)
{
    switch (src_type) {
        case INT4L_TYPE_BF16: return quantize_typed<INT4L_TYPE_BF16>(ctx, src, src_pitch, dst, stream);
        case INT4L_TYPE_F16: return quantize_typed<INT4L_TYPE_F16>(ctx, src, src_pitch, dst, stream);
        default: return quantize_typed<INT4L_TYPE_F32>(ctx, src, src_pitch, dst, stream);
    }
}

int launch_fp4_dequantize(DeviceCtx* ctx, const Fp4& src, void* dst, int dst_type, bool apply_tensor_scale, cudaStream_t stream)
{
    switch (dst_type) {
        case INT4L_TYPE_BF16: return dequantize_typed<INT4L_TYPE_BF16>(ctx, src, dst, apply_tensor_scale, stream);
        case INT4L_TYPE_F16: return dequantize_typed<INT4L_TYPE_F16>(ctx, src, dst, apply_tensor_scale, stream);
        default: return dequantize_typed<INT4L_TYPE_F32>(ctx, src, dst, apply_tensor_scale, stream);
    }
}

}  // namespace i4l
