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
#include "epilogue.cuh"
#include "fp4.cuh"

namespace i4l {

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // rows of a unit

template <int kType> struct Src;
template <> struct Src<INT4L_TYPE_BF16> { using T = __nv_bfloat16; };
template <> struct Src<INT4L_TYPE_F16> { using T = __half; };
template <> struct Src<INT4L_TYPE_F32> { using T = float; };

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

// Eight source elements and the largest magnitude among them as float bits (infinities and NaNs on top).
template <typename T> struct Eight;
template <> struct Eight<float> {
    float v[8];
    __device__ __forceinline__ float get(int e) const { return v[e]; }
    __device__ __forceinline__ uint32_t top() const
    {
        uint32_t t = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) t = max(t, __float_as_uint(v[e]) & 0x7FFFFFFFu);
        return t;
    }
};
template <> struct Eight<__nv_bfloat16> {
    uint32_t w[4];
    __device__ __forceinline__ float get(int e) const { return __uint_as_float((e & 1) ? w[e / 2] & 0xFFFF0000u : w[e / 2] << 16); }
    __device__ __forceinline__ uint32_t top() const
    {
        auto mag = [&](int i) { const uint32_t a = w[i] & 0x7FFF7FFFu; return *reinterpret_cast<const __nv_bfloat162*>(&a); };
        const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(mag(0), mag(1)), __hmax2_nan(mag(2), mag(3)));
        const uint32_t b = *reinterpret_cast<const uint32_t*>(&m);
        return max(b << 16, b & 0xFFFF0000u);
    }
};
template <> struct Eight<__half> {
    uint32_t w[4];
    __device__ __forceinline__ float get(int e) const
    {
        return __half2float(__ushort_as_half(static_cast<unsigned short>((e & 1) ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu)));
    }
    __device__ __forceinline__ uint32_t top() const
    {
        auto mag = [&](int i) { const uint32_t a = w[i] & 0x7FFF7FFFu; return *reinterpret_cast<const __half2*>(&a); };
        const __half2 m = __hmax2_nan(__hmax2_nan(mag(0), mag(1)), __hmax2_nan(mag(2), mag(3)));
        return max(__float_as_uint(__low2float(m)) & 0x7FFFFFFFu, __float_as_uint(__high2float(m)) & 0x7FFFFFFFu);
    }
};

// A warp's unit: 256 consecutive elements (eight per lane) of four consecutive rows.  Both kernels were first bound by
// instructions, most of them addresses: with a row of its own per step they took 143 (mxfp4), 236 (nvfp4) and 116
// (expansion) instructions for eight elements; a unit's rows share the address arithmetic.
struct Unit {
    int row0, col;
    __device__ __forceinline__ explicit Unit(int k)
    {
        const uint32_t u = blockIdx.x * (kThreads / 32) + threadIdx.x / 32, chunks = (k + 255u) / 256u;
        const uint32_t group = u / chunks;
        row0 = static_cast<int>(group * kUnroll);
        col = static_cast<int>((u - group * chunks) * 256 + (threadIdx.x & 31) * 8);
    }
};

// A lane's loads are 16 (or 32) bytes, the warp's code store 128, and a block's scale is agreed on by 4 (mxfp4) or 2
// (nvfp4) lanes, whose first writes the byte.  Rows are padded to 128 and scales to whole words with zeros, so that
// nothing in a scale tile is undefined.
template <int kType, bool kBlock16>
__global__ void __launch_bounds__(kThreads)
fp4_quantize_kernel(const typename Src<kType>::T* __restrict__ src, long long pitch, uint8_t* __restrict__ codes,
                    uint8_t* __restrict__ scales, const float* __restrict__ tensor_scale, int rows, int k)
{
    constexpr int kLanes = kBlock16 ? 2 : 4;  // lanes of a block
    using T = typename Src<kType>::T;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Unit u(k);
    if (u.row0 >= (rows + 127) / 128 * 128) return;  // (uniform over the warp)
    const int ktiles = fp4_ktiles(k, kBlock16);
    const bool in_k = u.col < k;
    Eight<T> v[kUnroll];
    {
        const T* p = src + u.row0 * pitch + u.col;
        const bool vec = ((reinterpret_cast<uintptr_t>(src) | (static_cast<uintptr_t>(pitch) * sizeof(T))) & 15u) == 0;
#pragma unroll
        for (int i = 0; i < kUnroll; ++i, p += pitch) {
            v[i] = Eight<T>{};
            if (!in_k || u.row0 + i >= rows) continue;
            if (vec) {
#pragma unroll
                for (int q = 0; q < static_cast<int>(sizeof(v[i]) / 16); ++q) reinterpret_cast<uint4*>(&v[i])[q] = __ldg(reinterpret_cast<const uint4*>(p) + q);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) reinterpret_cast<T*>(&v[i])[e] = p[e];
            }
        }
    }
    float inv = 1.0f;
    if (kBlock16 && tensor_scale != nullptr) {
        const float ts = __ldg(tensor_scale);
        inv = ts != 0.0f ? 1.0f / ts : 0.0f;
    }
    const int block = u.col / (8 * kLanes);
    uint8_t* scale_at = scales + fp4_scale_word(u.row0, block >> 2, ktiles) + (block & 3);  // row0 % 4 == 0: the next rows' are 16 bytes on
    const bool writes_scale = (threadIdx.x & (kLanes - 1)) == 0 && block < 4 * ktiles;
    uint8_t* code_at = codes + (static_cast<size_t>(u.row0) * k + u.col) / 2;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i, code_at += k / 2) {
        const bool live = in_k && u.row0 + i < rows;
        uint32_t top = v[i].top();
#pragma unroll
        for (int d = 1; d < kLanes; d *= 2) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        uint32_t byte;
        float x[8];
        if constexpr (kBlock16) {
            // Rounding is monotonic: the largest product is the product of the largest.
            top = __float_as_uint(__uint_as_float(top) * inv) & 0x7FFFFFFFu;
            // amax / 6, rounded to odd: with its last bit set where it is not exact, and on the exact quotient's side
            // of every float with a trailing zero bit.  (The product errs by at most 1.5 ulp, and the quotients
            // next to a tie between two e4m3 values lie at least 2/3 ulp from it, so stepping back once is enough.)
            // 24 such bits round to e4m3's 4 as the exact quotient does.
            const float a = __uint_as_float(top);
            const float q = a * (1.0f / 6.0f);
            const float rest = fmaf(-q, 6.0f, a);
            uint32_t odd = __float_as_uint(q) - (rest < 0.0f ? 1u : 0u);
            if (rest != 0.0f) odd |= 1u;
            byte = to_e4m3(__uint_as_float(odd));
            const float s = from_e4m3(byte);
            // x / s: a quotient from the approximate reciprocal and one residual step (Markstein, "Computation of
            // elementary functions on the IBM RISC System/6000", 1990).  A tie between two codes times s has at most
            // 7 bits, so it is itself a float, whose quotient comes out exact; the quotients of its neighbours lie
            // at least 1/1.875 = 0.53 ulp from the tie and are not rounded onto it.
            const float r = s > 0.0f ? __fdividef(1.0f, s) : 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float t = v[i].get(e) * inv;
                const float q0 = t * r;
                x[e] = copysignf(fmaf(fmaf(-q0, s, t), r, q0), t);  // (the residual step loses the sign of -0)
            }
            if (top >= 0x7F800000u) byte = 0x7Fu;
        } else {
            const int e8 = max(static_cast<int>(top >> 23) - 2, 0);
            byte = static_cast<uint32_t>(e8);
            // 2^(127 - e8), from 2^127 down to 2^-125: exact, and normal wherever a value survives
            const float r = __uint_as_float(static_cast<uint32_t>(254 - e8) << 23);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = v[i].get(e) * r;
            if (top >= 0x7F800000u) byte = 0xFFu;
        }
        if (live) *reinterpret_cast<uint32_t*>(code_at) = to_e2m1x8(x);
        if (writes_scale) scale_at[16 * i] = static_cast<uint8_t>(live ? byte : 0);
    }
}

// The same units: eight codes and their scale -> eight values per lane and row.
template <int kType, bool kBlock16>
__global__ void __launch_bounds__(kThreads)
fp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const float* __restrict__ tensor_scale,
                      int apply_tensor_scale, typename Src<kType>::T* __restrict__ dst, int rows, int k)
{
    using T = typename Src<kType>::T;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Unit u(k);
    if (u.row0 >= rows || u.col >= k) return;
    const int block = u.col / (kBlock16 ? 16 : 32);
    const uint8_t* scale_at = scales + fp4_scale_word(u.row0, block >> 2, fp4_ktiles(k, kBlock16)) + (block & 3);
    const size_t first = static_cast<size_t>(u.row0) * k + u.col;
    uint32_t word[kUnroll], byte[kUnroll];
    {
        const uint8_t* p = codes + first / 2;
#pragma unroll
        for (int i = 0; i < kUnroll; ++i, p += k / 2) {
            if (u.row0 + i >= rows) break;
            word[i] = __ldg(reinterpret_cast<const uint32_t*>(p));
            byte[i] = __ldg(scale_at + 16 * i);
        }
    }
    float ts = tensor_scale != nullptr ? __ldg(tensor_scale) : 1.0f;
    // Operands of the gradient products keep the tensor scale out (their epilogue applies it), but a matrix
    // whose tensor scale is 0 is 0 there too.
    if (!apply_tensor_scale) ts = ts == 0.0f ? 0.0f : 1.0f;
    T* d = dst + first;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i, d += k) {
        if (u.row0 + i >= rows) break;
        float s;
        if constexpr (kBlock16) {
            s = from_e4m3(byte[i]);  // 0x7F converts to NaN
        } else {
            // 2^(b - 127); 2^-127 is subnormal
            s = byte[i] == 0xFFu ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float(byte[i] ? byte[i] << 23 : 0x00400000u);
        }
        const bool scaled = kBlock16 && ts != 1.0f;
        uint32_t h2[4];  // the codes as eight halves
        asm("{\n\t"
            ".reg .b8 c0, c1, c2, c3;\n\t"
            "mov.b32 {c0, c1, c2, c3}, %4;\n\t"
            "cvt.rn.f16x2.e2m1x2 %0, c0;\n\t"
            "cvt.rn.f16x2.e2m1x2 %1, c1;\n\t"
            "cvt.rn.f16x2.e2m1x2 %2, c2;\n\t"
            "cvt.rn.f16x2.e2m1x2 %3, c3;\n\t"
            "}\n" : "=r"(h2[0]), "=r"(h2[1]), "=r"(h2[2]), "=r"(h2[3]) : "r"(word[i]));
        __align__(16) T out[8];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&h2[b]));
            float lo = c.x * s, hi = c.y * s;  // exact
            if (scaled) { lo *= ts; hi *= ts; }
            if constexpr (kType == INT4L_TYPE_BF16) reinterpret_cast<uint32_t*>(out)[b] = pack16<false>(lo, hi);
            else if constexpr (kType == INT4L_TYPE_F16) reinterpret_cast<uint32_t*>(out)[b] = pack16<true>(lo, hi);
            else { out[2 * b] = lo; out[2 * b + 1] = hi; }
        }
#pragma unroll
        for (int q = 0; q < static_cast<int>(sizeof(T)) / 2; ++q) reinterpret_cast<uint4*>(d)[q] = reinterpret_cast<const uint4*>(out)[q];
    }
}

template <typename... P, typename... A>
int launch_units(DeviceCtx* ctx, void (*kernel)(P...), long long rows, int k, cudaStream_t stream, A... args)
{
    const long long units = rows / kUnroll * ((k + 255) / 256), blocks = (units + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x1FFFFFFF) return INT4L_ERR_TOO_LARGE;  // (units are counted in 32 bits; 4 T elements)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    count_launch();
    if (e != cudaSuccess) { cudaGetLastError(); return INT4L_ERR_CUDA; }
    return INT4L_OK;
}

template <int kType>
int quantize_typed(DeviceCtx* ctx, const void* src, long long pitch, const Fp4& d, cudaStream_t stream)
{
    using T = typename Src<kType>::T;
    return launch_units(ctx, d.block16 ? fp4_quantize_kernel<kType, true> : fp4_quantize_kernel<kType, false>, (d.rows + 127ll) / 128 * 128, d.k, stream,
                        static_cast<const T*>(src), pitch, const_cast<uint8_t*>(d.codes), const_cast<uint8_t*>(d.scales), d.tensor_scale, d.rows, d.k);
}

template <int kType>
int dequantize_typed(DeviceCtx* ctx, const Fp4& s, void* dst, bool apply, cudaStream_t stream)
{
    using T = typename Src<kType>::T;
    return launch_units(ctx, s.block16 ? fp4_dequantize_kernel<kType, true> : fp4_dequantize_kernel<kType, false>, (s.rows + 3ll) / 4 * 4, s.k, stream,
                        s.codes, s.scales, s.tensor_scale, static_cast<int>(apply), static_cast<T*>(dst), s.rows, s.k);
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
