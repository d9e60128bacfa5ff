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
// Bound: HBM.  Each element is read once (2 or 4 bytes) and written once (half a byte and 1/32 or 1/16).  Measured at
// 8192 x 8192 bf16, four calls on end: 30.7 us mxfp4 (5.5 TB/s), 38.4 us nvfp4 (4.5; its divisions), 28.5 us expansion to bf16
// (32.8 with a tensor scale).
#include "fp4_expand.cuh"

namespace i4l {

namespace {

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

// kE elements per lane: 8, or 16, a whole nvfp4 block (its scale takes as many instructions as eight elements do).  A
// block's scale is agreed on by its lanes, whose first writes the byte.  Rows are padded to 128 and scales to whole words with zeros, so that
// nothing in a scale tile is undefined.
template <int kType, bool kBlock16, int kE>
__global__ void __launch_bounds__(kUnitThreads)
fp4_quantize_kernel(const typename Src<kType>::T* __restrict__ src, long long pitch, uint8_t* __restrict__ codes,
                    uint8_t* __restrict__ scales, const float* __restrict__ tensor_scale, int rows, int k)
{
    constexpr int kLanes = (kBlock16 ? 16 : 32) / kE;  // lanes of a block
    constexpr int kH = kE / 8;
    using T = typename Src<kType>::T;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Unit<kE> u(blockIdx.x, k);
    if (u.row0 >= (rows + 127) / 128 * 128) return;  // (uniform over the warp)
    const int ktiles = fp4_ktiles(k, kBlock16);
    const bool in_k = u.col < k;
    Eight<T> v[kUnitRows][kH];
    {
        const T* p = src + u.row0 * pitch + u.col;
        const bool vec = ((reinterpret_cast<uintptr_t>(src) | (static_cast<uintptr_t>(pitch) * sizeof(T))) & 15u) == 0;
#pragma unroll
        for (int i = 0; i < kUnitRows; ++i, p += pitch) {
#pragma unroll
            for (int h = 0; h < kH; ++h) {
                v[i][h] = Eight<T>{};
                if (!in_k || u.row0 + i >= rows) continue;
                if (vec) {
#pragma unroll
                    for (int q = 0; q < static_cast<int>(sizeof(Eight<T>) / 16); ++q)
                        reinterpret_cast<uint4*>(&v[i][h])[q] = __ldg(reinterpret_cast<const uint4*>(p + 8 * h) + q);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) reinterpret_cast<T*>(&v[i][h])[e] = p[8 * h + e];
                }
            }
        }
    }
    float inv = 1.0f;
    if (kBlock16 && tensor_scale != nullptr) {
        const float ts = __ldg(tensor_scale);
        inv = ts != 0.0f ? 1.0f / ts : 0.0f;
    }
    const int block = u.col / (kE * kLanes);
    uint8_t* scale_at = scales + fp4_scale_word(u.row0, block >> 2, ktiles) + (block & 3);  // row0 % 4 == 0: the next rows' are 16 bytes on
    const bool writes_scale = (threadIdx.x & (kLanes - 1)) == 0 && block < 4 * ktiles;
    uint8_t* code_at = codes + (static_cast<size_t>(u.row0) * k + u.col) / 2;
#pragma unroll
    for (int i = 0; i < kUnitRows; ++i, code_at += k / 2) {
        const bool live = in_k && u.row0 + i < rows;
        uint32_t top = v[i][0].top();
        if constexpr (kH == 2) top = max(top, v[i][1].top());
#pragma unroll
        for (int d = 1; d < kLanes; d *= 2) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
        uint32_t byte;
        float x[kH][8];
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
            for (int e = 0; e < kE; ++e) {
                const float t = v[i][e / 8].get(e & 7) * inv;
                const float q0 = t * r;
                x[e / 8][e & 7] = copysignf(fmaf(fmaf(-q0, s, t), r, q0), t);  // (the residual step loses the sign of -0)
            }
            if (top >= 0x7F800000u) byte = 0x7Fu;
        } else {
            const int e8 = max(static_cast<int>(top >> 23) - 2, 0);
            byte = static_cast<uint32_t>(e8);
            // 2^(127 - e8), from 2^127 down to 2^-125: exact, and normal wherever a value survives
            const float r = __uint_as_float(static_cast<uint32_t>(254 - e8) << 23);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[0][e] = v[i][0].get(e) * r;
            if (top >= 0x7F800000u) byte = 0xFFu;
        }
        if (live) {
            if constexpr (kH == 2) *reinterpret_cast<uint2*>(code_at) = make_uint2(to_e2m1x8(x[0]), to_e2m1x8(x[1]));
            else *reinterpret_cast<uint32_t*>(code_at) = to_e2m1x8(x[0]);
        }
        if (writes_scale) scale_at[16 * i] = static_cast<uint8_t>(live ? byte : 0);
    }
}

template <int kType, bool kBlock16>
__global__ void __launch_bounds__(kUnitThreads)
fp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, const float* __restrict__ tensor_scale,
                      typename Src<kType>::T* __restrict__ dst, int rows, int k)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    fp4_expand_block<kType, kBlock16>(blockIdx.x, codes, scales, tensor_scale, true, dst, rows, k);
}

template <typename... P, typename... A>
int launch_units(void (*kernel)(P...), long long rows, int k, int elems, cudaStream_t stream, A... args)
{
    const long long units = rows / kUnitRows * ((k + 32ll * elems - 1) / (32 * elems)), blocks = (units + kUnitThreads / 32 - 1) / (kUnitThreads / 32);
    if (blocks > 0x1FFFFFFF) return INT4L_ERR_TOO_LARGE;  // (units are counted in 32 bits; 4 T elements)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
    cfg.blockDim = dim3(kUnitThreads, 1, 1);
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
int quantize_typed(const void* src, long long pitch, const Fp4& d, cudaStream_t stream)
{
    using T = typename Src<kType>::T;
    const long long rows = (d.rows + 127ll) / 128 * 128;
    auto launch = [&](auto kernel, int elems) {
        return launch_units(kernel, rows, d.k, elems, stream, static_cast<const T*>(src), pitch, const_cast<uint8_t*>(d.codes),
                            const_cast<uint8_t*>(d.scales), d.tensor_scale, d.rows, d.k);
    };
    if (!d.block16) return launch(fp4_quantize_kernel<kType, false, 8>, 8);
    // 16 elements per lane take fewer instructions (8192 x 8192 bf16: 36.3 us against 41.1), 8 have the shorter way
    // where the GPU is not filled anyway (16 x 4096: 2.1 us against 2.7).
    return static_cast<long long>(d.rows) * d.k >= (1 << 20) ? launch(fp4_quantize_kernel<kType, true, 16>, 16)
                                                             : launch(fp4_quantize_kernel<kType, true, 8>, 8);
}

template <int kType>
int dequantize_typed(const Fp4& s, void* dst, cudaStream_t stream)
{
    using T = typename Src<kType>::T;
    return launch_units(s.block16 ? fp4_dequantize_kernel<kType, true> : fp4_dequantize_kernel<kType, false>, (s.rows + 3ll) / 4 * 4, s.k, 8, stream,
                        s.codes, s.scales, s.tensor_scale, static_cast<T*>(dst), s.rows, s.k);
}

}  // namespace

int launch_fp4_quantize(const void* src, int src_type, long long src_pitch, const Fp4& dst, cudaStream_t stream)
{
    switch (src_type) {
        case INT4L_TYPE_BF16: return quantize_typed<INT4L_TYPE_BF16>(src, src_pitch, dst, stream);
        case INT4L_TYPE_F16: return quantize_typed<INT4L_TYPE_F16>(src, src_pitch, dst, stream);
        default: return quantize_typed<INT4L_TYPE_F32>(src, src_pitch, dst, stream);
    }
}

int launch_fp4_dequantize(const Fp4& src, void* dst, int dst_type, cudaStream_t stream)
{
    switch (dst_type) {
        case INT4L_TYPE_BF16: return dequantize_typed<INT4L_TYPE_BF16>(src, dst, stream);
        case INT4L_TYPE_F16: return dequantize_typed<INT4L_TYPE_F16>(src, dst, stream);
        default: return dequantize_typed<INT4L_TYPE_F32>(src, dst, stream);
    }
}

}  // namespace i4l
