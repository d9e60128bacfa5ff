// Expansion of microscaled codes into floats (fp4.cuh), as a device function: it is a kernel of its own
// (fp4_quant.cu) and part of the preparation of a backward pass (gemm_grad.cu).
#pragma once

#include "epilogue.cuh"
#include "fp4.cuh"

namespace i4l {

constexpr int kUnitThreads = 256;
constexpr int kUnitRows = 4;  // rows of a unit

template <int kType> struct Src;
template <> struct Src<INT4L_TYPE_BF16> { using T = __nv_bfloat16; };
template <> struct Src<INT4L_TYPE_F16> { using T = __half; };
template <> struct Src<INT4L_TYPE_F32> { using T = float; };

__device__ __forceinline__ float from_e4m3(uint32_t byte)
{
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(byte)));
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h2 & 0xFFFFu)));
}

// The value of a scale byte, NaN included.
template <bool kBlock16>
__device__ __forceinline__ float fp4_scale(uint32_t byte)
{
    if constexpr (kBlock16) return from_e4m3(byte);  // 0x7F converts to NaN
    // 2^(b - 127); 2^-127 is subnormal
    return byte == 0xFFu ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// Eight codes -> eight halves.
__device__ __forceinline__ void fp4_codes_to_halves(uint32_t word, uint32_t (&h2)[4])
{
    asm("{\n\t"
        ".reg .b8 c0, c1, c2, c3;\n\t"
        "mov.b32 {c0, c1, c2, c3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, c0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, c1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, c3;\n\t"
        "}\n" : "=r"(h2[0]), "=r"(h2[1]), "=r"(h2[2]), "=r"(h2[3]) : "r"(word));
}

// a b in fp32.  kOdd: rounded to odd (cut off, the last bit set where something was cut), so that rounding the result to 16 bits
// rounds the product once: a product beside a tie does not land on it.  (A remainder below 2^-150 is lost, which takes a
// product below 2^-119.)  Three more instructions per value: 8192 x 8192 nvfp4 to bf16 28.7 -> 32.8 us.
template <bool kOdd>
__device__ __forceinline__ float times(float a, float b)
{
    if constexpr (!kOdd) return a * b;
    const float p = __fmul_rz(a, b);
    // (a NaN remainder comes with an infinite or NaN product, which stays as it is)
    return fabsf(fmaf(a, b, -p)) > 0.0f ? __uint_as_float(__float_as_uint(p) | 1u) : p;
}

// A warp's unit: 32 kE consecutive elements (kE per lane) of four consecutive rows.  Both kernels were first bound by
// instructions, most of them addresses: with a row of its own per step they took 143 (mxfp4), 236 (nvfp4) and 116
// (expansion) instructions for eight elements; a unit's rows share the address arithmetic.
template <int kE>
struct Unit {
    int row0, col;
    __device__ __forceinline__ Unit(uint32_t block, int k)
    {
        const uint32_t u = block * (kUnitThreads / 32) + threadIdx.x / 32, chunks = (k + 32u * kE - 1) / (32u * kE);
        const uint32_t group = u / chunks;
        row0 = static_cast<int>(group * kUnitRows);
        col = static_cast<int>((u - group * chunks) * (32 * kE) + (threadIdx.x & 31) * kE);
    }
};

// The units of one block: eight codes and their scale -> eight values per lane and row.
template <int kType, bool kBlock16>
__device__ __forceinline__ void fp4_expand_block(uint32_t block_index, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                 const float* __restrict__ tensor_scale, bool apply_tensor_scale,
                                                 typename Src<kType>::T* __restrict__ dst, int rows, int k)
{
    using T = typename Src<kType>::T;
    const Unit<8> u(block_index, k);
    if (u.row0 >= rows || u.col >= k) return;
    const int block = u.col / (kBlock16 ? 16 : 32);
    const uint8_t* scale_at = scales + fp4_scale_word(u.row0, block >> 2, fp4_ktiles(k, kBlock16)) + (block & 3);
    const size_t first = static_cast<size_t>(u.row0) * k + u.col;
    uint32_t word[kUnitRows], byte[kUnitRows];
    {
        const uint8_t* p = codes + first / 2;
#pragma unroll
        for (int i = 0; i < kUnitRows; ++i, p += k / 2) {
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
    for (int i = 0; i < kUnitRows; ++i, d += k) {
        if (u.row0 + i >= rows) break;
        const float s = fp4_scale<kBlock16>(byte[i]);
        const bool scaled = kBlock16 && ts != 1.0f;
        uint32_t h2[4];
        fp4_codes_to_halves(word[i], h2);
        __align__(16) T out[8];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&h2[b]));
            float lo = c.x * s, hi = c.y * s;  // exact
            if (scaled) { lo = times<kType != INT4L_TYPE_F32>(lo, ts); hi = times<kType != INT4L_TYPE_F32>(hi, ts); }
            if constexpr (kType == INT4L_TYPE_BF16) reinterpret_cast<uint32_t*>(out)[b] = pack16<false>(lo, hi);
            else if constexpr (kType == INT4L_TYPE_F16) reinterpret_cast<uint32_t*>(out)[b] = pack16<true>(lo, hi);
            else { out[2 * b] = lo; out[2 * b + 1] = hi; }
        }
#pragma unroll
        for (int q = 0; q < static_cast<int>(sizeof(T)) / 2; ++q) reinterpret_cast<uint4*>(d)[q] = reinterpret_cast<const uint4*>(out)[q];
    }
}

// Blocks that expand a rows x k matrix.
inline long long fp4_expand_blocks(int rows, int k) { return ((rows + 3ll) / 4 * ((k + 255) / 256) + kUnitThreads / 32 - 1) / (kUnitThreads / 32); }

}  // namespace i4l
