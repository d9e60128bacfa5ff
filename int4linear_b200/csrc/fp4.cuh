// Microscaled 4-bit floating point: the format's constants, its scale order, and the launchers of its kernels.
//
// A matrix is `rows` x `k` e2m1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign bit), packed like the signed
// 4-bit integers: two per byte, low nibble = even index, row pitch k / 2 bytes.  Every `block` consecutive
// elements of a row share one scale byte:
//     mxfp4  block 32, byte b stands for 2^(b - 127) (e8m0), 0xFF for NaN
//     nvfp4  block 16, an e4m3 value, and one float for the whole matrix (tensor_scale)
// Scale bytes lie in the order in which the tensor core's scale memory is filled: tiles of 128 rows x 4 scales,
// 512 bytes, element (r, j) of a tile at byte (r % 32) * 16 + (r / 32) * 4 + j; the tiles of one group of 128
// rows follow one another along k, the groups along the rows.  So the scales of a 128-row operand tile and one
// step of k are contiguous: one bulk copy brings them in, and one tcgen05.cp per 512 bytes puts them in place.
#pragma once

#include "common.h"

namespace i4l {

constexpr int kScaleTileBytes = 512;

// A checked int4_linear_fp4_matrix.
struct Fp4 {
    const uint8_t* codes = nullptr;
    const uint8_t* scales = nullptr;
    const float* tensor_scale = nullptr;  // device, may be null (1)
    int rows = 0, k = 0;
    bool block16 = false;                 // nvfp4
};

__host__ __device__ inline int fp4_block(bool block16) { return block16 ? 16 : 32; }
// Scale tiles along k.
__host__ __device__ inline int fp4_ktiles(int k, bool block16) { return (k + 4 * fp4_block(block16) - 1) / (4 * fp4_block(block16)); }

#ifdef __CUDACC__
// Byte offset of the scale word (4 scales) of `row` in scale tile `kt`.
__device__ __forceinline__ size_t fp4_scale_word(int row, int kt, int ktiles)
{
    return (static_cast<size_t>(row >> 7) * ktiles + kt) * kScaleTileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}
#endif

enum GateAct { kActNone = -1, kActSilu = 0, kActGelu = 1, kActGeluTanh = 2 };

// One product: y = x w^T (w_up null), or h = act(x w^T) * (x w_up^T).
struct Fp4Problem {
    Fp4 x, w, w_up;
    bool gated = false;
    int act = kActSilu;
    const float* bias = nullptr;   // n floats or null (product only)
    void* y = nullptr;             // m x n 16-bit floats
    void* keep_gate = nullptr;     // m x n, both or neither (gated only)
    void* keep_up = nullptr;
    int fp16 = 0;
    int m = 0, n = 0, k = 0;
};

int launch_fp4_quantize(DeviceCtx* ctx, const void* src, int src_type, long long src_pitch, const Fp4& dst, cudaStream_t stream);
int launch_fp4_dequantize(DeviceCtx* ctx, const Fp4& src, void* dst, int dst_type, bool apply_tensor_scale, cudaStream_t stream);
// The gradient products (gemm_grad.cu), bf16 operands and result, fp32 accumulation; alpha = num / den, a null
// pointer or a 0 in den counting as 1.
//     input gradient    dx[m x k] = alpha (d0[m x n] w0[n x k] + d1 w1)    (d1 / w1 null: one product)
//     weight gradient   dw[n x k] = alpha d0[m x n]^T x[m x k]
// d0 / d1 have a row pitch of `ld` elements (a multiple of 8).
struct GradProduct {
    bool weight = false;
    const void* d0 = nullptr; const void* d1 = nullptr;
    const void* b0 = nullptr; const void* b1 = nullptr;  // w0, w1, or x
    void* out = nullptr;
    int m = 0, n = 0, k = 0;
    long long ld = 0;
    const float* num = nullptr; const float* den = nullptr;
};
int setup_grad(DeviceCtx* ctx);
int launch_grad_product(DeviceCtx* ctx, const GradProduct& p, cudaStream_t stream);
// dg = dh u act'(g) f_g, du = dh act(g) f_u as bf16 with row pitch ld; f = the tensor scale of that weight (0 counts as 1).
int launch_gate_backward(DeviceCtx* ctx, const void* dh, const void* gate, const void* up, void* dg, void* du, int act,
                         const float* f_g, const float* f_u, int m, int n, long long ld, cudaStream_t stream);
int setup_fp4_gemm(DeviceCtx* ctx);
int launch_fp4_gemm(DeviceCtx* ctx, const Fp4Problem& p, cudaStream_t stream);
// Few rows of x (gemm_fp4_fewrows.cu).
int setup_fp4_fewrows(DeviceCtx* ctx);
bool fp4_fewrows_supports(const Fp4Problem& p);
int launch_fp4_fewrows(DeviceCtx* ctx, const Fp4Problem& p, cudaStream_t stream);

}  // namespace i4l
