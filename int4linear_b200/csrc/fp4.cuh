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

// Map of a matrix's scales: one row per group of 128 matrix rows, 8-byte elements (a box has at most 256); a box takes the scale
// tiles of one step of k (`step_bytes`) from `groups` groups.
inline int fp4_scale_map(DeviceCtx* ctx, CUtensorMap* out, const Fp4& q, int step_bytes, int groups)
{
    const uint64_t row_bytes = static_cast<uint64_t>(fp4_ktiles(q.k, q.block16)) * kScaleTileBytes;
    return encode_tensor_map_2d(ctx, out, q.scales, 8, row_bytes / 8, (q.rows + 127ll) / 128, row_bytes, step_bytes / 8, groups, false);
}

enum GateAct { kActSilu = INT4L_ACT_SILU, kActGelu = INT4L_ACT_GELU, kActGeluTanh = INT4L_ACT_GELU_TANH };

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

int launch_fp4_quantize(const void* src, int src_type, long long src_pitch, const Fp4& dst, cudaStream_t stream);
int launch_fp4_dequantize(const Fp4& src, void* dst, int dst_type, cudaStream_t stream);
// Backward pass of a product or a gated product (gemm_grad.cu); x, w, w_up and m, n, k as in `forward`.
struct Fp4Backward {
    Fp4Problem forward;
    const void* dy = nullptr;             // m x n bf16: the gradient of y or h
    const void* gate = nullptr;           // gated: the kept products
    const void* up = nullptr;
    void* dx = nullptr;                   // m x k, or null
    void* dw = nullptr;                   // n x k, or null (gated: the gate's, and dw_up with it)
    void* dw_up = nullptr;
    int terms = 0;                        // gated: bf16 terms of dg and du, 1 or 2, 0 by size
    uint8_t* workspace = nullptr;         // fp4_backward_workspace() bytes, 256-byte aligned
};
long long fp4_backward_workspace(long long m, long long n, long long k, bool gated, bool want_dx, bool want_dw, int terms);
int setup_fp4_backward(DeviceCtx* ctx);
int launch_fp4_backward(DeviceCtx* ctx, const Fp4Backward& b, cudaStream_t stream);
int setup_fp4_gemm(DeviceCtx* ctx);
int launch_fp4_gemm(DeviceCtx* ctx, const Fp4Problem& p, cudaStream_t stream);
// Few rows of x (gemm_fp4_fewrows.cu).
int setup_fp4_fewrows(DeviceCtx* ctx);
bool fp4_fewrows_preferred(const DeviceCtx* ctx, const Fp4Problem& p);
int launch_fp4_fewrows(DeviceCtx* ctx, const Fp4Problem& p, cudaStream_t stream);

}  // namespace i4l
