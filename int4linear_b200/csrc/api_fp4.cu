// C-ABI layer of the microscaled 4-bit floating-point operators (include/int4linear_b200.h): argument checks,
// workspace layout of the backward passes, and the order of their launches.
#include "fp4.cuh"

using namespace i4l;

namespace {

bool misaligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

int take_matrix(const int4_linear_fp4_matrix* q, Fp4* out)
{
    if (!q || !q->codes || !q->scales || q->rows <= 0 || q->k <= 0) return INT4L_ERR_INVALID_ARG;
    if (q->format != INT4L_FP4_MX && q->format != INT4L_FP4_NV) return INT4L_ERR_INVALID_ARG;
    if (q->format == INT4L_FP4_MX && q->tensor_scale) return INT4L_ERR_INVALID_ARG;
    if (q->k % 32 != 0) return INT4L_ERR_UNSUPPORTED;
    if (q->rows > INT4L_FP4_MAX_EXTENT || q->k > INT4L_FP4_MAX_EXTENT) return INT4L_ERR_TOO_LARGE;
    if (misaligned(q->codes, 16) || misaligned(q->scales, 16) || misaligned(q->tensor_scale, 4)) return INT4L_ERR_MISALIGNED;
    out->codes = static_cast<const uint8_t*>(q->codes);
    out->scales = static_cast<const uint8_t*>(q->scales);
    out->tensor_scale = q->tensor_scale;
    out->rows = q->rows;
    out->k = q->k;
    out->block16 = q->format == INT4L_FP4_NV;
    return INT4L_OK;
}

int element_bytes(int type) { return type == INT4L_TYPE_F32 ? 4 : 2; }

// x[m x k] and one or two w[n x k] of one format.
int take_operands(const int4_linear_fp4_matrix* x, const int4_linear_fp4_matrix* w, const int4_linear_fp4_matrix* w_up, bool gated, Fp4Problem* p)
{
    int rc = take_matrix(x, &p->x);
    if (rc == INT4L_OK) rc = take_matrix(w, &p->w);
    if (rc == INT4L_OK && gated) rc = take_matrix(w_up, &p->w_up);
    if (rc != INT4L_OK) return rc;
    if (p->x.k != p->w.k || p->x.block16 != p->w.block16) return INT4L_ERR_INVALID_ARG;
    if (gated && (p->w_up.k != p->x.k || p->w_up.rows != p->w.rows || p->w_up.block16 != p->x.block16)) return INT4L_ERR_INVALID_ARG;
    p->gated = gated;
    p->m = p->x.rows;
    p->n = p->w.rows;
    p->k = p->x.k;
    return INT4L_OK;
}

bool bad_act(int act) { return act != INT4L_ACT_SILU && act != INT4L_ACT_GELU && act != INT4L_ACT_GELU_TANH; }

// Takes INT4L_GRAD_*_TERM(S) out of a value: 1, 2, 0 for neither, -1 for both.
int take_terms(int* value)
{
    const int flags = *value & (INT4L_GRAD_ONE_TERM | INT4L_GRAD_TWO_TERMS);
    *value &= ~flags;
    return flags == 0 ? 0 : flags == INT4L_GRAD_ONE_TERM ? 1 : flags == INT4L_GRAD_TWO_TERMS ? 2 : -1;
}

int launch_product(DeviceCtx* ctx, const Fp4Problem& p, cudaStream_t stream)
{
    return fp4_fewrows_preferred(ctx, p) ? launch_fp4_fewrows(ctx, p, stream) : launch_fp4_gemm(ctx, p, stream);
}

// The common part of both backward passes.
int run_backward(Fp4Backward& b, void* workspace_d, long long workspace_bytes, void* stream)
{
    const Fp4Problem& p = b.forward;
    if (!b.dx && !b.dw) return INT4L_ERR_INVALID_ARG;
    if (misaligned(b.dx, 16) || misaligned(b.dw, 16) || misaligned(b.dw_up, 16) || misaligned(workspace_d, 256)) return INT4L_ERR_MISALIGNED;
    const long long need = fp4_backward_workspace(p.m, p.n, p.k, p.gated, b.dx != nullptr, b.dw != nullptr, b.terms);
    if (need > 0 && (!workspace_d || workspace_bytes < need)) return INT4L_ERR_INVALID_ARG;
    int rc = INT4L_OK;
    DeviceCtx* ctx = current_ctx(&rc);
    if (!ctx) return rc;
    b.workspace = static_cast<uint8_t*>(workspace_d);
    return launch_fp4_backward(ctx, b, static_cast<cudaStream_t>(stream));
}

}  // namespace

extern "C" {

long long int4_linear_fp4_scale_bytes(int rows, int k, int format)
{
    if (rows <= 0 || k <= 0 || k % 32 != 0 || (format != INT4L_FP4_MX && format != INT4L_FP4_NV)) return -INT4L_ERR_INVALID_ARG;
    return (rows + 127ll) / 128 * fp4_ktiles(k, format == INT4L_FP4_NV) * kScaleTileBytes;
}

int int4_linear_fp4_quantize_async(const void* src_d, int src_type, long long src_pitch, const int4_linear_fp4_matrix* dst, void* stream)
{
    Fp4 d;
    int rc = take_matrix(dst, &d);
    if (rc == INT4L_OK && (!src_d || src_type < INT4L_TYPE_BF16 || src_type > INT4L_TYPE_F32 || src_pitch < d.k)) rc = INT4L_ERR_INVALID_ARG;
    if (rc == INT4L_OK && misaligned(src_d, element_bytes(src_type))) rc = INT4L_ERR_MISALIGNED;
    if (rc != INT4L_OK) return record_status(rc);
    DeviceCtx* ctx = current_ctx(&rc);
    if (ctx) rc = launch_fp4_quantize(src_d, src_type, src_pitch, d, static_cast<cudaStream_t>(stream));
    return record_status(rc);
}

int int4_linear_fp4_dequantize_async(const int4_linear_fp4_matrix* src, void* dst_d, int dst_type, void* stream)
{
    Fp4 s;
    int rc = take_matrix(src, &s);
    if (rc == INT4L_OK && (!dst_d || dst_type < INT4L_TYPE_BF16 || dst_type > INT4L_TYPE_F32)) rc = INT4L_ERR_INVALID_ARG;
    if (rc == INT4L_OK && misaligned(dst_d, 16)) rc = INT4L_ERR_MISALIGNED;
    if (rc != INT4L_OK) return record_status(rc);
    DeviceCtx* ctx = current_ctx(&rc);
    if (ctx) rc = launch_fp4_dequantize(s, dst_d, dst_type, static_cast<cudaStream_t>(stream));
    return record_status(rc);
}

int int4_linear_fp4_launch_async(const int4_linear_fp4_matrix* x, const int4_linear_fp4_matrix* w, const float* bias_d,
                                 void* y_d, int y_type, void* stream)
{
    Fp4Problem p;
    int rc = take_operands(x, w, nullptr, false, &p);
    if (rc == INT4L_OK && (!y_d || (y_type != INT4L_TYPE_BF16 && y_type != INT4L_TYPE_F16))) rc = INT4L_ERR_INVALID_ARG;
    if (rc == INT4L_OK && (misaligned(y_d, 16) || misaligned(bias_d, 4))) rc = INT4L_ERR_MISALIGNED;
    if (rc != INT4L_OK) return record_status(rc);
    DeviceCtx* ctx = current_ctx(&rc);
    if (!ctx) return record_status(rc);
    p.bias = bias_d;
    p.y = y_d;
    p.fp16 = y_type == INT4L_TYPE_F16;
    return record_status(launch_product(ctx, p, static_cast<cudaStream_t>(stream)));
}

int int4_linear_fp4_gated_launch_async(const int4_linear_fp4_matrix* x, const int4_linear_fp4_matrix* w_gate,
                                       const int4_linear_fp4_matrix* w_up, int activation, void* h_d, void* gate_d, void* up_d,
                                       int h_type, void* stream)
{
    Fp4Problem p;
    int rc = take_operands(x, w_gate, w_up, true, &p);
    if (rc == INT4L_OK && (!h_d || !gate_d != !up_d || bad_act(activation) || (h_type != INT4L_TYPE_BF16 && h_type != INT4L_TYPE_F16)))
        rc = INT4L_ERR_INVALID_ARG;
    if (rc == INT4L_OK && (misaligned(h_d, 16) || misaligned(gate_d, 16) || misaligned(up_d, 16))) rc = INT4L_ERR_MISALIGNED;
    if (rc != INT4L_OK) return record_status(rc);
    DeviceCtx* ctx = current_ctx(&rc);
    if (!ctx) return record_status(rc);
    p.act = activation;
    p.y = h_d;
    p.keep_gate = gate_d;
    p.keep_up = up_d;
    p.fp16 = h_type == INT4L_TYPE_F16;
    return record_status(launch_product(ctx, p, static_cast<cudaStream_t>(stream)));
}

long long int4_linear_fp4_grad_workspace_bytes(int m, int n, int k, int gated, int want_dx, int want_dw)
{
    const int terms = take_terms(&gated);
    if (m <= 0 || n <= 0 || k <= 0 || terms < 0) return -INT4L_ERR_INVALID_ARG;
    if (m > INT4L_FP4_MAX_EXTENT || n > INT4L_FP4_MAX_EXTENT || k > INT4L_FP4_MAX_EXTENT) return -INT4L_ERR_TOO_LARGE;
    return fp4_backward_workspace(m, n, k, gated != 0, want_dx != 0, want_dw != 0, terms);
}

int int4_linear_fp4_grad_async(const void* dy_d, const int4_linear_fp4_matrix* x, const int4_linear_fp4_matrix* w,
                               void* dx_d, void* dw_d, void* workspace_d, long long workspace_bytes, void* stream)
{
    Fp4Backward b;
    int rc = take_operands(x, w, nullptr, false, &b.forward);
    if (rc == INT4L_OK && !dy_d) rc = INT4L_ERR_INVALID_ARG;
    if (rc == INT4L_OK && misaligned(dy_d, b.forward.n % 8 == 0 ? 16 : 2)) rc = INT4L_ERR_MISALIGNED;
    if (rc != INT4L_OK) return record_status(rc);
    b.dy = dy_d;
    b.dx = dx_d;
    b.dw = dw_d;
    return record_status(run_backward(b, workspace_d, workspace_bytes, stream));
}

int int4_linear_fp4_gated_grad_async(const void* dh_d, const void* gate_d, const void* up_d, const int4_linear_fp4_matrix* x,
                                     const int4_linear_fp4_matrix* w_gate, const int4_linear_fp4_matrix* w_up, int activation,
                                     void* dx_d, void* dw_gate_d, void* dw_up_d, void* workspace_d, long long workspace_bytes,
                                     void* stream)
{
    Fp4Backward b;
    b.terms = take_terms(&activation);
    int rc = take_operands(x, w_gate, w_up, true, &b.forward);
    if (rc == INT4L_OK && (!dh_d || !gate_d || !up_d || !dw_gate_d != !dw_up_d || bad_act(activation) || b.terms < 0)) rc = INT4L_ERR_INVALID_ARG;
    if (rc == INT4L_OK && (misaligned(dh_d, 2) || misaligned(gate_d, 2) || misaligned(up_d, 2))) rc = INT4L_ERR_MISALIGNED;
    if (rc != INT4L_OK) return record_status(rc);
    b.forward.act = activation;
    b.dy = dh_d;
    b.gate = gate_d;
    b.up = up_d;
    b.dx = dx_d;
    b.dw = dw_gate_d;
    b.dw_up = dw_up_d;
    return record_status(run_backward(b, workspace_d, workspace_bytes, stream));
}

}  // extern "C"
