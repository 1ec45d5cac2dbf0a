// Launch interfaces of the training operators: the vocabulary cross entropy (loss.hip, loss_mid.hip, loss_few.hip), the
// head's RMS norm (norm.hip), the norms around a residual block (residual.hip), AdamW and the gradients' norm
// (optim.hip) and the embedding table (table.hip), all on caller-owned device tensors.
#pragma once

#include "common.h"

namespace adn {

// Element types of the training operators' tensors (ADN_T_F32, ADN_T_BF16).
template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    return (float)v;
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    return (T)v;  // one rounding, to nearest even
}

inline int elem_bytes(uint32_t dtype) { return dtype == ADN_T_F32 ? 4 : 2; }

// Rows of `d` elements at `stride` elements, 16 bytes at a time: both the base and the stride allow
// it and a row is whole 16-byte pieces.
inline bool rows_vec16(const void *p, long stride, int d, int eb) {
    return ((uintptr_t)p % 16 == 0) && (stride * eb) % 16 == 0 && ((long)d * eb) % 16 == 0;
}

// f(T{}) for the tensors' element type
template <typename F>
void dispatch_type(uint32_t dtype, F &&f) {
    if (dtype == ADN_T_F32)
        f(float{});
    else
        f(__bf16{});
}

// ---- vocabulary cross entropy (loss.hip) ---------------------------------------------------
struct LossParams {
    int rows, d, vocab;
    uint32_t dtype;
    const void *x;
    long x_stride;
    const void *w;
    long w_stride;
    const float *bias;       // [vocab] or null
    const int32_t *targets;  // [rows], negative = no target
    const float *dloss;      // [rows] or null = 1
    float *loss, *lse;       // [rows], loss null: not wanted
    void *dx;
    long dx_stride;
    void *dw;
    long dw_stride;
    float *db;
    unsigned *err;
};
// Workspace of a call, in bytes, and the launches, which lay it out the same way.
size_t loss_workspace_bytes(const LossParams &p);
void launch_loss(const LossParams &p, void *ws, hipStream_t st);
// A few rows and small problems (loss_few.hip); the others go through the products of loss.hip.
bool loss_few_ok(const LossParams &p);
size_t loss_few_workspace_bytes(const LossParams &p);
void launch_loss_few(const LossParams &p, void *ws, hipStream_t st);

// Up to 64 rows that W's bytes bound (loss_mid.hip).
bool loss_mid_ok(const LossParams &p);
size_t loss_mid_workspace_bytes(const LossParams &p);
void launch_loss_mid(const LossParams &p, void *ws, hipStream_t st);

// ---- RMS norm of rows (norm.hip) -----------------------------------------------------------
struct NormParams {
    int rows, d;
    uint32_t dtype;
    const void *x;
    long x_stride;
    const float *gain;  // [d] or null = 1
    float eps;
    void *y;            // forward
    long y_stride;
    const void *dy;     // backward
    long dy_stride;
    void *dx;           // or null
    long dx_stride;
    float *dg;          // [d] or null
};
size_t norm_backward_workspace_bytes(const NormParams &p);
void launch_norm(const NormParams &p, hipStream_t st);
void launch_norm_backward(const NormParams &p, void *ws, hipStream_t st);

// ---- norms around a residual block (residual.hip) -------------------------------------------
struct ResidualParams {
    int rows, d;
    uint32_t dtype;
    uint32_t gate_kind;      // ADN_GATE_*
    bool sigmoid, post;      // the gate is given as logits; f is normed
    float keep, scale, eps;
    const void *x, *f, *gate;
    long x_stride, f_stride, gate_stride;
    const float *post_gain, *pre_gain;  // [d] or null = 1
    void *z, *y;             // forward: y null: not wanted; backward: z is read
    long z_stride, y_stride;
    const void *dz, *dy;     // backward: one of them may be null = 0
    long dz_stride, dy_stride;
    void *dx, *df, *dgate;   // each null: not wanted
    long dx_stride, df_stride, dgate_stride;
    float *dpost, *dpre;
};
void launch_residual(const ResidualParams &p, hipStream_t st);
size_t residual_backward_workspace_bytes(const ResidualParams &p);
void launch_residual_backward(const ResidualParams &p, void *ws, hipStream_t st);

// ---- AdamW over a list of tensors (optim.hip) ----------------------------------------------
struct OptTensor {  // one tensor of the list
    float *param;
    const void *grad;
    __bf16 *copy;            // or null
    void *m, *v;             // fp32, or e4m3 codes
    float *m_scale, *v_scale;
    int64_t n;
    int64_t block;           // the list's number of its first block of 256 values
    float lr_scale, decay;
    uint32_t grad_bf16;
    uint32_t pad;
};
struct OptChunk {  // a share of a tensor
    int32_t tensor, chunk;
};
struct OptPlan {  // the list as it stands on the device
    const OptTensor *tensors;
    const OptChunk *step_chunks, *norm_chunks;  // a workgroup's of the step, a wave's of the norm
    int n_step_chunks, step_values, n_norm_chunks, norm_values;
    int state_bits;
    bool streams;            // a step reads and writes past the caches
    double beta1, beta2, log_beta1, log_beta2;
    float eps;
    uint64_t seed;
    int32_t *step;
    double *partials;        // [OPT_NORM_BLOCKS]
    unsigned *ticket;        // [1 + OPT_TICKETS] at OPT_TICKET_PITCH, zero between calls
};
struct OptStep {
    double lr;
    const float *lr_device, *grad_norm;  // or null
    float max_norm, grad_scale;
};
constexpr int OPT_BLOCK = 256;         // values of an 8-bit state that share a scale
constexpr int OPT_NORM_BLOCKS = 512;   // most workgroups of the norm
constexpr int OPT_TICKETS = 32, OPT_TICKET_PITCH = 64;  // places at which workgroups count themselves, 256 bytes apart
int opt_step_values(int64_t total, bool eight);
int opt_norm_values(int64_t total);
void launch_grad_norm(const OptPlan &p, float *norm, hipStream_t st);
void launch_adamw(const OptPlan &p, const OptStep &s, hipStream_t st);

// ---- embedding table (table.hip) -----------------------------------------------------------
struct TableParams {
    int n, d, vocab;
    uint32_t dtype;
    const int32_t *tokens;  // [n], negative = none
    float scale;
    const void *src;        // lookup: the table [vocab] rows; gradient: dout [n] rows
    long src_stride;
    void *dst;              // lookup: out [n] rows; gradient: the table's gradient [vocab] rows
    long dst_stride;
    unsigned *err;
};
void launch_embed_lookup(const TableParams &p, hipStream_t st);
size_t embed_grad_workspace_bytes(const TableParams &p);
void launch_embed_grad(const TableParams &p, void *ws, hipStream_t st);

}  // namespace adn
