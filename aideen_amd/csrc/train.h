// Launch interfaces of the training operators (loss.hip, norm.hip, table.hip): the vocabulary
// cross entropy, the head's RMS norm and the embedding table, all on caller-owned device tensors.
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
