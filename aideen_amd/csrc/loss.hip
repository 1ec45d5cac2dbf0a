// Softmax cross entropy of the LM head over the whole vocabulary, with its gradients, without
// keeping the logits:
//
//   z = x W^T + b,  lse_i = log sum_v exp(z_iv),  loss_i = lse_i - z_i,t(i)
//   dz_iv = g_i (exp(z_iv - lse_i) - [v = t(i)])
//   dx = dz W,  dW = dz^T x,  db = sum_i dz_i
//
// The logits exist a piece of the vocabulary at a time: a first pass over the pieces merges each
// row's running maximum and sum of exponentials, a second one forms the piece's logits again, turns
// them into dz and multiplies it with both operands.  All sums in fp32.
#include <algorithm>

#include "train.h"

namespace adn {

namespace {

constexpr int NT = 256;
constexpr int BT = 64, BKS = 16;
constexpr size_t PIECE_BYTES = 256u << 20;

// C[i][j] = sum_k A(i,k) B(j,k) (+ bias[j], + C), A(i,k) = A[i ai + k ak], B(j,k) = B[j bj + k bk]:
// 64 x 64 blocks, 4 x 4 values a thread.
// Where `live` is set, terms k with live[k] < 0 are left out (rows without a target: their x is not read).
template <typename TA, typename TB, typename TC>
__global__ __launch_bounds__(NT) void k_tile_product(const TA *A, long ai, long ak, const TB *B, long bj, long bk, TC *C,
                                                     long ci, int M, int N, int K, const float *bias, bool add,
                                                     const int32_t *live) {
    __shared__ float As[BKS][BT + 1], Bs[BKS][BT + 1];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const long i0 = (long)blockIdx.y * BT, j0 = (long)blockIdx.x * BT;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += BKS) {
        for (int q = threadIdx.x; q < BT * BKS; q += NT) {
            // neighbouring threads along the operand's unit stride
            const int ka = ak == 1 ? q % BKS : q / BT, ia = ak == 1 ? q / BKS : q % BT;
            const int kb = bk == 1 ? q % BKS : q / BT, jb = bk == 1 ? q / BKS : q % BT;
            As[ka][ia] = i0 + ia < M && k0 + ka < K ? to_f32<TA>(A[(i0 + ia) * ai + (long)(k0 + ka) * ak]) : 0.0f;
            Bs[kb][jb] = j0 + jb < N && k0 + kb < K && (!live || live[k0 + kb] >= 0) ? to_f32<TB>(B[(j0 + jb) * bj + (long)(k0 + kb) * bk]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < BKS; ++k)
#pragma unroll
            for (int a = 0; a < 4; ++a)
#pragma unroll
                for (int b = 0; b < 4; ++b) acc[a][b] += As[k][ty + 16 * a] * Bs[k][tx + 16 * b];
        __syncthreads();
    }
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const long i = i0 + ty + 16 * a, j = j0 + tx + 16 * b;
            if (i < M && j < N) {
                float v = acc[a][b] + (bias ? bias[j] : 0.0f);
                if (add) v += to_f32<TC>(C[i * ci + j]);
                C[i * ci + j] = from_f32<TC>(v);
            }
        }
}

template <typename TA, typename TB, typename TC>
void tile_product(const TA *A, long ai, long ak, const TB *B, long bj, long bk, TC *C, long ci, int M, int N, int K,
                  const float *bias, bool add, hipStream_t st, const int32_t *live = nullptr) {
    const dim3 grid((unsigned)((N + BT - 1) / BT), (unsigned)((M + BT - 1) / BT));
    k_tile_product<TA, TB, TC><<<grid, NT, 0, st>>>(A, ai, ak, B, bj, bk, C, ci, M, N, K, bias, add, live);
}

__device__ __forceinline__ float block_max(float v, float *red) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < NT / 64; ++w) v = fmaxf(v, red[w]);
    return v;
}
__device__ __forceinline__ float block_sum(float v, float *red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < NT / 64; ++w) v += red[w];
    return v;
}

// Row i's target: its column, or -1 where it has none (negative, or beyond the vocabulary: an error
// that the next synchronisation reports).
__device__ __forceinline__ int target_of(const LossParams &p, int i) {
    const int t = p.targets[i];
    if (t >= p.vocab) {
        if (threadIdx.x == 0) atomicOr(p.err, ADN_DEVERR_TOKEN);
        return -1;
    }
    return t < 0 ? -1 : t;
}

// Merge a piece's logits [rows][n] into each row's maximum, sum and target logit; after the last
// piece the row's lse and loss.  A block a row.
__global__ __launch_bounds__(NT) void k_merge(LossParams p, const float *z, int v0, int n, float *stat, int last) {
    __shared__ float red[NT / 64];
    const int i = blockIdx.x, t = target_of(p, i);
    const float *row = z + (long)i * n;
    float m = -INFINITY;
    bool bad = false;  // fmaxf passes NaN over
    for (int c = threadIdx.x; c < n; c += NT) {
        m = fmaxf(m, row[c]);
        bad |= row[c] != row[c];
    }
    m = block_max(m, red);
    bad = __syncthreads_or(bad);
    const float om = v0 ? stat[i * 3L] : -INFINITY, os = v0 ? stat[i * 3L + 1] : 0.0f;
    const float ot = v0 ? stat[i * 3L + 2] : 0.0f;
    const float nm = fmaxf(m, om), ref = nm == -INFINITY ? 0.0f : nm;
    float s = 0.0f;
    for (int c = threadIdx.x; c < n; c += NT) s += expf(row[c] - ref);
    s = block_sum(s, red) + (v0 ? os * expf(om - ref) : 0.0f);
    if (bad) s = NAN;
    if (threadIdx.x) return;
    const float tz = t >= v0 && t < v0 + n ? row[t - v0] : ot;
    stat[i * 3L] = nm;
    stat[i * 3L + 1] = s;
    stat[i * 3L + 2] = tz;
    if (last) {
        const float lse = ref + logf(s);
        p.lse[i] = t < 0 ? 0.0f : lse;
        if (p.loss) p.loss[i] = t < 0 ? 0.0f : lse - tz;
    }
}

// z -> dz in place, and the block's columns' share of db is left to k_col_sums.
__global__ __launch_bounds__(NT) void k_dz(LossParams p, float *z, int v0, int n) {
    const int i = blockIdx.x, t = target_of(p, i);
    const float g = t < 0 ? 0.0f : p.dloss ? p.dloss[i] : 1.0f, lse = p.lse[i];
    float *row = z + (long)i * n;
    for (int c = threadIdx.x; c < n; c += NT)
        row[c] = t < 0 ? 0.0f : g * (expf(row[c] - lse) - (v0 + c == t ? 1.0f : 0.0f));
}

__global__ __launch_bounds__(NT) void k_col_sums(const float *z, int rows, int n, float *db) {
    const int c = blockIdx.x * NT + threadIdx.x;
    if (c >= n) return;
    float s = 0.0f;
    for (long i = 0; i < rows; ++i) s += z[i * n + c];
    db[c] = s;
}

template <typename T>
__global__ __launch_bounds__(NT) void k_round_rows(const float *src, int rows, int d, T *dst, long stride) {
    const long i = blockIdx.x;
    for (int c = threadIdx.x; c < d; c += NT) dst[i * stride + c] = from_f32<T>(src[i * d + c]);
}

struct LossLayout {
    int piece;
    size_t z, stat, lse, dx, bytes;
};
LossLayout loss_layout(const LossParams &p) {
    LossLayout L{};
    const long rows = std::max(1, p.rows);
    L.piece = (int)std::min<long>(p.vocab, std::max<long>(64, (long)(PIECE_BYTES / 4) / rows));
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += (bytes + 255) / 256 * 256;
        return r;
    };
    L.z = take((size_t)rows * L.piece * 4);
    L.stat = take((size_t)rows * 12);
    L.lse = take((size_t)rows * 4);
    L.dx = take(p.dx ? (size_t)rows * p.d * 4 : 0);
    L.bytes = at;
    return L;
}

}  // namespace

size_t loss_workspace_bytes(const LossParams &p) { return loss_layout(p).bytes; }

void launch_loss(const LossParams &q, void *ws, hipStream_t st) {
    LossParams p = q;
    const LossLayout L = loss_layout(p);
    char *w8 = (char *)ws;
    float *z = (float *)(w8 + L.z), *stat = (float *)(w8 + L.stat), *dxa = (float *)(w8 + L.dx);
    if (!p.lse) p.lse = (float *)(w8 + L.lse);
    dispatch_type(p.dtype, [&](auto ty) {
        typedef decltype(ty) T;
        const T *x = (const T *)p.x, *w = (const T *)p.w;
        for (int pass = 0; pass < (p.dx || p.dw || p.db ? 2 : 1); ++pass)
            for (int v0 = 0; v0 < p.vocab; v0 += L.piece) {
                const int n = std::min(L.piece, p.vocab - v0);
                if (p.rows) {
                    tile_product<T, T, float>(x, p.x_stride, 1, w + (long)v0 * p.w_stride, p.w_stride, 1, z, n, p.rows, n,
                                              p.d, p.bias ? p.bias + v0 : nullptr, false, st);
                    if (pass == 0) {
                        k_merge<<<p.rows, NT, 0, st>>>(p, z, v0, n, stat, v0 + n == p.vocab);
                        continue;
                    }
                    k_dz<<<p.rows, NT, 0, st>>>(p, z, v0, n);
                }
                if (pass == 0) continue;
                if (p.dx && p.rows)
                    tile_product<float, T, float>(z, n, 1, w + (long)v0 * p.w_stride, 1, p.w_stride, dxa, p.d, p.rows,
                                                  p.d, n, nullptr, v0 > 0, st);
                if (p.dw)
                    tile_product<float, T, T>(z, 1, n, x, 1, p.x_stride, (T *)p.dw + (long)v0 * p.dw_stride, p.dw_stride,
                                              n, p.d, p.rows, nullptr, false, st, p.targets);
                if (p.db) k_col_sums<<<(n + NT - 1) / NT, NT, 0, st>>>(z, p.rows, n, p.db + v0);
            }
        if (p.dx && p.rows) k_round_rows<T><<<p.rows, NT, 0, st>>>(dxa, p.rows, p.d, (T *)p.dx, p.dx_stride);
    });
}

}  // namespace adn
