// The vocabulary cross entropy (loss.hip has the mathematics) of a few rows, and of small problems: fp32
// arithmetic on the operands as they are, two launches each.
//
// A few rows (at most 8 of 512, 4 of 1024, 2 of 2048; 4 where loss_mid.hip can take more) read W at the rate of HBM whatever is done with it,
// so W is read once: the first kernel has R rows of x in registers, a wave takes one row of W at a time
// (its elements in the lanes), forms its R logits, and adds it, weighted by exp(z - m) with the running
// maximum m, to the wave's share of sum_v exp(z_v) w_v -- dx but for the target and the normalisation.
// The logits themselves (rows x vocab values, the one piece here) stay in the workspace for the second
// kernel, which forms lse from the blocks' shares, dx = g (sum / total - w_t), and dW = dz^T x and db
// row by row.  One row of 512 against 50257, 206 MB read and written: 58 us; through fp16 planes 157.
//
// Other small problems (rows x vocab x d at most SMALL, the logits in the workspace again) gain from the two
// launches, and from little code: a straight line of unrolled instructions that each wave runs once
// waits for its own fetch.  One kernel forms 4 x 64 logits a block with the tile's maxima and sums, one
// both gradients as the same sum, out[o][c] = sum_i coef[o][i] src[i][c] (dW: o an entry, i a row, src
// x; dx: o a row, i an entry, src W), 8 x 256 values a block.
#include <algorithm>

#include "train.h"

namespace adn {

namespace {

constexpr int NT = 256;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int MAX_SHARES = 512;     // blocks that share the vocabulary
constexpr int MAX_ROWS = 8;         // of the few
constexpr long SMALL = 1L << 23;
constexpr int SMALL_ROWS = 256, SMALL_VOCAB = 256;  // a block walks all of one of them

struct Few {
    LossParams p;
    int shares;           // blocks (small: tiles of 64 entries) that share the vocabulary
    float *z;             // [rows][vocab], in units of log 2
    float *pm, *ps;       // [rows][shares] maximum and sum of exponentials
    float *pdx;           // [shares][rows][d], or null
    int dx_blocks, dx_cols;  // second kernel: blocks of dx first; blocks a row of theirs (small: of either's)
    bool vecx, vecw, vecdw;
};

// Sum over the wave without LDS: the 16 lanes of a row by DPP, then the four rows' sums; wave-uniform.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float sum_lanes(float v) {
    v += dpp<0xB1>(v);   // quad_perm 1 0 3 2
    v += dpp<0x4E>(v);   // quad_perm 2 3 0 1
    v += dpp<0x141>(v);  // row_half_mirror
    v += dpp<0x140>(v);  // row_mirror
    auto row = [&](int l) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l)); };
    return (row(0) + row(16)) + (row(32) + row(48));
}

// A lane's E elements of a row: 16-byte pieces, 64 lanes side by side.
template <typename T, int E>
__device__ __forceinline__ int col_of(int lane, int e) {
    constexpr int W = 16 / (int)sizeof(T);
    return ((e / W) * 64 + lane) * W + e % W;
}
template <typename T, int E>
__device__ __forceinline__ void load_lane(const T *row, int d, int lane, bool vec, float (&v)[E]) {
    constexpr int W = 16 / (int)sizeof(T);
    typedef T V __attribute__((ext_vector_type(W)));
    if (vec) {
#pragma unroll
        for (int e = 0; e < E; e += W) {
            const int c = col_of<T, E>(lane, e);
            V x = {};
            if (c < d) x = *reinterpret_cast<const V *>(row + c);
#pragma unroll
            for (int j = 0; j < W; ++j) v[e + j] = to_f32<T>(x[j]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = col_of<T, E>(lane, e);
            v[e] = c < d ? to_f32<T>(row[c]) : 0.0f;
        }
    }
}
template <typename T, int E>
__device__ __forceinline__ void store_lane(T *row, int d, int lane, bool vec, const float (&v)[E]) {
    constexpr int W = 16 / (int)sizeof(T);
    typedef T V __attribute__((ext_vector_type(W)));
    if (vec) {
#pragma unroll
        for (int e = 0; e < E; e += W) {
            const int c = col_of<T, E>(lane, e);
            V x;
#pragma unroll
            for (int j = 0; j < W; ++j) x[j] = from_f32<T>(v[e + j]);
            if (c < d) *reinterpret_cast<V *>(row + c) = x;
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = col_of<T, E>(lane, e);
            if (c < d) row[c] = from_f32<T>(v[e]);
        }
    }
}

// Rows without a target are zeros, whatever stands in x (their x and targets are loaded side by side).
template <typename T, int R, int E>
__device__ __forceinline__ void load_rows(const Few &f, int lane, float (&x)[R][E]) {
    int t[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const long i = min(r, f.p.rows - 1);
        t[r] = f.p.targets[i];
        load_lane<T, E>((const T *)f.p.x + i * f.p.x_stride, f.p.d, lane, f.vecx, x[r]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (t[r] < 0 || t[r] >= f.p.vocab || r >= f.p.rows)
#pragma unroll
            for (int e = 0; e < E; ++e) x[r][e] = 0.0f;
}

template <typename T, int R, int E>
__global__ __launch_bounds__(NT) void k_few_logits(Few f) {
    constexpr int U = E <= 8 ? 4 : E <= 16 ? 2 : 1;  // rows of W in flight
    __shared__ float sm[4][R], ss[4][R];
    __shared__ float sacc[3][R][64][E + 1];
    const LossParams &p = f.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int share = blockIdx.x;
    if (share == 0 && (int)threadIdx.x < p.rows && p.targets[threadIdx.x] >= p.vocab) atomicOr(p.err, ADN_DEVERR_TOKEN);
    float x[R][E], acc[R][E], m[R], s[R];
    load_rows<T, R, E>(f, lane, x);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        s[r] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] = 0.0f;
    }
    const bool sum = f.pdx != nullptr;
    const int per = (p.vocab + f.shares - 1) / f.shares;
    const int v0 = share * per, v1 = min(p.vocab, v0 + per);
    // the waves of a block take every fourth row; the next U rows are loaded before these are used
    float wn[U][E], bn[U];
    auto fetch = [&](int vb) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int v = max(0, min(vb + 4 * u, v1 - 1));
            load_lane<T, E>((const T *)p.w + (long)v * p.w_stride, p.d, lane, f.vecw, wn[u]);
            bn[u] = p.bias ? p.bias[v] : 0.0f;
        }
    };
    fetch(v0 + wave);
    for (int vb = v0 + wave; vb < v1; vb += 4 * U) {
        float w[U][E], z[U][R], bias[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float b = bn[u];
            if (b < -1e38f && b > -INFINITY) b = -1e38f;  // the lowest value times log2(e) stays finite
            bias[u] = b * LOG2E;
#pragma unroll
            for (int e = 0; e < E; ++e) w[u][e] = wn[u][e];
        }
        if (vb + 4 * U < v1) fetch(vb + 4 * U);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float t = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) t += x[r][e] * w[u][e];
                t = __builtin_fmaf(sum_lanes(t), LOG2E, bias[u]);
                const bool in = vb + 4 * u < v1;
                if (in && lane == 0 && r < p.rows) f.z[(long)r * p.vocab + vb + 4 * u] = t;
                z[u][r] = in ? t : -INFINITY;
            }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = m[r];
#pragma unroll
            for (int u = 0; u < U; ++u) top = fmaxf(top, z[u][r]);
            if (top > m[r]) {
                const float k = __builtin_amdgcn_exp2f(m[r] - top);
                m[r] = top;
                s[r] *= k;
                if (sum)
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[r][e] *= k;
            }
            const float ref = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float q = __builtin_amdgcn_exp2f(z[u][r] - ref);
                s[r] += q;
                if (sum)
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[r][e] += q * w[u][e];
            }
        }
    }
    // the waves' shares, in order
    if (lane == 0)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            sm[wave][r] = m[r];
            ss[wave][r] = s[r];
        }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float top = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
        const float ref = top == -INFINITY ? 0.0f : top;
        const long i = r;
        if (threadIdx.x == 0 && i < p.rows) {
            float t = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) t += ss[w][r] * __builtin_amdgcn_exp2f(sm[w][r] - ref);
            f.pm[i * f.shares + share] = top;
            f.ps[i * f.shares + share] = t;
        }
        const float k = __builtin_amdgcn_exp2f(m[r] - ref);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] *= k;
        if (sum && wave)
#pragma unroll
            for (int e = 0; e < E; ++e) sacc[wave - 1][r][lane][e] = acc[r][e];
    }
    if (!sum) return;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const long i = r;
        if (i >= p.rows) break;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = col_of<T, E>(lane, e);
            const float t = acc[r][e] + sacc[0][r][lane][e] + sacc[1][r][lane][e] + sacc[2][r][lane][e];
            if (c < p.d) f.pdx[((long)share * p.rows + i) * p.d + c] = t;
        }
    }
}

// Blocks below dx_blocks: 64 columns of a row of dx.  The others: rows of dW and db, a wave VB at a
// time.  The first block also writes loss and lse.
template <typename T, int R, int E>
__global__ __launch_bounds__(NT) void k_few_grads(Few f) {
    constexpr int VB = E <= 8 ? 4 : E <= 16 ? 2 : 1;
    __shared__ float lse[MAX_ROWS], up[MAX_ROWS];  // up: g_i, 0 without a target
    __shared__ int tgt[MAX_ROWS];
    __shared__ float weight[MAX_SHARES];
    __shared__ float red[4][64];
    const LossParams &p = f.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const bool of_dx = (int)blockIdx.x < f.dx_blocks;
    const int my_row = of_dx ? (int)blockIdx.x / f.dx_cols : -1;
    for (int i = threadIdx.x; i < p.rows; i += NT) {
        const int t = p.targets[i];
        const bool there = t >= 0 && t < p.vocab;
        tgt[i] = there ? t : -1;
        up[i] = there ? (p.dloss ? p.dloss[i] : 1.0f) : 0.0f;
    }
    // lse of the rows that the block needs, a wave each
    for (int i = wave; i < p.rows; i += 4) {
        if (of_dx && blockIdx.x && i != my_row) continue;
        const float *pm = f.pm + (long)i * f.shares, *ps = f.ps + (long)i * f.shares;
        float a[MAX_SHARES / 64], b[MAX_SHARES / 64], m = -INFINITY, s = 0.0f;
#pragma unroll
        for (int u = 0; u < MAX_SHARES / 64; ++u) {
            const int q = lane + 64 * u;
            a[u] = q < f.shares ? pm[q] : -INFINITY;
            b[u] = q < f.shares ? ps[q] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < MAX_SHARES / 64; ++u) m = fmaxf(m, a[u]);
        m = wave_max(m);
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int u = 0; u < MAX_SHARES / 64; ++u) s += b[u] * __builtin_amdgcn_exp2f(a[u] - ref);
        s = sum_lanes(s);
        if (lane == 0) lse[i] = ref + log2f(s);
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < p.rows; i += NT) {
            const int t = tgt[i];
            if (p.lse) p.lse[i] = t >= 0 ? lse[i] * LN2 : 0.0f;
            if (p.loss) p.loss[i] = t >= 0 ? (lse[i] - f.z[(long)i * p.vocab + t]) * LN2 : 0.0f;
        }
    if (of_dx) {
        const int i = my_row, c = ((int)blockIdx.x % f.dx_cols) * 64 + lane;
        const int t = tgt[i];
        const float g = up[i], l = lse[i];
        for (int q = threadIdx.x; q < f.shares; q += NT) weight[q] = __builtin_amdgcn_exp2f(f.pm[(long)i * f.shares + q] - l);
        __syncthreads();
        float s = 0.0f;
        if (c < p.d) {
#pragma unroll 16
            for (int q = wave; q < f.shares; q += 4) s += weight[q] * f.pdx[((long)q * p.rows + i) * p.d + c];
        }
        red[wave][lane] = s;
        __syncthreads();
        if (wave || c >= p.d) return;
        s = red[0][lane] + red[1][lane] + red[2][lane] + red[3][lane];
        if (g != 0.0f)
            s = g * (s - to_f32<T>(((const T *)p.w)[(long)t * p.w_stride + c]));
        else
            s = 0.0f;
        ((T *)p.dx)[(long)i * p.dx_stride + c] = from_f32<T>(s);
        return;
    }
    if (!p.dw && !p.db) return;
    float x[R][E];
    load_rows<T, R, E>(f, lane, x);
    const int first = ((int)blockIdx.x - f.dx_blocks) * 4 + wave, step = ((int)gridDim.x - f.dx_blocks) * 4;
    for (int v0 = first * VB; v0 < p.vocab; v0 += step * VB) {
        float acc[VB][E], db[VB], z[R][VB];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int b = 0; b < VB; ++b) z[r][b] = f.z[(long)min(r, p.rows - 1) * p.vocab + min(v0 + b, p.vocab - 1)];
#pragma unroll
        for (int b = 0; b < VB; ++b) {
            db[b] = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[b][e] = 0.0f;
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float g = r < p.rows ? up[r] : 0.0f;
            if (g == 0.0f) continue;
            const int t = tgt[r];
            const float l = lse[r];
#pragma unroll
            for (int b = 0; b < VB; ++b) {
                const float dz = g * (__builtin_amdgcn_exp2f(z[r][b] - l) - (v0 + b == t ? 1.0f : 0.0f));
                db[b] += dz;
#pragma unroll
                for (int e = 0; e < E; ++e) acc[b][e] += dz * x[r][e];
            }
        }
#pragma unroll
        for (int b = 0; b < VB; ++b) {
            if (v0 + b >= p.vocab) break;
            if (p.dw) store_lane<T, E>((T *)p.dw + (long)(v0 + b) * p.dw_stride, p.d, lane, f.vecdw, acc[b]);
            if (p.db && lane == 0) p.db[v0 + b] = db[b];
        }
    }
}

// ---- small problems ------------------------------------------------------------------------
// Logits of 4 rows (a wave each) and 64 entries (a lane each), 64 columns of the operands in LDS at a
// time, the next ones loaded meanwhile.
template <typename T>
__global__ __launch_bounds__(NT) void k_small_logits(Few f) {
    __shared__ float ws[64][65], xs[4][64];
    const LossParams &p = f.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int v0 = blockIdx.x * 64, i = blockIdx.y * 4 + wave;
    const int t = i < p.rows ? p.targets[i] : -1;
    if (t >= p.vocab && blockIdx.x == 0 && lane == 0) atomicOr(p.err, ADN_DEVERR_TOKEN);
    const long ix = min(i, p.rows - 1);
    float wn[16], xn;
    auto fetch = [&](int k0) {
        const int c = k0 + lane;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const long v = min(v0 + wave * 16 + q, p.vocab - 1);
            wn[q] = c < p.d ? to_f32<T>(((const T *)p.w)[v * p.w_stride + c]) : 0.0f;
        }
        xn = c < p.d ? to_f32<T>(((const T *)p.x)[ix * p.x_stride + c]) : 0.0f;
    };
    fetch(0);
    float z = 0.0f;
    for (int k0 = 0; k0 < p.d; k0 += 64) {
        if (k0) __syncthreads();
#pragma unroll
        for (int q = 0; q < 16; ++q) ws[wave * 16 + q][lane] = wn[q];
        xs[wave][lane] = t >= 0 && t < p.vocab ? xn : 0.0f;
        __syncthreads();
        if (k0 + 64 < p.d) fetch(k0 + 64);
#pragma unroll 16
        for (int k = 0; k < 64; ++k) z += xs[wave][k] * ws[lane][k];
    }
    if (i >= p.rows) return;
    const int v = v0 + lane;
    float b = v < p.vocab ? (p.bias ? p.bias[v] : 0.0f) : -INFINITY;
    if (b < -1e38f && b > -INFINITY) b = -1e38f;  // the lowest value times log2(e) stays finite
    z = __builtin_fmaf(z, LOG2E, b * LOG2E);
    if (v < p.vocab) f.z[(long)i * p.vocab + v] = z;
    const float m = wave_max(z), ref = m == -INFINITY ? 0.0f : m;
    const float s = sum_lanes(__builtin_amdgcn_exp2f(z - ref));
    if (lane == 0) {
        f.pm[(long)i * f.shares + blockIdx.x] = m;
        f.ps[(long)i * f.shares + blockIdx.x] = s;
    }
}

// Blocks below dx_blocks: 8 rows of dx x 256 columns; the others: 8 rows of dW x 256 columns, the first
// columns' blocks db too.  The first block also writes loss and lse.
template <typename T>
__global__ __launch_bounds__(NT) void k_small_grads(Few f) {
    constexpr int O = 8, IC = 64;  // outputs a block, terms of the sum in LDS at a time
    __shared__ float lse[SMALL_ROWS], up[SMALL_ROWS];
    __shared__ int tgt[SMALL_ROWS];
    __shared__ float coef[IC][O];
    __shared__ int live[IC];
    const LossParams &p = f.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool of_dx = (int)blockIdx.x < f.dx_blocks;
    const int b = of_dx ? blockIdx.x : (int)blockIdx.x - f.dx_blocks;
    const int o0 = b / f.dx_cols * O, c = b % f.dx_cols * NT + tid;
    for (int i = tid; i < p.rows; i += NT) {
        if (of_dx && blockIdx.x && (i < o0 || i >= o0 + O)) continue;
        const int t = p.targets[i];
        const bool there = t >= 0 && t < p.vocab;
        tgt[i] = there ? t : -1;
        up[i] = there ? (p.dloss ? p.dloss[i] : 1.0f) : 0.0f;
        float m = -INFINITY, s = 0.0f;
        for (int q0 = 0; q0 < f.shares; q0 += 8) {
            float a[8], e[8], top = m;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const long at = (long)i * f.shares + min(q0 + u, f.shares - 1);
                a[u] = q0 + u < f.shares ? f.pm[at] : -INFINITY;
                e[u] = q0 + u < f.shares ? f.ps[at] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) top = fmaxf(top, a[u]);
            const float ref = top == -INFINITY ? 0.0f : top;
            s *= __builtin_amdgcn_exp2f(m - ref);
#pragma unroll
            for (int u = 0; u < 8; ++u) s += e[u] * __builtin_amdgcn_exp2f(a[u] - ref);
            m = top;
        }
        const float l = (m == -INFINITY ? 0.0f : m) + log2f(s);
        lse[i] = l;
        if (blockIdx.x == 0) {
            if (p.lse) p.lse[i] = there ? l * LN2 : 0.0f;
            if (p.loss) p.loss[i] = there ? (l - f.z[(long)i * p.vocab + t]) * LN2 : 0.0f;
        }
    }
    if (of_dx ? !p.dx : !p.dw && !p.db) return;
    const int n = of_dx ? p.vocab : p.rows;  // terms
    const int no = of_dx ? p.rows : p.vocab;
    const T *src = (const T *)(of_dx ? p.w : p.x);
    const long stride = of_dx ? p.w_stride : p.x_stride;
    float acc[O] = {}, db[2] = {0.0f, 0.0f};
    for (int i0 = 0; i0 < n; i0 += IC) {
        __syncthreads();
#pragma unroll
        for (int q = tid; q < IC * O; q += NT) {
            // neighbouring threads along the logits' rows
            const int k = of_dx ? q % IC : q / O, o = of_dx ? q / IC : q % O;
            const int row = of_dx ? o0 + o : i0 + k, v = of_dx ? i0 + k : o0 + o;
            float g = 0.0f;
            if (row < p.rows && v < p.vocab) g = up[row];
            coef[k][o] = g == 0.0f ? 0.0f
                                   : g * (__builtin_amdgcn_exp2f(f.z[(long)row * p.vocab + v] - lse[row]) - (v == tgt[row] ? 1.0f : 0.0f));
            if (o == 0) live[k] = of_dx ? v < p.vocab : g != 0.0f;
        }
        __syncthreads();
        if (p.db && !of_dx && b % f.dx_cols == 0) {
            db[0] += sum_lanes(coef[lane][2 * wave]);
            db[1] += sum_lanes(coef[lane][2 * wave + 1]);
        }
        if (c < p.d)
#pragma unroll 1
            for (int k0 = 0; k0 < IC; k0 += 16) {
                float x[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const int i = min(i0 + k0 + k, n - 1);
                    x[k] = to_f32<T>(src[i * stride + c]);
                }
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const float xv = live[k0 + k] ? x[k] : 0.0f;  // rows that give nothing are not read
#pragma unroll
                    for (int o = 0; o < O; ++o) acc[o] += coef[k0 + k][o] * xv;
                }
            }
    }
    if (p.db && !of_dx && b % f.dx_cols == 0 && lane == 0)
#pragma unroll
        for (int q = 0; q < 2; ++q)
            if (o0 + 2 * wave + q < p.vocab) p.db[o0 + 2 * wave + q] = db[q];
    if (c >= p.d) return;
#pragma unroll
    for (int o = 0; o < O; ++o) {
        if (o0 + o >= no) break;
        if (of_dx)
            ((T *)p.dx)[(o0 + o) * p.dx_stride + c] = from_f32<T>(up[o0 + o] == 0.0f ? 0.0f : acc[o]);
        else if (p.dw)
            ((T *)p.dw)[(long)(o0 + o) * p.dw_stride + c] = from_f32<T>(acc[o]);
    }
}

// Elements a lane holds of a row of d, and rows a block holds of them (64 registers).
int lane_elems(int d) { return d <= 512 ? 8 : d <= 1024 ? 16 : 32; }
int group_rows(int rows, int d) {
    const int most = 64 / lane_elems(d);
    int r = 1;
    while (r < rows && r < most) r *= 2;
    return r;
}

// f(T, R, E)
template <typename F>
void dispatch_few(const LossParams &p, F &&f) {
    using std::integral_constant;
    const int e = lane_elems(p.d), r = group_rows(p.rows, p.d);
    dispatch_type(p.dtype, [&](auto t) {
        auto with = [&](auto ec) {
            constexpr int E = decltype(ec)::value;
            if (r == 1)
                f(t, integral_constant<int, 1>{}, ec);
            else if (r == 2)
                f(t, integral_constant<int, 2>{}, ec);
            else if constexpr (E <= 16) {
                if (r == 4)
                    f(t, integral_constant<int, 4>{}, ec);
                else if constexpr (E <= 8)
                    f(t, integral_constant<int, 8>{}, ec);
            }
        };
        if (e == 8)
            with(integral_constant<int, 8>{});
        else if (e == 16)
            with(integral_constant<int, 16>{});
        else
            with(integral_constant<int, 32>{});
    });
}

// Five to eight rows need as many sums over the wave again: 512 columns of 50257 entries 113 to 119 us, of 8192
// 46, where loss_mid.hip takes 80 and 34.
bool few(const LossParams &p) {
    return p.d <= 2048 && p.rows <= std::min(64 / lane_elems(p.d), loss_mid_ok(p) ? 4 : MAX_ROWS);
}
// Up to 64 rows go to loss_mid.hip unless W is small: 128 entries of 128 columns 18 us here and 23 to 26 there
// (fp32), of 512 columns 23 and 25 to 31, 512 of 512 columns 48 and 26 to 31.  A block walks all rows or
// all entries 64 at a time: 512 rows of 64 against 65 entries 43 us here and 29 on loss.hip's products.
bool small(const LossParams &p) {
    return !few(p) && p.rows <= SMALL_ROWS && p.vocab <= SMALL_VOCAB && (long)p.rows * p.vocab * p.d <= SMALL &&
           !(loss_mid_ok(p) && (long)p.vocab * p.d > 1 << 16);
}

struct FewLayout {
    int shares;
    size_t z, pm, ps, pdx, bytes;
};
FewLayout few_layout(const LossParams &p) {
    FewLayout L{};
    // enough blocks to fill the chip, at least 4 rows of W each
    L.shares = small(p) ? (p.vocab + 63) / 64 : (int)std::min<long>(MAX_SHARES, ((long)p.vocab + 3) / 4);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += (bytes + 255) / 256 * 256;
        return r;
    };
    L.z = take((size_t)p.rows * p.vocab * 4);
    L.pm = take((size_t)p.rows * L.shares * 4);
    L.ps = take((size_t)p.rows * L.shares * 4);
    L.pdx = take(p.dx && !small(p) ? (size_t)L.shares * p.rows * p.d * 4 : 0);
    L.bytes = at;
    return L;
}

}  // namespace

bool loss_few_ok(const LossParams &p) {
    return few(p) || small(p);
}

size_t loss_few_workspace_bytes(const LossParams &p) { return few_layout(p).bytes; }

void launch_loss_few(const LossParams &p, void *ws, hipStream_t st) {
    const FewLayout L = few_layout(p);
    char *w = (char *)ws;
    Few f{};
    f.p = p;
    f.shares = L.shares;
    f.z = (float *)(w + L.z), f.pm = (float *)(w + L.pm), f.ps = (float *)(w + L.ps);
    if (small(p)) {
        f.dx_cols = (p.d + NT - 1) / NT;
        f.dx_blocks = p.dx ? (p.rows + 7) / 8 * f.dx_cols : 0;
        const int dw_blocks = p.dw || p.db ? (p.vocab + 7) / 8 * f.dx_cols : 0;
        dispatch_type(p.dtype, [&](auto t) {
            typedef decltype(t) T;
            k_small_logits<T><<<dim3((unsigned)L.shares, (unsigned)((p.rows + 3) / 4)), NT, 0, st>>>(f);
            k_small_grads<T><<<(unsigned)std::max(1, f.dx_blocks + dw_blocks), NT, 0, st>>>(f);
        });
        return;
    }
    f.pdx = p.dx ? (float *)(w + L.pdx) : nullptr;
    f.dx_cols = (p.d + 63) / 64;
    f.dx_blocks = p.dx ? p.rows * f.dx_cols : 0;
    const int eb = elem_bytes(p.dtype);
    f.vecx = rows_vec16(p.x, p.x_stride, p.d, eb);
    f.vecw = rows_vec16(p.w, p.w_stride, p.d, eb);
    f.vecdw = p.dw && rows_vec16(p.dw, p.dw_stride, p.d, eb);
    dispatch_few(p, [&](auto t, auto rc, auto ec) {
        typedef decltype(t) T;
        constexpr int R = decltype(rc)::value, E = decltype(ec)::value;
        k_few_logits<T, R, E><<<(unsigned)L.shares, NT, 0, st>>>(f);
        constexpr int VB = E <= 8 ? 4 : E <= 16 ? 2 : 1;
        // at most about a thousand blocks, of equal shares
        const long units = ((long)p.vocab + 4 * VB - 1) / (4 * VB), each = (units + 1023) / 1024;
        const int dw_blocks = p.dw || p.db ? (int)((units + each - 1) / each) : 0;
        k_few_grads<T, R, E><<<(unsigned)std::max(1, f.dx_blocks + dw_blocks), NT, 0, st>>>(f);
    });
}

}  // namespace adn
