// The vocabulary cross entropy (loss.hip has the mathematics) of up to 64 rows, more than loss_few.hip
// takes: what W's bytes bound.  W is read once for the logits and once for dx, dW is written once, and
// nothing is laid out anew but x.  16 rows of 512 against 50257 entries, 309 MB: 81 us (fp32; logits 25,
// gradients 44, 4.7 TB/s) or 52 (bf16), on the products of loss.hip 150 and 94; 64 rows 110 and 76 (195
// and 95).
//
// The products run on the bf16 MFMA.  A fp32 value is the exact sum of three bf16 ones of 8 bits each,
// cut off in registers on the way to the MFMA; six of the nine products are formed (what is left out is
// below 2^-21 of a product).  bf16 needs as many exponent bits as fp32, so no scale is looked for first,
// which would take another pass over W.  bf16 tensors are their own single plane, dz has two.
//
// The logits stay in the workspace: rows x vocab values are few bytes beside W's d x vocab.
#include <algorithm>

#include "train.h"

namespace adn {

namespace {

constexpr int NT = 256;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int MAX_ROWS = 64;
constexpr int TE = 64;        // entries a block of the logits takes
constexpr int DW_TE = 128;    // entries a block of dW takes, 32 a wave
constexpr int STRIP = 128;    // columns of dW's products, 4 adjacent ones a lane

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

struct Mid {
    LossParams p;
    int np32;             // rows padded: 32 or 64
    int tiles;            // blocks of the logits
    bf8 *xa, *xb;         // x's planes as MFMA operands (lane by lane): for the logits, for dW
    float *z;             // [tiles * TE][np32], in units of log 2
    float *pm, *ps;       // [rows][tiles]: maximum and sum of exponentials
    float *lse;           // [rows], in units of log 2
    float *part;          // [shares][rows][d]: dx's partial sums
    int shares, share;    // of the vocabulary, entries of one (a multiple of 64)
    int strips;           // column strips of dx
    int dx_blocks;
    int dw_groups;        // blocks that share the strips of DW_TE entries
    bool vecdw;
};

template <typename T>
constexpr int planes_of() {
    return sizeof(T) == 4 ? 3 : 1;
}
template <typename T>
constexpr int dz_planes() {
    return sizeof(T) == 4 ? 3 : 2;
}

// v as a sum of PL bf16 vectors: 8 bits at a time, cut off (three hold an fp32 value exactly), the last
// of two rounded.
template <int PL>
__device__ __forceinline__ void split8(const float (&v)[8], bf8 (&out)[PL]) {
    float a[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = v[j];
#pragma unroll
    for (int q = 0; q < PL; ++q) {
        if (PL == 2 && q == 1) {
#pragma unroll
            for (int j = 0; j < 8; ++j) out[q][j] = (__bf16)a[j];
            continue;
        }
        uint4v w;
#pragma unroll
        for (int u = 0; u < 4; ++u)
            w[u] = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, a[2 * u + 1]), __builtin_bit_cast(unsigned, a[2 * u]), 0x07060302u);
        out[q] = __builtin_bit_cast(bf8, w);
        if (q + 1 < PL)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                a[j] -= __builtin_bit_cast(float, __builtin_bit_cast(unsigned, a[j]) & 0xffff0000u);
    }
}

// acc += a b over the planes, the smallest products first
template <int PA, int PB>
__device__ __forceinline__ void mfma(const bf8 (&a)[PA], const bf8 (&b)[PB], f16v &acc) {
    constexpr int M = PA > PB ? PA : PB;
#pragma unroll
    for (int s = M - 1; s >= 0; --s)
#pragma unroll
        for (int q = 0; q <= s; ++q)
            if (q < PA && s - q < PB) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[q], b[s - q], acc, 0, 0, 0);
}

__device__ __forceinline__ int target_of(const LossParams &p, int i) {
    const int t = i < p.rows ? p.targets[i] : -1;
    return t < p.vocab ? t : -1;
}
__device__ __forceinline__ float upstream_of(const LossParams &p, int i) {
    return target_of(p, i) < 0 ? 0.0f : p.dloss ? p.dloss[i] : 1.0f;
}

// x as operands, a wave 64 lanes x 8 values.  For the logits, operand (k block, tile of 32 rows): a lane 8
// columns of its row; for dW, operand (k block of 16 rows, strip, j): a lane 8 rows of the column
// strip + 4 lane + j.  Rows without a target (dW: without an upstream gradient) are zeros.
template <typename T>
__global__ __launch_bounds__(NT) void k_mid_prep(Mid m, int na, int nb) {
    constexpr int PL = planes_of<T>();
    const LossParams &p = m.p;
    const int lane = threadIdx.x & 63, r = lane & 31, hh = lane >> 5;
    int f = blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
    if (f >= na + nb) return;
    const T *x = (const T *)p.x;
    float v[8];
    bf8 o[PL];
    bf8 *dst;
    if (f < na) {
        const int nt = m.np32 / 32, i = f % nt * 32 + r, c = f / nt * 16 + hh * 8;
        const int at = min(i, p.rows - 1);  // x and targets are loaded side by side
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = to_f32<T>(x[at * p.x_stride + c + e]);
        if (target_of(p, i) < 0)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.0f;
        dst = m.xa + (long)f * PL * 64;
    } else {
        f -= na;
        const int ks = m.np32 / 16, j = f % 4, k = f / 4 % ks, c = f / 4 / ks * STRIP + 4 * r + j;
        const int cc = min(c, p.d - 1);
        int t[8];
        float g[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int i = min(k * 16 + hh * 8 + e, p.rows - 1);
            v[e] = to_f32<T>(x[i * p.x_stride + cc]);
            t[e] = p.targets[i];
            g[e] = p.dloss ? p.dloss[i] : 1.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c >= p.d || k * 16 + hh * 8 + e >= p.rows || t[e] < 0 || t[e] >= p.vocab || g[e] == 0.0f) v[e] = 0.0f;
        dst = m.xb + (long)f * PL * 64;
    }
    split8<PL>(v, o);
#pragma unroll
    for (int q = 0; q < PL; ++q) dst[q * 64 + lane] = o[q];
}

// Logits of TE entries, with each row's maximum and sum of exponentials over them.  The waves divide
// the columns: a wave takes 128 bytes of the TE rows of W at a time, loaded 8 lanes a row, through 8 KB
// of LDS of its own (chunks of 16 bytes swizzled by the row) into MFMA operands.  The next 8 KB and
// operands of x are loaded meanwhile; there is no barrier before the waves' sums are added.
template <typename T, int TN>
__global__ __launch_bounds__(NT, 2) void k_mid_logits(Mid m) {
    constexpr int PL = planes_of<T>(), KS = sizeof(T) == 4 ? 2 : 4;  // k blocks of 16 in 128 bytes
    __shared__ __attribute__((aligned(16))) char lds[4][TE * 128];
    __shared__ float red[2][8][32];
    const LossParams &p = m.p;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int v0 = blockIdx.x * TE, steps = p.d * (int)sizeof(T) / 128;
    const char *src[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
        src[u] = (const char *)p.w + (long)min(v0 + u * 8 + (lane >> 3), p.vocab - 1) * p.w_stride * (long)sizeof(T) + (lane & 7) * 16;
    uint4v wn[8];
    bf8 xn[KS][TN][PL];
    auto fetch = [&](int kt) {
#pragma unroll
        for (int u = 0; u < 8; ++u) wn[u] = *reinterpret_cast<const uint4v *>(src[u] + kt * 128);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int q = 0; q < PL; ++q) xn[s][j][q] = m.xa[(((long)kt * KS + s) * TN + j) * PL * 64 + q * 64 + lane];
    };
    f16v acc[2][TN];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    char *mine = lds[wave];
    if (wave < steps) fetch(wave);
    for (int kt = wave; kt < steps; kt += 4) {
#pragma unroll
        for (int u = 0; u < 8; ++u)
            *reinterpret_cast<uint4v *>(mine + (u * 8 + (lane >> 3)) * 128 + (((lane & 7) ^ (lane >> 3)) * 16)) = wn[u];
        bf8 x[KS][TN][PL];
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int q = 0; q < PL; ++q) x[s][j][q] = xn[s][j][q];
        if (kt + 4 < steps) fetch(kt + 4);
        // a wave's LDS operations run in order; the fences keep the compiler to it
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const char *row = mine + (i * 32 + r) * 128;
                bf8 a[PL];
                if constexpr (PL == 3) {
                    float v[8];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const floatx4 t = *reinterpret_cast<const floatx4 *>(row + (((s * 4 + hh * 2 + h) ^ (r & 7)) * 16));
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[4 * h + e] = t[e];
                    }
                    split8<PL>(v, a);
                } else {
                    a[0] = *reinterpret_cast<const bf8 *>(row + (((s * 2 + hh) ^ (r & 7)) * 16));
                }
#pragma unroll
                for (int j = 0; j < TN; ++j) mfma<PL, PL>(a, x[s][j], acc[i][j]);
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    // the waves' sums, 32 rows of x at a time: [entry][row] in each wave's own 8 KB
    const int i = tid & 31, g = tid >> 5;  // a thread's row, its 8 entries
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        float *w = reinterpret_cast<float *>(mine);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) w[(t * 32 + 8 * (e / 4) + 4 * hh + e % 4) * 32 + r] = acc[t][j][e];
        __syncthreads();
        float z[8], mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int at = (g * 8 + e) * 32 + i, v = v0 + g * 8 + e;
            float s = 0.0f;
#pragma unroll
            for (int q = 0; q < 4; ++q) s += reinterpret_cast<const float *>(lds[q])[at];
            float b = v < p.vocab ? (p.bias ? p.bias[v] : 0.0f) : -INFINITY;
            if (b < -1e38f && b > -INFINITY) b = -1e38f;  // the lowest value times log2(e) stays finite
            z[e] = __builtin_fmaf(s, LOG2E, b * LOG2E);
            m.z[(long)v * m.np32 + j * 32 + i] = z[e];
            mx = fmaxf(mx, z[e]);
        }
        const float ref = mx == -INFINITY ? 0.0f : mx;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s += __builtin_amdgcn_exp2f(z[e] - ref);
        red[0][g][i] = mx;
        red[1][g][i] = s;
        __syncthreads();
        if (tid < 32 && j * 32 + i < p.rows) {
#pragma unroll
            for (int q = 1; q < 8; ++q) mx = fmaxf(mx, red[0][q][i]);
            const float top = mx == -INFINITY ? 0.0f : mx;
            s = 0.0f;
#pragma unroll
            for (int q = 0; q < 8; ++q) s += red[1][q][i] * __builtin_amdgcn_exp2f(red[0][q][i] - top);
            m.pm[(long)(j * 32 + i) * m.tiles + blockIdx.x] = mx;
            m.ps[(long)(j * 32 + i) * m.tiles + blockIdx.x] = s;
        }
    }
}

// lse and loss, a block a row
__global__ __launch_bounds__(NT) void k_mid_rows(Mid m) {
    __shared__ float sm[4], ss[4];
    const LossParams &p = m.p;
    const int i = blockIdx.x, tid = threadIdx.x;
    const float *pm = m.pm + (long)i * m.tiles, *ps = m.ps + (long)i * m.tiles;
    float mx = -INFINITY, s = 0.0f;
    for (int t0 = tid; t0 < m.tiles; t0 += NT * 4) {
        float a[4], b[4], top = mx;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int t = min(t0 + u * NT, m.tiles - 1);
            a[u] = pm[t];
            b[u] = ps[t];
            if (t0 + u * NT >= m.tiles) a[u] = -INFINITY, b[u] = 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) top = fmaxf(top, a[u]);
        const float ref = top == -INFINITY ? 0.0f : top;
        s *= __builtin_amdgcn_exp2f(mx - ref);
#pragma unroll
        for (int u = 0; u < 4; ++u) s += b[u] * __builtin_amdgcn_exp2f(a[u] - ref);
        mx = top;
    }
    const float top = wave_max(mx);
    const float ref = top == -INFINITY ? 0.0f : top;
    s = wave_sum(s * __builtin_amdgcn_exp2f(mx - ref));
    if ((tid & 63) == 0) {
        sm[tid >> 6] = top;
        ss[tid >> 6] = s;
    }
    __syncthreads();
    if (tid) return;
    mx = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    const float all = mx == -INFINITY ? 0.0f : mx;
    s = 0.0f;
#pragma unroll
    for (int q = 0; q < 4; ++q) s += ss[q] * __builtin_amdgcn_exp2f(sm[q] - all);
    const float lse = all + log2f(s);
    m.lse[i] = lse;
    const int t = target_of(p, i);
    if (p.targets[i] >= p.vocab) atomicOr(p.err, ADN_DEVERR_TOKEN);
    if (p.lse) p.lse[i] = t >= 0 ? lse * LN2 : 0.0f;
    if (p.loss) p.loss[i] = t >= 0 ? (lse - m.z[(long)t * m.np32 + i]) * LN2 : 0.0f;
}

// Blocks below dx_blocks: a share of the vocabulary's part of dx, 32 CW columns (CW adjacent ones a
// lane, so that a row of W is read in whole lines straight into MFMA operands: a lane 8 entries of its
// columns).  The waves take 16 entries each in turn.  The others: dW and db of DW_TE entries.
template <typename T, int TN, int CW>
__global__ __launch_bounds__(NT, 2) void k_mid_grads(Mid m) {
    constexpr int PW = planes_of<T>(), PZ = dz_planes<T>();
    typedef T VC __attribute__((ext_vector_type(CW)));
    typedef T V4 __attribute__((ext_vector_type(4)));
    __shared__ __attribute__((aligned(16))) float lse_s[MAX_ROWS], g_s[MAX_ROWS];
    __shared__ __attribute__((aligned(16))) int t_s[MAX_ROWS];
    __shared__ float sum[3][TN * 32][32 * CW];
    const LossParams &p = m.p;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid < TN * 32) {
        lse_s[tid] = tid < p.rows ? m.lse[tid] : 0.0f;
        g_s[tid] = upstream_of(p, tid);
        t_s[tid] = target_of(p, tid);
    }
    __syncthreads();
    if ((int)blockIdx.x < m.dx_blocks) {
        const int strip = blockIdx.x % m.strips, q = blockIdx.x / m.strips;
        const int c = strip * 32 * CW + r * CW, a0 = q * m.share, a1 = min(a0 + m.share, m.tiles * TE);
        const bool in = c < p.d;
        float lse[TN], up[TN];
        int tgt[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            lse[j] = lse_s[j * 32 + r];
            up[j] = g_s[j * 32 + r];
            tgt[j] = t_s[j * 32 + r];
        }
        f16v acc[TN][CW];
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int k = 0; k < CW; ++k)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[j][k][e] = 0.0f;
        VC wn[8];
        float zn[TN][8];
        auto fetch = [&](int v) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const long at = min(v + hh * 8 + e, p.vocab - 1);
                wn[e] = *reinterpret_cast<const VC *>((const T *)p.w + at * p.w_stride + (in ? c : 0));
#pragma unroll
                for (int j = 0; j < TN; ++j) zn[j][e] = m.z[(long)(v + hh * 8 + e) * m.np32 + j * 32 + r];
            }
        };
        if (a0 + wave * 16 < a1) fetch(a0 + wave * 16);
        for (int v = a0 + wave * 16; v < a1; v += 64) {
            bf8 b[CW][PW], a[TN][PZ];
#pragma unroll
            for (int k = 0; k < CW; ++k) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = to_f32<T>(wn[e][k]);
                split8<PW>(x, b[k]);
            }
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float dz = up[j] * (__builtin_amdgcn_exp2f(zn[j][e] - lse[j]) - (v + hh * 8 + e == tgt[j] ? 1.0f : 0.0f));
                    x[e] = up[j] == 0.0f ? 0.0f : dz;
                }
                split8<PZ>(x, a[j]);
            }
            if (v + 64 < a1) fetch(v + 64);
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int k = 0; k < CW; ++k) mfma<PZ, PW>(a[j], b[k], acc[j][k]);
        }
        // the waves' sums in order
        if (wave)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e)
#pragma unroll
                    for (int k = 0; k < CW; ++k) sum[wave - 1][j * 32 + 8 * (e / 4) + 4 * hh + e % 4][r * CW + k] = acc[j][k][e];
        __syncthreads();
        if (wave || !in) return;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int i = j * 32 + 8 * (e / 4) + 4 * hh + e % 4;
                if (i >= p.rows) continue;
#pragma unroll
                for (int k = 0; k < CW; ++k) {
                    float s = acc[j][k][e];
#pragma unroll
                    for (int w = 0; w < 3; ++w) s += sum[w][i][r * CW + k];
                    m.part[((long)q * p.rows + i) * p.d + c + k] = s;
                }
            }
        return;
    }
    const int b = (int)blockIdx.x - m.dx_blocks, group = b % m.dw_groups;
    const int v0 = b / m.dw_groups * DW_TE + wave * 32, v = v0 + r;
    if (v0 >= p.vocab) return;
    bf8 a[TN * 2][PZ];
    float db = 0.0f;
#pragma unroll
    for (int k = 0; k < TN * 2; ++k) {
        const int i0 = k * 16 + hh * 8;
        float x[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const floatx4 z = *reinterpret_cast<const floatx4 *>(m.z + (long)min(v, p.vocab - 1) * m.np32 + i0 + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = i0 + 4 * h + e;
                const float g = g_s[i];
                const float dz = g * (__builtin_amdgcn_exp2f(z[e] - lse_s[i]) - (v == t_s[i] ? 1.0f : 0.0f));
                x[4 * h + e] = g == 0.0f ? 0.0f : dz;
                db += x[4 * h + e];
            }
        }
        split8<PZ>(x, a[k]);
    }
    db += __shfl_xor(db, 32, 64);
    if (p.db && group == 0 && hh == 0 && v < p.vocab) p.db[v] = db;
    if (!p.dw) return;
    T *dw = (T *)p.dw + (long)v0 * p.dw_stride;
    for (int s = group; s * STRIP < p.d; s += m.dw_groups) {
        f16v acc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < TN * 2; ++k) {
            bf8 x[4][PW];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int q = 0; q < PW; ++q) x[j][q] = m.xb[((((long)s * (TN * 2) + k) * 4 + j) * PW + q) * 64 + lane];
#pragma unroll
            for (int j = 0; j < 4; ++j) mfma<PZ, PW>(a[k], x[j], acc[j]);
        }
        const int c = s * STRIP + 4 * r;
        if (c >= p.d) continue;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int o = 8 * (e / 4) + 4 * hh + e % 4;
            if (v0 + o >= p.vocab) continue;
            T *dst = dw + (long)o * p.dw_stride + c;
            V4 w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = from_f32<T>(acc[j][e]);
            if (m.vecdw) {
                *reinterpret_cast<V4 *>(dst) = w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) dst[j] = w[j];
            }
        }
    }
}

// dx from the shares: 64 columns of a row a block, its waves a quarter of the shares each
template <typename T>
__global__ __launch_bounds__(NT) void k_mid_join(Mid m) {
    __shared__ float red[4][64];
    const LossParams &p = m.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = blockIdx.y, c = blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (c < p.d) {
#pragma unroll 16
        for (int q = wave; q < m.shares; q += 4) s += m.part[((long)q * p.rows + i) * p.d + c];
    }
    red[wave][lane] = s;
    __syncthreads();
    if (wave || c >= p.d) return;
    s = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
    ((T *)p.dx)[(long)i * p.dx_stride + c] = from_f32<T>(s);
}

struct MidLayout {
    int np32, tiles, cw, strips, shares, share;
    size_t xa, xb, z, pm, ps, lse, part, bytes;
};
MidLayout mid_layout(const LossParams &p) {
    MidLayout L{};
    L.np32 = p.rows <= 32 ? 32 : 64;
    L.tiles = (p.vocab + TE - 1) / TE;
    L.cw = L.np32 == 32 ? 4 : 2;
    L.strips = (p.d + 32 * L.cw - 1) / (32 * L.cw);
    // blocks for two a CU, shares of 64 entries at least
    const int want = std::max(1, 512 / L.strips);
    L.share = (int)(((long)L.tiles + want - 1) / want) * TE;
    L.shares = (L.tiles * TE + L.share - 1) / L.share;
    const int pl = p.dtype == ADN_T_F32 ? 3 : 1;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += (bytes + 1023) / 1024 * 1024;
        return r;
    };
    L.xa = take((size_t)L.np32 * p.d * 2 * pl);
    L.xb = take(p.dw ? (size_t)L.np32 * ((p.d + STRIP - 1) / STRIP) * STRIP * 2 * pl : 0);
    L.z = take((size_t)L.tiles * TE * L.np32 * 4);
    L.pm = take((size_t)p.rows * L.tiles * 4);
    L.ps = take((size_t)p.rows * L.tiles * 4);
    L.lse = take(MAX_ROWS * 4);
    L.part = take(p.dx ? (size_t)L.shares * p.rows * p.d * 4 : 0);
    L.bytes = at;
    return L;
}

template <typename T, int TN>
void run_mid(const LossParams &p, const MidLayout &L, char *ws, hipStream_t st) {
    Mid m{};
    m.p = p;
    m.np32 = L.np32, m.tiles = L.tiles;
    m.xa = (bf8 *)(ws + L.xa), m.xb = (bf8 *)(ws + L.xb);
    m.z = (float *)(ws + L.z), m.pm = (float *)(ws + L.pm), m.ps = (float *)(ws + L.ps), m.lse = (float *)(ws + L.lse);
    m.part = (float *)(ws + L.part);
    m.shares = L.shares, m.share = L.share, m.strips = L.strips;
    m.dx_blocks = p.dx ? L.shares * L.strips : 0;
    m.vecdw = p.dw && (uintptr_t)p.dw % 16 == 0 && p.dw_stride * (long)sizeof(T) % 16 == 0;
    const int na = p.d / 16 * TN, nb = p.dw ? (p.d + STRIP - 1) / STRIP * 4 * TN * 2 : 0;
    k_mid_prep<T><<<(unsigned)((na + nb + 3) / 4), NT, 0, st>>>(m, na, nb);
    k_mid_logits<T, TN><<<(unsigned)L.tiles, NT, 0, st>>>(m);
    k_mid_rows<<<(unsigned)p.rows, NT, 0, st>>>(m);
    // few entries: their columns are divided over more blocks, two a CU in all
    const int entry_blocks = (p.vocab + DW_TE - 1) / DW_TE;
    m.dw_groups = p.dw ? std::max(1, std::min((p.d + STRIP - 1) / STRIP, 512 / entry_blocks)) : 1;
    const int dw_blocks = p.dw || p.db ? entry_blocks * m.dw_groups : 0;
    if (m.dx_blocks + dw_blocks) k_mid_grads<T, TN, TN == 1 ? 4 : 2><<<(unsigned)(m.dx_blocks + dw_blocks), NT, 0, st>>>(m);
    if (p.dx) k_mid_join<T><<<dim3((unsigned)((p.d + 63) / 64), (unsigned)p.rows), NT, 0, st>>>(m);
}

}  // namespace

// Rows of W in whole 128-byte pieces, each 16-byte aligned.
bool loss_mid_ok(const LossParams &p) {
    const int eb = elem_bytes(p.dtype);
    return p.rows <= MAX_ROWS && p.d * eb % 128 == 0 && rows_vec16(p.w, p.w_stride, p.d, eb);
}

size_t loss_mid_workspace_bytes(const LossParams &p) { return mid_layout(p).bytes; }

void launch_loss_mid(const LossParams &p, void *ws, hipStream_t st) {
    const MidLayout L = mid_layout(p);
    dispatch_type(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        if (L.np32 == 32)
            run_mid<T, 1>(p, L, (char *)ws, st);
        else
            run_mid<T, 2>(p, L, (char *)ws, st);
    });
}

}  // namespace adn
