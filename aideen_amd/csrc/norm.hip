// RMS norm of rows with a gain (the LM head's norm, lm_head.rs:35-54), forward and backward:
//
//   r = 1 / sqrt(mean(x^2) + eps),  y = x r g
//   a = dy g,  dx = r (a - x r^2 mean(a x)),  dg = sum over the rows of dy x r
//
// A team of lanes owns a row: E elements a lane, held in registers, so that a row is read once
// (backward: x and dy once, dx written once) and HBM is the bound.  Sums in fp32.  A row of up to
// 2048 elements is a wave's (its sums need no barrier), a longer one a block's.  In the backward
// pass a team walks its share of the rows and keeps the gain's gradient of its columns in
// registers; the teams' sums are written as partials and added in a fixed order, so the result
// does not depend on the schedule.
#include <algorithm>

#include "train.h"

namespace adn {

namespace {

constexpr int NB = 256;          // threads a block
constexpr int DG_BLOCKS = 512;   // most blocks of the backward pass = partial rows of dg

template <typename T, int W>
struct VecOf {
    typedef T type __attribute__((ext_vector_type(W)));
};

// Where a lane's element e of a row stands: whole 16-byte pieces (VEC: 4 fp32 or 8 bf16 values
// each) or single elements, `TEAM` lanes side by side in both.
template <typename T, int TEAM, bool VEC>
struct Cols {
    static constexpr int W = VEC ? 16 / (int)sizeof(T) : 1;
    __device__ __forceinline__ static int col(int lane, int e) { return ((e / W) * TEAM + lane) * W + e % W; }
};

// A lane's share of a row as it is loaded: E elements in pieces of W.
template <typename T, int TEAM, int E, bool VEC>
struct Row {
    typedef Cols<T, TEAM, VEC> C;
    typedef typename VecOf<T, C::W>::type V;
    V v[E / C::W];
    __device__ __forceinline__ void load(const T *row, int d, int lane) {
#pragma unroll
        for (int q = 0; q < E / C::W; ++q) {
            const int c = C::col(lane, q * C::W);
            v[q] = V{};
            if (c < d) v[q] = *reinterpret_cast<const V *>(row + c);
        }
    }
    __device__ __forceinline__ float operator[](int e) const { return to_f32<T>(v[e / C::W][e % C::W]); }
};

template <typename T, int TEAM, int E, bool VEC>
__device__ __forceinline__ void store_row(T *row, int d, int lane, const float (&v)[E]) {
    typedef Cols<T, TEAM, VEC> C;
    if constexpr (VEC) {
        typedef typename VecOf<T, C::W>::type V;
#pragma unroll
        for (int e = 0; e < E; e += C::W) {
            const int c = C::col(lane, e);
            if (c < d) {
                V x;
#pragma unroll
                for (int j = 0; j < C::W; ++j) x[j] = from_f32<T>(v[e + j]);
                *reinterpret_cast<V *>(row + c) = x;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = C::col(lane, e);
            if (c < d) row[c] = from_f32<T>(v[e]);
        }
    }
}

// The gain of a lane's columns (1 where there is none; 0 beyond the row is never used).
template <typename T, int TEAM, int E, bool VEC>
__device__ __forceinline__ void load_gain(const float *gain, int d, int lane, float (&g)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = Cols<T, TEAM, VEC>::col(lane, e);
        g[e] = gain && c < d ? gain[c] : 1.0f;
    }
}

// Sums of N values over the team; every lane of it gets them.
template <int TEAM, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float (*red)[NB / 64]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if constexpr (TEAM > 64) {
        __syncthreads();  // the last row's sums have been read
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) red[i][threadIdx.x >> 6] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < TEAM / 64; ++w) s += red[i][w];
            v[i] = s;
        }
    }
}

template <typename T, int TEAM, int E, bool VEC>
__global__ __launch_bounds__(NB) void k_rms_norm(NormParams p) {
    __shared__ float red[1][NB / 64];
    const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
    const long row = (long)blockIdx.x * (NB / TEAM) + team;
    if (row >= p.rows) return;  // a whole wave (TEAM 64) or never (a block a row)
    Row<T, TEAM, E, VEC> x;
    float v[E], g[E];
    x.load((const T *)p.x + row * p.x_stride, p.d, lane);
    load_gain<T, TEAM, E, VEC>(p.gain, p.d, lane, g);
    float s[1] = {0.0f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] = x[e];
        s[0] += v[e] * v[e];
    }
    team_sum<TEAM, 1>(s, red);
    const float r = 1.0f / sqrtf(s[0] / (float)p.d + p.eps);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = v[e] * r * g[e];
    store_row<T, TEAM, E, VEC>((T *)p.y + row * p.y_stride, p.d, lane, v);
}

template <typename T, int TEAM, int E, bool VEC>
__global__ __launch_bounds__(NB) void k_rms_norm_back(NormParams p, float *part) {
    __shared__ float red[2][NB / 64];
    constexpr int TEAMS = NB / TEAM;
    const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
    float g[E], dg[E];
    load_gain<T, TEAM, E, VEC>(p.gain, p.d, lane, g);
#pragma unroll
    for (int e = 0; e < E; ++e) dg[e] = 0.0f;
    // the next row is loaded while this one is used
    const long step = (long)gridDim.x * TEAMS;
    long row = (long)blockIdx.x * TEAMS + team;
    Row<T, TEAM, E, VEC> xn, dyn;
    if (row < p.rows) {
        xn.load((const T *)p.x + row * p.x_stride, p.d, lane);
        dyn.load((const T *)p.dy + row * p.dy_stride, p.d, lane);
    }
    for (; row < p.rows; row += step) {
        const Row<T, TEAM, E, VEC> x = xn, dy = dyn;
        if (row + step < p.rows) {
            xn.load((const T *)p.x + (row + step) * p.x_stride, p.d, lane);
            dyn.load((const T *)p.dy + (row + step) * p.dy_stride, p.d, lane);
        }
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e) {
            s[0] += x[e] * x[e];
            s[1] += dy[e] * g[e] * x[e];
        }
        team_sum<TEAM, 2>(s, red);
        const float r = 1.0f / sqrtf(s[0] / (float)p.d + p.eps);
        const float k = r * r * (s[1] / (float)p.d);
        float dx[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            dg[e] += dy[e] * (x[e] * r);
            dx[e] = r * (dy[e] * g[e] - x[e] * k);
        }
        if (p.dx) store_row<T, TEAM, E, VEC>((T *)p.dx + row * p.dx_stride, p.d, lane, dx);
    }
    if (!part) return;
    // the block's teams in order, then one partial row a block
    if constexpr (TEAMS > 1) {
        __shared__ float sum[TEAMS][64][E + 1];
#pragma unroll
        for (int e = 0; e < E; ++e) sum[team][lane][e] = dg[e];
        __syncthreads();
        if (team) return;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            dg[e] = sum[0][lane][e];
#pragma unroll
            for (int t = 1; t < TEAMS; ++t) dg[e] += sum[t][lane][e];
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = Cols<T, TEAM, VEC>::col(lane, e);
        if (c < p.d) part[(long)blockIdx.x * p.d + c] = dg[e];
    }
}

// dst[c] = sum over the n partial rows: 16 waves of a block each take a share of the rows of 64 columns
// in order, then the shares in order.
__global__ __launch_bounds__(1024) void k_sum_rows(const float *part, int n, int d, float *dst) {
    constexpr int WAVES = 16;
    __shared__ float red[WAVES][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;
    const int per = (n + WAVES - 1) / WAVES;
    const int a = w * per, b = min(n, a + per);
    float s = 0.0f;
    if (c < d) {
#pragma unroll 16
        for (int i = a; i < b; ++i) s += part[(long)i * d + c];
    }
    red[w][lane] = s;
    __syncthreads();
    if (w == 0 && c < d) {
#pragma unroll
        for (int q = 1; q < WAVES; ++q) s += red[q][lane];
        dst[c] = s;
    }
}

// f(TEAM, E): the smallest team and share that hold a row (E a multiple of 8: whole 16-byte pieces)
template <typename F>
void dispatch_row(int d, F &&f) {
    using std::integral_constant;
    if (d <= 512)
        f(integral_constant<int, 64>{}, integral_constant<int, 8>{});
    else if (d <= 1024)
        f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
    else if (d <= 2048)
        f(integral_constant<int, 64>{}, integral_constant<int, 32>{});
    else
        f(integral_constant<int, 256>{}, integral_constant<int, 32>{});
}

int back_blocks(const NormParams &p) {
    const int teams = p.d <= 2048 ? NB / 64 : 1;
    return (int)std::min<long>(DG_BLOCKS, ((long)p.rows + teams - 1) / teams);
}

}  // namespace

void launch_norm(const NormParams &p, hipStream_t st) {
    if (p.rows == 0) return;
    const int eb = elem_bytes(p.dtype);
    const bool vec = rows_vec16(p.x, p.x_stride, p.d, eb) && rows_vec16(p.y, p.y_stride, p.d, eb);
    // a launch has less than 2^32 threads: 2^23 rows at a time, a block a row at most
    NormParams q = p;
    for (int row = 0; row < p.rows; row += 1 << 23) {
        q.rows = std::min(p.rows - row, 1 << 23);
        q.x = (const char *)p.x + row * p.x_stride * eb;
        q.y = (char *)p.y + row * p.y_stride * eb;
        dispatch_type(p.dtype, [&](auto t) {
            typedef decltype(t) T;
            dispatch_row(p.d, [&](auto team, auto e) {
                constexpr int TEAM = decltype(team)::value, E = decltype(e)::value;
                const dim3 grid((unsigned)(((long)q.rows * TEAM + NB - 1) / NB));
                if (vec)
                    k_rms_norm<T, TEAM, E, true><<<grid, NB, 0, st>>>(q);
                else
                    k_rms_norm<T, TEAM, E, false><<<grid, NB, 0, st>>>(q);
            });
        });
    }
}

size_t norm_backward_workspace_bytes(const NormParams &p) {
    return p.dg ? (size_t)back_blocks(p) * p.d * sizeof(float) : 0;
}

void launch_norm_backward(const NormParams &p, void *ws, hipStream_t st) {
    const int eb = elem_bytes(p.dtype), blocks = back_blocks(p);
    const bool vec = rows_vec16(p.x, p.x_stride, p.d, eb) && rows_vec16(p.dy, p.dy_stride, p.d, eb) &&
                     (!p.dx || rows_vec16(p.dx, p.dx_stride, p.d, eb));
    float *part = p.dg ? (float *)ws : nullptr;
    if (blocks)
        dispatch_type(p.dtype, [&](auto t) {
            typedef decltype(t) T;
            dispatch_row(p.d, [&](auto team, auto e) {
                constexpr int TEAM = decltype(team)::value, E = decltype(e)::value;
                if (vec)
                    k_rms_norm_back<T, TEAM, E, true><<<blocks, NB, 0, st>>>(p, part);
                else
                    k_rms_norm_back<T, TEAM, E, false><<<blocks, NB, 0, st>>>(p, part);
            });
        });
    if (p.dg) k_sum_rows<<<(p.d + 63) / 64, 1024, 0, st>>>(part, blocks, p.d, p.dg);
}

}  // namespace adn
