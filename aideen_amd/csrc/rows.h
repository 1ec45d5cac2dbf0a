// Rows held in registers by teams of lanes (norm.hip, residual.hip): where a lane's elements stand,
// their loads and stores, sums over a team.
#pragma once

#include "train.h"

namespace adn {

namespace {

constexpr int NB = 256;          // threads a block

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

}  // namespace

// dst[i][c] = the sum over the n partial rows part[i][.][c], for the dst that are not null (norm.hip)
struct SumRows {
    float *dst[3];
};
void launch_sum_rows(const float *part, int n, int d, const SumRows &to, int vectors, hipStream_t st);

}  // namespace adn
