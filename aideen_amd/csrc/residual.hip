// The norms around a residual block, forward and backward, each row in one pass:
//
//   n = f rf gp  (rf = 1 / sqrt(mean(f^2) + eps); n = f without the norm)
//   z = keep x + scale s n,   s the gate (1 without one; sigmoid of it where it is given as logits)
//   y = z rz gq,  rz = 1 / sqrt(mean(z^2) + eps)
//
//   D = dz + rz (a - z rz^2 mean(a z)),  a = dy gq
//   dx = keep D,  ds = scale D n (times s (1 - s) for logits),  dn = scale D s
//   df = rf (b - f rf^2 mean(b f)),  b = dn gp;   dgp = sum over the rows of dn f rf;  dgq of dy z rz
//
// A team of lanes owns a row and keeps all of its tensors in registers between the reductions, so
// that each is read or written once and HBM is the bound.  Sums in fp32.  Rows of up to 512
// elements are a wave's (no barriers), longer ones a block's of 2, 4 or 8 waves.  A team walks its share of
// the rows, the next one loaded while one is used; in the backward pass it keeps the column sums in
// registers, the blocks' sums are written as partials and added in a fixed order.
#include <algorithm>

#include "train.h"

namespace adn {

namespace {

// Blocks of a launch, which walk the rows: two a CU, or three in the forward pass of longer rows.  More rows in flight
// read no faster and spread the memory's open pages (8192 x 512 fp32 forward: 512 blocks 13.8 us, 1024 15.2, 2048 19.5;
// 32749 x 2048 bf16, a gate an element and without one: 512 blocks 138 and 114, 768 123 and 94, 1024 125 and 97; backward: 256
// blocks 268, 512 217, 1024 239, 2048 243).  Rows by single elements alone would have more: 20000 x 1535 bf16 forward 65,
// with 1024 blocks 58.
constexpr int ROW_BLOCKS = 512, WIDE_BLOCKS = 768;  // forward: of rows of a wave, and longer ones
constexpr int NB = 256;           // threads of a block of four waves' teams
constexpr int MAX_TEAM = 512;     // lanes of the longest rows
constexpr int COL_BLOCKS = 512;  // most blocks of the backward pass = partial rows of a column sum

// A lane's elements of a row.
constexpr int elements(int team) { return team < MAX_TEAM ? 8 : 16; }

// A block's threads: four teams of a wave, or one of more waves.
constexpr int block_threads(int team) { return team > 64 ? team : NB; }

// The gate's value s and ds / dgate.  The exponential is taken of -|g|: it cannot overflow, and
// s (1 - s) = t / (1 + t)^2 loses nothing where s is near 1.  exp(a) = 2^e (1 + ln 2 r), e the rounded and r what the
// rounding of a log2(e) leaves; 2^e and the reciprocal to 1 ulp (a gate below 2^-126 is 0).
__device__ __forceinline__ float gate_value(float g, bool sigmoid, float &slope) {
    if (!sigmoid) {
        slope = 1.0f;
        return g;
    }
    constexpr float LOG2E = 1.44269502f, REST = 1.92596303e-8f, LN2 = 0.693147182f;
    const float a = -fabsf(g) < -150.0f ? -150.0f : -fabsf(g);  // below, the exponential is 0 (and a NaN stays)
    const float e = a * LOG2E, r = fmaf(a, REST, fmaf(a, LOG2E, -e));
    const float p = __builtin_amdgcn_exp2f(e), t = fmaf(p, LN2 * r, p), i = __builtin_amdgcn_rcpf(1.0f + t);
    slope = t * i * i;
    return g >= 0.0f ? i : t * i;
}

// Sums of N values over the team, in every lane of it: six steps across a wave's lanes, then (teams of
// several waves) a place in LDS a wave.  `turn` alternates from call to call, so that one barrier a call is
// enough: a place is written again two calls later, behind the barrier of the call between, which a
// wave reaches when it has read what stood there.
template <int TEAM, int N>
__device__ __forceinline__ void team_add(float (&v)[N], float (*red)[3][MAX_TEAM / 64], int &turn) {
#define ADN_DPP_ADD(ctrl, rows) \
    _Pragma("unroll") for (int i = 0; i < N; ++i) \
        v[i] += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v[i]), ctrl, rows, 0xF, true))
    ADN_DPP_ADD(0x111, 0xF);  // from the lane one, two, four, eight to the left in a row of 16
    ADN_DPP_ADD(0x112, 0xF);
    ADN_DPP_ADD(0x114, 0xF);
    ADN_DPP_ADD(0x118, 0xF);
    ADN_DPP_ADD(0x142, 0xA);  // a row's last lane to the next row, then to the upper half
    ADN_DPP_ADD(0x143, 0xC);
#undef ADN_DPP_ADD
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v[i]), 63));
    if constexpr (TEAM > 64) {  // the team is the block
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) red[turn][i][threadIdx.x >> 6] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < TEAM / 64; ++w) s += red[turn][i][w];
            v[i] = s;
        }
        turn ^= 1;
    }
}

// A lane's share of a row: E elements, TEAM lanes side by side, in whole aligned pieces of 16 bytes (VEC) or by single elements.
// Pieces that are not aligned cost more than elements do (8191 x 777 fp32 backward 45 us by elements, 82 by pieces at any address; 20000 x 1535
// bf16 133 and 405).  STREAM: past the caches, as all stores of pieces go.
template <typename T, int TEAM, bool VEC>
struct Row {
    static constexpr int E = elements(TEAM), W = VEC ? 16 / (int)sizeof(T) : 1;
    typedef T V __attribute__((ext_vector_type(W)));
    V v[E / W];
    __device__ __forceinline__ static int col(int lane, int e) { return ((e / W) * TEAM + lane) * W + e % W; }
    __device__ __forceinline__ float operator[](int e) const { return to_f32<T>(v[e / W][e % W]); }
    template <bool STREAM>
    __device__ __forceinline__ void load(const T *row, int d, int lane) {
#pragma unroll
        for (int q = 0; q < E / W; ++q) {
            const int c = col(lane, q * W);
            v[q] = V{};
            if (c < d) {
                if constexpr (STREAM)
                    v[q] = __builtin_nontemporal_load(reinterpret_cast<const V *>(row + c));
                else
                    v[q] = *reinterpret_cast<const V *>(row + c);
            }
        }
    }
    __device__ __forceinline__ static void store(T *row, int d, int lane, const float (&x)[E]) {
#pragma unroll
        for (int q = 0; q < E / W; ++q) {
            const int c = col(lane, q * W);
            V y;
#pragma unroll
            for (int j = 0; j < W; ++j) y[j] = from_f32<T>(x[q * W + j]);
            if (c < d) {
                if constexpr (VEC)
                    __builtin_nontemporal_store(y, reinterpret_cast<V *>(row + c));
                else
                    *reinterpret_cast<V *>(row + c) = y;
            }
        }
    }
};

// What a lane has of a row's inputs, loaded ahead.
template <typename T, int TEAM, bool VEC, bool STREAM, bool BACK>
struct Inputs {
    typedef Row<T, TEAM, VEC> R;
    R a, f, g, dz, dy;  // a: x, or z in the backward pass
    float row_gate;
    __device__ __forceinline__ void load(const ResidualParams &p, long row, int lane) {
        auto take = [&](R &r, const void *base, long stride) {
            r.template load<STREAM>((const T *)base + row * stride, p.d, lane);
        };
        take(f, p.f, p.f_stride);
        if constexpr (BACK) {
            if (p.dy) take(a, p.z, p.z_stride), take(dy, p.dy, p.dy_stride);
            if (p.dz) take(dz, p.dz, p.dz_stride);
        } else {
            take(a, p.x, p.x_stride);
        }
        if (p.gate_kind == ADN_GATE_ELEMENT) take(g, p.gate, p.gate_stride);
        if (p.gate_kind == ADN_GATE_ROW) row_gate = ((const float *)p.gate)[row];
    }
};

template <typename T, int TEAM, bool VEC, bool STREAM>
__global__ __launch_bounds__(block_threads(TEAM)) void k_residual(ResidualParams p) {
    __shared__ float red[2][3][MAX_TEAM / 64];
    typedef Row<T, TEAM, VEC> C;
    constexpr int E = elements(TEAM), TEAMS = block_threads(TEAM) / TEAM;
    const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
    const long step = (long)gridDim.x * TEAMS;
    long row = (long)blockIdx.x * TEAMS + team;
    if (row >= p.rows) return;  // a whole wave (TEAM 64) or never (a block a row)
    Inputs<T, TEAM, VEC, STREAM, false> in, next;
    in.load(p, row, lane);
    float w[E], gq[E], slope;  // scale, the gain and a gate of the channels
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = C::col(lane, e);
        w[e] = p.scale;
        gq[e] = 1.0f;
        if (c < p.d) {
            if (p.post_gain) w[e] *= p.post_gain[c];
            if (p.gate_kind == ADN_GATE_CHANNEL) w[e] *= gate_value(((const float *)p.gate)[c], p.sigmoid, slope);
            if (p.pre_gain) gq[e] = p.pre_gain[c];
        }
    }
    const float inv_d = 1.0f / (float)p.d;
    int turn = 0;
    for (; row < p.rows; row += step) {
        if (row + step < p.rows) next.load(p, row + step, lane);
        float rf = 1.0f;
        if (p.post) {
            float s[1] = {0.0f};
#pragma unroll
            for (int e = 0; e < E; ++e) s[0] += in.f[e] * in.f[e];
            team_add<TEAM, 1>(s, red, turn);
            rf = 1.0f / sqrtf(s[0] * inv_d + p.eps);
        }
        if (p.gate_kind == ADN_GATE_ROW) rf *= gate_value(in.row_gate, p.sigmoid, slope);
        float v[E], s[1] = {0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float n = in.f[e] * rf * w[e];
            if (p.gate_kind == ADN_GATE_ELEMENT) n *= gate_value(in.g[e], p.sigmoid, slope);
            v[e] = p.keep * in.a[e] + n;
            s[0] += v[e] * v[e];
        }
        if (p.z) C::store((T *)p.z + row * p.z_stride, p.d, lane, v);
        if (p.y) {
            team_add<TEAM, 1>(s, red, turn);
            const float rz = 1.0f / sqrtf(s[0] * inv_d + p.eps);
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] *= rz * gq[e];
            C::store((T *)p.y + row * p.y_stride, p.d, lane, v);
        }
        in = next;
    }
}

// The column sums need two accumulators: A, the sum of u f rf (u = scale D, times a row's or an element's gate), which is
// dgp but for a channel's gate, and that gate's gradient but for dgp's factor; and dgq.
template <typename T, int TEAM, bool VEC, bool STREAM, uint32_t GATE>
__global__ __launch_bounds__(block_threads(TEAM)) void k_residual_back(ResidualParams p, float *part) {
    __shared__ float red[2][3][MAX_TEAM / 64];
    typedef Row<T, TEAM, VEC> C;
    constexpr int E = elements(TEAM), TEAMS = block_threads(TEAM) / TEAM;
    p.gate_kind = GATE;
    const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
    const long step = (long)gridDim.x * TEAMS;
    long row = (long)blockIdx.x * TEAMS + team;
    constexpr bool AHEAD = TEAM < MAX_TEAM;  // the next row is loaded while this one is used, where there are registers
    Inputs<T, TEAM, VEC, STREAM, true> in, next;
    if (AHEAD && row < p.rows) in.load(p, row, lane);
    float w[E], gq[E], A[E], dgq[E], slope;  // w: the gain, times a gate of the channels
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = C::col(lane, e);
        w[e] = gq[e] = 1.0f;
        A[e] = dgq[e] = 0.0f;
        if (c < p.d) {
            if (p.post_gain) w[e] = p.post_gain[c];
            if (GATE == ADN_GATE_CHANNEL) w[e] *= gate_value(((const float *)p.gate)[c], p.sigmoid, slope);
            if (p.pre_gain) gq[e] = p.pre_gain[c];
        }
    }
    const float inv_d = 1.0f / (float)p.d;
    int turn = 0;
    for (; row < p.rows; row += step) {
        if (!AHEAD)
            in.load(p, row, lane);
        else if (row + step < p.rows)
            next.load(p, row + step, lane);
        float s[3] = {0.0f, 0.0f, 0.0f};
        if (p.dy) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                s[0] += in.a[e] * in.a[e];
                s[1] += in.dy[e] * gq[e] * in.a[e];
            }
        }
        if (p.post) {
#pragma unroll
            for (int e = 0; e < E; ++e) s[2] += in.f[e] * in.f[e];
        }
        team_add<TEAM, 3>(s, red, turn);
        const float rf = p.post ? 1.0f / sqrtf(s[2] * inv_d + p.eps) : 1.0f;
        float D[E];
#pragma unroll
        for (int e = 0; e < E; ++e) D[e] = p.dz ? in.dz[e] : 0.0f;
        if (p.dy) {
            const float rz = 1.0f / sqrtf(s[0] * inv_d + p.eps), k = rz * rz * (s[1] * inv_d);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                dgq[e] += in.dy[e] * (in.a[e] * rz);
                D[e] += rz * (in.dy[e] * gq[e] - in.a[e] * k);
            }
        }
        if (p.dx) {
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = p.keep * D[e];
            C::store((T *)p.dx + row * p.dx_stride, p.d, lane, v);
        }
        // D becomes b = scale D s gp
        float slope_r = 1.0f, gate_r = 1.0f, t[2] = {0.0f, 0.0f};
        if (GATE == ADN_GATE_ROW) gate_r = gate_value(in.row_gate, p.sigmoid, slope_r);
        float dg[GATE == ADN_GATE_ELEMENT ? E : 1];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float fr = in.f[e] * rf;
            float u = p.scale * D[e];
            if (GATE == ADN_GATE_ROW) {
                t[1] += u * fr * w[e];
                u *= gate_r;
            }
            if constexpr (GATE == ADN_GATE_ELEMENT) {
                const float g = gate_value(in.g[e], p.sigmoid, slope);
                dg[e] = u * fr * w[e] * slope;
                u *= g;
            }
            A[e] += u * fr;
            D[e] = u * w[e];
            t[0] += D[e] * in.f[e];
        }
        if constexpr (GATE == ADN_GATE_ELEMENT)
            if (p.dgate) C::store((T *)p.dgate + row * p.dgate_stride, p.d, lane, dg);
        team_add<TEAM, 2>(t, red, turn);
        if (GATE == ADN_GATE_ROW && p.dgate && lane == 0) ((float *)p.dgate)[row] = t[1] * slope_r;
        if (p.df) {
            if (p.post) {  // without the norm df is b, whatever f holds
                const float k = rf * rf * (t[0] * inv_d);
#pragma unroll
                for (int e = 0; e < E; ++e) D[e] = rf * (D[e] - in.f[e] * k);
            }
            C::store((T *)p.df + row * p.df_stride, p.d, lane, D);
        }
        if (AHEAD) in = next;
    }
    if (!part) return;
    // the block's teams in order, then one partial row a block of A and of dgq
    if constexpr (TEAMS > 1) {
        __shared__ float sum[TEAMS][64][2 * E + 1];
#pragma unroll
        for (int e = 0; e < E; ++e) sum[team][lane][e] = A[e], sum[team][lane][E + e] = dgq[e];
        __syncthreads();
        if (team) return;
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int q = 1; q < TEAMS; ++q) A[e] += sum[q][lane][e], dgq[e] += sum[q][lane][E + e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = C::col(lane, e);
        if (c < p.d) {
            part[(long)blockIdx.x * p.d + c] = A[e];
            part[((long)gridDim.x + blockIdx.x) * p.d + c] = dgq[e];
        }
    }
}

// The column sums: 64 threads a column each take every 64th of its n partial sums in order, then a tree.  Behind
// them A's factors: dgp = A times a channel's gate, that gate's gradient = A times the gain (and the slope).
__global__ __launch_bounds__(1024) void k_residual_join(ResidualParams p, const float *part, int n) {
    constexpr int COLS = 16, GROUPS = 64;
    __shared__ float red[GROUPS][COLS + 1];
    const int col = threadIdx.x % COLS, g = threadIdx.x / COLS, c = blockIdx.x * COLS + col;
    const bool second = blockIdx.y;
    const float *src = part + (second ? (long)n * p.d : 0);
    float s = 0.0f;
    if (c < p.d) {
#pragma unroll 8
        for (int i = g; i < n; i += GROUPS) s += src[(long)i * p.d + c];
    }
    red[g][col] = s;
#pragma unroll
    for (int k = GROUPS / 2; k; k >>= 1) {
        __syncthreads();
        if (g < k) red[g][col] += red[g + k][col];
    }
    if (g || c >= p.d) return;
    s = red[0][col];
    if (second) {
        if (p.dpre) p.dpre[c] = s;
        return;
    }
    float gate = 1.0f, slope = 1.0f;
    const bool channel = p.gate_kind == ADN_GATE_CHANNEL;
    if (channel) gate = gate_value(((const float *)p.gate)[c], p.sigmoid, slope);
    if (p.dpost) p.dpost[c] = s * gate;
    if (p.dgate && channel) ((float *)p.dgate)[c] = s * (p.post_gain ? p.post_gain[c] : 1.0f) * slope;
}

// f(TEAM): the smallest team that holds a row
template <typename F>
void dispatch_row(int d, F &&f) {
    using std::integral_constant;
    if (d <= 64 * elements(64))
        f(integral_constant<int, 64>{});
    else if (d <= 128 * elements(128))
        f(integral_constant<int, 128>{});
    else if (d <= 256 * elements(256))
        f(integral_constant<int, 256>{});
    else
        f(integral_constant<int, MAX_TEAM>{});
}

bool column_sums(const ResidualParams &p) { return p.dpost || p.dpre || (p.dgate && p.gate_kind == ADN_GATE_CHANNEL); }

// A call reads past the caches where three of its matrices (backward six) are more than their 256 MB; it has up to five (up to
// eight).  What is best depends on what the call finds there: rows of 512 fp32, forward with z alone, us through the caches and past
// them, 84 MB a matrix: 38 and 41 behind a call on the same tensors, 47 and 42 behind one on others; 101 MB: 45 and 49, 56 and 51;
// 17 MB: 9.0 and 9.6, 10.1 and 11.3.  Backward, 42 MB: 42 and 48, 52 and 49; 50 MB: 49 and 56, 61 and 57.
bool streams(const ResidualParams &p, int matrices) {
    return (double)p.rows * p.d * elem_bytes(p.dtype) * matrices > 256e6;
}

int back_blocks(const ResidualParams &p) {
    const int teams = p.d <= 64 * elements(64) ? NB / 64 : 1;
    return (int)std::min<long>(COL_BLOCKS, ((long)p.rows + teams - 1) / teams);
}

// f(GATE) for the kind of gate
template <typename F>
void dispatch_gate(uint32_t kind, F &&f) {
    using std::integral_constant;
    if (kind == ADN_GATE_NONE)
        f(integral_constant<uint32_t, ADN_GATE_NONE>{});
    else if (kind == ADN_GATE_CHANNEL)
        f(integral_constant<uint32_t, ADN_GATE_CHANNEL>{});
    else if (kind == ADN_GATE_ROW)
        f(integral_constant<uint32_t, ADN_GATE_ROW>{});
    else
        f(integral_constant<uint32_t, ADN_GATE_ELEMENT>{});
}

}  // namespace

void launch_residual(const ResidualParams &p, hipStream_t st) {
    if (p.rows == 0) return;
    const int eb = elem_bytes(p.dtype);
    auto ok = [&](const void *q, long stride) { return !q || rows_vec16(q, stride, p.d, eb); };
    const bool vec = ok(p.x, p.x_stride) && ok(p.f, p.f_stride) && ok(p.z, p.z_stride) && ok(p.y, p.y_stride) &&
                     (p.gate_kind != ADN_GATE_ELEMENT || ok(p.gate, p.gate_stride));
    dispatch_type(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        dispatch_row(p.d, [&](auto team) {
            constexpr int TEAM = decltype(team)::value, BLOCK = block_threads(TEAM);
            const unsigned grid = (unsigned)std::min<long>(((long)p.rows * TEAM + BLOCK - 1) / BLOCK, TEAM > 64 ? WIDE_BLOCKS : ROW_BLOCKS);
            if (vec && streams(p, 3))
                k_residual<T, TEAM, true, true><<<grid, BLOCK, 0, st>>>(p);
            else if (vec)
                k_residual<T, TEAM, true, false><<<grid, BLOCK, 0, st>>>(p);
            else
                k_residual<T, TEAM, false, false><<<grid, BLOCK, 0, st>>>(p);
        });
    });
}

size_t residual_backward_workspace_bytes(const ResidualParams &p) {
    return column_sums(p) ? (size_t)2 * back_blocks(p) * p.d * sizeof(float) : 0;
}

void launch_residual_backward(const ResidualParams &p, void *ws, hipStream_t st) {
    const int blocks = back_blocks(p), eb = elem_bytes(p.dtype);
    auto ok = [&](const void *q, long stride) { return !q || rows_vec16(q, stride, p.d, eb); };
    const bool vec = ok(p.z, p.z_stride) && ok(p.f, p.f_stride) && ok(p.dz, p.dz_stride) && ok(p.dy, p.dy_stride) && ok(p.dx, p.dx_stride) &&
                     ok(p.df, p.df_stride) && (p.gate_kind != ADN_GATE_ELEMENT || (ok(p.gate, p.gate_stride) && ok(p.dgate, p.dgate_stride)));
    float *part = column_sums(p) ? (float *)ws : nullptr;
    if (blocks)
        dispatch_type(p.dtype, [&](auto t) {
            typedef decltype(t) T;
            dispatch_row(p.d, [&](auto team) {
                constexpr int TEAM = decltype(team)::value, BLOCK = block_threads(TEAM);
                dispatch_gate(p.gate_kind, [&](auto gate) {
                    constexpr uint32_t GATE = decltype(gate)::value;
                    if (vec && streams(p, 6))
                        k_residual_back<T, TEAM, true, true, GATE><<<blocks, BLOCK, 0, st>>>(p, part);
                    else if (vec)
                        k_residual_back<T, TEAM, true, false, GATE><<<blocks, BLOCK, 0, st>>>(p, part);
                    else
                        k_residual_back<T, TEAM, false, false, GATE><<<blocks, BLOCK, 0, st>>>(p, part);
                });
            });
        });
    if (column_sums(p)) k_residual_join<<<dim3((p.d + 15) / 16, 2), 1024, 0, st>>>(p, part, blocks);
}

}  // namespace adn
