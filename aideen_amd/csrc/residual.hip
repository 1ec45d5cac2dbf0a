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
// that each is read or written once and HBM is the bound.  Sums in fp32.  Rows of up to 1024
// elements are a wave's (no barriers), longer ones a block's.  In the backward pass a team walks its
// share of the rows and keeps the column sums in registers; the blocks' sums are written as partials
// and added in a fixed order.
#include <algorithm>

#include "rows.h"

namespace adn {

namespace {

constexpr int COL_BLOCKS = 512;  // most blocks of the backward pass = partial rows of a column sum

// The gate's value s and ds / dgate.  The exponential is taken of -|g|: it cannot overflow, and
// s (1 - s) = t / (1 + t)^2 loses nothing where s is near 1.
__device__ __forceinline__ float gate_value(float g, bool sigmoid, float &slope) {
    if (!sigmoid) {
        slope = 1.0f;
        return g;
    }
    const float t = expf(-fabsf(g)), i = 1.0f / (1.0f + t);
    slope = t * i * i;
    return g >= 0.0f ? i : t * i;
}

template <typename T, int TEAM, int E, bool VEC>
__global__ __launch_bounds__(NB) void k_residual(ResidualParams p) {
    __shared__ float red[1][NB / 64];
    typedef Cols<T, TEAM, VEC> C;
    const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
    const long row = (long)blockIdx.x * (NB / TEAM) + team;
    if (row >= p.rows) return;  // a whole wave (TEAM 64) or never (a block a row)
    Row<T, TEAM, E, VEC> x, f, gr;
    x.load((const T *)p.x + row * p.x_stride, p.d, lane);
    f.load((const T *)p.f + row * p.f_stride, p.d, lane);
    if (p.gate_kind == ADN_GATE_ELEMENT) gr.load((const T *)p.gate + row * p.gate_stride, p.d, lane);
    float slope, row_gate = 1.0f;
    if (p.gate_kind == ADN_GATE_ROW) row_gate = gate_value(((const float *)p.gate)[row], p.sigmoid, slope);
    float rf = 1.0f;
    if (p.post) {
        float s[1] = {0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e) s[0] += f[e] * f[e];
        team_sum<TEAM, 1>(s, red);
        rf = 1.0f / sqrtf(s[0] / (float)p.d + p.eps);
    }
    float v[E], s[1] = {0.0f};
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = C::col(lane, e);
        float n = f[e] * rf, g = row_gate;
        if (p.post_gain && c < p.d) n *= p.post_gain[c];
        if (p.gate_kind == ADN_GATE_CHANNEL)
            g = c < p.d ? gate_value(((const float *)p.gate)[c], p.sigmoid, slope) : 0.0f;
        else if (p.gate_kind == ADN_GATE_ELEMENT)
            g = gate_value(gr[e], p.sigmoid, slope);
        v[e] = c < p.d ? p.keep * x[e] + p.scale * g * n : 0.0f;
        s[0] += v[e] * v[e];
    }
    if (p.z) store_row<T, TEAM, E, VEC>((T *)p.z + row * p.z_stride, p.d, lane, v);
    if (!p.y) return;
    team_sum<TEAM, 1>(s, red);
    const float rz = 1.0f / sqrtf(s[0] / (float)p.d + p.eps);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = C::col(lane, e);
        v[e] *= rz;
        if (p.pre_gain && c < p.d) v[e] *= p.pre_gain[c];
    }
    store_row<T, TEAM, E, VEC>((T *)p.y + row * p.y_stride, p.d, lane, v);
}

template <typename T, int TEAM, int E, bool VEC>
__global__ __launch_bounds__(NB) void k_residual_back(ResidualParams p, float *part) {
    __shared__ float red[2][NB / 64];
    typedef Cols<T, TEAM, VEC> C;
    constexpr int TEAMS = NB / TEAM;
    const int team = threadIdx.x / TEAM, lane = threadIdx.x % TEAM;
    const bool channel = p.gate_kind == ADN_GATE_CHANNEL, element = p.gate_kind == ADN_GATE_ELEMENT;
    float gp[E], gq[E], gc[E], slope_c[E], dgp[E], dgq[E], dgc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int c = C::col(lane, e);
        gp[e] = p.post_gain && c < p.d ? p.post_gain[c] : 1.0f;
        gq[e] = p.pre_gain && c < p.d ? p.pre_gain[c] : 1.0f;
        gc[e] = slope_c[e] = 1.0f;
        if (channel && c < p.d) gc[e] = gate_value(((const float *)p.gate)[c], p.sigmoid, slope_c[e]);
        dgp[e] = dgq[e] = dgc[e] = 0.0f;
    }
    const float inv_d = 1.0f / (float)p.d;
    for (long row = (long)blockIdx.x * TEAMS + team; row < p.rows; row += (long)gridDim.x * TEAMS) {
        Row<T, TEAM, E, VEC> z, f, dz, dy, gr;
        z.load((const T *)p.z + row * p.z_stride, p.d, lane);
        f.load((const T *)p.f + row * p.f_stride, p.d, lane);
        if (p.dz) dz.load((const T *)p.dz + row * p.dz_stride, p.d, lane);
        if (p.dy) dy.load((const T *)p.dy + row * p.dy_stride, p.d, lane);
        if (element) gr.load((const T *)p.gate + row * p.gate_stride, p.d, lane);
        float slope_r = 1.0f, gate_r = 1.0f;
        if (p.gate_kind == ADN_GATE_ROW) gate_r = gate_value(((const float *)p.gate)[row], p.sigmoid, slope_r);
        float D[E];
#pragma unroll
        for (int e = 0; e < E; ++e) D[e] = p.dz ? dz[e] : 0.0f;
        float rf = 1.0f;
        if (p.dy) {
            float s[2] = {0.0f, 0.0f};
#pragma unroll
            for (int e = 0; e < E; ++e) {
                s[0] += z[e] * z[e];
                s[1] += dy[e] * gq[e] * z[e];
            }
            team_sum<TEAM, 2>(s, red);
            const float rz = 1.0f / sqrtf(s[0] * inv_d + p.eps), k = rz * rz * (s[1] * inv_d);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                dgq[e] += dy[e] * (z[e] * rz);
                D[e] += rz * (dy[e] * gq[e] - z[e] * k);
            }
        }
        if (p.post) {
            float s[1] = {0.0f};
#pragma unroll
            for (int e = 0; e < E; ++e) s[0] += f[e] * f[e];
            team_sum<TEAM, 1>(s, red);
            rf = 1.0f / sqrtf(s[0] * inv_d + p.eps);
        }
        if (p.dx) {
            float v[E];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = p.keep * D[e];
            store_row<T, TEAM, E, VEC>((T *)p.dx + row * p.dx_stride, p.d, lane, v);
        }
        // dn, then b = dn gp in D's place; the gate's gradient
        float dg[E], s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float g = gate_r, slope = slope_r;
            if (channel) g = gc[e], slope = slope_c[e];
            if (element) g = gate_value(gr[e], p.sigmoid, slope);
            const float fr = f[e] * rf, u = p.scale * D[e], dn = u * g;
            dg[e] = u * (fr * gp[e]) * slope;
            s[1] += dg[e];
            dgc[e] += dg[e];
            dgp[e] += dn * fr;
            D[e] = dn * gp[e];
            s[0] += D[e] * f[e];
        }
        if (p.dgate && element) store_row<T, TEAM, E, VEC>((T *)p.dgate + row * p.dgate_stride, p.d, lane, dg);
        team_sum<TEAM, 2>(s, red);
        if (p.dgate && p.gate_kind == ADN_GATE_ROW && lane == 0) ((float *)p.dgate)[row] = s[1];
        if (p.df) {
            const float k = p.post ? rf * rf * (s[0] * inv_d) : 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) D[e] = rf * (D[e] - f[e] * k);
            store_row<T, TEAM, E, VEC>((T *)p.df + row * p.df_stride, p.d, lane, D);
        }
    }
    if (!part) return;
    // the block's teams in order, then one partial row a block, for each of the three sums that is wanted
    __shared__ float sum[TEAMS > 1 ? TEAMS : 1][64][E + 1];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        if (!(i == 0 ? p.dpost != nullptr : i == 1 ? p.dpre != nullptr : p.dgate && channel)) continue;
        float t[E];
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = i == 0 ? dgp[e] : i == 1 ? dgq[e] : dgc[e];
        if constexpr (TEAMS > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < E; ++e) sum[team][lane][e] = t[e];
            __syncthreads();
            if (team == 0) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    t[e] = sum[0][lane][e];
#pragma unroll
                    for (int q = 1; q < TEAMS; ++q) t[e] += sum[q][lane][e];
                }
            }
        }
        if (team == 0)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int c = C::col(lane, e);
                if (c < p.d) part[((long)i * gridDim.x + blockIdx.x) * p.d + c] = t[e];
            }
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
        f(integral_constant<int, 256>{}, integral_constant<int, 8>{});
    else
        f(integral_constant<int, 256>{}, integral_constant<int, 32>{});
}

bool column_sums(const ResidualParams &p) { return p.dpost || p.dpre || (p.dgate && p.gate_kind == ADN_GATE_CHANNEL); }

int back_blocks(const ResidualParams &p) {
    const int teams = p.d <= 1024 ? NB / 64 : 1;
    return (int)std::min<long>(COL_BLOCKS, ((long)p.rows + teams - 1) / teams);
}

}  // namespace

void launch_residual(const ResidualParams &p, hipStream_t st) {
    if (p.rows == 0) return;
    const int eb = elem_bytes(p.dtype);
    const bool element = p.gate_kind == ADN_GATE_ELEMENT;
    const bool vec = rows_vec16(p.x, p.x_stride, p.d, eb) && rows_vec16(p.f, p.f_stride, p.d, eb) &&
                     (!p.z || rows_vec16(p.z, p.z_stride, p.d, eb)) && (!p.y || rows_vec16(p.y, p.y_stride, p.d, eb)) &&
                     (!element || rows_vec16(p.gate, p.gate_stride, p.d, eb));
    // a launch has less than 2^32 threads: 2^23 rows at a time, a block a row at most
    ResidualParams q = p;
    for (int row = 0; row < p.rows; row += 1 << 23) {
        q.rows = std::min(p.rows - row, 1 << 23);
        q.x = (const char *)p.x + row * p.x_stride * eb;
        q.f = (const char *)p.f + row * p.f_stride * eb;
        if (p.z) q.z = (char *)p.z + row * p.z_stride * eb;
        if (p.y) q.y = (char *)p.y + row * p.y_stride * eb;
        if (element) q.gate = (const char *)p.gate + row * p.gate_stride * eb;
        if (p.gate_kind == ADN_GATE_ROW) q.gate = (const float *)p.gate + row;
        dispatch_type(p.dtype, [&](auto t) {
            typedef decltype(t) T;
            dispatch_row(p.d, [&](auto team, auto e) {
                constexpr int TEAM = decltype(team)::value, E = decltype(e)::value;
                const dim3 grid((unsigned)(((long)q.rows * TEAM + NB - 1) / NB));
                if (vec)
                    k_residual<T, TEAM, E, true><<<grid, NB, 0, st>>>(q);
                else
                    k_residual<T, TEAM, E, false><<<grid, NB, 0, st>>>(q);
            });
        });
    }
}

size_t residual_backward_workspace_bytes(const ResidualParams &p) {
    return column_sums(p) ? (size_t)3 * back_blocks(p) * p.d * sizeof(float) : 0;
}

void launch_residual_backward(const ResidualParams &p, void *ws, hipStream_t st) {
    const int eb = elem_bytes(p.dtype), blocks = back_blocks(p);
    const bool element = p.gate_kind == ADN_GATE_ELEMENT;
    auto ok = [&](const void *q, long stride) { return !q || rows_vec16(q, stride, p.d, eb); };
    const bool vec = ok(p.z, p.z_stride) && ok(p.f, p.f_stride) && ok(p.dz, p.dz_stride) && ok(p.dy, p.dy_stride) &&
                     ok(p.dx, p.dx_stride) && ok(p.df, p.df_stride) &&
                     (!element || (ok(p.gate, p.gate_stride) && ok(p.dgate, p.dgate_stride)));
    float *part = column_sums(p) ? (float *)ws : nullptr;
    if (blocks)
        dispatch_type(p.dtype, [&](auto t) {
            typedef decltype(t) T;
            dispatch_row(p.d, [&](auto team, auto e) {
                constexpr int TEAM = decltype(team)::value, E = decltype(e)::value;
                if (vec)
                    k_residual_back<T, TEAM, E, true><<<blocks, NB, 0, st>>>(p, part);
                else
                    k_residual_back<T, TEAM, E, false><<<blocks, NB, 0, st>>>(p, part);
            });
        });
    if (part)
        launch_sum_rows(part, blocks, p.d, SumRows{{p.dpost, p.dpre, p.gate_kind == ADN_GATE_CHANNEL ? (float *)p.dgate : nullptr}},
                        3, st);
}

}  // namespace adn
