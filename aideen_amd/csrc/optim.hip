// AdamW over a list of tensors, and the norm of all of the list's gradients:
//
//   t = step + 1,  g = coef grad,  coef = grad_scale min(1, max_norm / (norm grad_scale + 1e-6))
//   m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p -= lr (m / (1 - b1^t) / (sqrt(v / (1 - b2^t)) + eps) + decay p),  copy = bf16(p)
//
// The list is a table on the device: a record a tensor and a pair (tensor, chunk) a workgroup, so
// that one launch serves any number of tensors of any sizes.  Every value is read and written once;
// HBM is the bound.
//
// States in 8 bits: 256 consecutive values of a tensor share a scale, a power of two 2^(E-7) where E
// is the exponent of the largest magnitude; a value is an e4m3 code times the scale, the largest in
// [128, 256].  A wave holds such a block, four values a lane.  The new moments are formed in 64 bits
// (their products and sums rounded one by one), and rounded to codes stochastically: with b2 = 0.999 a
// step moves v by a thousandth of g^2 - v, and rounding to nearest, half a code's step being 3 to 6 %,
// would not let it move at all until g^2 passes 30 to 60 v; a rounding whose expectation is the value
// follows the average.  The 16 random bits a value are a hash of the seed, the step, the block's number
// in the list and the place in the block, so that equal calls give equal bits.  In 64 bits the decision
// depends on no rounding that another order of the same sums would change (in 32 it would, once in a
// million values).  A v that is not zero never gets the code zero: its update would be m / eps.
#include <algorithm>

#include "train.h"

namespace adn {

namespace {

constexpr int NB = 256;          // threads a block
constexpr int V = 4;             // values a lane
constexpr int MIN_EXPONENT = -110;  // of a block: the smallest code times its scale is a normal fp32 number

typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32_any __attribute__((aligned(1)));

// SplitMix64's finaliser (Steele, Lea, Flood 2014)
__device__ __forceinline__ uint64_t mix64(uint64_t x) {
    x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
    x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
    return x ^ (x >> 31);
}
constexpr uint64_t GOLDEN = 0x9E3779B97F4A7C15ull;

// 32 random bits of place i of a block whose hash is a (two multiplications, shifts of 16, 15, 16)
__device__ __forceinline__ uint32_t mix32(uint32_t a, uint32_t i) {
    uint32_t r = a + i * 0x9E3779B9u;
    r = (r ^ (r >> 16)) * 0x7FEB352Du;
    r = (r ^ (r >> 15)) * 0x846CA68Bu;
    return r ^ (r >> 16);
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off, 64));
    return v;
}

// The e4m3 code (without its sign) of a magnitude whose high word is `hi`, in a block of exponent E:
// `r` in [0, 2^17) is added below the code's last bit before the rest is cut off.
__device__ __forceinline__ uint32_t code_of(uint32_t hi, int E, uint32_t r) {
    const int k = (int)hi - ((1023 + E - 14) << 20);  // exponent with e4m3's bias, and 20 bits of mantissa
    const int below = 1 - (k >> 20);                  // binades below the smallest normal code
    const uint32_t sub = ((hi & 0xFFFFF) | 0x100000) >> min(below, 31);
    return ((below > 0 ? sub : (uint32_t)k) + r) >> 17;
}

template <typename T>
__device__ __forceinline__ void load4(const T *p, int n, float (&v)[V]) {
    if (n >= V) {
        if constexpr (sizeof(T) == 4) {
            const f32x4 x = *reinterpret_cast<const f32x4 *>(p);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = x[j];
        } else {
            const bf16x4 x = *reinterpret_cast<const bf16x4 *>(p);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = (float)x[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = j < n ? (float)p[j] : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store4(T *p, int n, const float (&v)[V]) {
    if (n >= V) {
        if constexpr (sizeof(T) == 4) {
            f32x4 x;
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = v[j];
            *reinterpret_cast<f32x4 *>(p) = x;
        } else {
            bf16x4 x;
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = (__bf16)v[j];
            *reinterpret_cast<bf16x4 *>(p) = x;
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < n) p[j] = (T)v[j];
    }
}

__device__ __forceinline__ uint32_t load_codes(const uint8_t *p, int n) {
    if (n >= V) return *reinterpret_cast<const u32_any *>(p);
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < n) w |= (uint32_t)p[j] << (8 * j);
    return w;
}

__device__ __forceinline__ void store_codes(uint8_t *p, int n, uint32_t w) {
    if (n >= V) {
        *reinterpret_cast<u32_any *>(p) = w;
        return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < n) p[j] = (uint8_t)(w >> (8 * j));
}

__device__ __forceinline__ void decode4(uint32_t w, float scale, float (&v)[V]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    v[0] = a[0] * scale, v[1] = a[1] * scale, v[2] = b[0] * scale, v[3] = b[1] * scale;
}

// A new moment in 64 bits, b old + (1 - b) g, rounded after each operation (a fused one would round ties of
// short operands otherwise than the definition).
__device__ __forceinline__ double moment(double b, double old, double g, double square) {
#pragma clang fp contract(off)
    const double kept = b * old;
    double more = (1.0 - b) * g;
    more = more * square;
    return kept + more;
}

// The step's scalars, one thread: the counter, the bias corrections, the clipping coefficient.
__global__ void k_adamw_begin(OptPlan p, OptStep s) {
    OptScalars o;
    const float norm = s.grad_norm ? *s.grad_norm : 0.0f;
    o.skip = !(fabsf(norm) < INFINITY);
    const int done = max(*p.step, 0), t = done < INT32_MAX ? done + 1 : done;
    o.coef = (double)s.grad_scale;
    if (s.max_norm > 0.0f) o.coef *= fmin(1.0, (double)s.max_norm / ((double)norm * (double)s.grad_scale + 1e-6));
    o.lr = (float)(s.lr_device ? (double)*s.lr_device : s.lr);
    o.inv_bc1 = (float)(1.0 / (1.0 - pow(p.beta1, (double)t)));
    o.inv_sqrt_bc2 = (float)(1.0 / sqrt(1.0 - pow(p.beta2, (double)t)));
    o.key = mix64(p.seed + (uint64_t)(int64_t)(t - 1) * GOLDEN);
    *p.scalars = o;
    if (!o.skip) *p.step = t;
}

// p - lr (m / bc1 / (sqrt(v / bc2) + eps) + decay p)
__device__ __forceinline__ float stepped(float p, float m, float v, const OptScalars &o, float lr, float decay, float eps) {
    const float away = m * o.inv_bc1 / (sqrtf(v) * o.inv_sqrt_bc2 + eps);
    return p - lr * (away + decay * p);
}

template <bool EIGHT>
__global__ __launch_bounds__(NB) void k_adamw(OptPlan P) {
    const OptScalars o = *P.scalars;
    if (o.skip) return;
    const OptChunk ck = P.chunks[blockIdx.x];
    const OptTensor t = P.tensors[ck.tensor];
    const int lane = threadIdx.x & 63;
    const int64_t begin = (int64_t)ck.chunk * P.chunk_values;
    const int64_t end = min(begin + P.chunk_values, t.n);
    const float lr = o.lr * t.lr_scale;
    for (int64_t b = begin + (threadIdx.x >> 6) * OPT_BLOCK; b < end; b += (NB / 64) * OPT_BLOCK) {
        const int64_t i = b + lane * V;
        const int n = (int)min<int64_t>(max<int64_t>(t.n - i, 0), V);  // this lane's values
        float p[V], g[V], m[V], v[V];
        load4(t.param + i, n, p);
        if (t.grad_bf16)
            load4((const __bf16 *)t.grad + i, n, g);
        else
            load4((const float *)t.grad + i, n, g);
        if constexpr (EIGHT) {
            uint8_t *m8 = (uint8_t *)t.m + i, *v8 = (uint8_t *)t.v + i;
            const int64_t blk = b / OPT_BLOCK;
            decode4(load_codes(m8, n), t.m_scale[blk], m);
            decode4(load_codes(v8, n), t.v_scale[blk], v);
            double md[V], vd[V];
            uint32_t mtop = 0, vtop = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const double gd = (double)g[j] * o.coef;
                md[j] = moment(P.beta1, m[j], gd, 1.0);
                vd[j] = moment(P.beta2, v[j], gd, gd);
                if (j >= n) md[j] = vd[j] = 0.0;
                mtop = max(mtop, (uint32_t)__double2hiint(md[j]) & 0x7FFFFFFFu);
                vtop = max(vtop, (uint32_t)__double2hiint(vd[j]) & 0x7FFFFFFFu);
            }
            mtop = wave_max_u32(mtop), vtop = wave_max_u32(vtop);
            const int me = max((int)(mtop >> 20) - 1023, MIN_EXPONENT), ve = max((int)(vtop >> 20) - 1023, MIN_EXPONENT);
            const uint32_t a = (uint32_t)mix64(o.key + (uint64_t)(t.block + blk + 1) * GOLDEN);
            uint32_t mw = 0, vw = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const uint32_t r = mix32(a, lane * V + j);
                const uint32_t mh = (uint32_t)__double2hiint(md[j]), vh = (uint32_t)__double2hiint(vd[j]);
                const uint32_t mc = code_of(mh & 0x7FFFFFFFu, me, (r & 0xFFFFu) << 1) | (mh >> 24 & 0x80u);
                uint32_t vc = code_of(vh & 0x7FFFFFFFu, ve, (r >> 16) << 1);
                if (vc == 0 && vd[j] > 0.0) vc = 1;
                mw |= mc << (8 * j), vw |= vc << (8 * j);
                m[j] = (float)md[j], v[j] = (float)vd[j];
            }
            // a block that holds a value beyond fp32, an infinity or a NaN is not a number as a whole
            const bool mbad = me > 127, vbad = ve > 127;
            store_codes(m8, n, mbad ? 0 : mw);
            store_codes(v8, n, vbad ? 0 : vw);
            if (lane == 0) {
                t.m_scale[blk] = mbad ? NAN : __uint_as_float((uint32_t)(me - 7 + 127) << 23);
                t.v_scale[blk] = vbad ? NAN : __uint_as_float((uint32_t)(ve - 7 + 127) << 23);
            }
        } else {
            const float b1 = (float)P.beta1, c1 = (float)(1.0 - P.beta1), b2 = (float)P.beta2, c2 = (float)(1.0 - P.beta2);
            const float coef = (float)o.coef;
            load4((const float *)t.m + i, n, m);
            load4((const float *)t.v + i, n, v);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float gj = g[j] * coef;
                m[j] = b1 * m[j] + c1 * gj;
                v[j] = b2 * v[j] + c2 * gj * gj;
            }
            store4((float *)t.m + i, n, m);
            store4((float *)t.v + i, n, v);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) p[j] = stepped(p[j], m[j], v[j], o, lr, t.decay, P.eps);
        store4(t.param + i, n, p);
        if (t.copy) store4(t.copy + i, n, p);
    }
}

// Sum of the squares of all gradients in 64 bits (no overflow, and no order that matters to fp32): each
// workgroup's chunks in order, then the workgroups' sums in order by the last one to finish.
__global__ __launch_bounds__(NB) void k_grad_norm(OptPlan P, float *norm) {
    __shared__ double red[NB / 64];
    __shared__ bool last;
    double s = 0.0;
    for (int c = blockIdx.x; c < P.n_chunks; c += gridDim.x) {
        const OptChunk ck = P.chunks[c];
        const OptTensor &t = P.tensors[ck.tensor];
        const int64_t begin = (int64_t)ck.chunk * P.chunk_values, n = t.n;
        const int64_t end = min(begin + P.chunk_values, n);
        for (int64_t i = begin + threadIdx.x * V; i < end; i += NB * V) {
            float g[V];
            const int k = (int)min<int64_t>(n - i, V);
            if (t.grad_bf16)
                load4((const __bf16 *)t.grad + i, k, g);
            else
                load4((const float *)t.grad + i, k, g);
#pragma unroll
            for (int j = 0; j < V; ++j) s += (double)g[j] * (double)g[j];
        }
    }
    auto block_sum = [&](double x) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0.0;
        for (int w = 0; w < NB / 64; ++w) x += red[w];
        return x;
    };
    s = block_sum(s);
    if (threadIdx.x == 0) {
        __hip_atomic_store(&P.partials[blockIdx.x], s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(P.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    s = 0.0;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += NB)
        s += __hip_atomic_load(&P.partials[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s = block_sum(s);
    if (threadIdx.x == 0) {
        *norm = (float)sqrt(s);
        __hip_atomic_store(P.ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

}  // namespace

// Values a workgroup: enough workgroups to fill the GPU, and no more than 2^31 of them.
int opt_chunk_values(int64_t total) {
    constexpr int64_t LEAST = NB * V, MOST = 16 * NB * V;
    const int64_t per = total / 4096 / LEAST * LEAST;
    return (int)std::min(std::max(per, LEAST), MOST);
}

void launch_grad_norm(const OptPlan &p, float *norm, hipStream_t st) {
    const int blocks = std::max(1, std::min(p.n_chunks, OPT_NORM_BLOCKS));
    k_grad_norm<<<blocks, NB, 0, st>>>(p, norm);
}

void launch_adamw(const OptPlan &p, const OptStep &s, hipStream_t st) {
    k_adamw_begin<<<1, 1, 0, st>>>(p, s);
    if (p.n_chunks == 0) return;
    if (p.state_bits == 8)
        k_adamw<true><<<p.n_chunks, NB, 0, st>>>(p);
    else
        k_adamw<false><<<p.n_chunks, NB, 0, st>>>(p);
}

}  // namespace adn
