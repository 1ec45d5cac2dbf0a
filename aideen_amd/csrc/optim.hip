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

// SplitMix64's finaliser (Steele, Lea, Flood 2014)
__device__ __forceinline__ uint64_t mix64(uint64_t x) {
    x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
    x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
    return x ^ (x >> 31);
}
constexpr uint64_t GOLDEN = 0x9E3779B97F4A7C15ull;

// 32 random bits of place i of a block whose hash is a: a bijection of two multiplications between shifts of 16, 15 and 16, with the
// constants that C. Wellons found by a search for the least bias (Prospecting for hash functions, 2018)
__device__ __forceinline__ uint32_t mix32(uint32_t a, uint32_t i) {
    uint32_t r = a + i * 0x9E3779B9u;
    r = (r ^ (r >> 16)) * 0x7FEB352Du;
    r = (r ^ (r >> 15)) * 0x846CA68Bu;
    return r ^ (r >> 16);
}

// The e4m3 code (without its sign) of the magnitude x, whose high word is `hi`, in a block of exponent E:
// `r` in [0, 2^17) is added below the code's last bit before the rest is cut off.  The high word of a
// normal code holds it behind a change of bias; below those, x to_steps (2^(33-E)) counts 2^-17 of a step.
__device__ __forceinline__ uint32_t code_of(double x, uint32_t hi, int E, double to_steps, uint32_t r) {
    const int k = (int)hi - ((1023 + E - 14) << 20);
    const uint32_t below = (uint32_t)fmin(fabs(x) * to_steps, 0x1p20);
    return ((k < 1 << 20 ? below : (uint32_t)k) + r) >> 17;
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

struct Scalars {
    double coef;
    uint64_t key;
    float lr, inv_bc1, inv_sqrt_bc2;
    int t;
    bool skip;
};

// What a step takes from the device: the counter, the bias corrections, the clipping coefficient.
__device__ __forceinline__ Scalars scalars(const OptPlan &P, const OptStep &S) {
    Scalars o;
    const float norm = S.grad_norm ? *S.grad_norm : 0.0f;
    const int done = max(*P.step, 0);
    asm volatile("" ::"s"(done));  // it has arrived: the workgroup may say that it has read the counter
    o.skip = !(fabsf(norm) < INFINITY);
    o.t = done < INT32_MAX ? done + 1 : done;
    o.coef = (double)S.grad_scale;
    if (S.max_norm > 0.0f) o.coef *= fmin(1.0, (double)S.max_norm / ((double)norm * (double)S.grad_scale + 1e-6));
    o.lr = (float)(S.lr_device ? (double)*S.lr_device : S.lr);
    // 1 - b^t = -expm1(t log b), as exact in fp32 as its argument
    o.inv_bc1 = -__builtin_amdgcn_rcpf(expm1f((float)(o.t * P.log_beta1)));
    o.inv_sqrt_bc2 = __builtin_amdgcn_rsqf(-expm1f((float)(o.t * P.log_beta2)));
    o.key = mix64(P.seed + (uint64_t)(int64_t)(o.t - 1) * GOLDEN);
    return o;
}

// True in the last workgroup of the grid that comes here (one thread of each calls it).  One address
// takes a read-modify-write in about 10 ns from the whole chip (512 workgroups at one: 5 us), so a
// group of the workgroups counts at a place of its own and its last one at a common place.
__device__ __forceinline__ bool last_of_grid(unsigned *ticket) {
    const unsigned group = blockIdx.x % OPT_TICKETS, groups = min((unsigned)OPT_TICKETS, gridDim.x);
    const unsigned members = (gridDim.x - group + OPT_TICKETS - 1) / OPT_TICKETS;
    unsigned *mine = ticket + (1 + group) * OPT_TICKET_PITCH;
    if (__hip_atomic_fetch_add(mine, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != members - 1) return false;
    __hip_atomic_store(mine, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != groups - 1) return false;
    __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return true;
}

// p - lr (m / bc1 / (sqrt(v / bc2) + eps) + decay p), the root and the reciprocal to 1 ulp.  The root
// instruction takes numbers below 2^-126 for zero: what is lost, less than 2^-63 / sqrt(bc2), is nothing
// beside an eps of 2^25 times that.
__device__ __forceinline__ void stepped(float (&p)[V], const float (&m)[V], const float (&v)[V], const Scalars &o, float lr,
                                        float decay, float eps) {
    float root[V];
    if (eps >= 0x1p-38f * o.inv_sqrt_bc2) {
#pragma unroll
        for (int j = 0; j < V; ++j) root[j] = __builtin_amdgcn_sqrtf(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) root[j] = sqrtf(v[j]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float away = m[j] * o.inv_bc1 * __builtin_amdgcn_rcpf(fmaf(root[j], o.inv_sqrt_bc2, eps));
        p[j] = fmaf(-lr, fmaf(decay, p[j], away), p[j]);
    }
}

// The largest of the wave's values, the same in every lane and known to be so.
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
#define ADN_DPP_MAX(ctrl, rows) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xF, true))
    ADN_DPP_MAX(0x111, 0xF);  // from the lane one, two, four, eight to the left in a row of 16
    ADN_DPP_MAX(0x112, 0xF);
    ADN_DPP_MAX(0x114, 0xF);
    ADN_DPP_MAX(0x118, 0xF);
    ADN_DPP_MAX(0x142, 0xA);  // a row's last lane to the next row, then to the upper half
    ADN_DPP_MAX(0x143, 0xC);
#undef ADN_DPP_MAX
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// A pointer that is known to be to global memory (one that was loaded from a record is not).
template <typename T>
using global_ptr = __attribute__((address_space(1))) T *;

// A lane's four values of a block, as they are loaded: of a WHOLE block four neighbours, at any address (60 M parameters one
// element off the alignment 288 us, aligned 270; in 8 bits 199 and 165, by single values 244); of a tensor's last
// block every 64th, of those that there are.
template <typename T, bool WHOLE, bool NT>
struct Four {
    typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    vec x;
    __device__ __forceinline__ void load(const T *p, int lane, int n) {
        if constexpr (WHOLE && NT) {
            x = __builtin_nontemporal_load((global_ptr<const vec>)(p + lane * V));
        } else if constexpr (WHOLE) {
            x = *(global_ptr<const vec>)(p + lane * V);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) x[j] = lane + 64 * j < n ? ((global_ptr<const T>)p)[lane + 64 * j] : (T)0;
        }
    }
    __device__ __forceinline__ void store(T *p, int lane, int n) const {
        if constexpr (WHOLE && NT) {
            __builtin_nontemporal_store(x, (global_ptr<vec>)(p + lane * V));
        } else if constexpr (WHOLE) {
            *(global_ptr<vec>)(p + lane * V) = x;
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (lane + 64 * j < n) ((global_ptr<T>)p)[lane + 64 * j] = x[j];
        }
    }
};

// A block of 256 values of a tensor (or what the tensor has left), loaded and stepped.
template <bool EIGHT, bool BF16, bool WHOLE, bool NT>
struct Block {
    typedef std::conditional_t<EIGHT, uint8_t, float> S;
    typedef std::conditional_t<BF16, __bf16, float> G;
    Four<float, WHOLE, NT> p;
    Four<G, WHOLE, NT> g;
    Four<S, WHOLE, NT> m, v;
    float ms, vs;

    __device__ __forceinline__ static int count(const OptTensor &t, int64_t blk) {
        return WHOLE ? OPT_BLOCK : (int)min<int64_t>(t.n - blk * OPT_BLOCK, OPT_BLOCK);
    }
    // the place in its block of a lane's value j
    __device__ __forceinline__ static int place(int lane, int j) { return WHOLE ? lane * V + j : lane + 64 * j; }

    __device__ __forceinline__ void load(const OptTensor &t, int64_t blk, int lane) {
        const int64_t i = blk * OPT_BLOCK;
        const int n = count(t, blk);
        g.load((const G *)t.grad + i, lane, n);
        m.load((const S *)t.m + i, lane, n);
        v.load((const S *)t.v + i, lane, n);
        p.load(t.param + i, lane, n);
        if constexpr (EIGHT) ms = ((global_ptr<const float>)t.m_scale)[blk], vs = ((global_ptr<const float>)t.v_scale)[blk];
    }

    __device__ __forceinline__ void step(const OptPlan &P, const OptTensor &t, const Scalars &o, float lr, int64_t blk, int lane) {
        const int64_t i = blk * OPT_BLOCK;
        const int n = count(t, blk);
        float mf[V], vf[V];
        if constexpr (EIGHT) {
            decode4(__builtin_bit_cast(uint32_t, m.x), ms, mf);
            decode4(__builtin_bit_cast(uint32_t, v.x), vs, vf);
            double md[V], vd[V];
            uint32_t mtop = 0, vtop = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const double gd = (double)(float)g.x[j] * o.coef;
                md[j] = moment(P.beta1, mf[j], gd, 1.0);
                vd[j] = moment(P.beta2, vf[j], gd, gd);
                if (!WHOLE && place(lane, j) >= n) md[j] = vd[j] = 0.0;
                mtop = max(mtop, (uint32_t)__double2hiint(md[j]) & 0x7FFFFFFFu);
                vtop = max(vtop, (uint32_t)__double2hiint(vd[j]) & 0x7FFFFFFFu);
            }
            mtop = wave_max_u32(mtop), vtop = wave_max_u32(vtop);
            const int me = max((int)(mtop >> 20) - 1023, MIN_EXPONENT), ve = max((int)(vtop >> 20) - 1023, MIN_EXPONENT);
            const uint32_t a = (uint32_t)mix64(o.key + (uint64_t)(t.block + blk + 1) * GOLDEN);
            const double m_steps = __hiloint2double((1023 + 33 - me) << 20, 0), v_steps = __hiloint2double((1023 + 33 - ve) << 20, 0);
            uint32_t mw = 0, vw = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const uint32_t r = mix32(a, place(lane, j));
                const uint32_t mh = (uint32_t)__double2hiint(md[j]), vh = (uint32_t)__double2hiint(vd[j]);
                const uint32_t mc = code_of(md[j], mh & 0x7FFFFFFFu, me, m_steps, (r & 0xFFFFu) << 1) | (mh >> 24 & 0x80u);
                const uint32_t vc = max(code_of(vd[j], vh, ve, v_steps, (r >> 16) << 1), min(vh, 1u));
                mw |= mc << (8 * j), vw |= vc << (8 * j);
                mf[j] = (float)md[j], vf[j] = (float)vd[j];
            }
            // a block that holds 2^127 or more (its largest code could be 2^128), an infinity or a NaN is not a number as a whole
            const bool mbad = me > 126, vbad = ve > 126;
            typedef typename Four<S, WHOLE, NT>::vec codes;
            m.x = __builtin_bit_cast(codes, mbad ? 0 : mw), v.x = __builtin_bit_cast(codes, vbad ? 0 : vw);
            if (lane == 0) {
                ((global_ptr<float>)t.m_scale)[blk] = mbad ? NAN : __uint_as_float((uint32_t)(me - 7 + 127) << 23);
                ((global_ptr<float>)t.v_scale)[blk] = vbad ? NAN : __uint_as_float((uint32_t)(ve - 7 + 127) << 23);
            }
        } else {
            const float b1 = (float)P.beta1, c1 = (float)(1.0 - P.beta1), b2 = (float)P.beta2, c2 = (float)(1.0 - P.beta2);
            // a coefficient below fp32's normal numbers would lose bits: its power of two is a factor of its own
            const bool below = o.coef < 0x1p-126;
            const float low = below ? 0x1p-126f : 1.0f, coef = (float)(below ? o.coef * 0x1p126 : o.coef);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float gj = (float)g.x[j] * coef * low;
                // fused as written: a block's bits do not depend on how it is loaded
                m.x[j] = mf[j] = fmaf(b1, m.x[j], c1 * gj);
                v.x[j] = vf[j] = fmaf(b2, v.x[j], c2 * gj * gj);
            }
        }
        m.store((S *)t.m + i, lane, n);
        v.store((S *)t.v + i, lane, n);
        float pf[V];
#pragma unroll
        for (int j = 0; j < V; ++j) pf[j] = p.x[j];
        stepped(pf, mf, vf, o, lr, t.decay, P.eps);
#pragma unroll
        for (int j = 0; j < V; ++j) p.x[j] = pf[j];
        p.store(t.param + i, lane, n);
        if (t.copy) {
            Four<__bf16, WHOLE, NT> c;
#pragma unroll
            for (int j = 0; j < V; ++j) c.x[j] = (__bf16)p.x[j];
            c.store(t.copy + i, lane, n);
        }
    }
};

// A workgroup's chunk: its waves take the chunk's blocks in turn.  The first is loaded before the step's
// scalars are asked for, so that the two round trips are one (3.1 M parameters in 701 tensors, 8 bits:
// 18.8 -> 16.3 us).
template <bool EIGHT, bool BF16, bool NT>
__device__ __forceinline__ void step_chunk(const OptPlan &P, const OptStep &S, const OptTensor &t, int chunk) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t per = P.step_values / OPT_BLOCK, first = chunk * per;
    const int64_t last = min(first + per, (t.n + OPT_BLOCK - 1) / OPT_BLOCK), end = min(last, t.n / OPT_BLOCK);  // all, and the whole ones
    Block<EIGHT, BF16, true, NT> block;
    int64_t b = first + wave;
    if (b < end) block.load(t, b, lane);
    const Scalars o = scalars(P, S);
    if (o.skip) return;
    // every workgroup has read the counter once the last one comes here: it sets the next count
    __syncthreads();
    if (threadIdx.x == 0 && last_of_grid(P.ticket)) *P.step = o.t;
    const float lr = o.lr * t.lr_scale;
    while (b < end) {
        block.step(P, t, o, lr, b, lane);
        b += NB / 64;
        if (b < end) block.load(t, b, lane);
    }
    if (b < last) {  // the tensor's last block, where it does not fill it
        Block<EIGHT, BF16, false, NT> rest;
        rest.load(t, b, lane);
        rest.step(P, t, o, lr, b, lane);
    }
}

template <bool EIGHT, bool NT>
__global__ __launch_bounds__(NB) void k_adamw(OptPlan P, OptStep S) {
    const OptChunk ck = P.step_chunks[blockIdx.x];
    const OptTensor t = P.tensors[ck.tensor];
    if (t.grad_bf16)
        step_chunk<EIGHT, true, NT>(P, S, t, ck.chunk);
    else
        step_chunk<EIGHT, false, NT>(P, S, t, ck.chunk);
}

// An empty list's step.
__global__ void k_adamw_count(OptPlan P, OptStep S) {
    const Scalars o = scalars(P, S);
    if (!o.skip) *P.step = o.t;
}

// The squares of R times 64 lanes' 16 bytes, all loaded before the first is used.
template <typename T, int R>
__device__ __forceinline__ void add_squares(const T *g, double (&s)[4]) {
    constexpr int W = 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(W), aligned(sizeof(T))));
    vec x[R];
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = *reinterpret_cast<const vec *>(g + r * 64 * W);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < W; ++j) s[j & 3] += (double)(float)x[r][j] * (double)(float)x[r][j];
}

template <typename T>
__device__ __forceinline__ void add_squares(const T *g, int64_t n, int lane, double (&s)[4]) {
    constexpr int W = 16 / (int)sizeof(T), R = 4;
    int64_t i = 0;
    for (; i + R * 64 * W <= n; i += R * 64 * W) add_squares<T, R>(g + i + lane * W, s);
    for (; i + 64 * W <= n; i += 64 * W) add_squares<T, 1>(g + i + lane * W, s);
    for (i += lane; i < n; i += 64) s[0] += (double)(float)g[i] * (double)(float)g[i];
}

// Sum of the squares of all gradients in 64 bits (no overflow, and no order that matters to fp32): each
// wave's chunks in order, then the workgroups' sums in order by the last one to finish.  A sum is
// handed over by a read-modify-write of its place, and the workgroup counted once that has returned,
// so that no cache has to be written back (with a release of the caches in each of 1850 workgroups the
// kernel took 47 us for 1.9 M values, now 5).  The order is the hardware's, not the memory model's, which knows no order of
// relaxed operations on two places: an agent-scope read-modify-write is carried out where all XCDs see it before
// it returns its old value, the use of that value keeps the count behind it, and the sums are read by agent-scope loads.
__global__ __launch_bounds__(NB) void k_grad_norm(OptPlan P, float *norm) {
    __shared__ double red[NB / 64];
    __shared__ bool last;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double s4[4] = {0.0, 0.0, 0.0, 0.0};
    for (int c = blockIdx.x * (NB / 64) + wave; c < P.n_norm_chunks; c += gridDim.x * (NB / 64)) {
        const OptChunk ck = P.norm_chunks[c];
        const OptTensor &t = P.tensors[ck.tensor];
        const int64_t begin = (int64_t)ck.chunk * P.norm_values, n = min((int64_t)P.norm_values, t.n - begin);
        if (t.grad_bf16)
            add_squares((const __bf16 *)t.grad + begin, n, lane, s4);
        else
            add_squares((const float *)t.grad + begin, n, lane, s4);
    }
    auto block_sum = [&](double x) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, 64);
        __syncthreads();
        if (lane == 0) red[wave] = x;
        __syncthreads();
        x = 0.0;
        for (int w = 0; w < NB / 64; ++w) x += red[w];
        return x;
    };
    double s = block_sum((s4[0] + s4[1]) + (s4[2] + s4[3]));
    if (threadIdx.x == 0) {
        const uint64_t before = __hip_atomic_exchange((uint64_t *)&P.partials[blockIdx.x], (uint64_t)__double_as_longlong(s), __ATOMIC_RELAXED,
                                                      __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("" ::"v"(before) : "memory");  // the exchange has returned before the counter is raised
        last = last_of_grid(P.ticket);
    }
    __syncthreads();
    if (!last) return;
    s = 0.0;
    for (unsigned i = threadIdx.x; i < gridDim.x; i += NB)
        s += __hip_atomic_load(&P.partials[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s = block_sum(s);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

}  // namespace

// Values of a workgroup's chunk in a step.  With fp32 states one block a wave: more blocks a workgroup, or
// more workgroups in flight, spread the open pages of seven streams (65 M parameters: 16 blocks a wave 351 us, 4 322, 1
// 307).  With 8-bit states three where there are enough, as the scalars' arithmetic counts (65 M: 1 block 198 us,
// 3 178, 8 187; 206 M: 618, 565, 617).
int opt_step_values(int64_t total, bool eight) {
    constexpr int LEAST = NB * V;
    return eight && total >= (int64_t)4096 * 3 * LEAST ? 3 * LEAST : LEAST;
}

// Values of a wave's chunk in the norm: 2048 waves, up to 16 thousand values at a time.
int opt_norm_values(int64_t total) {
    constexpr int64_t LEAST = NB * V, MOST = 16 * NB * V;
    return (int)std::min(std::max(total / (OPT_NORM_BLOCKS * (NB / 64)) / LEAST * LEAST, LEAST), MOST);
}

void launch_grad_norm(const OptPlan &p, float *norm, hipStream_t st) {
    const int blocks = std::max(1, std::min((p.n_norm_chunks + NB / 64 - 1) / (NB / 64), OPT_NORM_BLOCKS));
    k_grad_norm<<<blocks, NB, 0, st>>>(p, norm);
}

// A list of more than 8 M parameters (16 M with 8 bits) is read and written past the caches: with lists that take turns, us
// through them and past them, fp32 states 6 M 31 and 32, 8 M 44 and 41, 12 M 68 and 61, 48 M 262 and 224; 8 bits 8 M 30 and 30, 12 M 44
// and 40, 20 M 68 and 61; 1.9 M behind a step of its own 11.4 and 12.8.  With fp32 states
// 32 KB of LDS that nothing uses then keep the workgroups at five a CU, for the same reason as the chunks:
// 65 M 308 -> 287 us (8 a CU; 6: 304, 4: 289, 2: 340), 206 M with bf16 gradients and copies 977 -> 929.
void launch_adamw(const OptPlan &p, const OptStep &s, hipStream_t st) {
    const int wg = p.n_step_chunks;
    constexpr int FEWER = 32768;
    if (wg == 0)
        k_adamw_count<<<1, 1, 0, st>>>(p, s);
    else if (p.state_bits == 8)
        p.streams ? k_adamw<true, true><<<wg, NB, 0, st>>>(p, s) : k_adamw<true, false><<<wg, NB, 0, st>>>(p, s);
    else
        p.streams ? k_adamw<false, true><<<wg, NB, FEWER, st>>>(p, s) : k_adamw<false, false><<<wg, NB, 0, st>>>(p, s);
}

}  // namespace adn
