// The embedding table as a trained tensor: scaled lookup (Tokenizer::embed_sequence,
// tokenizer.rs:151-159, with a factor) and its gradient
//
//   out[i] = scale E[tok_i]            dE[v] = scale sum over i with tok_i = v of dout[i]
//
// The gradient adds each table row's positions in a fixed order, so it is the same bits on every run.
//
// Up to FEW positions: one launch.  A block a position compares its token with all the others (eight
// 64-bit masks a wave).  The blocks of a token share its columns, 64 lanes' at a time: a wave adds all the
// rows of its columns where they are few, an eighth of them where they are many (4096 positions of 2048
// columns on 65 tokens, the most frequent a fifth: 79 us with one block a token, 17 shared).  Other blocks
// write zeros where no token is, which is most of the time: 256 positions of 512 columns of 50257 entries
// 16 us (6.3 TB/s), 4096 30 us (sorted 46).
//
// More: the positions are sorted by token (a stable radix sort of 8 bits a pass), the sorted list is
// cut into chunks, a wave adds one chunk's rows in order and stores the table rows that begin and end
// in it; of a row that crosses chunks every chunk stores a partial sum, and a last kernel adds those in
// chunk order (a frequent token has thousands of positions).  The sort's launches are short and leave
// most of the chip idle: their other blocks write the table's zeros, the larger part of all bytes.
#include <algorithm>

#include "train.h"

namespace adn {

namespace {

constexpr int NT = 256;
constexpr int RADIX = 256;
constexpr int TILE = 1024;                // keys a block of a radix pass
constexpr int W_KEYS = TILE / (NT / 64);  // consecutive keys a wave of it
constexpr int OWN_PREFIX = 128;           // blocks up to which each forms its own offsets
constexpr int FW = 8;                     // waves of a block of the few
constexpr int FEW = FW * 8 * 64;
constexpr int C0 = 32;                    // sorted entries a wave adds at a time

// The key of position i: its token, or `vocab` (sorted behind every token) where it has none.
__device__ __forceinline__ unsigned key_of(const int32_t *tokens, long i, int vocab, unsigned *err) {
    const int t = tokens[i];
    if (t >= vocab) {
        if (err) atomicOr(err, ADN_DEVERR_TOKEN);
        return (unsigned)vocab;
    }
    return t < 0 ? (unsigned)vocab : (unsigned)t;
}

template <typename T, int W>
struct VecT {
    typedef T type __attribute__((ext_vector_type(W)));
};

// out[i] = scale E[tok_i], a wave a row
template <typename T, bool VEC>
__global__ __launch_bounds__(NT) void k_lookup(TableParams p) {
    const long i = (long)blockIdx.x * (NT / 64) + (threadIdx.x >> 6);
    if (i >= p.n) return;
    const int lane = threadIdx.x & 63;
    const unsigned key = key_of(p.tokens, i, p.vocab, lane == 0 ? p.err : nullptr);
    const bool there = key < (unsigned)p.vocab;
    const T *src = (const T *)p.src + (there ? (long)key * p.src_stride : 0);
    T *dst = (T *)p.dst + i * p.dst_stride;
    constexpr int W = VEC ? 16 / (int)sizeof(T) : 1;
    typedef typename VecT<T, W>::type V;
    for (int c = lane * W; c < p.d; c += 64 * W) {
        V v = *reinterpret_cast<const V *>(src + c);
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = from_f32<T>(there ? to_f32<T>(v[j]) * p.scale : 0.0f);
        *reinterpret_cast<V *>(dst + c) = v;
    }
}

// Zeros in rows v0 + first, + step, ... below v1 of the table, a wave a row.
template <typename T, bool VEC>
__device__ __forceinline__ void zero_rows(T *dst, long stride, int d, long v0, long v1, long first, long step) {
    constexpr int W = VEC ? 16 / (int)sizeof(T) : 1;
    typedef typename VecT<T, W>::type V;
    V z;
#pragma unroll
    for (int j = 0; j < W; ++j) z[j] = from_f32<T>(0.0f);
    const int lane = threadIdx.x & 63;
    for (long v = v0 + first; v < v1; v += step)
        for (int c = lane * W; c < d; c += 64 * W) *reinterpret_cast<V *>(dst + v * stride + c) = z;
}

// ---- few positions -------------------------------------------------------------------------
// Blocks below n: position blockIdx.x.  The others: FEW_ROWS rows of the table each.
constexpr int FEW_ROWS = 64;
template <typename T, bool VEC>
__global__ __launch_bounds__(64 * FW) void k_grad_few(TableParams p) {
    constexpr int W = VEC ? 16 / (int)sizeof(T) : 1, LOADS = 16;
    typedef typename VecT<T, W>::type V;
    __shared__ int list[FEW];
    __shared__ int cnt[FW], ahead[FW];
    __shared__ int here[FEW_ROWS];
    __shared__ float part[FW - 1][64 * W];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if ((int)blockIdx.x >= p.n) {
        const long v0 = (long)((int)blockIdx.x - p.n) * FEW_ROWS, v1 = min(v0 + FEW_ROWS, (long)p.vocab);
        if (tid < FEW_ROWS) here[tid] = 0;
        __syncthreads();
#pragma unroll 8
        for (int i = tid; i < p.n; i += 64 * FW) {
            const int t = p.tokens[i];
            if (t >= v0 && t < v1) here[t - v0] = 1;
        }
        __syncthreads();
        for (long v = v0 + wave; v < v1; v += FW)
            if (!here[v - v0]) zero_rows<T, VEC>((T *)p.dst, p.dst_stride, p.d, v, v + 1, 0, 1);
        return;
    }
    // the positions of this token in order: wave w looks at [w S, (w + 1) S)
    const int S = ((p.n + FW - 1) / FW + 63) / 64 * 64;  // at most 8 x 64
    int t[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int i = wave * S + u * 64 + lane;
        t[u] = u * 64 < S && i < p.n ? p.tokens[i] : -1;
    }
    const int me = p.tokens[blockIdx.x];
    if (me >= p.vocab && tid == 0) atomicOr(p.err, ADN_DEVERR_TOKEN);
    if (me < 0 || me >= p.vocab) return;
    int mine = 0, before = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        mine += __popcll(__ballot(t[u] == me));
        before += __popcll(__ballot(t[u] == me && wave * S + u * 64 + lane < (int)blockIdx.x));
    }
    if (lane == 0) {
        cnt[wave] = mine;
        ahead[wave] = before;
    }
    __syncthreads();
    int m = 0, at = 0, rank = 0;
#pragma unroll
    for (int w = 0; w < FW; ++w) {
        if (w == wave) at = m;
        m += cnt[w];
        rank += ahead[w];
    }
    // the token's blocks, one a position, share its columns: a wave a strip of 64 lanes' where the rows are
    // few, else a block a strip, its waves an eighth of the rows each
    const int strips = (p.d + 64 * W - 1) / (64 * W);
    const bool light = m <= LOADS;
    const int sharers = min(m, light ? (strips + FW - 1) / FW : strips);
    if (rank >= sharers) return;  // (all waves agree)
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const unsigned long long hit = __ballot(t[u] == me);
        if (t[u] == me) list[at + __popcll(hit & ((1ull << lane) - 1))] = wave * S + u * 64 + lane;
        at += __popcll(hit);
    }
    __syncthreads();
    const int per = light ? m : (m + FW - 1) / FW, a = light ? 0 : min(m, wave * per), b = min(m, a + per);
    for (int s = light ? rank * FW + wave : rank; s < strips; s += light ? sharers * FW : sharers) {
        const int c = (s * 64 + lane) * W;
        float acc[W];
#pragma unroll
        for (int j = 0; j < W; ++j) acc[j] = 0.0f;
        if (c < p.d)
            for (int e0 = a; e0 < b; e0 += LOADS) {
                V v[LOADS];
#pragma unroll
                for (int u = 0; u < LOADS; ++u)
                    if (e0 + u < b) v[u] = *reinterpret_cast<const V *>((const T *)p.src + (long)list[e0 + u] * p.src_stride + c);
#pragma unroll
                for (int u = 0; u < LOADS; ++u)
                    if (e0 + u < b)
#pragma unroll
                        for (int j = 0; j < W; ++j) acc[j] += to_f32<T>(v[u][j]);
            }
        if (!light) {  // the waves' sums in order
            __syncthreads();
            if (wave)
#pragma unroll
                for (int j = 0; j < W; ++j) part[wave - 1][lane * W + j] = acc[j];
            __syncthreads();
            if (wave) continue;
#pragma unroll
            for (int q = 0; q < FW - 1; ++q)
#pragma unroll
                for (int j = 0; j < W; ++j) acc[j] += part[q][lane * W + j];
        }
        if (c < p.d) {
            V o;
#pragma unroll
            for (int j = 0; j < W; ++j) o[j] = from_f32<T>(acc[j] * p.scale);
            *reinterpret_cast<V *>((T *)p.dst + (long)me * p.dst_stride + c) = o;
        }
    }
}

// ---- radix sort of (token, position) -------------------------------------------------------
struct Sort {
    const int32_t *tokens;
    int n, vocab, nblocks;      // blocks of TILE keys
    int passes;
    unsigned *keys[2];          // keys and positions, alternating
    int32_t *pos[2];
    unsigned *cnt;              // [digit][block]: counts of a pass
    bool own_prefix;            // offsets formed by the moving blocks, else in place by k_scan
    unsigned *err;
    // zeros of the table, written by the launches' other blocks: a share of the rows each
    void *dst;
    long dst_stride;
    int d;
    bool vec;
    int launch, launches;
};

template <typename T>
__device__ __forceinline__ void sort_zero(const Sort &s) {
    const long v0 = (long)s.vocab * s.launch / s.launches, v1 = (long)s.vocab * (s.launch + 1) / s.launches;
    const long first = ((long)blockIdx.x - s.nblocks) * (NT / 64) + (threadIdx.x >> 6);
    const long step = ((long)gridDim.x - s.nblocks) * (NT / 64);
    if (s.vec)
        zero_rows<T, true>((T *)s.dst, s.dst_stride, s.d, v0, v1, first, step);
    else
        zero_rows<T, false>((T *)s.dst, s.dst_stride, s.d, v0, v1, first, step);
}

// cnt[digit][block] = keys of the block's tile with the pass's digit (the first pass forms the keys from
// the tokens).  Counting a pass's digits while the pass before it moves the keys was 60 us slower at
// 32768 positions: a few digits are most of the keys, and their counters take one atomic at a time.
template <typename T>
__global__ __launch_bounds__(NT) void k_radix_count(Sort s, int pass) {
    if ((int)blockIdx.x >= s.nblocks) return sort_zero<T>(s);
    __shared__ unsigned h[RADIX];
    h[threadIdx.x] = 0;
    __syncthreads();
    const unsigned *keys = s.keys[(pass & 1) ^ 1];
    const long base = (long)blockIdx.x * TILE;
    unsigned k[TILE / NT];
#pragma unroll
    for (int j = 0; j < TILE / NT; ++j) {
        const long i = base + j * NT + threadIdx.x;
        k[j] = i >= s.n ? 0 : pass ? keys[i] : key_of(s.tokens, i, s.vocab, s.err);
    }
#pragma unroll
    for (int j = 0; j < TILE / NT; ++j)
        if (base + j * NT + threadIdx.x < s.n) atomicAdd(&h[(k[j] >> (8 * pass)) & (RADIX - 1)], 1u);
    __syncthreads();
    s.cnt[(long)threadIdx.x * s.nblocks + blockIdx.x] = h[threadIdx.x];
}

// Exclusive prefix sum in place over `m` counts (a multiple of 8), one block, 8 counts a thread.
__global__ __launch_bounds__(1024) void k_scan(unsigned *cnt, long m) {
    typedef unsigned uint4v __attribute__((ext_vector_type(4)));
    __shared__ unsigned wsum[16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    unsigned carry = 0;
    uint4v next[2] = {};
    auto fetch = [&](long i) {
        if (i < m)
#pragma unroll
            for (int h = 0; h < 2; ++h) next[h] = *reinterpret_cast<const uint4v *>(cnt + i + 4 * h);
        else
            next[0] = next[1] = uint4v{};
    };
    fetch((long)threadIdx.x * 8);
    for (long base = 0; base < m; base += 1024 * 8) {
        const long i = base + (long)threadIdx.x * 8;
        uint4v v[2] = {next[0], next[1]};
        fetch(i + 1024 * 8);
        unsigned sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned c = v[j / 4][j % 4];
            v[j / 4][j % 4] = sum;
            sum += c;
        }
        unsigned s = sum;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const unsigned o = __shfl_up(s, off, 64);
            if (lane >= off) s += o;
        }
        if (lane == 63) wsum[w] = s;
        __syncthreads();
        unsigned before = carry, all = 0;
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            before += q < w ? wsum[q] : 0;
            all += wsum[q];
        }
        carry += all;
        before += s - sum;
        if (i < m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                v[h] += before;
                *reinterpret_cast<uint4v *>(cnt + i + 4 * h) = v[h];
            }
        __syncthreads();
    }
}

// Moves each key and its position to its place: the number of smaller digits, of its digit in earlier
// blocks, and its rank among the tile's keys of that digit (stable).
template <typename T>
__global__ __launch_bounds__(NT) void k_radix_move(Sort s, int pass) {
    if ((int)blockIdx.x >= s.nblocks) return sort_zero<T>(s);
    __shared__ unsigned at[NT / 64][RADIX];  // next place of each wave's keys of a digit
    __shared__ unsigned wsum[NT / 64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, shift = 8 * pass;
    const unsigned *cnt = s.cnt, *keys = s.keys[(pass & 1) ^ 1];
    const int32_t *pos = s.pos[(pass & 1) ^ 1];
    unsigned *keys_out = s.keys[pass & 1];
    int32_t *pos_out = s.pos[pass & 1];
#pragma unroll
    for (int q = 0; q < NT / 64; ++q) at[q][threadIdx.x] = 0;
    // keys of the digit threadIdx.x: in earlier blocks, and in all
    unsigned before = 0, all = 0;
    if (s.own_prefix) {
#pragma unroll 16
        for (int b = 0; b < s.nblocks; ++b) {
            const unsigned c = cnt[(long)threadIdx.x * s.nblocks + b];
            before += b < (int)blockIdx.x ? c : 0;
            all += c;
        }
    } else {
        before = cnt[(long)threadIdx.x * s.nblocks + blockIdx.x];
    }
    const long base = (long)blockIdx.x * TILE + (long)w * W_KEYS;
    unsigned key[W_KEYS / 64];
    int32_t from[W_KEYS / 64];
#pragma unroll
    for (int j = 0; j < W_KEYS / 64; ++j) {
        const long i = base + j * 64 + lane;
        key[j] = 0;
        from[j] = (int32_t)i;
        if (i < s.n) {
            key[j] = pass ? keys[i] : key_of(s.tokens, i, s.vocab, nullptr);
            if (pass) from[j] = pos[i];
        }
    }
    if (s.own_prefix) {  // plus the keys of smaller digits
        unsigned sum = all;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const unsigned o = __shfl_up(sum, off, 64);
            if (lane >= off) sum += o;
        }
        if (lane == 63) wsum[w] = sum;
        __syncthreads();
        before += sum - all;
        for (int q = 0; q < w; ++q) before += wsum[q];
    } else {
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < W_KEYS / 64; ++j)
        if (base + j * 64 + lane < s.n) atomicAdd(&at[w][(key[j] >> shift) & (RADIX - 1)], 1u);
    __syncthreads();
#pragma unroll
    for (int q = 0; q < NT / 64; ++q) {
        const unsigned c = at[q][threadIdx.x];
        at[q][threadIdx.x] = before;
        before += c;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < W_KEYS / 64; ++j) {
        const bool in = base + j * 64 + lane < s.n;
        const unsigned dig = (key[j] >> shift) & (RADIX - 1);
        unsigned long long same = __ballot(in);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const unsigned long long m = __ballot((dig >> b) & 1);
            same &= (dig >> b) & 1 ? m : ~m;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        unsigned o = 0;
        if (in) o = at[w][dig];
        // every lane has read the place before the first of a digit moves it on (the wave's LDS operations
        // run in order; the fences keep the compiler to it)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (in && rank == 0) at[w][dig] = o + (unsigned)__popcll(same);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if (in) {
            keys_out[o + rank] = key[j];
            pos_out[o + rank] = from[j];
        }
    }
}

// ---- sums of the sorted rows ----------------------------------------------------------------
// A wave adds the rows of sorted entries [chunk C, + C) in order, 64 W columns from strip * 64 W.
// part[chunk][0]: the sum of a table row that began in an earlier chunk; part[chunk][1]: of one
// that begins here and goes on in the next.
template <typename T, bool VEC>
__global__ __launch_bounds__(64) void k_chunk_sums(TableParams p, const unsigned *keys, const int32_t *pos, int C,
                                                   float *part) {
    constexpr int W = VEC ? 16 / (int)sizeof(T) : 1;
    typedef typename VecT<T, W>::type V;
    const int lane = threadIdx.x;
    const long chunk = blockIdx.x, a = chunk * C;
    const long b = a + C < p.n ? a + C : (long)p.n;
    const int c = (int)(blockIdx.y * 64 + lane) * W;
    const bool in = c < p.d;
    const int cc = in ? c : 0;  // lanes beyond the row load what they do not use
    float acc[W];
#pragma unroll
    for (int j = 0; j < W; ++j) acc[j] = 0.0f;
    bool began = a == 0;  // the current table row begins in this chunk
    // C0 entries: keys of entries e0 - 1 .. e0 + C0 in the lanes 0 .. C0 + 1, positions in 0 .. C0 - 1
    for (long e0 = a; e0 < b; e0 += C0) {
        const long ke = e0 - 1 + lane;
        const int kl = lane < C0 + 2 && ke >= 0 && ke < p.n ? (int)keys[ke] : -1;
        const int pl = lane < C0 && e0 + lane < b ? pos[e0 + lane] : 0;
        if (e0 == a && a > 0) began = __builtin_amdgcn_readlane(kl, 0) != __builtin_amdgcn_readlane(kl, 1);
        if (__builtin_amdgcn_readlane(kl, 1) >= p.vocab) break;  // positions without a token are the last ones
#pragma unroll
        for (int g = 0; g < C0; g += 8) {
            if (e0 + g >= b) break;
            V v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const long at = __builtin_amdgcn_readlane(pl, g + u);  // 0 behind the end: not used
                v[u] = *reinterpret_cast<const V *>((const T *)p.src + at * p.src_stride + cc);
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int k = __builtin_amdgcn_readlane(kl, g + u + 1), kn = __builtin_amdgcn_readlane(kl, g + u + 2);
                if (e0 + g + u >= b || k >= p.vocab) break;
#pragma unroll
                for (int j = 0; j < W; ++j) acc[j] += to_f32<T>(v[u][j]);
                const bool last = kn != k;  // the table row's last position
                if (!last && e0 + g + u + 1 < b) continue;
                if (in) {
                    if (last && began) {
                        V o;
#pragma unroll
                        for (int j = 0; j < W; ++j) o[j] = from_f32<T>(acc[j] * p.scale);
                        *reinterpret_cast<V *>((T *)p.dst + (long)k * p.dst_stride + c) = o;
                    } else {
                        float *q = part + (chunk * 2 + (began ? 1 : 0)) * p.d + c;
#pragma unroll
                        for (int j = 0; j < W; ++j) q[j] = acc[j];
                    }
                }
#pragma unroll
                for (int j = 0; j < W; ++j) acc[j] = 0.0f;
                began = true;
            }
        }
    }
}

// Table rows that begin in a chunk and end in a later one: their partial sums in chunk order, the
// waves a quarter of the chunks each.
template <typename T>
__global__ __launch_bounds__(NT) void k_join_sums(TableParams p, const unsigned *keys, int C, const float *part) {
    __shared__ float sum[3][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long chunk = blockIdx.x, a = chunk * C, b = a + C;
    if (b >= p.n) return;
    // the chunks that begin with the row: chunk + 1 .. chunk + m (64 of them looked at beside the rest)
    const long chunks = (p.n + C - 1) / C;
    const unsigned k = keys[b - 1], kb = keys[b], ka = keys[a], kz = keys[a > 0 ? a - 1 : 0];
    unsigned ahead = keys[min((chunk + 1 + lane) * C, (long)p.n - 1)];
    if (k >= (unsigned)p.vocab || kb != k) return;  // nothing goes on
    if (a > 0 && ka == k && kz == k) return;        // it began in an earlier chunk
    long m = 0;
    for (;;) {
        const unsigned long long on = __ballot(chunk + 1 + m + lane < chunks && ahead == k);
        m += on == ~0ull ? 64 : __ffsll(~on) - 1;
        if (on != ~0ull) break;
        ahead = keys[min((chunk + 1 + m + lane) * C, (long)p.n - 1)];
    }
    const int c = (int)(blockIdx.y * 64 + lane);
    const long per = (m + 3) / 4, q0 = chunk + 1 + min(m, wave * per), q1 = chunk + 1 + min(m, (wave + 1) * per);
    float acc = 0.0f;
    if (c < p.d) {
        if (wave == 0) acc = part[(chunk * 2 + 1) * p.d + c];
#pragma unroll 16
        for (long q = q0; q < q1; ++q) acc += part[q * 2 * p.d + c];
    }
    if (wave) sum[wave - 1][lane] = acc;
    __syncthreads();
    if (wave || c >= p.d) return;
    acc = ((acc + sum[0][lane]) + sum[1][lane]) + sum[2][lane];
    ((T *)p.dst)[(long)k * p.dst_stride + c] = from_f32<T>(acc * p.scale);
}

// Sorted entries a chunk: C0, more where there would be over 2048 chunks (a frequent token's partial
// sums are added one after another).
int chunk_len(long n) { return (int)((std::max<long>(C0, (n + 2047) / 2048) + C0 - 1) / C0 * C0); }

struct GradLayout {
    size_t keys[2], pos[2], cnt, part, bytes;
    int nblocks;
};
GradLayout grad_layout(const TableParams &p) {
    GradLayout L{};
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += (bytes + 255) / 256 * 256;
        return r;
    };
    L.nblocks = (int)(((long)p.n + TILE - 1) / TILE);
    for (int i = 0; i < 2; ++i) {
        L.keys[i] = take((size_t)p.n * 4);
        L.pos[i] = take((size_t)p.n * 4);
    }
    L.cnt = take((size_t)RADIX * L.nblocks * 4);
    const long C = chunk_len(p.n);
    L.part = take((size_t)((p.n + C - 1) / C) * 2 * p.d * 4);
    L.bytes = at;
    return L;
}

}  // namespace

void launch_embed_lookup(const TableParams &p, hipStream_t st) {
    if (p.n == 0) return;
    const int eb = elem_bytes(p.dtype);
    const bool vec = rows_vec16(p.src, p.src_stride, p.d, eb) && rows_vec16(p.dst, p.dst_stride, p.d, eb);
    const unsigned grid = (unsigned)(((long)p.n + NT / 64 - 1) / (NT / 64));
    dispatch_type(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        if (vec)
            k_lookup<T, true><<<grid, NT, 0, st>>>(p);
        else
            k_lookup<T, false><<<grid, NT, 0, st>>>(p);
    });
}

size_t embed_grad_workspace_bytes(const TableParams &p) { return p.n <= FEW ? 0 : grad_layout(p).bytes; }

void launch_embed_grad(const TableParams &p, void *ws, hipStream_t st) {
    const int eb = elem_bytes(p.dtype);
    const bool vdst = rows_vec16(p.dst, p.dst_stride, p.d, eb);
    const bool vec = vdst && rows_vec16(p.src, p.src_stride, p.d, eb);
    if (p.n <= FEW) {
        dispatch_type(p.dtype, [&](auto t) {
            typedef decltype(t) T;
            const unsigned grid = (unsigned)(p.n + (p.vocab + FEW_ROWS - 1) / FEW_ROWS);
            if (vec)
                k_grad_few<T, true><<<grid, 64 * FW, 0, st>>>(p);
            else
                k_grad_few<T, false><<<grid, 64 * FW, 0, st>>>(p);
        });
        return;
    }
    const GradLayout L = grad_layout(p);
    char *w = (char *)ws;
    Sort s{};
    s.tokens = p.tokens, s.n = p.n, s.vocab = p.vocab, s.nblocks = L.nblocks;
    for (int i = 0; i < 2; ++i) {
        s.keys[i] = (unsigned *)(w + L.keys[i]);
        s.pos[i] = (int32_t *)(w + L.pos[i]);
    }
    s.cnt = (unsigned *)(w + L.cnt);
    s.passes = 1;
    while (s.passes < 4 && (p.vocab >> (8 * s.passes)) > 0) ++s.passes;  // keys are 0 .. vocab
    s.own_prefix = L.nblocks <= OWN_PREFIX;
    s.err = p.err;
    s.dst = p.dst, s.dst_stride = p.dst_stride, s.d = p.d, s.vec = vdst;
    s.launches = 2 * s.passes;
    float *part = (float *)(w + L.part);
    const int C = chunk_len(p.n);
    const unsigned chunks = (unsigned)(((long)p.n + C - 1) / C);
    const long counts = (long)RADIX * L.nblocks;
    dispatch_type(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        // zero-writing blocks: a wave has about eight rows of a launch's share
        const unsigned zb = (unsigned)std::max<long>(1, std::min<long>(1024, p.vocab / (s.launches * 32L)));
        for (int pass = 0; pass < s.passes; ++pass) {
            s.launch = 2 * pass;
            k_radix_count<T><<<L.nblocks + zb, NT, 0, st>>>(s, pass);
            if (!s.own_prefix) k_scan<<<1, 1024, 0, st>>>(s.cnt, counts);
            s.launch = 2 * pass + 1;
            k_radix_move<T><<<L.nblocks + zb, NT, 0, st>>>(s, pass);
        }
        const unsigned *keys = s.keys[(s.passes & 1) ^ 1];
        const int32_t *pos = s.pos[(s.passes & 1) ^ 1];
        const int W = vec ? 16 / (int)sizeof(T) : 1;
        const dim3 grid(chunks, (unsigned)((p.d + 64 * W - 1) / (64 * W)));
        if (vec)
            k_chunk_sums<T, true><<<grid, 64, 0, st>>>(p, keys, pos, C, part);
        else
            k_chunk_sums<T, false><<<grid, 64, 0, st>>>(p, keys, pos, C, part);
        k_join_sums<T><<<dim3(chunks, (unsigned)((p.d + 63) / 64)), NT, 0, st>>>(p, keys, C, part);
    });
}

}  // namespace adn
