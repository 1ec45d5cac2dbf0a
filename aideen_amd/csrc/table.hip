// The embedding table as a trained tensor: scaled lookup (Tokenizer::embed_sequence,
// tokenizer.rs:151-159, with a factor) and its gradient
//
//   out[i] = scale E[tok_i]            dE[v] = scale sum over i with tok_i = v of dout[i]
//
// The gradient adds each table row's positions in ascending order, so it is the same bits on every
// run: the positions are sorted by token (a stable radix sort of 8 bits a pass), the sorted list is
// cut into chunks, a wave adds one chunk's rows in order and stores the table rows that begin and
// end in it; of a row that crosses chunks every chunk stores a partial sum, and a second kernel
// adds those in chunk order.  Rows without a token are zeros, written by a fill of the whole table.
#include <algorithm>

#include "train.h"

namespace adn {

namespace {

constexpr int NT = 256;
constexpr int RADIX = 256;
constexpr int TILE = 2048;            // keys a block of a radix pass
constexpr int W_KEYS = TILE / (NT / 64);  // consecutive keys a wave of it

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

// ---- radix sort of (token, position) -------------------------------------------------------
// cnt[digit][block] = keys of the block's tile with that digit.  First pass: the keys are formed
// from the tokens (and the positions are their indexes).
template <bool FIRST>
__global__ __launch_bounds__(NT) void k_radix_count(const unsigned *keys, const int32_t *tokens, int n, int vocab,
                                                    int shift, unsigned *cnt, int nblocks, unsigned *err) {
    __shared__ unsigned h[RADIX];
    h[threadIdx.x] = 0;
    __syncthreads();
    const long base = (long)blockIdx.x * TILE;
    for (int j = threadIdx.x; j < TILE; j += NT) {
        const long i = base + j;
        if (i < n) {
            const unsigned k = FIRST ? key_of(tokens, i, vocab, err) : keys[i];
            atomicAdd(&h[(k >> shift) & (RADIX - 1)], 1u);
        }
    }
    __syncthreads();
    cnt[(long)threadIdx.x * nblocks + blockIdx.x] = h[threadIdx.x];
}

// Exclusive prefix sum in place over `m` counts, one block.
__global__ __launch_bounds__(1024) void k_scan(unsigned *cnt, long m) {
    __shared__ unsigned wsum[16];
    __shared__ unsigned carry;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (threadIdx.x == 0) carry = 0;
    __syncthreads();
    for (long base = 0; base < m; base += 1024) {
        const long i = base + threadIdx.x;
        const unsigned v = i < m ? cnt[i] : 0;
        unsigned s = v;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const unsigned o = __shfl_up(s, off, 64);
            if (lane >= off) s += o;
        }
        if (lane == 63) wsum[w] = s;
        __syncthreads();
        unsigned before = carry;
        for (int q = 0; q < w; ++q) before += wsum[q];
        if (i < m) cnt[i] = before + s - v;
        __syncthreads();
        if (threadIdx.x == 1023) carry = before + s;
        __syncthreads();
    }
}

// Moves each key and its position to its place: offset[digit][block] plus its rank among the
// tile's keys of that digit, in order (stable).
template <bool FIRST>
__global__ __launch_bounds__(NT) void k_radix_move(const unsigned *keys, const int32_t *pos, const int32_t *tokens,
                                                   int n, int vocab, int shift, const unsigned *offset, int nblocks,
                                                   unsigned *keys_out, int32_t *pos_out) {
    __shared__ unsigned at[NT / 64][RADIX];  // next place of each wave's keys of a digit
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int q = 0; q < NT / 64; ++q) at[q][threadIdx.x] = 0;
    __syncthreads();
    const long base = (long)blockIdx.x * TILE + (long)w * W_KEYS;
    unsigned key[W_KEYS / 64];
#pragma unroll
    for (int j = 0; j < W_KEYS / 64; ++j) {
        const long i = base + j * 64 + lane;
        key[j] = 0;
        if (i < n) {
            key[j] = FIRST ? key_of(tokens, i, vocab, nullptr) : keys[i];
            atomicAdd(&at[w][(key[j] >> shift) & (RADIX - 1)], 1u);
        }
    }
    __syncthreads();
    {
        unsigned o = offset[(long)threadIdx.x * nblocks + blockIdx.x];
#pragma unroll
        for (int q = 0; q < NT / 64; ++q) {
            const unsigned c = at[q][threadIdx.x];
            at[q][threadIdx.x] = o;
            o += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < W_KEYS / 64; ++j) {
        const long i = base + j * 64 + lane;
        const bool in = i < n;
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
        __builtin_amdgcn_wave_barrier();  // every lane has read the place before the first of a digit moves it on
        if (in && rank == 0) at[w][dig] = o + (unsigned)__popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (in) {
            keys_out[o + rank] = key[j];
            pos_out[o + rank] = FIRST ? (int32_t)i : pos[i];
        }
    }
}

// ---- sums of the sorted rows ----------------------------------------------------------------
template <typename T, bool VEC>
__global__ __launch_bounds__(NT) void k_zero_table(T *dst, int vocab, int d, long stride) {
    constexpr int W = VEC ? 16 / (int)sizeof(T) : 1;
    typedef typename VecT<T, W>::type V;
    V z;
#pragma unroll
    for (int j = 0; j < W; ++j) z[j] = from_f32<T>(0.0f);
    const int lane = threadIdx.x & 63;
    for (long v = (long)blockIdx.x * (NT / 64) + (threadIdx.x >> 6); v < vocab; v += (long)gridDim.x * (NT / 64))
        for (int c = lane * W; c < d; c += 64 * W) *reinterpret_cast<V *>(dst + v * stride + c) = z;
}

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
    const unsigned none = (unsigned)p.vocab;
    float acc[W];
#pragma unroll
    for (int j = 0; j < W; ++j) acc[j] = 0.0f;
    bool began = a == 0 || keys[a - 1] != keys[a];  // the current table row begins in this chunk
    for (long e = a; e < b; ++e) {
        const unsigned k = keys[e];
        if (k >= none) break;  // positions without a token are the last ones
        if (in) {
            const V v = *reinterpret_cast<const V *>((const T *)p.src + (long)pos[e] * p.src_stride + c);
#pragma unroll
            for (int j = 0; j < W; ++j) acc[j] += to_f32<T>(v[j]);
        }
        const bool last = e + 1 == p.n || keys[e + 1] != k;  // the table row's last position
        if (!last && e + 1 < b) continue;
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

// Table rows that begin in a chunk and end in a later one: their partial sums in chunk order.
template <typename T>
__global__ __launch_bounds__(64) void k_join_sums(TableParams p, const unsigned *keys, int C, const float *part) {
    const long chunk = blockIdx.x, a = chunk * C, b = a + C;
    if (b >= p.n) return;
    const unsigned k = keys[b - 1];
    if (k >= (unsigned)p.vocab || keys[b] != k) return;       // nothing goes on
    if (keys[a] == k && a > 0 && keys[a - 1] == k) return;    // it began in an earlier chunk
    // the chunks that hold the rest: from the next one to the one with its last position
    long lo = b, hi = p.n;  // first sorted entry behind it
    while (lo < hi) {
        const long mid = (lo + hi) / 2;
        if (keys[mid] <= k)
            lo = mid + 1;
        else
            hi = mid;
    }
    const long end = (lo - 1) / C;
    const int c = (int)(blockIdx.y * 64 + threadIdx.x);
    if (c >= p.d) return;
    float acc = part[(chunk * 2 + 1) * p.d + c];
#pragma unroll 8
    for (long q = chunk + 1; q <= end; ++q) acc += part[q * 2 * p.d + c];
    ((T *)p.dst)[(long)k * p.dst_stride + c] = from_f32<T>(acc * p.scale);
}

// Sorted entries a chunk: 32, more where there would be over 2048 chunks (a frequent token's
// partial sums are added one after another).
int chunk_len(long n) { return (int)std::max<long>(32, (n + 2047) / 2048); }

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

size_t embed_grad_workspace_bytes(const TableParams &p) { return grad_layout(p).bytes; }

void launch_embed_grad(const TableParams &p, void *ws, hipStream_t st) {
    const int eb = elem_bytes(p.dtype);
    const bool vdst = rows_vec16(p.dst, p.dst_stride, p.d, eb);
    dispatch_type(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        const unsigned grid = (unsigned)std::min<long>(2048, ((long)p.vocab + NT / 64 - 1) / (NT / 64));
        if (vdst)
            k_zero_table<T, true><<<grid, NT, 0, st>>>((T *)p.dst, p.vocab, p.d, p.dst_stride);
        else
            k_zero_table<T, false><<<grid, NT, 0, st>>>((T *)p.dst, p.vocab, p.d, p.dst_stride);
    });
    if (p.n == 0) return;
    const GradLayout L = grad_layout(p);
    char *w = (char *)ws;
    unsigned *keys[2] = {(unsigned *)(w + L.keys[0]), (unsigned *)(w + L.keys[1])};
    int32_t *pos[2] = {(int32_t *)(w + L.pos[0]), (int32_t *)(w + L.pos[1])};
    unsigned *cnt = (unsigned *)(w + L.cnt);
    float *part = (float *)(w + L.part);
    int cur = 0;
    for (int shift = 0; shift < 32 && (shift == 0 || (p.vocab >> shift) > 0); shift += 8) {  // keys are 0 .. vocab
        const int nxt = shift ? cur ^ 1 : 0;
        if (shift == 0) {
            k_radix_count<true><<<L.nblocks, NT, 0, st>>>(nullptr, p.tokens, p.n, p.vocab, 0, cnt, L.nblocks, p.err);
            k_scan<<<1, 1024, 0, st>>>(cnt, (long)RADIX * L.nblocks);
            k_radix_move<true><<<L.nblocks, NT, 0, st>>>(nullptr, nullptr, p.tokens, p.n, p.vocab, 0, cnt, L.nblocks,
                                                         keys[nxt], pos[nxt]);
        } else {
            k_radix_count<false><<<L.nblocks, NT, 0, st>>>(keys[cur], nullptr, p.n, p.vocab, shift, cnt, L.nblocks,
                                                           nullptr);
            k_scan<<<1, 1024, 0, st>>>(cnt, (long)RADIX * L.nblocks);
            k_radix_move<false><<<L.nblocks, NT, 0, st>>>(keys[cur], pos[cur], nullptr, p.n, p.vocab, shift, cnt,
                                                          L.nblocks, keys[nxt], pos[nxt]);
        }
        cur = nxt;
    }
    const int C = chunk_len(p.n);
    const unsigned chunks = (unsigned)(((long)p.n + C - 1) / C);
    const bool vec = vdst && rows_vec16(p.src, p.src_stride, p.d, eb);
    dispatch_type(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        const int W = vec ? 16 / (int)sizeof(T) : 1;
        const dim3 grid(chunks, (unsigned)((p.d + 64 * W - 1) / (64 * W)));
        if (vec)
            k_chunk_sums<T, true><<<grid, 64, 0, st>>>(p, keys[cur], pos[cur], C, part);
        else
            k_chunk_sums<T, false><<<grid, 64, 0, st>>>(p, keys[cur], pos[cur], C, part);
        k_join_sums<T><<<dim3(chunks, (unsigned)((p.d + 63) / 64)), 64, 0, st>>>(p, keys[cur], C, part);
    });
}

}  // namespace adn
