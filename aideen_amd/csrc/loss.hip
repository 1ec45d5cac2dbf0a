// Softmax cross entropy of the LM head over the whole vocabulary, with its gradients, keeping the
// logits only where they are few:
//
//   z = x W^T + b,  lse_i = log sum_v exp(z_iv),  loss_i = lse_i - z_i,t(i)
//   dz_iv = g_i (exp(z_iv - lse_i) - [v = t(i)])
//   dx = dz W,  dW = dz^T x,  db = sum_i dz_i
//
// Four products on the fp16 MFMA, 2 n V d operations each (n rows, V entries, width d): the logits
// for lse (stored nowhere: their epilogue leaves each row's maximum and sum of exponentials per 256
// entries), then a piece of the vocabulary at a time the logits again, whose epilogue stores the
// piece's dz, and dz W and dz^T x from it.  A piece's dz takes at most PIECE_BYTES, or 256 entries of
// every row where those are more (beyond 2^18 rows of fp32), and is there twice, for dx and for dW.
// What grows with n V in the workspace is the statistics, 8 bytes a row and 256 entries, and db's
// partial sums, 4 bytes an entry and tile of rows.  Forming the logits twice costs a third more
// operations than keeping them, n V values of 4 bytes, which is done up to PIECE_BYTES where it
// saves time (loss_plan).
//
// Operands are fp16 planes.  fp32 tensors: two planes, hi = f16(s x) and lo = f16(s x - hi), three
// products hi hi + hi lo + lo hi (the split of the forward's products: 2^-22 of a product is lost).
// bf16 tensors: one plane, exact (8 of 11 bits), one product.  dz is rounded to the same number of
// planes: 22 bits or 11, where bf16 outputs keep 8.  The scales are powers of two.  W has one, by its
// largest value (values below 2^-36 of it are lost, to the same absolute error as the rest).  Every row
// of x has its own for the logits, 2^f_i, by the row's largest value, so that a row's size does not
// matter to another row's loss.  dz_i is stored as (softmax - onehot) / c_i, c_i in [1, 2) the mantissa of
// 1 - softmax_i,t(i): the target's value is then a power of two, rounded by nothing.  With g_i = m_i 2^e_i
// in it (a mean's 1 / n is alike for all rows) or without c_i (the softmax of an untrained head is too), one
// plane would round all targets the same way, up to 3e-4 of the whole gradient.  dx takes c_i g_i in fp32
// behind its product, so that g_i does not matter to another row's dx either; dW sums over the rows, its
// planes of x hold x_i c_i m_i 2^(e_i + F), one F for all, by the largest |x_i| 2^e_i.  All sums are fp32.
//
// fp16's smallest step leaves a small probability few bits (2^-39 under the scale of 2^14: 1e-10 to 2 %), which
// is nothing in dx_i, a sum over all entries, and everything in dW's row of a rare entry.  So the logits' epilogue
// takes each entry's maximum over its rows (32 to 128), and where one of 256 entries is that small stores the
// tile's dz for dW apart, each entry times a power of two of its own (MAX_D).  dW's product takes such blocks to
// the entry's largest over its rows on the way to the MFMA, and its sums back at the end; the other blocks are
// dx's, so that a head with few rare entries pays for the maxima and some shares of dW (8192 x 512 fp32 1 %,
// 4096 x 2048 bf16 nothing, 531 x 1024 bf16 2 %, calls of 50 us 2 us; with rare entries everywhere 8, 4 and 9 %).
// dx has planes that no other row matters to.
//
// Layout.  Every plane is stored as blocks of 32 rows x 16 columns, 1 KB each, the blocks of 32 rows
// one after another along the columns; rows and columns are padded with zeros.  A block is what one
// direct global->LDS load of a wave moves.  The one image serves a product over the columns (a lane
// reads 8 consecutive columns of its row, ds_read_b128) and a product over the rows (the transposing
// ds_read_b64_tr_b16: a group of 16 lanes reads 4 rows of 16 columns, 128 adjacent bytes, and each
// lane gets one column), so x, W and dz are laid out once and no operand is ever transposed in memory.
#include <algorithm>
#include <cmath>

#include "gemm_common.h"
#include "train.h"

namespace adn {

namespace {

using gemm::lds_barrier;

constexpr int NT = 256;             // threads a workgroup: 4 waves
constexpr size_t PIECE_BYTES = 256u << 20;
constexpr int BM = 128;             // rows of a gradient tile
constexpr int TV = 256;             // entries a workgroup of the logits' product covers
constexpr int NW = 4;               // waves of a workgroup
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int XR = 8;               // rows of x a block splits
constexpr long SAMPLE_FROM = 32L << 20;  // bytes of W from which its scale is taken from a sample
constexpr int W_BLOCKS = 1024;      // blocks of the pass over |W|, one partial each

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) short4v lds_short4;

template <int N>
__device__ __forceinline__ void wait_vmcnt() {  // the other counters left alone
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// 16 bytes a lane from base + off (base wave-uniform, off in bytes) to the LDS address `lds` + 16 lane.
// In assembly so that the compiler does not take the transposing LDS reads for uses of it and wait for
// every load in flight before each: the waits are wait_vmcnt's.  It has no register output.  The compiler
// does not see into it, so it keeps the wait states itself: one between the write of m0 and its use, five
// before a scalar base that a vector instruction may just have written.
__device__ __forceinline__ void load_lds(const void *base, unsigned off, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(base)
                 : "memory", "m0");
}

// The same with 4 bytes a lane, to `lds` + 4 lane.
__device__ __forceinline__ void load_lds4(const void *base, unsigned off, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, %2"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(base)
                 : "memory", "m0");
}

// e of |g| = m 2^e, m in [1, 2); 0 for zero and what is not finite
__device__ __forceinline__ int exp_of(float g) {
    const float a = fabsf(g);
    return a > 0.0f && a < INFINITY ? ilogbf(a) : 0;
}

__device__ __forceinline__ float finite_abs(float v) {
    const float a = fabsf(v);
    return a < INFINITY ? a : 0.0f;  // NaN and inf stay in their own rows
}

// A product rounded to fp32 before it is split: left to itself the compiler rounds the product of the one use
// straight to fp16 and of the other by way of fp32, and the two halves no longer belong together.
__device__ __forceinline__ float rounded(float v) {
    asm("" : "+v"(v));
    return v;
}

// The mantissa of v, in [1, 2); 1 for zero.
__device__ __forceinline__ float mantissa(float v) {
    return __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, v) & 0x007fffffu) | 0x3f800000u);
}
// c_i of a row: of its softmax at the target, less one
__device__ __forceinline__ float row_unit(float z_target, float lse) {
    return mantissa(__builtin_amdgcn_exp2f(z_target - lse) - 1.0f);
}
// c_i m_i
__device__ __forceinline__ float row_factor(float g, float c) { return ldexpf(g, -exp_of(g)) * c; }
constexpr int DZ_EXP = 14;  // (softmax - onehot) / c is stored times 2^14, at most 2^14
// For dW an entry's values of a tile of rows are stored times 2^D more, D > 0 where the largest of them is so
// small that the planes' smallest step, 2^-39, would cost it bits: with two planes (22 bits) 16 below 2^-16, and
// with either number 24 below 2^-24.  Down to 2^-24 the factor is an fp16 value.
constexpr int MAX_D = 24;

// Exponent that takes a magnitude to [2^14, 2^15); 0 for zero and what is not finite.
__device__ __forceinline__ int scale_exp(float mx) {
    if (!(mx > 0.0f) || mx == INFINITY) return 0;
    return 15 - (ilogbf(mx) + 1);
}

__device__ __forceinline__ float block_max256(float v, float *red) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// W's scale is taken from a sample of its rows, HEAD powers of two below what their largest value allows,
// so that W is not read once for its scale alone; the kernels that split W find its largest value on the
// way, and are launched once more for a W that the sample's scale does not fit (they end at once for
// one that it does): 256 rows of 512 against 50257 entries, losses alone, 69 us for 60.
constexpr int HEAD = 3;
// The exponent from the sample's partial maxima (0 where they are: W's own are needed); `redo`: from what
// the first launch reported, false where that is nothing.
__device__ __forceinline__ bool scale_of_w(const float *part, int n, int head, const unsigned *w_max, bool redo, float *red,
                                           int &kw, bool &blank) {
    if (redo) {
        kw = scale_exp(__builtin_bit_cast(float, *w_max));
        return *w_max != 0;
    }
    float m = 0.0f;
    for (int i = threadIdx.x; i < n; i += NT) m = fmaxf(m, part[i]);
    m = block_max256(m, red);
    kw = m > 0.0f ? scale_exp(m) - head : 0;
    blank = m == 0.0f;
    return true;
}
// Reports the largest value of a share of W that the sample's scale does not fit (blank: any).
__device__ __forceinline__ void report_w(float top, int kw, bool blank, unsigned *w_max) {
    if (blank ? top > 0.0f : ldexpf(top, kw) > 65000.0f) atomicMax(w_max, __builtin_bit_cast(unsigned, top));
}

// Chunk (8 halves) of a block's row r that holds columns [0, 8) in the LDS image of an operand read
// along its columns: the b128 reads of 32 consecutive rows then use every bank alike.
__device__ __forceinline__ int swz(int r) { return ((r >> 2) ^ (r >> 3)) & 1; }

// A blocked matrix: planes `plane` halves apart, `ncb` column blocks in a row of blocks.
struct Planes {
    const _Float16 *p;
    long plane;
    int ncb;
};

// What the products share.  Rows (M) are the MFMA's rows, held in a lane's registers; columns (N)
// its columns, one a lane.
struct LossGemm {
    Planes A, B;
    int nM, nN, S;       // tiles of rows and columns, shares of K
    int K;               // length of the product (a multiple of the slice), the same for every share but the last
    int Ks;              // length of a share
    int a_row0;          // first row of A (entries of the piece), a multiple of 32
    // logits
    const float *bias;
    const int32_t *f;    // [rows padded] exponents of the rows' scales
    const int32_t *tgt;  // [rows padded] targets, -1 = none
    const int32_t *kw_dev;  // exponent of W's scale
    int vocab, rows;
    float *part_m, *part_s, *ztgt;      // [tile][rows padded]: maximum and sum of exponentials; the target's logit
    long rows_pad;
    const void *w_raw;                  // LOGITS_RAW: W's rows as they are, their stride in bytes, the
    unsigned w_stride;                  //   partial maxima of |W|
    const float *w_part;
    int w_blocks, w_head, w_redo;       //   of the sampled rows (scale_of_w)
    unsigned *w_max;
    float *out_loss, *out_lse;          // LOGITS_ALL: [rows] or null
    float *z;                           // kept logits, a workgroup's registers as they are, or null
    const float *lse, *g, *c, *h;       // per row: lse (in units of log 2), g_i = m_i 2^e_i, c_i, c_i m_i
    float *out_c, *out_h;               // LOGITS_ALL: the last two
    _Float16 *dz, *dzw;                 // planes of the piece, blocks of rows x entries: for dx, for dW (or null)
    long dz_plane;
    _Float16 *fx;                       // of dzw, [group of rows][entries of the piece]: 2^-D
    int *scaled;                        // [group of rows][TV entries]: dzw is not dz; where it is, dzw is not written
    long fx_ld;
    int fx_log;                         // GRAD: rows of a group = 2^fx_log
    const _Float16 *plain;              // GRAD dW: A's planes of blocks that are not scaled
    int dz_ncb;
    float *db_part;                     // [row tile][entries padded]
    long db_ld;
    // gradients
    float *part;                        // [share][rows][ld] partial sums, or null: dst is written
    long part_ld;
    int add;                            // the partial sums are added to
    void *dst;                          // [rows] of the result
    long dst_stride;
    int out_rows, out_cols;
    const int32_t *e_all;               // exponent of dst's values (dx: of g and kw_dev)
};

// The logits' epilogues: each row's maximum and sum of a tile of entries (RAW: W's rows read as they are
// and split on the way to the MFMA, for losses alone, where planes of W would be read once); dz of a
// piece, from the product again or (KEPT) from the logits that the first pass kept; both in one where a
// tile holds the whole vocabulary.
enum { LOGITS_STATS = 0, LOGITS_DZ = 1, GRAD = 2, LOGITS_RAW = 3, LOGITS_ALL = 4, LOGITS_KEPT = 5 };

// The two gradients of a piece in one launch: tiles of the one with the longer shares first.
struct LossGrads {
    LossGemm dw, dx;
    int first;     // workgroups of the first gradient
    int dx_first;
};

// One tile: WGM x WGN waves of WTM x WTN MFMA tiles of 32x32.  NP planes an operand; a k slice is
// 16 KB values (24 KB of LDS for either NP at the largest tile: three slices and two workgroups a
// CU, so that one's epilogue runs under the other's MFMAs).  TRA / TRB: the operand's rows are the
// product's K.
template <int NP, int WTM, int WTN, int WGM, int WGN, int EXTRA = 0>  // EXTRA: halves beside a slice
struct Tile {
    static constexpr int KB = NP == 2 ? 1 : 2;
    static constexpr int TM = WGM * WTM * 32, TN = WGN * WTN * 32;
    static constexpr int A_BLK = TM / 32 * KB, B_BLK = TN / 32 * KB;  // 1 KB loads a plane and slice
    static constexpr int SLICE = NP * (A_BLK + B_BLK) * 512;           // halves of a k slice
    // slices of the LDS ring: what half of a CU's LDS holds, three to six
    static constexpr int FIT = 80 * 512 / (SLICE + EXTRA), STAGES = FIT < 3 ? 3 : FIT > 6 ? 6 : FIT;
    static constexpr int RING = STAGES * SLICE, LDS = STAGES * (SLICE + EXTRA);
    static_assert(WGM * WGN == 4, "four waves");
    static_assert(LDS * 2 <= 80 * 1024, "two workgroups a CU");
};
constexpr int FX = 128;  // factors of a slice of dW's dz: one an entry of the tile

template <int MODE, typename T, int NP, int WTM, int WTN, int WGM, int WGN, bool TRA, bool TRB>
__device__ __forceinline__ void loss_tile(const LossGemm &p, int bid, _Float16 *ring) {
    typedef Tile<NP, WTM, WTN, WGM, WGN, MODE == GRAD ? FX : 0> G;
    constexpr bool FACT = MODE == GRAD && TRA;  // dW: dz's groups of rows have scales of their own
    constexpr int KB = G::KB, TM = G::TM, TN = G::TN, A_BLK = G::A_BLK, B_BLK = G::B_BLK, STAGES = G::STAGES;
    constexpr int A_PW = (A_BLK + NW - 1) / NW, B_PW = (B_BLK + NW - 1) / NW;
    constexpr int LOADS = NP * (A_PW + B_PW);
    constexpr int A_SZ = A_BLK * 512, B_SZ = B_BLK * 512;      // halves a plane and slice
    constexpr int SLICE = G::SLICE;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WGN, wn = wave % WGN;
    const int r = lane & 31, hh = lane >> 5;
    int s, mt, nt;
    gemm::map_block(bid, p.nM * p.nN * p.S, p.nM, p.nN, s, mt, nt);
    const int k0 = s * p.Ks;
    const int nk = (min(p.Ks, p.K - k0)) / (16 * KB);

    // Direct global->LDS loads of a slice.  A load's address is a wave-uniform base plus a byte offset of
    // the lane that is the same for every load of an operand.
    auto lane_off = [&](bool tr) -> unsigned {
        if (!tr) return (lane >> 1) * 32 + (((lane & 1) ^ swz(lane >> 1)) * 16);  // a block, its rows' chunks swizzled
        // rows k of odd column blocks stand at k ^ 4, so that the two 128-byte pieces that 32 lanes
        // read at once (4 rows of neighbouring column blocks) are in different halves of the banks
        if constexpr (KB == 2) return (lane ^ ((wave & 1) * 8)) * 16;             // a block of 32 k x 16 columns
        return (lane >> 5) * 1024 + ((lane & 31) ^ ((lane >> 5) * 8)) * 16;       // 16 k of two neighbouring blocks
    };
    // base of load idx at slice 0, in halves
    auto src_of = [&](bool tr, int idx, int tile0, const Planes &P) -> long {
        if (!tr) return ((long)(tile0 / 32 + idx / KB) * P.ncb + k0 / 16 + idx % KB) * 512;  // (row block, k block)
        // columns past the matrix (a multiple of 32 wide) read its last blocks: outputs that are not stored
        if constexpr (KB == 2) return ((long)(k0 / 32) * P.ncb + min(tile0 / 16 + idx, P.ncb - 2 + (idx & 1))) * 512;
        return (long)min(tile0 / 16 + 2 * idx, P.ncb - 2) * 512;  // the k block and half: step_of
    };
    // slice kt's offset from slice 0
    auto step_of = [&](bool tr, int kt, const Planes &P) -> long {
        if (!tr) return (long)kt * KB * 512;
        if constexpr (KB == 2) return (long)kt * P.ncb * 512;
        const int k = k0 / 16 + kt;
        return (long)(k >> 1) * P.ncb * 512 + (k & 1) * 256;
    };
    // a plane's slice of the tile is A_BLK (B_BLK) KB in either order; where the waves outnumber its
    // loads some are issued twice, to the same place
    constexpr bool RAW = MODE == LOGITS_RAW;
    long asrc[A_PW], bsrc[B_PW];
    // RAW: load idx is 16 rows of 64 bytes (4 chunks, swizzled by the row), a lane a chunk
    constexpr int R_PW = NP * A_PW;
    unsigned roff[RAW ? R_PW : 1];
    const char *rbase = nullptr;
    int kw_raw = 0;
    float top_raw = 0.0f;
    bool blank_raw = false;
    auto swz4 = [](int row) { return ((row >> 1) ^ (row >> 2)) & 3; };
    if constexpr (RAW) {
        static_assert(A_BLK * NP % NW == 0, "whole loads a wave");
        const int row0 = p.a_row0 + mt * TM;
        rbase = (const char *)p.w_raw + (long)row0 * p.w_stride;
#pragma unroll
        for (int j = 0; j < R_PW; ++j) {
            const int row = (wave + NW * j) * 16 + (lane >> 2);
            roff[j] = (unsigned)min(row, p.vocab - 1 - row0) * p.w_stride + (((lane & 3) ^ swz4(row)) * 16);
        }
        if (!scale_of_w(p.w_part, p.w_blocks, p.w_head, p.w_max, p.w_redo, reinterpret_cast<float *>(ring), kw_raw, blank_raw))
            return;
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < A_PW; ++j) asrc[j] = src_of(TRA, (wave + NW * j) % A_BLK, p.a_row0 + mt * TM, p.A);
#pragma unroll
    for (int j = 0; j < B_PW; ++j) bsrc[j] = src_of(TRB, (wave + NW * j) % B_BLK, nt * TN, p.B);
    // FACT: which of 64 groups of rows are scaled, from the share's on; of the slices issued last
    const int g1 = FACT ? (k0 + nk * 16 * KB - 1) >> p.fx_log : 0;
    auto scaled_groups = [&](int g0) -> unsigned long long {
        const int g = g0 + lane;
        return __ballot(g <= g1 && p.scaled[(long)min(g, g1) * (p.fx_ld / TV) + mt / (TV / TM)]);
    };
    int mask_g0 = FACT ? k0 >> p.fx_log : 0;
    unsigned long long mask = FACT ? scaled_groups(mask_g0) : 0;
    unsigned bits = 0;
    const unsigned aoff = lane_off(TRA), boff = lane_off(TRB);
    const unsigned ring0 = (unsigned)(uintptr_t)(lds_void *)ring;
    // sc (dW): scaled blocks and their factors are looked out for
    auto issue = [&](int kt, auto sc) {
        constexpr bool SC = decltype(sc)::value;
        const unsigned base = ring0 + (kt % STAGES) * (SLICE * 2);
        const _Float16 *Ap = FACT && !SC ? p.plain : p.A.p;
        if constexpr (SC) {
            const int g = (k0 + kt * 16 * KB) >> p.fx_log;
            if (g - mask_g0 >= 64) mask = scaled_groups(mask_g0 += 64);
            const unsigned bit = (unsigned)(mask >> (g - mask_g0)) & 1;
            if (!bit) Ap = p.plain;
            bits = bits << 1 | bit;
        }
        Ap += step_of(TRA, kt, p.A);
        const _Float16 *Bp = p.B.p + step_of(TRB, kt, p.B);
        if constexpr (RAW) {
#pragma unroll
            for (int j = 0; j < R_PW; ++j) load_lds(rbase + kt * 64, roff[j], base + (wave + NW * j) * 1024);
        }
#pragma unroll
        for (int q = 0; q < NP; ++q) {
#pragma unroll
            for (int j = 0; !RAW && j < A_PW; ++j)
                load_lds(Ap + q * p.A.plane + asrc[j], aoff, base + (q * A_SZ + ((wave + NW * j) % A_BLK) * 512) * 2);
#pragma unroll
            for (int j = 0; j < B_PW; ++j)
                load_lds(Bp + q * p.B.plane + bsrc[j], boff,
                         base + (NP * A_SZ + q * B_SZ + ((wave + NW * j) % B_BLK) * 512) * 2);
        }
        if constexpr (SC) {
            static_assert(TM == FX, "a factor an entry");
            load_lds4(p.fx + (long)((k0 + kt * 16 * KB) >> p.fx_log) * p.fx_ld + mt * TM, lane * 4,
                      ring0 + (G::RING + kt % STAGES * FX) * 2);
        }
    };
    // MFMA operand of 32 rows (columns) `t` of the tile, k block kb of the slice
    auto frag = [&](const _Float16 *img, bool tr, int t, int kb) -> half8 {
        if (!tr) return *reinterpret_cast<const half8 *>(img + (t * KB + kb) * 512 + r * 16 + ((hh ^ swz(r)) * 8));
        const int odd = (lane >> 4) & 1;
        const int at = (2 * t + odd) * (KB * 256) + (kb * 16 + 8 * hh + ((lane >> 2) & 3) + 4 * odd) * 16 + (lane & 3) * 4;
        const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(img + at));
        const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4 *)(img + (at ^ 64)));
        return __builtin_bit_cast(half8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };

    // RAW: the planes of 32 rows' 8 values a lane, split here
    auto raw_frag = [&](const _Float16 *img, int t, int kb, half8 &hi, half8 &lo) {
        const int row = t * 32 + r;
        const char *at = (const char *)img + row * 64;
        float v[8];
        if constexpr (NP == 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const floatx4 x = *reinterpret_cast<const floatx4 *>(at + (((2 * hh + h) ^ swz4(row)) * 16));
#pragma unroll
                for (int u = 0; u < 4; ++u) v[4 * h + u] = x[u];
            }
        } else {
            typedef T V8 __attribute__((ext_vector_type(16 / sizeof(T))));
            const V8 x = *reinterpret_cast<const V8 *>(at + (((2 * kb + hh) ^ swz4(row)) * 16));
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = to_f32<T>(x[u % (16 / (int)sizeof(T))]);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            top_raw = fmaxf(top_raw, finite_abs(v[u]));
            const float x = ldexpf(v[u], kw_raw);
            hi[u] = (_Float16)x;
            if constexpr (NP == 2) lo[u] = (_Float16)(x - (float)hi[u]);  // (one plane: lo is hi)
        }
    };

    floatx16 acc[WTM][WTN];
#pragma unroll
    for (int i = 0; i < WTM; ++i)
#pragma unroll
        for (int j = 0; j < WTN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    float fmost[WTM], fless[WTM];  // FACT: a lane's entries' largest factor, and its inverse
    unsigned long long any = 0;    // FACT: a block of the share's is scaled
    // KEPT: this tile's logits, 16 bytes a lane side by side
    const auto kept = [&](int i, int j, int e4) -> floatx4 * {
        const long tile = (long)(p.a_row0 / TV + mt) * p.nN + nt;
        return reinterpret_cast<floatx4 *>(p.z) + (((tile * NW + wave) * WTM + i) * WTN + j) * 256 + e4 * 64 + lane;
    };
    if constexpr (MODE == LOGITS_KEPT) {
#pragma unroll
        for (int i = 0; i < WTM; ++i)
#pragma unroll
            for (int j = 0; j < WTN; ++j)
#pragma unroll
                for (int e4 = 0; e4 < 4; ++e4) {
                    const floatx4 t = *kept(i, j, e4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][4 * e4 + e] = t[e];
                }
    } else {
        auto product = [&](auto sc) {
            constexpr bool SC = decltype(sc)::value;
            constexpr int IN_FLIGHT = (STAGES - 2) * (LOADS + SC);
#pragma unroll
            for (int t = 0; t < STAGES - 1; ++t)
                if (t < nk) issue(t, sc);
            for (int kt = 0; kt < nk; ++kt) {
                // slice kt is in LDS once this wave's later loads are all that is in flight; the barrier
                // covers the other waves' loads, and their reads of the slot that is loaded next
                if (kt + STAGES - 2 < nk)
                    wait_vmcnt<IN_FLIGHT>();
                else
                    wait_vmcnt<0>();
                lds_barrier();
                if (kt + STAGES - 1 < nk) issue(kt + STAGES - 1, sc);
                const _Float16 *base = ring + (kt % STAGES) * SLICE;
                const bool scaled = SC && (bits >> (min(kt + STAGES - 1, nk - 1) - kt) & 1);
                _Float16 fac[WTM];
                if (scaled)
#pragma unroll
                    for (int i = 0; i < WTM; ++i)
                        fac[i] = (_Float16)((float)ring[G::RING + kt % STAGES * FX + (wm * WTM + i) * 32 + r] * fless[i]);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) {
                    half8 a[NP][WTM];
                    if constexpr (RAW) {
#pragma unroll
                        for (int i = 0; i < WTM; ++i) raw_frag(base, wm * WTM + i, kb, a[0][i], a[NP - 1][i]);
                    } else {
#pragma unroll
                        for (int q = 0; q < NP; ++q)
#pragma unroll
                            for (int i = 0; i < WTM; ++i) a[q][i] = frag(base + q * A_SZ, TRA, wm * WTM + i, kb);
                    }
                    half8 b[NP][WTN];
#pragma unroll
                    for (int j = 0; j < WTN; ++j)
#pragma unroll
                        for (int q = 0; q < NP; ++q) b[q][j] = frag(base + NP * A_SZ + q * B_SZ, TRB, wn * WTN + j, kb);
                    if (scaled)
#pragma unroll
                        for (int q = 0; q < NP; ++q)
#pragma unroll
                            for (int i = 0; i < WTM; ++i) a[q][i] *= fac[i];
                    // all of a k block's reads before its first MFMA: left to itself the compiler reads the last
                    // columns halfway and waits there (8192 x 512 fp32 4600 us for 4505, 4096 x 2048 bf16 3285 for 3218)
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 0; j < WTN; ++j) {
#pragma unroll
                        for (int i = 0; i < WTM; ++i) {
                            if constexpr (NP == 2) {
                                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1][i], b[0][j], acc[i][j], 0, 0, 0);
                                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0][i], b[1][j], acc[i][j], 0, 0, 0);
                            }
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0][i], b[0][j], acc[i][j], 0, 0, 0);
                        }
                    }
                }
            }
        };
        // dW: the marks of the share's blocks.  The product that looks out for scaled ones costs 10 % more
        // whether there are any or not, so that shares without one take the other.
        for (int g = k0 >> p.fx_log; FACT && g <= g1; g += 64) any |= g == mask_g0 ? mask : scaled_groups(g);
        if constexpr (FACT)
            if (any) {
                // the largest factor 2^-D of a lane's entries over the share's rows: scaled blocks are taken to its scale
#pragma unroll
                for (int i = 0; i < WTM; ++i) fmost[i] = 0.0f;
                const _Float16 *f = p.fx + mt * TM + wm * WTM * 32 + r;
#pragma unroll 16
                for (int g = mask_g0 + hh; g <= g1; g += 2)
#pragma unroll
                    for (int i = 0; i < WTM; ++i) fmost[i] = fmaxf(fmost[i], (float)f[g * p.fx_ld + i * 32]);
#pragma unroll
                for (int i = 0; i < WTM; ++i) fmost[i] = fmaxf(fmost[i], __shfl_xor(fmost[i], 32, 64));
#pragma unroll
                for (int i = 0; i < WTM; ++i) fless[i] = 1.0f / fmost[i];
                product(std::true_type{});
            }
        if (!any) product(std::false_type{});
    }
    if constexpr (RAW) {
        if (p.w_head && !p.w_redo && nt == 0) {
            const float top = wave_max(top_raw);
            if (lane == 0) report_w(top, kw_raw, blank_raw, p.w_max);
        }
    }
    lds_barrier();  // every wave is done with the ring

    // Output layout of a 32x32 tile: lane holds column r; register e row 8 (e / 4) + 4 hh + e % 4.
    if constexpr (MODE == GRAD) {
        if (any) {  // the entries' scales, by way of LDS from a lane an entry to the sums' registers
            float *own = reinterpret_cast<float *>(ring) + wave * (WTM * 32);
            if (hh == 0)
#pragma unroll
                for (int i = 0; i < WTM; ++i) own[i * 32 + r] = fmost[i];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < WTM; ++i)
#pragma unroll
                for (int e4 = 0; e4 < 4; ++e4) {
                    const floatx4 t = *reinterpret_cast<const floatx4 *>(own + i * 32 + 8 * e4 + 4 * hh);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int j = 0; j < WTN; ++j) acc[i][j][4 * e4 + e] *= t[e];
                }
        }
        const int ec = p.e_all ? *p.e_all : p.g ? *p.kw_dev : 0;  // g: dx, a row's own exponent
        const long r0 = (long)mt * TM + wm * WTM * 32 + 4 * hh;
        const int c0 = nt * TN + wn * WTN * 32 + r;
        auto store = [&](auto whole) {
            constexpr bool W = decltype(whole)::value;  // an interior tile: nothing to check
#pragma unroll
            for (int i = 0; i < WTM; ++i) {
                auto in = [&](int rr, int j) { return W || (r0 + i * 32 + rr < p.out_rows && c0 + 32 * j < p.out_cols); };
                if (p.part) {
                    float *o = p.part + ((long)s * p.out_rows + r0 + i * 32) * p.part_ld + c0;
                    if (p.add) {  // the earlier sums of 32 rows are loaded before the first store
#pragma unroll
                        for (int e = 0; e < 16; ++e)
#pragma unroll
                            for (int j = 0; j < WTN; ++j) {
                                const int rr = 8 * (e / 4) + e % 4;
                                if (in(rr, j)) acc[i][j][e] += o[rr * p.part_ld + 32 * j];
                            }
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e)
#pragma unroll
                        for (int j = 0; j < WTN; ++j) {
                            const int rr = 8 * (e / 4) + e % 4;
                            if (in(rr, j)) o[rr * p.part_ld + 32 * j] = acc[i][j][e];
                        }
                } else {
                    int er[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) er[e] = ec;
                    if (p.g) {  // the rows' factors, loaded before the first store
                        float g[16], h[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            g[e] = p.g[r0 + i * 32 + 8 * (e / 4) + e % 4];
                            h[e] = p.h[r0 + i * 32 + 8 * (e / 4) + e % 4];
                        }
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            er[e] = exp_of(g[e]) - DZ_EXP - ec;
#pragma unroll
                            for (int j = 0; j < WTN; ++j) acc[i][j][e] *= h[e];
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int rr = 8 * (e / 4) + e % 4;
                        T *o = (T *)p.dst + (r0 + i * 32 + rr) * p.dst_stride + c0;
#pragma unroll
                        for (int j = 0; j < WTN; ++j)
                            if (in(rr, j)) o[32 * j] = from_f32<T>(ldexpf(acc[i][j][e], er[e]));
                    }
                }
            }
        };
        if ((long)mt * TM + TM <= p.out_rows && nt * TN + TN <= p.out_cols)
            store(std::integral_constant<bool, true>{});
        else
            store(std::integral_constant<bool, false>{});
    } else {
        static_assert(TM == TV && WGN == 1, "a wave's columns are the tile's");
        constexpr bool KEPT = MODE == LOGITS_KEPT;
        // the tile's biases; entries beyond the vocabulary get -inf: no part of any sum.  From here on
        // logits are in units of log 2 (z log2(e)), what exp2 takes.
        float *bias_l = reinterpret_cast<float *>(ring);                   // [TM]
        const int v0 = p.a_row0 + mt * TM;
        for (int c = tid; !KEPT && c < TM; c += NT) {
            float b = v0 + c < p.vocab ? (p.bias ? p.bias[v0 + c] : 0.0f) : -INFINITY;
            if (b < -1e38f && b > -INFINITY) b = -1e38f;  // the type's lowest value stays finite
            bias_l[c] = b * LOG2E;
        }
        lds_barrier();
        const int kw = RAW ? kw_raw : *p.kw_dev;
        const int w0 = v0 + wm * WTM * 32;  // the wave's first entry
        float unscale[WTN];
#pragma unroll
        for (int j = 0; !KEPT && j < WTN; ++j) unscale[j] = ldexpf(LOG2E, -(p.f[nt * TN + j * 32 + r] + kw));
#pragma unroll
        for (int i = 0; !KEPT && i < WTM; ++i)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
                const floatx4 b = *reinterpret_cast<const floatx4 *>(bias_l + (wm * WTM + i) * 32 + 8 * e4 + 4 * hh);
#pragma unroll
                for (int j = 0; j < WTN; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[i][j][4 * e4 + e] = __builtin_fmaf(acc[i][j][4 * e4 + e], unscale[j], b[e]);
                if constexpr (MODE == LOGITS_STATS)
                    if (p.z)
#pragma unroll
                        for (int j = 0; j < WTN; ++j)
                            *kept(i, j, e4) = floatx4{acc[i][j][4 * e4], acc[i][j][4 * e4 + 1], acc[i][j][4 * e4 + 2], acc[i][j][4 * e4 + 3]};
            }
        float *red_m = bias_l + TM, *red_s = red_m + 4 * TN, *zt = red_s + 4 * TN;  // [wave][TN] twice, [TN]
        if constexpr (MODE != LOGITS_DZ && !KEPT) {
#pragma unroll
            for (int j = 0; j < WTN; ++j) {
                const long m = (long)nt * TN + j * 32 + r;
                float mx = acc[0][j][0];
#pragma unroll
                for (int i = 0; i < WTM; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) mx = fmaxf(mx, acc[i][j][e]);
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const float ref = mx == -INFINITY ? 0.0f : mx;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < WTM; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        sum += __builtin_amdgcn_exp2f(acc[i][j][e] - ref);
                sum += __shfl_xor(sum, 32, 64);
                if (hh == 0) {
                    red_m[wave * TN + j * 32 + r] = mx;
                    red_s[wave * TN + j * 32 + r] = sum;
                }
                // the target's logit, by the one lane that holds it
                const int t = p.tgt[m] - w0;
                if (__any(t >= 0 && t < WTM * 32))
#pragma unroll
                    for (int i = 0; i < WTM; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (t == i * 32 + 8 * (e / 4) + 4 * hh + e % 4) 
                                *(MODE == LOGITS_ALL ? zt + j * 32 + r : p.ztgt + m) = acc[i][j][e];
            }
            lds_barrier();
            for (int c = tid; MODE != LOGITS_ALL && c < TN; c += NT) {
                float mx = red_m[c];
#pragma unroll
                for (int w = 1; w < 4; ++w) mx = fmaxf(mx, red_m[w * TN + c]);
                const float ref = mx == -INFINITY ? 0.0f : mx;
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    sum += red_s[w * TN + c] * __builtin_amdgcn_exp2f(red_m[w * TN + c] - ref);
                const long o = (long)mt * p.rows_pad + nt * TN + c;
                p.part_m[o] = mx;
                p.part_s[o] = sum;
            }
        }
        if constexpr (MODE == LOGITS_DZ || MODE == LOGITS_ALL || KEPT) {
            const bool grads = p.dz || p.dzw || p.db_part;
            float *any_l = zt + TN, *scale = any_l + 4 + wave * (WTM * 32);     // dzw: [wave]; [WTM * 32 entries]
            float *colsum = any_l + 4 + 4 * (WTM * 32) + wave * (32 * WTM * 33);  // db: [WTM * 32 entries][32 + 1]
            float unit_l[WTN];  // LOGITS_ALL: c
            // 32 rows x 32 entries of a lane's values as blocks: a register pair of 8 values becomes the two
            // 16-byte chunks of a block's row (columns 0-7 in the lower half of the wave, 8-15 in the upper one)
            auto put = [&](_Float16 *dst, int i, int j, auto value) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    unsigned pk[NP][4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        unsigned w[NP] = {};
#pragma unroll
                        for (int v = 0; v < 2; ++v) {
                            const float x = value(8 * h + 2 * u + v);  // (a power of two times a value: rounded once)
                            const _Float16 hi = (_Float16)x;
                            w[0] |= (unsigned)__builtin_bit_cast(unsigned short, hi) << (16 * v);
                            if constexpr (NP == 2)
                                w[1] |= (unsigned)__builtin_bit_cast(unsigned short, (_Float16)(x - (float)hi)) << (16 * v);
                        }
#pragma unroll
                        for (int q = 0; q < NP; ++q) pk[q][u] = w[q];
                    }
                    const long blk = (long)(nt * (TN / 32) + j) * p.dz_ncb + (long)mt * (TM / 16) + (wm * WTM + i) * 2 + h;
#pragma unroll
                    for (int q = 0; q < NP; ++q) {
                        const auto x0 = __builtin_amdgcn_permlane32_swap(pk[q][0], pk[q][2], false, false);
                        const auto x1 = __builtin_amdgcn_permlane32_swap(pk[q][1], pk[q][3], false, false);
                        const uint4v o = {x0[0], x1[0], x0[1], x1[1]};
                        *reinterpret_cast<uint4v *>(dst + q * p.dz_plane + blk * 512 + r * 16 + hh * 8) = o;
                    }
                    __builtin_amdgcn_sched_barrier(0);  // one pair after the other: 128 values are held besides
                }
            };
#pragma unroll
            for (int j = 0; j < WTN; ++j) {
                const long m = (long)nt * TN + j * 32 + r;
                const float gm = p.g[m];
                const int tm = p.tgt[m], t = tm - w0;
                float lse, cm;
                if constexpr (MODE == LOGITS_ALL) {
                    float mx = red_m[j * 32 + r];
#pragma unroll
                    for (int w = 1; w < 4; ++w) mx = fmaxf(mx, red_m[w * TN + j * 32 + r]);
                    const float ref = mx == -INFINITY ? 0.0f : mx;
                    float sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        sum += red_s[w * TN + j * 32 + r] * __builtin_amdgcn_exp2f(red_m[w * TN + j * 32 + r] - ref);
                    lse = ref + log2f(sum);
                    const float z = tm >= 0 ? zt[j * 32 + r] : lse;
                    cm = row_unit(z, lse);
                    if (wave == 0 && hh == 0) {
                        if (p.out_lse && m < p.rows) p.out_lse[m] = tm >= 0 ? lse * LN2 : 0.0f;
                        if (p.out_loss && m < p.rows) p.out_loss[m] = tm >= 0 ? (lse - z) * LN2 : 0.0f;
                        if (grads) p.out_c[m] = cm, p.out_h[m] = row_factor(gm, cm);
                    }
                    unit_l[j] = cm;
                    if (!grads) continue;
                } else {
                    lse = p.lse[m];
                    cm = p.c[m];
                }
                const float unit = 1.0f / cm;
                const bool off = gm == 0.0f;  // no target, or nothing from upstream: exactly zero
#pragma unroll
                for (int i = 0; i < WTM; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        acc[i][j][e] = __builtin_amdgcn_exp2f(acc[i][j][e] - lse);
                if (__any(t >= 0 && t < WTM * 32))
#pragma unroll
                    for (int i = 0; i < WTM; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (t == i * 32 + 8 * (e / 4) + 4 * hh + e % 4) acc[i][j][e] -= 1.0f;
#pragma unroll
                for (int i = 0; i < WTM; ++i) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[i][j][e] = off ? 0.0f : rounded(acc[i][j][e] * unit);
                    if (p.dz) put(p.dz, i, j, [&](int e) { return acc[i][j][e] * (float)(1 << DZ_EXP); });
                }
            }
            if (grads && p.db_part) {  // each entry's sum over the tile's rows, lanes in order
                float gm[WTN], cm[WTN];
#pragma unroll
                for (int j = 0; j < WTN; ++j) {
                    const long m = (long)nt * TN + j * 32 + r;
                    gm[j] = p.g[m];
                    if constexpr (MODE == LOGITS_ALL)
                        cm[j] = unit_l[j];
                    else
                        cm[j] = p.c[m];
                }
#pragma unroll
                for (int i = 0; i < WTM; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float t = acc[i][0][e] * gm[0] * cm[0];
#pragma unroll
                        for (int j = 1; j < WTN; ++j) t += acc[i][j][e] * gm[j] * cm[j];
                        colsum[(i * 32 + 8 * (e / 4) + 4 * hh + e % 4) * 33 + r] = t;
                    }
                lds_barrier();
                if (lane < WTM * 32) {
                    float t = 0.0f;
#pragma unroll
                    for (int c = 0; c < 32; ++c) t += colsum[lane * 33 + c];
                    p.db_part[(long)nt * p.db_ld + v0 + wm * WTM * 32 + lane] = t;
                }
            }
            if (p.dzw) {
                // an entry's largest value over the tile's rows: those of a lane, then over the 32 lanes of a half wave,
                // which divide the 32 values a lane holds between them a bit at a time, so that lane r ends with value r
                static_assert(WTM == 2, "32 values a lane");
                float top[32];
#pragma unroll
                for (int q = 0; q < 32; ++q) {
                    top[q] = fabsf(acc[q / 16][0][q % 16]);
#pragma unroll
                    for (int j = 1; j < WTN; ++j) top[q] = fmaxf(top[q], fabsf(acc[q / 16][j][q % 16]));
                }
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    const auto x = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, top[q]),
                                                                    __builtin_bit_cast(unsigned, top[q + 16]), false, false);
                    top[q] = fmaxf(__builtin_bit_cast(float, (unsigned)x[0]), __builtin_bit_cast(float, (unsigned)x[1]));
                }
                auto halve = [&](auto n, auto ctrl) {  // lanes that differ in bit n, for n = 4 in all three lower bits
                    constexpr int N = decltype(n)::value, C = decltype(ctrl)::value;
#pragma unroll
                    for (int q = 0; q < N; ++q) {
                        const float mine = lane & N ? top[q + N] : top[q], other = lane & N ? top[q] : top[q + N];
                        const int moved = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, other), C, 0xF, 0xF, true);
                        top[q] = fmaxf(mine, __builtin_bit_cast(float, moved));
                    }
                };
                using std::integral_constant;
                halve(integral_constant<int, 8>{}, integral_constant<int, 0x128>{});  // row_ror 8
                halve(integral_constant<int, 4>{}, integral_constant<int, 0x141>{});  // row_half_mirror
                halve(integral_constant<int, 2>{}, integral_constant<int, 0x4E>{});   // quad_perm 2 3 0 1
                halve(integral_constant<int, 1>{}, integral_constant<int, 0xB1>{});   // quad_perm 1 0 3 2
                const float most = top[0];
                const int D = most < 0x1p-24f ? MAX_D : NP == 2 && most < 0x1p-16f ? 16 : 0;
                const int at = (r >> 4) * 32 + 8 * ((r & 15) >> 2) + 4 * hh + (r & 3);
                scale[at] = ldexpf(1.0f, DZ_EXP + D);
                p.fx[(long)nt * p.fx_ld + mt * TM + wm * (WTM * 32) + at] = (_Float16)ldexpf(1.0f, -D);
                const bool any_here = __any(D > 0 && most > 0.0f);
                if (lane == 0) any_l[wave] = any_here ? 1.0f : 0.0f;
                lds_barrier();
                const bool any = any_l[0] + any_l[1] + any_l[2] + any_l[3] > 0.0f;
                if (tid == 0) p.scaled[(long)nt * (p.fx_ld / TV) + mt] = any;
                if (p.dz && !any) return;  // dz serves dW too
#pragma unroll
                for (int i = 0; i < WTM; ++i) {
                    float f[16];
#pragma unroll
                    for (int e4 = 0; e4 < 4; ++e4) {
                        const floatx4 t = *reinterpret_cast<const floatx4 *>(scale + i * 32 + 8 * e4 + 4 * hh);
#pragma unroll
                        for (int e = 0; e < 4; ++e) f[4 * e4 + e] = t[e];
                    }
#pragma unroll
                    for (int j = 0; j < WTN; ++j) put(p.dzw, i, j, [&](int e) { return acc[i][j][e] * f[e]; });
                }
            }
        }
    }
}

template <int MODE, typename T, int NP, int WTN>
__global__ __launch_bounds__(NT, 2) void k_loss_logits(LossGemm p) {
    __shared__ __attribute__((aligned(1024))) _Float16 ring[Tile<NP, 2, WTN, 4, 1>::RING];
    loss_tile<MODE, T, NP, 2, WTN, 4, 1, false, false>(p, blockIdx.x, ring);
}

template <typename T, int NP, int WTM, int WTN, int WGM, int WGN>
__global__ __launch_bounds__(NT, 2) void k_loss_grads(LossGrads p) {
    __shared__ __attribute__((aligned(1024))) _Float16 ring[Tile<NP, WTM, WTN, WGM, WGN, FX>::LDS];
    const int b = blockIdx.x;
    if ((b < p.first) == (p.dx_first != 0))
        loss_tile<GRAD, T, NP, WTM, WTN, WGM, WGN, false, true>(p.dx, p.dx_first ? b : b - p.first, ring);
    else
        loss_tile<GRAD, T, NP, WTM, WTN, WGM, WGN, true, true>(p.dw, p.dx_first ? b - p.first : b, ring);
}

// ---- operands ------------------------------------------------------------------------------
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *row, int c, int d, float (&v)[8]) {
    if constexpr (VEC) {
        if (c + 8 <= d) {
            typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
            for (int q = 0; q < (int)sizeof(T) / 2; ++q) {
                const V x = *reinterpret_cast<const V *>(row + c + q * (16 / (int)sizeof(T)));
#pragma unroll
                for (int j = 0; j < 16 / (int)sizeof(T); ++j) v[q * (16 / (int)sizeof(T)) + j] = to_f32<T>(x[j]);
            }
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < d ? to_f32<T>(row[c + j]) : 0.0f;
}

// v 2^ex f
template <int NP>
__device__ __forceinline__ void store_planes(_Float16 *dst, long plane, const float (&v)[8], int ex, float f = 1.0f) {
    half8 hi, lo;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float x = rounded(ldexpf(v[j], ex) * f);
        hi[j] = (_Float16)x;
        if constexpr (NP == 2) lo[j] = (_Float16)(x - (float)hi[j]);
    }
    *reinterpret_cast<half8 *>(dst) = hi;
    if constexpr (NP == 2) *reinterpret_cast<half8 *>(dst + plane) = lo;
}

struct Prep {
    const void *x;
    long x_stride;
    const void *w;
    long w_stride;
    int rows, d, vocab, dcb;     // dcb: column blocks of a row of width d
    int w_blocks, row_blocks;    // blocks of the pass over |W|; blocks of XR rows of x
    int w_sample, w_step, w_head;  // rows of that pass, one of every w_step; HEAD, or 0: all of them
    unsigned *w_max;             // W's largest value, found by the split (w_head)
    int w_rows, w_cols;          // blocks of 32 rows of W, and blocks that share the columns of each
    const int32_t *targets;
    const float *dloss;
    unsigned *err;
    _Float16 *xp, *x2p, *wp;     // x for the logits, x for dW (null: not wanted), W
    long x_plane, w_plane;
    float *w_part;               // [w_blocks] largest |w| of each block's share
    int32_t *f, *tgt;            // [rows padded]
    float *g, *gmax;             // [rows padded], [row blocks]: largest |x_i| 2^e_i
    float *c, *h;                // [rows padded]: c_i, c_i m_i
    int32_t *kw, *e_dw;          // exponent of W's scale; of dW's results
};

// The planes of XR rows of x, row r times 2^ex[r] (zeros where live[r] < 0): chunk (column block, row,
// half) by chunk, neighbouring threads side by side.  XR = 8: four blocks share a block row of 32, so
// that 4096 rows fill the chip.
template <typename T, int NP, bool VECX>
__device__ __forceinline__ void split_rows(const Prep &p, _Float16 *dst, long rb, const int *live, const int *ex) {
    const long row0 = rb * XR;
    dst += row0 / 32 * p.dcb * 512 + row0 % 32 * 16;
#pragma unroll 4
    for (int ch = threadIdx.x; ch < p.dcb * 2 * XR; ch += NT) {
        const int cb = ch / (2 * XR), rl = (ch >> 1) % XR, c = cb * 16 + (ch & 1) * 8;
        float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (live[rl] >= 0) load8<T, VECX>((const T *)p.x + (row0 + rl) * p.x_stride, c, p.d, x);
        store_planes<NP>(dst + (long)cb * 512 + rl * 16 + (ch & 1) * 8, p.x_plane, x, ex[rl]);
    }
}

// The planes of x for dW, rows [rb XR, + XR), from k_loss_prep's maxima.  factors(f) writes the rows' c_i m_i; what
// does not depend on them is loaded before.
template <typename T, int NP, bool VECX, typename F>
__device__ __forceinline__ void split_x2(const Prep &p, long rb, F &&factors) {
    constexpr int AHEAD = 2;  // chunks of x a thread loads ahead
    __shared__ float top[NT / 64], f[XR];
    __shared__ int live[XR], ex[XR];
    const int tid = threadIdx.x, total = p.dcb * 2 * XR;
    float m = 0.0f, x[AHEAD][8];
    for (int i = tid; i < p.row_blocks; i += NT) m = fmaxf(m, p.gmax[i]);
    const auto row_of = [&](int ch) { return (const T *)p.x + min(rb * XR + (ch >> 1) % XR, (long)p.rows - 1) * p.x_stride; };
    const auto col_of = [&](int ch) { return ch / (2 * XR) * 16 + (ch & 1) * 8; };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
        if (tid + u * NT < total) load8<T, VECX>(row_of(tid + u * NT), col_of(tid + u * NT), p.d, x[u]);
    const float g = tid < XR ? p.g[rb * XR + tid] : 0.0f;
    factors(f);
    m = wave_max(m);
    if ((tid & 63) == 0) top[tid >> 6] = m;
    if (tid < XR) {
        ex[tid] = exp_of(g);
        live[tid] = g == 0.0f ? -1 : 0;  // a row that gives nothing is not in the scale's range
    }
    __syncthreads();
    const int e = scale_exp(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]))) - 2;  // c_i m_i < 4
    if (rb == 0 && tid == 0) *p.e_dw = -DZ_EXP - e;
    const long row0 = rb * XR;
    _Float16 *dst = p.x2p + row0 / 32 * p.dcb * 512 + row0 % 32 * 16;
    auto put = [&](int ch, float (&v)[8]) {
        const int rl = (ch >> 1) % XR;
        if (live[rl] < 0)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        store_planes<NP>(dst + (long)(ch / (2 * XR)) * 512 + rl * 16 + (ch & 1) * 8, p.x_plane, v, ex[rl] + e, f[rl]);
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
        if (tid + u * NT < total) put(tid + u * NT, x[u]);
#pragma unroll 4
    for (int ch = tid + AHEAD * NT; ch < total; ch += NT) {
        float v[8];
        load8<T, VECX>(row_of(ch), col_of(ch), p.d, v);
        put(ch, v);
    }
}

// The first row_blocks blocks: XR rows of x each, split into planes with a scale of their own; rows
// without a target are zeros and are not read.  The others: the largest |w| of a share of W.
template <typename T, int NP, bool VECX, bool VECW>
__global__ __launch_bounds__(NT) void k_loss_prep(Prep p) {
    __shared__ float red[4];
    __shared__ float rmax[XR];
    __shared__ int fx[XR], tg[XR];
    const int tid = threadIdx.x;
    if ((int)blockIdx.x >= p.row_blocks) {
        float m = 0.0f;
        const int nch = (p.d + 7) / 8, b = blockIdx.x - p.row_blocks;
        const long total = (long)p.w_sample * nch, step = (long)p.w_blocks * NT;
        // four chunks in flight
        for (long i = (long)b * NT + tid; i < total; i += 4 * step) {
            float x[4][8];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const long k = min(i + u * step, total - 1), v = k / nch;
                load8<T, VECW>((const T *)p.w + v * p.w_step * p.w_stride, (int)(k - v * nch) * 8, p.d, x[u]);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(x[u][j]));
        }
        m = block_max256(m, red);
        if (tid == 0) p.w_part[b] = m;
        if (tid == 0 && b == 0) *p.w_max = 0;
        return;
    }
    const int rb = blockIdx.x;
    {
        constexpr int PER = NT / XR;  // threads a row: half a wave
        const int rl = tid / PER, part = tid % PER;
        const long i = (long)rb * XR + rl;
        int t = i < p.rows ? p.targets[i] : -1;
        if (t >= p.vocab) {
            if (part == 0) atomicOr(p.err, ADN_DEVERR_TOKEN);
            t = -1;
        }
        if (t < 0) t = -1;
        float m = 0.0f;
        if (t >= 0)
#pragma unroll 4
            for (int c = part * 8; c < p.d; c += 8 * PER) {
                float x[8];
                load8<T, VECX>((const T *)p.x + i * p.x_stride, c, p.d, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(x[j]));
            }
#pragma unroll
        for (int off = PER / 2; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        if (part == 0) {
            const float g = t < 0 ? 0.0f : p.dloss ? p.dloss[i] : 1.0f;
            tg[rl] = t;
            fx[rl] = scale_exp(m);
            p.f[i] = fx[rl];
            p.tgt[i] = t;
            p.g[i] = g;
            rmax[rl] = g == 0.0f ? 0.0f : fminf(ldexpf(m, exp_of(g)), 0x1p127f);
        }
    }
    __syncthreads();
    if (tid == 0) {
        float m = rmax[0];
#pragma unroll
        for (int r = 1; r < XR; ++r) m = fmaxf(m, rmax[r]);
        p.gmax[rb] = m;
    }
    split_rows<T, NP, VECX>(p, p.xp, rb, tg, fx);
}

// W's planes, from k_loss_prep's maxima: each block those of every so many-th block of 32 rows, of a share
// of the columns where W has few rows.
template <typename T, int NP, bool VECW>
__global__ __launch_bounds__(NT) void k_loss_split(Prep p, int redo) {
    __shared__ float red[4];
    const int tid = threadIdx.x;
    int e;
    bool blank = false;
    if (!scale_of_w(p.w_part, p.w_blocks, p.w_head, p.w_max, redo, red, e, blank)) return;
    if (blockIdx.x == 0 && tid == 0) *p.kw = e;
    float top = 0.0f;
    const int b = blockIdx.x, part = b % p.w_cols, per = (p.dcb + p.w_cols - 1) / p.w_cols;
    const int ch1 = min((part + 1) * per, p.dcb) * 64;
    for (long rb = b / p.w_cols; rb < p.w_rows; rb += (int)gridDim.x / p.w_cols)
        for (int ch = part * per * 64 + tid; ch < ch1; ch += NT) {
            const int cb = ch >> 6, rl = (ch >> 1) & 31, c = cb * 16 + (ch & 1) * 8;
            const long v = rb * 32 + rl;
            float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (v < p.vocab) load8<T, VECW>((const T *)p.w + v * p.w_stride, c, p.d, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, finite_abs(x[j]));
            store_planes<NP>(p.wp + (rb * p.dcb) * 512 + (long)ch * 8, p.w_plane, x, e);
        }
    if (p.w_head && !redo) {
        top = block_max256(top, red);
        if (tid == 0) report_w(top, e, blank, p.w_max);
    }
}

// ---- rows: lse and loss from the tiles' partials -------------------------------------------
struct Rows {
    int rows, tiles;
    long rows_pad;
    const float *part_m, *part_s, *ztgt;
    const int32_t *tgt;
    float *lse;               // [rows padded], in units of log 2
    float *out_loss, *out_lse;
};

// XR rows a block; 32 threads share a row's tiles, eight loads in flight each: a row's 8 in a wave, the waves then.
// Where dW is wanted, then the rows' planes of x for it.
template <typename T, int NP, bool VECX>
__global__ __launch_bounds__(NT) void k_loss_rows(Rows p, Prep pr) {
    constexpr int PARTS = NT / XR;
    __shared__ float sm[NT / 64][XR], ss[NT / 64][XR];
    const int rl = threadIdx.x % XR, part = threadIdx.x / XR, wave = threadIdx.x >> 6;
    const long i = (long)blockIdx.x * XR + rl;
    auto stats = [&](float *f) {
        const bool there = p.tgt[i] >= 0;
        const float zt = p.ztgt[i], g = pr.g[i];
        float mx = -INFINITY, s = 0.0f;
        for (int t0 = part; t0 < p.tiles; t0 += PARTS * 8) {
            float m[8], v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int t = t0 + PARTS * u;
                const long o = (long)min(t, p.tiles - 1) * p.rows_pad + i;
                m[u] = p.part_m[o];
                v[u] = p.part_s[o];
                if (t >= p.tiles) m[u] = -INFINITY, v[u] = 0.0f;
            }
            float nm = mx;
#pragma unroll
            for (int u = 0; u < 8; ++u) nm = fmaxf(nm, m[u]);
            const float ref = nm == -INFINITY ? 0.0f : nm;
            s *= __builtin_amdgcn_exp2f(mx - ref);
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u] * __builtin_amdgcn_exp2f(m[u] - ref);
            mx = nm;
        }
        float top = mx;
#pragma unroll
        for (int off = XR; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
        s *= __builtin_amdgcn_exp2f(mx - (top == -INFINITY ? 0.0f : top));
#pragma unroll
        for (int off = XR; off < 64; off <<= 1) s += __shfl_xor(s, off, 64);
        if (part % (64 / XR) == 0) {
            sm[wave][rl] = top;
            ss[wave][rl] = s;
        }
        __syncthreads();
        if (part) return;
        mx = fmaxf(fmaxf(sm[0][rl], sm[1][rl]), fmaxf(sm[2][rl], sm[3][rl]));
        const float ref = mx == -INFINITY ? 0.0f : mx;
        s = 0.0f;
#pragma unroll
        for (int q = 0; q < NT / 64; ++q) s += ss[q][rl] * __builtin_amdgcn_exp2f(sm[q][rl] - ref);
        const float lse = ref + log2f(s);
        const float z = there ? zt : lse, c = row_unit(z, lse);
        p.lse[i] = lse;
        pr.c[i] = c;
        pr.h[i] = row_factor(g, c);
        if (f) f[rl] = row_factor(g, c);
        if (i < p.rows) {
            if (p.out_lse) p.out_lse[i] = there ? lse * LN2 : 0.0f;
            if (p.out_loss) p.out_loss[i] = there ? (lse - z) * LN2 : 0.0f;
        }
    };
    if (pr.x2p)
        split_x2<T, NP, VECX>(pr, blockIdx.x, stats);
    else
        stats(nullptr);
}

// Those planes by themselves, where one tile of the logits' product was the whole vocabulary.
template <typename T, int NP, bool VECX>
__global__ __launch_bounds__(NT) void k_loss_x2(Prep p) {
    split_x2<T, NP, VECX>(p, blockIdx.x, [&](float *f) {
        if (threadIdx.x < XR) f[threadIdx.x] = p.h[(long)blockIdx.x * XR + threadIdx.x];
    });
}

// ---- shares of the gradients ---------------------------------------------------------------
// dst[row][col] = sum over the shares, in order, times 2^exponent: of dW all alike (e_all), of dx a
// row's own, e_i - 14 - kw (g), and c_i m_i (h).  Blocks from n_blocks on: db, the tiles' sums in order.
struct Join {
    const float *part;
    int S, rows, d;
    void *dst;
    long stride;
    bool vec;            // rows of whole fours, aligned as such
    const int32_t *e_all, *kw;
    const float *g, *h;
    int n_blocks;
    const float *db_part;
    int db_tiles, vocab;
    long db_ld;
    float *db;
};
template <typename T>
__global__ __launch_bounds__(NT) void k_loss_join(Join p) {
    if ((int)blockIdx.x >= p.n_blocks) {  // 64 entries, the waves a quarter of the tiles each
        __shared__ float red[4][64];
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int v = ((int)blockIdx.x - p.n_blocks) * 64 + lane;
        const int per = (p.db_tiles + 3) / 4, t1 = min(p.db_tiles, (wave + 1) * per);
        float s = 0.0f;
        if (v < p.vocab) {
#pragma unroll 16
            for (int t = wave * per; t < t1; ++t) s += p.db_part[t * p.db_ld + v];
        }
        red[wave][lane] = s;
        __syncthreads();
        if (wave == 0 && v < p.vocab) p.db[v] = ((s + red[1][lane]) + red[2][lane]) + red[3][lane];
        return;
    }
    const long n = (long)p.rows * p.d;
    typedef T V4 __attribute__((ext_vector_type(4)));
    if (p.vec) {  // four columns a thread
        for (long i = (long)blockIdx.x * NT + threadIdx.x; i < n / 4; i += (long)p.n_blocks * NT) {
            floatx4 s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
            for (int q = 0; q < p.S; ++q) s += *reinterpret_cast<const floatx4 *>(p.part + q * n + i * 4);
            const long row = n / 4 <= 0xffffffffl ? (unsigned)i / (unsigned)(p.d / 4) : i / (p.d / 4);
            const int e = p.g ? exp_of(p.g[row]) - DZ_EXP - *p.kw : *p.e_all;
            const float h = p.g ? p.h[row] : 1.0f;
            V4 o;
#pragma unroll
            for (int u = 0; u < 4; ++u) o[u] = from_f32<T>(ldexpf(s[u] * h, e));
            *reinterpret_cast<V4 *>((T *)p.dst + row * p.stride + (i * 4 - row * p.d)) = o;
        }
        return;
    }
    for (long i = (long)blockIdx.x * NT + threadIdx.x; i < n; i += (long)p.n_blocks * NT) {
        float s = 0.0f;
#pragma unroll 8
        for (int q = 0; q < p.S; ++q) s += p.part[q * n + i];
        const long row = i / p.d;
        const int e = p.g ? exp_of(p.g[row]) - DZ_EXP - *p.kw : *p.e_all;
        ((T *)p.dst)[row * p.stride + (i - row * p.d)] = from_f32<T>(ldexpf(s * (p.g ? p.h[row] : 1.0f), e));
    }
}

template <typename T>
__global__ __launch_bounds__(NT) void k_loss_zero(T *dst, long rows, int d, long stride) {
    for (long i = (long)blockIdx.x * NT + threadIdx.x; i < rows * d; i += (long)gridDim.x * NT)
        dst[i / d * stride + i % d] = from_f32<T>(0.0f);
}

// ---- plan ----------------------------------------------------------------------------------
constexpr int SLOTS = 512;  // workgroups that run at once: two a CU
long round_up(long n, long to) { return (n + to - 1) / to * to; }

struct LossPlan {
    bool raw;                // losses alone: W goes to the product as it is
    bool keep;               // the logits are kept for dz
    bool dx_whole;           // dx is written by its product
    int np, tn;              // planes; rows a workgroup of the logits' product covers
    int dcb;                 // column blocks of width d
    long rows_pad, v_pad;    // rows of the planes of x (and dz), of W
    int v_tiles;             // tiles of TV entries
    int piece;               // entries a piece, a multiple of TV
    int w_blocks, w_sample, w_step, w_head;
    int bn;                  // columns of a gradient tile
    int dx_split, dx_ks, dw_split, dw_ks;
    size_t xp, x2p, wp, w_part, f, tgt, g, gmax, kw, w_max, part_m, part_s, ztgt, lse, c, h, e_dw, z, dz, dzw, fx, scaled, dx_part, dw_part, db_part, bytes;
};

// K of `len` (a multiple of 32) in at most `want` shares of whole 32s, each not empty
void split_k(long len, long want, int *split, int *share) {
    *share = (int)round_up((len + want - 1) / want, 32);
    *split = (int)((len + *share - 1) / *share);
}

// Rows a workgroup of the logits' product covers.  A k slice takes a tile of 128, 64 or 32 rows about 0.8,
// 0.5 or 0.38 us, whether the chip is full (then its products) or not (then a round trip): 2000 rows
// against 512 entries run 26 us on 128 rows a tile and 13 on 32, 8192 against 50257 best on 128.
int pick_tn(long rows, long v_tiles) {
    int best = 128;
    double least = INFINITY;
    for (int tn : {128, 64, 32}) {
        const double n = (double)((rows + tn - 1) / tn * v_tiles) / SLOTS;
        const double t = (n <= 1 ? 1.0 : n + 0.3) * (tn == 128 ? 0.8 : tn == 64 ? 0.5 : 0.38);
        if (t < least) least = t, best = tn;
    }
    return best;
}

// Time of n1 units of length a and then n2 of length b (a >= b) on SLOTS slots, in order.
double makespan(long n1, double a, long n2, double b) {
    const long full = n1 / SLOTS, m1 = n1 % SLOTS, free = SLOTS - m1;
    const long fit = m1 ? free * (long)(a / b) : 0;  // units of b done beside the last a's
    double t = full * a;
    if (n2 <= fit) return t + std::max(m1 ? a : 0.0, (double)((n2 + free - 1) / free) * b);
    return t + (m1 ? a : 0.0) + (double)((n2 - fit + SLOTS - 1) / SLOTS) * b;
}

// Columns of the gradients' tiles and the shares of their K: the choice with the shortest estimated time of
// the common launch, in values of K of a unit of 128 x 256.  A narrower tile takes 0.62 (128 columns) or
// 0.45 (64) of it a value of K (2000 rows against 512 entries of 512: 103, 99 and 96 us a call), a
// prologue and epilogue as long as 60 values and 140 more for the stores of 256 columns.  Partial sums
// are written and read again: two passes of their bytes at 5 TB/s, where a value of K takes a unit about
// 0.044 us (two planes) or 0.022 us (one).
struct GradSizes {
    int np, d;
    long dx_rows, dx_k, dx_elems;  // 128-row tiles, length of the sum, elements of dx; 0: not wanted
    bool whole;                    // one piece: dx of one share is written as it is
    long dw_rows, dw_k, dw_elems;  // of a piece of dW
};
struct GradPick {
    int bn, dx_split, dx_ks, dw_split, dw_ks;
};
GradPick pick_grads(const GradSizes &g) {
    constexpr int SHARES[] = {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 24, 32, 48, 64, 96, 128, 192, 256};
    const double join = 8.0 / (g.np == 2 ? 2.2e5 : 1.1e5);  // K values an element of a share
    double best = INFINITY;
    GradPick pick{};
    for (int bn : {256, 128, 64}) {
        if (bn > 64 && g.d <= bn / 2) continue;
        const double unit = bn == 256 ? 1.0 : bn == 128 ? 0.62 : 0.45, epi = 60 + 140.0 * bn / 256;
        const long nbn = (g.d + bn - 1) / bn;
        for (int sx : SHARES) {
            if (sx > 1 && g.dx_k / sx < 256) break;
            int nx = 0, kx = 32;
            if (g.dx_rows) split_k(g.dx_k, sx, &nx, &kx);
            for (int sw : SHARES) {
                if (sw > 1 && g.dw_k / sw < 256) break;
                int nw = 0, kw = 32;
                if (g.dw_rows) split_k(g.dw_k, sw, &nw, &kw);
                const double a = kx * unit + epi, b = kw * unit + epi;
                const long ux = g.dx_rows * nbn * nx, uw = g.dw_rows * nbn * nw;
                double t = a >= b ? makespan(ux, a, uw, b) : makespan(uw, b, ux, a);
                t += join * ((double)g.dx_elems * (g.whole && nx == 1 ? 0 : nx) + (nw > 1 ? (double)g.dw_elems * nw : 0.0));
                if (t < best) {
                    best = t;
                    pick = {bn, nx, kx, nw, kw};
                }
            }
        }
    }
    return pick;
}

LossPlan loss_plan(const LossParams &p) {
    LossPlan L{};
    const bool grads = p.dx || p.dw || p.db;
    L.np = p.dtype == ADN_T_F32 ? 2 : 1;
    L.tn = pick_tn(p.rows, round_up(p.vocab, TV) / TV);
    L.dcb = (int)(round_up(p.d, 32) / 16);
    L.rows_pad = round_up(p.rows, BM);
    {   // rows of W in whole slices of 16-byte pieces, a tile's offsets in 32 bits (256 rows of 512 against
        // 50257: 107 us with planes of W, 71 without, before the scale was sampled)
        const long bytes = p.w_stride * elem_bytes(p.dtype);
        L.raw = !grads && p.vocab > TV && p.d % (L.np == 2 ? 16 : 32) == 0 && (uintptr_t)p.w % 16 == 0 && bytes % 16 == 0 &&
                bytes < (1L << 31) / TV;
    }
    L.v_pad = round_up(p.vocab, TV);
    L.v_tiles = (int)(L.v_pad / TV);
    const long fit = (long)(PIECE_BYTES / (L.np * 2)) / L.rows_pad / TV * TV;
    const long npieces = (L.v_pad + std::max<long>(TV, fit) - 1) / std::max<long>(TV, fit);
    L.piece = (int)round_up((L.v_pad + npieces - 1) / npieces, TV);
    {   // W's scale from one row in 32 where W is large: 128 rows against 50257 entries 328 -> 294 us (fp32, d =
        // 1024), 98 -> 94 (bf16, 512); below, the launch costs what it saves (8192 entries: 60 and 62, 46 and 48)
        const bool all = (long)p.vocab * p.d * elem_bytes(p.dtype) < SAMPLE_FROM;
        L.w_step = all ? 1 : 32;
        L.w_sample = (p.vocab + L.w_step - 1) / L.w_step;
        L.w_head = all ? 0 : HEAD;
        L.w_blocks = (int)std::min<long>(W_BLOCKS, ((long)L.w_sample * ((p.d + 7) / 8) + NT * 4 - 1) / (NT * 4));
    }
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t r = at;
        at += (bytes + 1023) / 1024 * 1024;
        return r;
    };
    L.xp = take((size_t)L.rows_pad * L.dcb * 32 * L.np);
    L.x2p = take(p.dw ? (size_t)L.rows_pad * L.dcb * 32 * L.np : 0);
    L.wp = take(L.raw ? 0 : (size_t)L.v_pad * L.dcb * 32 * L.np);
    L.w_part = take(W_BLOCKS * 4);
    L.f = take(L.rows_pad * 4);
    L.tgt = take(L.rows_pad * 4);
    L.g = take(L.rows_pad * 4);
    L.gmax = take(L.rows_pad / XR * 4);
    L.kw = take(4);
    L.w_max = take(4);
    L.part_m = take((size_t)L.v_tiles * L.rows_pad * 4);
    L.part_s = take((size_t)L.v_tiles * L.rows_pad * 4);
    L.ztgt = take(L.rows_pad * 4);
    L.lse = take(L.rows_pad * 4);
    L.c = take(L.rows_pad * 4);
    L.h = take(L.rows_pad * 4);
    L.e_dw = take(4);
    {   // Logits of no more bytes than a piece of dz are kept where their product takes longer than writing and
        // reading them: 512 rows against 50257 entries 1389 -> 1122 us (fp32, d = 2048), 391 -> 353 (512), 152 ->
        // 163 (128); 592 -> 530 (bf16, 2048), 185 -> 188 (512).  A few of them stay in the caches: 512 rows
        // against 2000 entries 158 -> 121 (fp32, 2048), 47 -> 45 (128), 50 -> 46 (bf16, 512).
        const long bytes = L.rows_pad * L.v_pad * 4;
        L.keep = grads && L.v_tiles > 1 && bytes <= ((long)p.d * (L.np == 2 ? 3 : 1) >= 1024 ? (long)PIECE_BYTES : 16L << 20);
    }
    L.z = take(L.keep ? (size_t)round_up(p.rows, L.tn) * L.v_pad * 4 : 0);
    if (grads) {
        if (p.dx) L.dz = take((size_t)L.rows_pad * L.piece * 2 * L.np);
        if (p.dw) {
            L.dzw = take((size_t)L.rows_pad * L.piece * 2 * L.np);
            L.fx = take((size_t)(L.rows_pad / L.tn) * L.piece * 2);
            L.scaled = take((size_t)(L.rows_pad / L.tn) * (L.piece / TV) * 4);
        }
        GradSizes g{L.np, p.d};
        if (p.dx) g.dx_rows = round_up(p.rows, BM) / BM, g.dx_k = L.piece, g.dx_elems = (long)p.rows * p.d;
        if (p.dw) {
            const long n = std::min<long>(L.piece, p.vocab);
            g.dw_rows = round_up(n, BM) / BM, g.dw_k = round_up(p.rows, 32), g.dw_elems = n * p.d;
        }
        g.whole = L.piece == L.v_pad;
        const GradPick k = pick_grads(g);
        L.bn = k.bn, L.dx_split = k.dx_split, L.dx_ks = k.dx_ks, L.dw_split = k.dw_split, L.dw_ks = k.dw_ks;
        L.dx_whole = p.dx && g.whole && L.dx_split == 1;
        if (p.dx && !L.dx_whole) L.dx_part = take((size_t)L.dx_split * p.rows * p.d * 4);
        if (p.dw && L.dw_split > 1) L.dw_part = take((size_t)L.dw_split * L.piece * p.d * 4);
        if (p.db) L.db_part = take((size_t)(L.rows_pad / L.tn) * L.v_pad * 4);
    }
    L.bytes = at;
    return L;
}

// A launch has less than 2^32 threads: the pass over the whole vocabulary (2^20 rows against 2^19 entries are 2^24
// workgroups) is launched a range of its tiles at a time.  A piece's tiles are fewer.
constexpr long MOST_BLOCKS = (1L << 32) / NT - 1;

template <int MODE, typename T, int NP>
void launch_logits(LossGemm g, int tn, hipStream_t st) {
    const int tiles = g.nM, most = (int)std::min<long>(tiles, MOST_BLOCKS / g.nN);
    for (int m = 0; m < tiles; m += most) {
        g.nM = std::min(most, tiles - m);
        const unsigned grid = (unsigned)(g.nM * g.nN);
        if (tn == 128)
            k_loss_logits<MODE, T, NP, 4><<<grid, NT, 0, st>>>(g);
        else if (tn == 64)
            k_loss_logits<MODE, T, NP, 2><<<grid, NT, 0, st>>>(g);
        else
            k_loss_logits<MODE, T, NP, 1><<<grid, NT, 0, st>>>(g);
        g.a_row0 += most * TV;
        g.part_m += most * g.rows_pad, g.part_s += most * g.rows_pad;
    }
}

template <typename T, int NP>
void launch_grads(LossGrads &g, int bn, hipStream_t st) {
    const int ndx = g.dx.nM * g.dx.nN * g.dx.S, ndw = g.dw.nM * g.dw.nN * g.dw.S;  // 0: not wanted
    g.dx_first = ndx && (!ndw || g.dx.Ks >= g.dw.Ks);
    g.first = g.dx_first ? ndx : ndw;
    const unsigned grid = (unsigned)(ndx + ndw);
    if (bn == 256)
        k_loss_grads<T, NP, 2, 4, 2, 2><<<grid, NT, 0, st>>>(g);
    else if (bn == 128)
        k_loss_grads<T, NP, 2, 2, 2, 2><<<grid, NT, 0, st>>>(g);
    else
        k_loss_grads<T, NP, 1, 2, 4, 1><<<grid, NT, 0, st>>>(g);
}

int join_blocks(long n) { return (int)std::min<long>(2048, (n + NT - 1) / NT); }
bool join_vec(const Join &j, int eb) {
    return j.d % 4 == 0 && (uintptr_t)j.dst % (4 * eb) == 0 && j.stride % 4 == 0;
}

template <typename T, int NP>
void run_loss(const LossParams &p, const LossPlan &L, char *ws, hipStream_t st) {
    const int eb = elem_bytes(p.dtype);
    // rows of whole 16-byte pieces are loaded 8 values at a time (the tail of a row by itself)
    const bool vx = (uintptr_t)p.x % 16 == 0 && p.x_stride * eb % 16 == 0;
    const bool vw = (uintptr_t)p.w % 16 == 0 && p.w_stride * eb % 16 == 0;
    Prep r{};
    r.x = p.x, r.x_stride = p.x_stride, r.w = p.w, r.w_stride = p.w_stride;
    r.rows = p.rows, r.d = p.d, r.vocab = p.vocab, r.dcb = L.dcb;
    r.w_blocks = L.w_blocks, r.row_blocks = (int)(L.rows_pad / XR), r.w_rows = (int)(L.v_pad / 32);
    r.w_cols = std::max(1, std::min(1024 / r.w_rows, L.dcb / 4));  // 1142 rows of 2048: 20 us for 8
    r.targets = p.targets, r.dloss = p.dloss, r.err = p.err;
    r.xp = (_Float16 *)(ws + L.xp), r.x2p = p.dw ? (_Float16 *)(ws + L.x2p) : nullptr, r.wp = (_Float16 *)(ws + L.wp);
    r.x_plane = L.rows_pad * L.dcb * 16, r.w_plane = L.v_pad * L.dcb * 16;
    r.w_part = (float *)(ws + L.w_part);
    r.w_sample = L.w_sample, r.w_step = L.w_step, r.w_head = L.w_head, r.w_max = (unsigned *)(ws + L.w_max);
    r.f = (int32_t *)(ws + L.f), r.tgt = (int32_t *)(ws + L.tgt);
    r.g = (float *)(ws + L.g), r.gmax = (float *)(ws + L.gmax);
    r.c = (float *)(ws + L.c), r.h = (float *)(ws + L.h);
    r.kw = (int32_t *)(ws + L.kw), r.e_dw = (int32_t *)(ws + L.e_dw);
    const bool grads = p.dx || p.dw || p.db;
    const unsigned prep_grid = (unsigned)(r.row_blocks + r.w_blocks);
    auto prep = [&](auto vecx, auto vecw) {
        constexpr bool VX = decltype(vecx)::value, VW = decltype(vecw)::value;
        k_loss_prep<T, NP, VX, VW><<<prep_grid, NT, 0, st>>>(r);
        if (L.raw) return;
        k_loss_split<T, NP, VW><<<(unsigned)(r.w_rows * r.w_cols), NT, 0, st>>>(r, 0);
        if (L.w_head) k_loss_split<T, NP, VW><<<std::min(r.w_rows, 1024) * r.w_cols, NT, 0, st>>>(r, 1);
    };
    using std::bool_constant;
    if (vx && vw)
        prep(bool_constant<true>{}, bool_constant<true>{});
    else if (vx)
        prep(bool_constant<true>{}, bool_constant<false>{});
    else if (vw)
        prep(bool_constant<false>{}, bool_constant<true>{});
    else
        prep(bool_constant<false>{}, bool_constant<false>{});

    const Planes X{r.xp, r.x_plane, L.dcb}, X2{r.x2p, r.x_plane, L.dcb}, W{r.wp, r.w_plane, L.dcb};
    LossGemm z{};
    z.A = W, z.B = X;
    z.nM = L.v_tiles, z.nN = (int)(round_up(p.rows, L.tn) / L.tn), z.S = 1;
    z.K = z.Ks = L.dcb * 16;
    z.bias = p.bias, z.f = r.f, z.tgt = r.tgt, z.kw_dev = r.kw;
    z.vocab = p.vocab, z.rows = p.rows, z.rows_pad = L.rows_pad;
    z.part_m = (float *)(ws + L.part_m), z.part_s = (float *)(ws + L.part_s), z.ztgt = (float *)(ws + L.ztgt);
    z.g = r.g, z.c = z.out_c = r.c, z.h = z.out_h = r.h;
    const unsigned row_grid = (unsigned)(round_up(p.rows, L.tn) / XR);
    if (grads) {
        z.dz = p.dx ? (_Float16 *)(ws + L.dz) : nullptr, z.dzw = p.dw ? (_Float16 *)(ws + L.dzw) : nullptr;
        z.dz_plane = L.rows_pad * L.piece, z.dz_ncb = L.piece / 16;
        z.fx = (_Float16 *)(ws + L.fx), z.fx_ld = L.piece, z.scaled = (int *)(ws + L.scaled);
        z.db_part = p.db ? (float *)(ws + L.db_part) : nullptr, z.db_ld = L.v_pad;
    }
    const bool all = L.v_tiles == 1;  // one tile holds the vocabulary: one pass
    if (all) {
        z.out_loss = p.loss, z.out_lse = p.lse;
        launch_logits<LOGITS_ALL, T, NP>(z, L.tn, st);
        if (r.x2p) vx ? k_loss_x2<T, NP, true><<<row_grid, NT, 0, st>>>(r) : k_loss_x2<T, NP, false><<<row_grid, NT, 0, st>>>(r);
    } else {
        if (L.raw) {
            z.K = z.Ks = p.d;
            z.w_raw = p.w, z.w_stride = (unsigned)(p.w_stride * eb), z.w_part = r.w_part, z.w_blocks = r.w_blocks;
            z.w_head = L.w_head, z.w_max = r.w_max;
            launch_logits<LOGITS_RAW, T, NP>(z, L.tn, st);
            if (L.w_head) {
                z.w_redo = 1;
                launch_logits<LOGITS_RAW, T, NP>(z, L.tn, st);
            }
        } else {
            z.z = L.keep ? (float *)(ws + L.z) : nullptr;
            launch_logits<LOGITS_STATS, T, NP>(z, L.tn, st);
        }
        Rows q{};
        q.rows = p.rows, q.tiles = L.v_tiles, q.rows_pad = L.rows_pad;
        q.part_m = z.part_m, q.part_s = z.part_s, q.ztgt = z.ztgt, q.tgt = r.tgt;
        q.lse = (float *)(ws + L.lse), q.out_loss = p.loss, q.out_lse = p.lse;
        vx ? k_loss_rows<T, NP, true><<<row_grid, NT, 0, st>>>(q, r) : k_loss_rows<T, NP, false><<<row_grid, NT, 0, st>>>(q, r);
        z.lse = q.lse;
    }
    if (!grads) return;

    const int nbn = (p.d + L.bn - 1) / L.bn;
    for (long v0 = 0; v0 < L.v_pad; v0 += L.piece) {
        const int n = (int)std::min<long>(L.piece, L.v_pad - v0);  // entries of the piece, padded
        z.a_row0 = (int)v0;
        z.nM = n / TV;
        if (L.keep)
            launch_logits<LOGITS_KEPT, T, NP>(z, L.tn, st);
        else if (!all)
            launch_logits<LOGITS_DZ, T, NP>(z, L.tn, st);
        const int live = (int)std::min<long>(n, p.vocab - v0);
        T *dst = p.dw ? (T *)p.dw + v0 * p.dw_stride : nullptr;
        LossGrads g{};
        if (p.dx) {
            LossGemm &x = g.dx;
            x.A = Planes{z.dz, z.dz_plane, z.dz_ncb}, x.B = W;
            x.B.p += v0 / 32 * (long)W.ncb * 512;
            x.nM = (int)(round_up(p.rows, BM) / BM), x.nN = nbn, x.S = (n + L.dx_ks - 1) / L.dx_ks;
            x.K = n, x.Ks = L.dx_ks;
            if (L.dx_whole)
                x.dst = p.dx, x.dst_stride = p.dx_stride, x.g = r.g, x.h = r.h, x.kw_dev = r.kw;
            else
                x.part = (float *)(ws + L.dx_part), x.part_ld = p.d, x.add = v0 > 0;
            x.out_rows = p.rows, x.out_cols = p.d;
        }
        if (p.dw) {
            LossGemm &w = g.dw;
            w.A = Planes{z.dzw, z.dz_plane, z.dz_ncb}, w.B = X2;
            w.plain = p.dx ? z.dz : z.dzw;
            w.scaled = z.scaled, w.fx = z.fx, w.fx_ld = z.fx_ld, w.fx_log = L.tn == 128 ? 7 : L.tn == 64 ? 6 : 5;
            w.nM = (live + BM - 1) / BM, w.nN = nbn, w.S = L.dw_split;
            w.K = (int)round_up(p.rows, 32), w.Ks = L.dw_ks;
            w.out_rows = live, w.out_cols = p.d;
            if (L.dw_split > 1)
                w.part = (float *)(ws + L.dw_part), w.part_ld = p.d;
            else
                w.dst = dst, w.dst_stride = p.dw_stride, w.e_all = r.e_dw;
        }
        if (p.dx || p.dw) launch_grads<T, NP>(g, L.bn, st);
        if (p.dw && L.dw_split > 1) {
            Join j{};
            j.part = g.dw.part, j.S = L.dw_split, j.rows = live, j.d = p.d, j.dst = dst, j.stride = p.dw_stride;
            j.vec = join_vec(j, eb);
            j.e_all = r.e_dw, j.n_blocks = join_blocks((long)live * p.d / (j.vec ? 4 : 1));
            k_loss_join<T><<<j.n_blocks, NT, 0, st>>>(j);
        }
    }
    const bool join_dx = p.dx && !L.dx_whole;
    if (!join_dx && !p.db) return;
    Join j{};
    j.part = (float *)(ws + L.dx_part), j.S = L.dx_split, j.rows = p.rows, j.d = p.d, j.dst = p.dx, j.stride = p.dx_stride;
    j.vec = join_vec(j, eb);
    j.g = r.g, j.h = r.h, j.kw = r.kw, j.n_blocks = join_dx ? join_blocks((long)p.rows * p.d / (j.vec ? 4 : 1)) : 0;
    j.db_part = z.db_part, j.db_tiles = z.nN, j.db_ld = z.db_ld, j.vocab = p.vocab, j.db = p.db;
    k_loss_join<T><<<j.n_blocks + (p.db ? (p.vocab + 63) / 64 : 0), NT, 0, st>>>(j);
}

}  // namespace

size_t loss_workspace_bytes(const LossParams &p) {
    return p.rows == 0 ? 0
           : loss_few_ok(p) ? loss_few_workspace_bytes(p)
           : loss_mid_ok(p) ? loss_mid_workspace_bytes(p)
                            : loss_plan(p).bytes;
}

void launch_loss(const LossParams &p, void *ws, hipStream_t st) {
    if (p.rows && loss_few_ok(p)) return launch_loss_few(p, ws, st);
    if (p.rows && loss_mid_ok(p)) return launch_loss_mid(p, ws, st);
    dispatch_type(p.dtype, [&](auto ty) {
        typedef decltype(ty) T;
        if (p.rows == 0) {  // no row: the sums over the rows are zero
            if (p.dw) k_loss_zero<T><<<2048, NT, 0, st>>>((T *)p.dw, p.vocab, p.d, p.dw_stride);
            if (p.db) k_loss_zero<float><<<256, NT, 0, st>>>(p.db, 1, p.vocab, p.vocab);
            return;
        }
        run_loss<T, std::is_same<T, float>::value ? 2 : 1>(p, loss_plan(p), (char *)ws, st);
    });
}

}  // namespace adn
