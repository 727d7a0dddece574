/*
 * gfx950 kernels between the q/k/v projections and the output projection:
 * rotary embedding with the write into a paged cache (rope_kernel), and causal
 * attention over packed prompts and over a paged cache (attention_kernel, with
 * attention_join_kernel where the keys of a row tile are cut into pieces and
 * attention_image_kernel before long prompts).
 *
 * What bounds attention (28 query and 4 key heads of 128 unless said; a copy
 * reaches 4.6 TB/s here and an 8192^3 f16 product 1.1 PFLOP/s):
 *   one token each of 64 sequences of 1 to 8191 keys, f16 cache: the stream of
 *   keys and values, 494 MB in 98 us with the join, 5.0 TB/s;
 *   a prompt of 8192: the matrix cores, 1.44 T operations (three products of
 *   limbs each) in 1.27 to 1.38 ms by card, 1.13 PFLOP/s at best, at 2.0 GHz, where
 *   the power limit holds the clock;
 *   512 tokens over 16100, f16 cache: the matrix cores, 0.23 T (two products) in
 *   245 to 255 us, 0.94 PFLOP/s with the pieces' results and their join;
 *   small calls: their chain of memory round trips (lengths, page table, keys)
 *   and a second launch for the join: one token over 777 keys, 14 and 2 heads of
 *   64, 9 + 3 us.
 */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "qmv_kernels.h"

namespace qmv {

typedef float f4_t __attribute__((ext_vector_type(4)));

/* Nearest, ties to even; NaN stays NaN. */
__device__ __forceinline__ uint16_t to_bf16(float v)
{
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)(u >> 16 | 0x40u);
    return (uint16_t)((u + 0x7fffu + (u >> 16 & 1u)) >> 16);
}

template <int TYPE> __device__ __forceinline__ void store_kv(void *base, int64_t i, float v)
{
    if (TYPE == QMV_KV_F32) ((float *)base)[i] = v;
    else if (TYPE == QMV_KV_F16) ((_Float16 *)base)[i] = (_Float16)v;
    else ((uint16_t *)base)[i] = to_bf16(v);
}

/* The sequence of token t: the last whose start is at most t, if it reaches
 * that far; else -1. */
__device__ __forceinline__ int sequence_of(const AttnTokens &a, int t)
{
    int lo = 0, hi = a.count; /* starts[lo] <= t < starts[hi], as far as starts rises */
    if (a.starts[0] > t || a.starts[a.count] <= t) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    return a.starts[lo + 1] > t ? lo : -1;
}

/* Where key `j` of sequence s and of head h begins in a paged cache, -1 if its
 * page is outside the cache or the table. */
__device__ __forceinline__ int64_t key_at(const AttnTokens &a, int s, int j, int h)
{
    const int page = j / a.page_size;
    if (page >= a.table_stride) return -1;
    const int at = a.table[(int64_t)s * a.table_stride + page];
    if (at < 0 || at >= a.pages) return -1;
    return (int64_t)at * a.page_stride + (int64_t)h * a.head_stride + (int64_t)(j - page * a.page_size) * a.token_stride;
}

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef float f2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef short s4_t __attribute__((ext_vector_type(4)));

#define QMV_LDS __attribute__((address_space(3)))

/* Barrier for data exchanged through LDS: waits for this wave's LDS
 * operations, not for the global loads of the next tile. */
__device__ __forceinline__ void lds_barrier()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F); /* lgkmcnt(0) */
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

/* The values of the lanes that share lane % RW (32 or 16), joined by f. */
template <int RW, typename F> __device__ __forceinline__ float join_lanes(float x, F f)
{
    if (RW == 16) {
        const auto q = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = f(__uint_as_float(q[0]), __uint_as_float(q[1]));
    }
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int RW> __device__ __forceinline__ float max_lanes(float x)
{
    return join_lanes<RW>(x, [](float a, float b) { return fmaxf(a, b); });
}
template <int RW> __device__ __forceinline__ float sum_lanes(float x)
{
    return join_lanes<RW>(x, [](float a, float b) { return a + b; });
}

/* Matrix products of RW columns, D (RW x RW) += A B: a lane holds 8 elements of
 * the contraction of one row of A and of one column of B, lane % RW, those
 * from 8 (lane / RW) on (of 16 with RW = 32, of 32 with RW = 16); and of D's
 * column lane % RW the rows 4 (lane / RW) + 256 / RW j + i in register 4 j + i. */
template <int RW> struct Product;
template <> struct Product<32> {
    typedef float acc_t __attribute__((ext_vector_type(16)));
    static __device__ __forceinline__ acc_t run(h8_t a, h8_t b, acc_t c)
    {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <> struct Product<16> {
    typedef float acc_t __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ acc_t run(h8_t a, h8_t b, acc_t c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

/* The largest of the wave's unsigned values, in every lane. */
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
#define QMV_STEP(CTRL) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false));
    QMV_STEP(0x111) /* row_shr 1, 2, 4, 8: lane 15 of each row has the row's */
    QMV_STEP(0x112)
    QMV_STEP(0x114)
    QMV_STEP(0x118)
    QMV_STEP(0x142) /* row_bcast 15, 31: lane 63 has all */
    QMV_STEP(0x143)
#undef QMV_STEP
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

__device__ __forceinline__ int64_t shfl64(int64_t v, int lane)
{
    const int lo = __shfl((int)(uint32_t)v, lane), hi = __shfl((int)(v >> 32), lane);
    return (int64_t)((uint64_t)(uint32_t)hi << 32 | (uint32_t)lo);
}

/* Sums over the lanes up to each: of row_shr 1, 2, 4, 8 within rows of 16, then
 * of the rows before. */
template <typename T> __device__ __forceinline__ T scan_lanes(T v)
{
#define QMV_STEP(CTRL, ROWS) \
    v += __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
    QMV_STEP(0x111, 0xf)
    QMV_STEP(0x112, 0xf)
    QMV_STEP(0x114, 0xf)
    QMV_STEP(0x118, 0xf)
    QMV_STEP(0x142, 0xa)
    QMV_STEP(0x143, 0xc)
#undef QMV_STEP
    return v;
}
template <typename T> __device__ __forceinline__ T lane_of(T v, int lane)
{
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

/* ---- attention -----------------------------------------------------------------
 *
 * A workgroup takes a tile of RW WR rows of one sequence and key head, a row
 * being a new token and one of the group's query heads, so every key and value
 * that it reads serves the whole group; and a range of keys. A wave holds RW
 * rows (32, or 16 where a sequence has no more); WK waves take turns along the
 * keys. Per 32 keys it computes
 *   S^T = K Q^T   (matrix rows: keys; columns: rows of the tile)
 *   O^T += V^T P^T
 * A lane has scores of one row in its registers, and the registers that S^T
 * leaves are the operand that O^T's product takes, with no exchange between
 * lanes, if V's keys are read in the same order. The running maximum is joined
 * over the lanes of a row, the sum at the end.
 *
 * Numbers. Products are of f16 with fp32 sums. q (times scale and log2 e) and
 * the weights are two f16 limbs each, x = hi + lo, after a power of two has
 * brought a row's largest |q| to [2^14, 2^15) and the weights to at most 2^15:
 * 22 bits, or 2^-39 of the largest. f16 keys and values are operands as they
 * are; those of bf16 are one limb and of f32 two, scaled in blocks of 16
 * tokens by a power of two in the same way. The product of two low limbs (2^-22
 * of the whole) is left out. A block's scale of the keys is a factor of its
 * scores; that of the values is added to the exponents of its weights, and
 * taken out again where the weights are summed.
 *
 * Two references, both whole numbers, so that moving them rounds nothing: the
 * weights' sum l is of 2^(score - m - 9), m following the running maximum of
 * the scores; O is relative to 2^(m + rm), which follows that of score plus the
 * exponent of a block's values. (Of f16 values, which have no exponents, one
 * reference r is both.) They move only when the maximum is more than 2^4 over
 * them, so that most tiles leave O as it is.
 *
 * Where the values of a row's blocks differ much in size (by more than 2^kApart
 * between their largest), the smaller ones' weights would lose places in limbs
 * beside the larger's reference. From there on a wave takes the blocks one after
 * the other, each relative to its own largest: O is brought down to that
 * reference and the next block's raises it again, exactly, down to 2^-kReach of
 * the row's largest product of weight and value so far; products below that are
 * left out of O, their weights still summed in l. The same where scores are so
 * large (2^22) that an exponent added to them would be rounded away. Against one
 * reference for both, which left l to the weights of the largest values (values
 * of 1e30 beside zeros: off by any factor; one channel of 2^30 in 16 tokens: the
 * others off by 1e-2): 1.3 to 1.7% of a long prompt, 3% of the 0.5B prompts. */

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNothing = -3.40282347e38f; /* r, m before any key: no finite score is below it */
constexpr float kNoScale = -1000.f;         /* rm before any key */
constexpr float kApart = 10.f, kReach = 60.f;
constexpr float kShift = 11.f; /* weights are at most 2^(kShift + kSlack) */
constexpr float kSlack = 4.f;

/* 2^n as a float, -126 <= n <= 127. */
__device__ __forceinline__ float power_of_two(int n) { return __uint_as_float((uint32_t)(n + 127) << 23); }

/* The n with |x| 2^n in [2^14, 2^15) for the bits of a finite |x|, at most
 * `most`. */
__device__ __forceinline__ int scale_of(uint32_t bits, int most) { return min(14 - ((int)(bits >> 23) - 127), most); }

/* Eight values as two limbs. In pairs, so that a limb is rounded once, packed;
 * v - hi is one instruction as a multiply-add of a half and floats, if the
 * compiler does not know that the factor is -1. */
__device__ __forceinline__ void limbs_of(const float *x, h8_t *hi, h8_t *lo)
{
    float minus;
    asm("s_mov_b32 %0, -1.0" : "=s"(minus));
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const f2_t v = {x[i], x[i + 1]};
        const h2_t h = __builtin_convertvector(v, h2_t);
        const f2_t rest = {fmaf((float)h[0], minus, v[0]), fmaf((float)h[1], minus, v[1])};
        const h2_t l = __builtin_convertvector(rest, h2_t);
        (*hi)[i] = h[0];
        (*hi)[i + 1] = h[1];
        (*lo)[i] = l[0];
        (*lo)[i + 1] = l[1];
    }
}

/* What lanes read for keys past the end (zeros), and for keys whose page is not
 * there (NaN in every type: the rows that attend them become NaN). */
__device__ const u4_t kNoPiece[4] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {~0u, ~0u, ~0u, ~0u}, {~0u, ~0u, ~0u, ~0u}};
constexpr int64_t kPastEnd = -2, kNoPage = -1;

/* Pieces of 8 elements that a lane loads, as 16-byte words. */
template <int TYPE> struct Raw {
    static constexpr int WORDS = TYPE == QMV_KV_F32 ? 2 : 1;
    static constexpr uint32_t INF = TYPE == QMV_KV_F32 ? 0x7f800000u : TYPE == QMV_KV_F16 ? 0x7c00u : 0x7f80u;
    u4_t w[WORDS];

    /* The largest magnitude's bits (f16, bf16: its code); at least INF where an
     * element is not finite. */
    __device__ __forceinline__ uint32_t top() const
    {
        uint32_t m = 0;
        if (TYPE == QMV_KV_F32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, w[i >> 2][i & 3] & 0x7fffffffu);
            return m;
        }
        typedef uint16_t s2_t __attribute__((ext_vector_type(2)));
        s2_t m2 = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) m2 = __builtin_elementwise_max(m2, __builtin_bit_cast(s2_t, w[0][i] & 0x7fff7fffu));
        return max(m2[0], m2[1]);
    }

    /* The same of the finite ones. */
    __device__ __forceinline__ uint32_t top_finite() const
    {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t x = TYPE == QMV_KV_F32 ? w[i >> 2][i & 3] & 0x7fffffffu : w[0][i >> 1] >> 16 * (i & 1) & 0x7fffu;
            m = max(m, x >= INF ? 0u : x);
        }
        return m;
    }

    /* f(element) for those that are not finite, which become zero. */
    template <typename F> __device__ __forceinline__ void clear_odd(F f)
    {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            constexpr bool wide = TYPE == QMV_KV_F32;
            const uint32_t x = w[wide ? e >> 2 : 0][wide ? e & 3 : e >> 1];
            const uint32_t mask = wide ? INF : INF << 16 * (e & 1);
            if ((x & mask) == mask) {
                w[wide ? e >> 2 : 0][wide ? e & 3 : e >> 1] = wide ? 0u : x & 0xffff0000u >> 16 * (e & 1);
                f(e);
            }
        }
    }

    /* As f16 limbs, after a factor 2^n (not of f16), to `to` and to + apart. */
    __device__ __forceinline__ void put(unsigned char *to, int apart, int n) const
    {
        if (TYPE == QMV_KV_F16) {
            *(u4_t *)to = w[0];
        } else if (TYPE == QMV_KV_BF16) {
            h8_t h;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const f2_t v = {__uint_as_float(w[0][e] << 16) * power_of_two(n),
                                __uint_as_float(w[0][e] & 0xffff0000u) * power_of_two(n)};
                const h2_t h2 = __builtin_convertvector(v, h2_t);
                h[2 * e] = h2[0];
                h[2 * e + 1] = h2[1];
            }
            *(h8_t *)to = h;
        } else {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e >> 2][e & 3]) * power_of_two(n);
            h8_t hi, lo;
            limbs_of(x, &hi, &lo);
            *(h8_t *)to = hi;
            *(h8_t *)(to + apart) = lo;
        }
    }
};

/* A tile in LDS is rows of keys. Piece c of a key is at place c ^ turn(key):
 * neither the loads of one piece of 32 keys nor the transposing loads of a few
 * pieces of eight meet in a bank (none counted with 32 rows a wave). */
template <int DP> __device__ __forceinline__ int turn_of(int key)
{
    return DP == 128 ? (key & 3) << 2 | (key >> 2 & 3) : (key >> 1 & 1) << 2 | (key >> 2 & 3);
}
constexpr int kMostKeys = 126, kMostValues = 100; /* most factors of scale_of */
constexpr int kZeroValues = 12; /* the factor of a block of zeros: what values near one have, so that they are not apart */

struct AttnItem {
    int s, start, n, len; /* the sequence, its first token, new tokens and length (cut to its pages) */
    int first;            /* position of its first new token */
    int tiles;            /* its row tiles */
    int tile, tile_at;    /* one of them; among all sequences' */
    int split, chunk;     /* keys [split * chunk, ...) */
};

/* What attention_list_kernel finds: pieces and row tiles of a key head, and keys
 * of a piece at most. */
struct AttnLists {
    int items, tiles, chunk;
};

/* What the pieces' join has to know of a row tile whose keys are cut. */
struct AttnJoin {
    int start, n, first, tile; /* as in AttnItem */
    int pieces;                /* 0: not cut */
    int item, apart;    /* the first piece's number, and what the next ones' are apart */
};

/* A sequence as the kernels see it: cut to the call's tokens and its pages. */
struct AttnSequence {
    int start, n, len, first, tiles; /* as in AttnItem */
};
template <int BM> __device__ __forceinline__ AttnSequence sequence_at(const AttnTokens &a, int s)
{
    AttnSequence q = {};
    if (s >= a.count) return q;
    const int room = a.page_size ? a.table_stride * a.page_size : INT32_MAX; /* at most 2^30, or no limit */
    q.start = min(max(a.starts[s], 0), a.tokens);
    q.n = max(min(a.starts[s + 1], a.tokens) - q.start, 0);
    q.len = a.lengths ? max(a.lengths[s], 0) : q.n;
    q.first = q.len - q.n;
    if (q.len > room) q.len = room + 1; /* one key past the table: its rows are NaN */
    q.tiles = (q.n * (a.heads / a.kv_heads) + BM - 1) / BM;
    return q;
}

/* What a sequence's tiles attend, or more. */
__device__ __forceinline__ float work_of(const AttnTokens &a, const AttnSequence &q)
{
    return (float)q.tiles * (a.page_size ? (float)q.len : 0.5f * (float)q.len);
}

/* Keys of a piece at most, from the sums over all sequences and the longest
 * that brings tokens; `even`: their new tokens are alike. A whole wave asks. The
 * sums are of floats, whose rounding the one piece beyond plan_attention's count
 * allows for.
 *
 * Where the lengths are alike (and slots is set: up to 32 rows over f16 or bf16) each
 * lane takes a number of pieces per tile and says what it costs: rounds of the
 * workgroups that run at once, each as long as its keys and 64 more for its
 * start, less where a single round leaves compute units to one workgroup, which
 * streams up to 1 / 0.58 times as fast as two. 28 and 4 heads of 128, f16, with
 * and without (us): 64 sequences of 1000 keys 33 / 42, of 4000 108 / 121, 16 of
 * 4000 33 / 41. */
template <int STEP> __device__ __forceinline__ int chunk_of(const AttnParams &p, float work, float tiles, int longest, bool even)
{
    const int whole = INT32_MAX / STEP * STEP;
    if (p.target == 0) return whole;
    const bool alike = even && tiles * (float)longest <= 1.1f * work;
    const int pieces = (alike ? p.alike : p.target) / p.t.kv_heads;
    if (p.slots && alike && tiles * 64.f >= (float)pieces) {
        const int lane = threadIdx.x & 63, n = lane + 1;
        const int keys = max((longest / n + STEP) / STEP * STEP, STEP); /* n of them reach `longest` */
        const float items = tiles * (float)n, load = items * (float)p.t.kv_heads / (float)p.slots;
        const float cost = (float)(keys + 64) * (load > 1.f ? ceilf(load) : fmaxf(load, 0.58f));
        const bool fits = lane == 0 || (items <= (float)pieces && keys >= p.least);
        /* the cheapest, of the same cost the fewest pieces */
        const uint32_t worth = fits ? ~(__float_as_uint(cost) & ~63u | (uint32_t)lane) : 0u;
        const int best = (int)(~wave_max(worth) & 63u);
        return lane_of(keys, best);
    }
    /* pieces beside the tiles' last ones, which may be short */
    const float each = work / (float)max(max(pieces - (int)tiles, pieces / 2), 1);
    return each < 1e9f ? max(((int)each + STEP) / STEP * STEP, p.least) : whole;
}

__device__ __forceinline__ int splits_of(const AttnSequence &q, int chunk)
{
    return max((int)(((uint32_t)q.len + (uint32_t)chunk - 1) / (uint32_t)chunk), 1);
}

/* The `mine`-th piece of sequence s: the first pieces of all its row tiles, the
 * later ones (which attend more) first, then their second pieces, and so on.
 * Consecutive workgroups run on different XCDs, and with a tile's pieces side by
 * side those that have no keys were all on the same four (a prompt of 4096, 7B,
 * 542 us in two pieces a tile). */
template <int STEP> __device__ __forceinline__ void piece_of(const AttnSequence &q, int s, int splits, int mine, int tiles_before, AttnItem *out)
{
    const int nth = mine % q.tiles;
    out->s = s;
    out->start = q.start;
    out->n = q.n;
    out->len = q.len;
    out->first = q.first;
    /* pieces of one length, not all but the last of a whole chunk */
    out->chunk = ((max(q.len, 1) + splits - 1) / splits + STEP - 1) / STEP * STEP;
    out->tiles = q.tiles;
    out->split = mine / q.tiles;
    out->tile = q.tiles - 1 - nth;
    out->tile_at = tiles_before + out->tile;
}

/* The `item`-th piece of a key head's work, sequence after sequence, by one wave.
 * Every workgroup takes the same sums over all lengths. *tiles_all: row tiles in
 * all, or 0 where the starts fall so that there would be more rows than the
 * call's. */
template <int BM, int STEP>
__device__ __forceinline__ bool find_item(const AttnParams &p, int item, int lane, AttnItem *out, int *tiles_all)
{
    const AttnTokens &a = p.t;
    if (p.lists) { /* attention_list_kernel has looked already */
        const AttnLists &lists = *p.lists;
        *tiles_all = lists.tiles;
        if (item >= lists.items) return false;
        const int s = __builtin_amdgcn_readfirstlane(p.sequence_of_item[item]);
        const AttnSequence q = sequence_at<BM>(a, s);
        const int2 before = p.before[s];
        piece_of<STEP>(q, s, splits_of(q, lists.chunk), item - before.x, before.y, out);
        return true;
    }
    AttnSequence q;
    float work = 0.f, rows = 0.f, tiles = 0.f, busy = 0.f;
    int longest = 0, most = 0;
    for (int s0 = 0; s0 < a.count; s0 += 64) {
        q = sequence_at<BM>(a, s0 + lane);
        longest = max(longest, q.n > 0 ? q.len : 0);
        most = max(most, q.n);
        busy += q.n > 0 ? 1.f : 0.f;
        work += work_of(a, q);
        rows += (float)q.n;
        tiles += (float)q.tiles;
    }
    work = lane_of(scan_lanes(work), 63);
    rows = lane_of(scan_lanes(rows), 63);
    tiles = lane_of(scan_lanes(tiles), 63);
    *tiles_all = 0;
    if (rows > (float)a.tokens) return false;
    bool even = true;
    if (p.alike != p.target) even = (float)wave_max((uint32_t)most) * lane_of(scan_lanes(busy), 63) <= 1.1f * rows;
    const int chunk = chunk_of<STEP>(p, work, tiles, (int)wave_max((uint32_t)longest), even);
    int before = 0, tiles_before = 0;
    bool found = false;
    for (int s0 = 0; s0 < a.count; s0 += 64) {
        if (a.count > 64) q = sequence_at<BM>(a, s0 + lane);
        const int splits = splits_of(q, chunk);
        const int items = q.tiles * splits;
        const int sum = scan_lanes(items), tsum = scan_lanes(q.tiles);
        const uint64_t hit = __ballot(before + sum > item);
        if (hit && !found) {
            const int at = __builtin_ctzll(hit);
            const AttnSequence mine = {lane_of(q.start, at), lane_of(q.n, at), lane_of(q.len, at), lane_of(q.first, at),
                                       lane_of(q.tiles, at)};
            piece_of<STEP>(mine, s0 + at, lane_of(splits, at), item - before - (lane_of(sum, at) - lane_of(items, at)),
                           tiles_before + lane_of(tsum, at) - mine.tiles, out);
            found = true;
        }
        before += lane_of(sum, 63);
        tiles_before += lane_of(tsum, 63);
        if (found && item > 0) break; /* the first workgroup counts all tiles */
    }
    *tiles_all = tiles_before;
    return found;
}

/* Many sequences: what find_item would look for in every workgroup, once. One
 * workgroup: the sums and the chunk, then 1024 sequences at a time the items
 * and tiles before each and each item's sequence. (8192 sequences of 200 keys,
 * 28 and 4 heads: 9.7 ms without.) */
template <int BM, int STEP> __global__ __launch_bounds__(1024) void attention_list_kernel(AttnParams p)
{
    __shared__ float sums[4][16];
    __shared__ int longests[16], mosts[16], ends[1024], tile_ends[16], item_ends[16];
    const AttnTokens &a = p.t;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    float work = 0.f, rows = 0.f, tiles = 0.f, busy = 0.f;
    int longest = 0, most = 0;
    for (int s = tid; s < a.count; s += 1024) {
        const AttnSequence q = sequence_at<BM>(a, s);
        longest = max(longest, q.n > 0 ? q.len : 0);
        most = max(most, q.n);
        busy += q.n > 0 ? 1.f : 0.f;
        work += work_of(a, q);
        rows += (float)q.n;
        tiles += (float)q.tiles;
    }
    work = scan_lanes(work);
    rows = scan_lanes(rows);
    tiles = scan_lanes(tiles);
    busy = scan_lanes(busy);
    longest = (int)wave_max((uint32_t)longest);
    most = (int)wave_max((uint32_t)most);
    if (lane == 63) {
        longests[wave] = longest;
        mosts[wave] = most;
        sums[3][wave] = busy;
        sums[0][wave] = work;
        sums[1][wave] = rows;
        sums[2][wave] = tiles;
    }
    __syncthreads();
    work = rows = tiles = busy = 0.f;
    for (int i = 0; i < 16; ++i) {
        work += sums[0][i];
        rows += sums[1][i];
        tiles += sums[2][i];
        busy += sums[3][i];
        longest = max(longest, longests[i]);
        most = max(most, mosts[i]);
    }
    const int chunk = chunk_of<STEP>(p, work, tiles, longest, (float)most * busy <= 1.1f * rows || p.alike == p.target);
    const bool valid = rows <= (float)a.tokens;
    int items_before = 0, tiles_before = 0;
    for (int s0 = 0; valid && s0 < a.count; s0 += 1024) {
        const AttnSequence q = sequence_at<BM>(a, s0 + tid);
        const int items = q.tiles * splits_of(q, chunk);
        int sum = scan_lanes(items), tsum = scan_lanes(q.tiles);
        if (lane == 63) {
            item_ends[wave] = sum;
            tile_ends[wave] = tsum;
        }
        __syncthreads();
        int all = 0, tall = 0;
        for (int i = 0; i < 16; ++i) {
            if (i < wave) {
                sum += item_ends[i];
                tsum += tile_ends[i];
            }
            all += item_ends[i];
            tall += tile_ends[i];
        }
        ends[tid] = sum;
        if (s0 + tid < a.count) p.before[s0 + tid] = int2{items_before + sum - items, tiles_before + tsum - q.tiles};
        __syncthreads();
        for (int i = tid; i < all; i += 1024) {
            if (items_before + i >= p.most_items) break;
            int lo = 0, hi = 1023; /* the first sequence whose items end past i */
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (ends[mid] > i) hi = mid;
                else lo = mid + 1;
            }
            p.sequence_of_item[items_before + i] = s0 + lo;
        }
        items_before += all;
        tiles_before += tall;
        __syncthreads();
    }
    if (tid == 0) *p.lists = AttnLists{min(items_before, p.most_items), tiles_before, chunk};
}

/* Long prompts: their keys and values are split into limbs once, as images of
 * the tiles in LDS: K high, K low, V high, V low, and a head of floats: the
 * blocks' factors of the keys, exponents of the values, and whether any value
 * is not finite. Sequence s has its tiles from start / 64 + s on. */
constexpr int kImageKeys = 64, kImageHead = 64;
__host__ __device__ constexpr int64_t image_bytes(int dp) { return kImageKeys * dp * 2 * 4 + kImageHead * 4; }

template <int DP> __global__ __launch_bounds__(256) void attention_image_kernel(AttnParams p)
{
    constexpr int SLOTS = DP / 32, PIECES = DP / 8, PER = 64 / PIECES, MAT = kImageKeys * DP * 2;
    __shared__ int odd_waves[4];
    const AttnTokens &a = p.t;
    const int lane = threadIdx.x & 63, b = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); /* a block of 16 keys */
    const int kvh = blockIdx.x % a.kv_heads, at = blockIdx.x / a.kv_heads;
    auto start_of = [&](int s) { return min(max(a.starts[s], 0), a.tokens); };
    int lo = 0, hi = a.count; /* the last sequence that begins at this tile or before */
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start_of(mid) / kImageKeys + mid <= at) lo = mid;
        else hi = mid;
    }
    const int start = start_of(lo), n = start_of(lo + 1) - start, first = (at - start / kImageKeys - lo) * kImageKeys;
    if (first < 0 || first >= n) return;
    unsigned char *const image = p.image + (int64_t)blockIdx.x * image_bytes(DP);
    float *const head = (float *)(image + 4 * MAT);
    const int piece = lane % PIECES, sub = lane / PIECES;
    Raw<QMV_KV_F32> raw[2][SLOTS];
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
        const int j = first + 16 * b + i * PER + sub;
        const bool there = j < n && 8 * piece < a.dim;
        const int64_t column = (int64_t)kvh * a.dim + 8 * piece;
        const u4_t *k = there ? (const u4_t *)((const float *)p.k + (start + j) * p.k_stride + column) : kNoPiece;
        const u4_t *v = there ? (const u4_t *)((const float *)p.v + (start + j) * p.v_stride + column) : kNoPiece;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            raw[0][i].w[r] = k[r];
            raw[1][i].w[r] = v[r];
        }
    }
    bool odd_values = false;
#pragma unroll
    for (int values = 0; values < 2; ++values) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) top = max(top, raw[values][i].top());
        top = wave_max(top);
        if (top >= Raw<QMV_KV_F32>::INF) {
            if (values) {
                odd_values = true;
#pragma unroll
                for (int i = 0; i < SLOTS; ++i) raw[1][i].clear_odd([](int) {});
            }
            top = 0;
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) top = max(top, raw[values][i].top_finite());
            top = wave_max(top);
        }
        const int n2 = values && top == 0 ? kZeroValues : scale_of(top, values ? kMostValues : kMostKeys);
        if (lane == 0) head[4 * values + b] = values ? (float)-n2 : power_of_two(-n2);
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            const int key = i * PER + sub;
            raw[values][i].put(image + 2 * values * MAT + (16 * b + key) * DP * 2 + ((piece ^ turn_of<DP>(key)) << 4), MAT, n2);
        }
    }
    if (lane == 0) odd_waves[b] = odd_values;
    __syncthreads();
    if (threadIdx.x < kImageHead - 8)
        head[8 + threadIdx.x] = threadIdx.x == 4 && (odd_waves[0] | odd_waves[1] | odd_waves[2] | odd_waves[3]) ? 1.f : 0.f;
}

/* DP: head_dim padded to 64 or 128; RW: rows of a wave; WR waves along the
 * rows, WK along the keys. */
template <int TYPE, int DP, int RW, int WR, int WK> struct AttnShape {
    static constexpr bool IMAGE = TYPE == QMV_KV_IMAGE;
    static constexpr int NL = TYPE == QMV_KV_F32 || IMAGE ? 2 : 1; /* limbs of keys and values */
    static constexpr int KT = WR >= 4 ? 64 : 32;            /* keys a wave takes per tile */
    static constexpr int NB = KT / 16;                      /* blocks of 16 keys */
    static constexpr int UNITS = 2 * NB / WR;               /* blocks (of keys, of values) a wave loads */
    static constexpr int SLOTS = DP / 32;                   /* pieces of 8 elements a lane loads per block */
    static constexpr int MAT = KT * DP * 2;                 /* bytes of a limb of keys or of values */
    static constexpr int TILE = 2 * NL * MAT;
    static constexpr int ROWS = RW * WR;
    static constexpr int JOIN = WK > 1 ? WK * (RW * DP * 4) : 0; /* the waves' O, where they meet */
    static constexpr int TILES = IMAGE ? 2 : WK;
    static constexpr int LDS = TILES * TILE > JOIN ? TILES * TILE : JOIN;
    static constexpr int PEAKS = TYPE == QMV_KV_F16 ? 1 : WR * WK * RW;
};

template <class S, int DP, int RW, int WK> struct AttnShared {
    __attribute__((aligned(16))) unsigned char lds[S::LDS];
    /* of the keys: factors; of the values: exponents; of an image: its whole head */
    float scales[S::TILES][S::IMAGE ? kImageHead : 2 * S::NB];
    int first_odd[DP]; /* the first key whose value is not finite there */
    int any_odd;
    float joined[WK > 1 ? WK : 1][2][RW];
    /* Each row's highest rm so far, where blocks are taken one after the other;
     * a row's lanes write the same. */
    float peaks[S::PEAKS];
};

/* One piece; LAYOUT: rows of a tile as its result's place in the workspace. */
template <int TYPE, int DP, int RW, int WR, int WK, int LAYOUT>
__device__ __forceinline__ void attend_piece(const AttnParams &p, const AttnItem &it, int item, int kvh,
                                             AttnShared<AttnShape<TYPE, DP, RW, WR, WK>, DP, RW, WK> &shared)
{
    using S = AttnShape<TYPE, DP, RW, WR, WK>;
    using P = Product<RW>;
    using acc_t = typename P::acc_t;
    constexpr bool IMAGE = S::IMAGE;
    constexpr int KT = S::KT, NB = S::NB, UNITS = S::UNITS, SLOTS = S::SLOTS, MAT = S::MAT, NL = S::NL;
    constexpr int THREADS = 64 * WR * WK, WIDE = 512 / RW; /* of a product's contraction */
    constexpr int STEPS = DP / WIDE, DB = DP / RW, REGS = RW * RW / 64, SCORES = RW / 2;
    constexpr int PARTIAL = LAYOUT * DP + 2 * LAYOUT; /* floats of a piece's result */
    auto &lds = shared.lds;
    auto &scales = shared.scales;
    auto &first_odd = shared.first_odd;
    auto &any_odd = shared.any_odd;
    auto &joined = shared.joined;
    constexpr bool SCALED = TYPE != QMV_KV_F16;
    float *const peak = shared.peaks + (SCALED ? (threadIdx.x >> 6) * RW + threadIdx.x % RW : 0);

    const AttnTokens &a = p.t;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave % WR, wk = wave / WR, part_of = lane / RW, col = lane % RW;
    const int group = a.heads / a.kv_heads, dim = a.dim;
    for (int i = tid; i < DP; i += THREADS) first_odd[i] = INT32_MAX;
    if (tid == 0) any_odd = 0;
    if (SCALED) *peak = kNoScale;
    lds_barrier();

    /* the keys of this piece */
    const int last_token = min(it.n - 1, (it.tile * S::ROWS + S::ROWS - 1) / group);
    const int keys = max(min(it.first + last_token + 1, it.len), 0);
    const int pieces = max((int)(((int64_t)keys + it.chunk - 1) / it.chunk), 1);
    if (it.split >= pieces) return;
    if (p.target && kvh == 0 && it.split == 0 && tid == 0)
        p.joins[1 + it.tile_at] = AttnJoin{it.start, it.n, it.first, it.tile, pieces > 1 ? pieces : 0, item, it.tiles};
    const int begin = it.split * it.chunk, end = min((int64_t)keys, (int64_t)begin + it.chunk);
    const int unmasked = it.first + it.tile * S::ROWS / group; /* every row attends keys up to here */

    /* this lane's row */
    const int row = it.tile * S::ROWS + wr * RW + col;
    const int token = row / group, head = kvh * group + row % group;
    const bool real = token < it.n;
    const int pos = real ? it.first + token : -1;
    /* A wave without rows only loads: 24 of 128 rows over 4000 keys 179 us
     * otherwise, 169 so. */
    const bool works = WR == 1 || it.tile * S::ROWS + wr * RW < it.n * group;

    /* ---- tiles: loads into registers, then as f16 limbs into LDS ---- */
    unsigned char *tile = lds + (IMAGE ? 0 : wk * S::TILE);
    int buf = IMAGE ? 0 : wk;
    constexpr int PIECES = DP / 8, PER = 64 / PIECES; /* of a key; keys per slot */
    const int piece = lane % PIECES, sub = lane / PIECES;
    constexpr int OWN = WR == 1 ? KT : 16; /* keys whose places a wave looks up */
    const int own_first = WR == 1 ? 0 : 16 * (wr % NB);

    /* Where lane's key (own_first + lane % OWN) of the tile at k0 begins, of a
     * prompt its row. */
    auto place = [&](int k0) -> int64_t {
        const int j = k0 + own_first + (lane & (OWN - 1));
        if (j >= end) return kPastEnd;
        if (a.page_size == 0) return it.start + j;
        const int64_t at = key_at(a, it.s, j, kvh);
        if (at < 0 && a.status) *a.status = 0;
        return at;
    };
    Raw<TYPE> raw[UNITS][SLOTS];
    /* Tiles of 16 and 32 rows load past the caches, since most often one tile
     * reads a key there: 64 sequences of 4000 keys, 28 and 4 heads of 128, f16, 108
     * us without and 97 with, of 1000 keys 35 and 35. Not of fp32, whose lanes take
     * 32 bytes of a line in two loads (64 of 2000: 129 and 139), nor tiles of more
     * rows, which share keys (4 sequences of 8000 under 28 tiles each 38 and 41).
     * A sequence of several such tiles, in a call whose average chose them, shares
     * keys all the same, and reads them from memory each time. */
    constexpr bool STREAM = WR == 1 && TYPE != QMV_KV_F32;
    auto unit_block = [&](int u) { return WR == 1 ? u % NB : wr % NB; };
    auto unit_values = [&](int u) { return WR == 1 ? u >= NB : UNITS == 1 ? wr >= NB : u == 1; };
    auto load = [&](int64_t at) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const unsigned char *base = (const unsigned char *)(unit_values(u) ? p.v : p.k);
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                int64_t from = shfl64(at, (WR == 1 ? 16 * unit_block(u) : 0) + i * PER + sub);
                if (a.page_size == 0 && from >= 0) /* both under 2^31 */
                    from = (int64_t)((uint64_t)(uint32_t)from * (uint32_t)(unit_values(u) ? p.v_stride : p.k_stride)) + kvh * dim;
                const unsigned char *src = base + (from + 8 * piece) * (TYPE == QMV_KV_F32 ? 4 : 2);
                if (from < 0 || 8 * piece >= dim)
                    src = (const unsigned char *)(kNoPiece + (from == kNoPage && !unit_values(u) && 8 * piece < dim ? 2 : 0));
#pragma unroll
                for (int r = 0; r < Raw<TYPE>::WORDS; ++r)
                    raw[u][i].w[r] = STREAM ? __builtin_nontemporal_load((const u4_t *)src + r) : ((const u4_t *)src)[r];
            }
        }
    };
    auto store = [&](int k0) {
        const bool masked = k0 + KT - 1 > unmasked;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const int b = unit_block(u);
            const bool values = unit_values(u);
            int n = 0;
            if (TYPE != QMV_KV_F16 || (values && masked)) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < SLOTS; ++i) top = max(top, raw[u][i].top());
                top = wave_max(top);
                if (top >= Raw<TYPE>::INF) {
                    /* A value that is not finite must not reach the rows that do not
                     * attend it, and 0 * inf is NaN: where some do not, zero takes
                     * its place here, and the rows that do are marked at the end. */
                    if (values && masked) {
                        any_odd = 1;
#pragma unroll
                        for (int i = 0; i < SLOTS; ++i)
                            raw[u][i].clear_odd([&](int e) { atomicMin(&first_odd[8 * piece + e], k0 + 16 * b + i * PER + sub); });
                    }
                    top = 0;
#pragma unroll
                    for (int i = 0; i < SLOTS; ++i) top = max(top, raw[u][i].top_finite());
                    top = wave_max(top);
                }
                if (TYPE != QMV_KV_F16) {
                    n = values && top == 0 ? kZeroValues : scale_of(TYPE == QMV_KV_BF16 ? top << 16 : top, values ? kMostValues : kMostKeys);
                    if (lane == 0) scales[wk][values ? NB + b : b] = values ? (float)-n : power_of_two(-n);
                }
            }
            unsigned char *to = tile + (values ? NL * MAT : 0) + 16 * b * DP * 2;
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) {
                const int key = i * PER + sub;
                raw[u][i].put(to + key * DP * 2 + ((piece ^ turn_of<DP>(key)) << 4), MAT, n);
            }
        }
    };

    /* An image's tile goes to LDS as it is. */
    const int64_t image_at = IMAGE ? it.start / KT + it.s : 0;
    auto fetch = [&](int k0, int buf) {
        constexpr int MINE = S::TILE / (WR * WK);
        const unsigned char *src = p.image + ((image_at + k0 / KT) * a.kv_heads + kvh) * image_bytes(DP);
        unsigned char *to = lds + buf * S::TILE + wave * MINE;
        typedef __attribute__((address_space(1))) void *from_t;
        typedef QMV_LDS void *to_t;
#pragma unroll
        for (int i = 0; i < MINE; i += 1024)
            __builtin_amdgcn_global_load_lds((from_t)(src + wave * MINE + i + lane * 16), (to_t)(to + i), 16, 0, 0);
        if (wave == 0) __builtin_amdgcn_global_load_lds((from_t)(src + S::TILE + lane * 4), (to_t)&scales[buf][0], 4, 0, 0);
    };

    constexpr int STEP = KT * WK;
    int k0 = begin + wk * KT;
    int64_t next = 0;
    if constexpr (IMAGE) {
        if (begin < end) fetch(begin, 0);
    } else {
        next = place(k0);
        if (begin < end) load(next);
        next = place(k0 + STEP);
    }

    /* q as two limbs, 8 elements of each step */
    h8_t qhi[STEPS], qlo[STEPS];
    float q_back;
    {
        const float *q = p.q + (int64_t)(it.start + token) * p.q_stride + (int64_t)head * dim;
        const float by = p.scale * kLog2e;
        float x[STEPS][8];
        uint32_t bits = 0;
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
            const int d = WIDE * st + 8 * part_of;
            f4_t u = {0, 0, 0, 0}, v = {0, 0, 0, 0};
            if (real && d < dim) {
                u = *(const f4_t *)(q + d);
                v = *(const f4_t *)(q + d + 4);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[st][i] = (i < 4 ? u[i & 3] : v[i & 3]) * by;
                const uint32_t m = __float_as_uint(x[st][i]) & 0x7fffffffu;
                if (m < 0x7f800000u) bits = max(bits, m);
            }
        }
        const int n = scale_of(__float_as_uint(max_lanes<RW>(__uint_as_float(bits))), 126);
        q_back = power_of_two(-n);
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[st][i] *= power_of_two(n);
            limbs_of(x[st], &qhi[st], &qlo[st]);
        }
    }

    /* ---- a tile's products ---- */
    acc_t o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = acc_t{0};
    float m = kNothing, rm = SCALED ? kNoScale : 0.f, l = 0.f; /* of f16 values m is r */
    float limit = kNothing;                                    /* m + rm + kSlack */
    /* Key 32 sb + score_key(i) of a tile is the one of score register i. */
    auto score_key = [&](int i) { return (256 / RW) * (i >> 2) + 4 * part_of + (i & 3); };
    const int k_at = col * DP * 2 + ((part_of ^ turn_of<DP>(col)) << 4);
    /* K of RW keys, one step of the contraction. */
    auto k_frag = [&](int limb, int kb, int st) -> h8_t {
        return *(const h8_t *)(tile + limb * MAT + kb * RW * DP * 2 + (k_at ^ st * (WIDE * 2)));
    };
    const int kk = (lane & 15) >> 2; /* this lane's key of four in a transposing load */
    int v_at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int key = 256 / RW * i + 4 * part_of + kk;
        const int at = (RW == 32 ? (lane >> 4 & 1) << 1 : 0) | (lane >> 1 & 1); /* pieces within the product's rows */
        v_at[i] = key * DP * 2 + ((at ^ turn_of<DP>(key)) << 4) + (lane & 1) * 8;
    }
    /* V^T of one step of keys and RW elements: 8 keys of one element a lane, in
     * the order in which the scores are in its registers. */
    auto v_frag = [&](int limb, int step, int db) -> h8_t {
        const unsigned char *base = tile + (NL + limb) * MAT + step * WIDE * DP * 2;
        typedef QMV_LDS s4_t *ptr;
        const s4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(base + (v_at[0] ^ db * (RW * 2))));
        const s4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(base + (v_at[1] ^ db * (RW * 2))));
        const h4_t hx = __builtin_bit_cast(h4_t, x), hy = __builtin_bit_cast(h4_t, y);
        return h8_t{hx[0], hx[1], hx[2], hx[3], hy[0], hy[1], hy[2], hy[3]};
    };
    constexpr int EACH = SCORES / 2; /* scores of a block of 16 keys */
    constexpr int VS = 32 / WIDE;    /* steps of 8 scores a lane */
    bool apart = false;
    /* 32 keys; of blocks taken one after the other (apart) the first or the
     * second. */
    auto pass = [&](int k0, int sb, int only) {
        /* Unknown to the compiler, so that it does not keep the masks of all
         * scores between the two (93 spilled scalar registers at 128 rows). */
        if (SCALED) asm volatile("" : "+s"(k0));
        float c[SCORES];
        __builtin_amdgcn_s_setprio(1); /* these products before the other waves' softmax: 1% of a long prompt */
#pragma unroll
        for (int kb = 0; kb < 32 / RW; ++kb) {
            acc_t x = {0};
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                const h8_t hi = k_frag(0, 32 / RW * sb + kb, st);
                x = P::run(hi, qhi[st], x);
                x = P::run(hi, qlo[st], x);
                if (NL == 2) x = P::run(k_frag(1, 32 / RW * sb + kb, st), qhi[st], x);
            }
#pragma unroll
            for (int i = 0; i < REGS; ++i) c[REGS * kb + i] = x[i];
        }
        __builtin_amdgcn_s_setprio(0);
        const int first = k0 + 32 * sb;
        const bool masked = first + 31 > unmasked;
        if (masked) {
#pragma unroll
            for (int i = 0; i < SCORES; ++i)
                if (first + score_key(i) > pos) c[i] = -INFINITY;
        }
        float by[2], add[2], most[2];
        float top = -INFINITY;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            if (SCALED) {
                /* within the finite positive floats, so that a masked score stays -inf */
                by[g] = fminf(fmaxf(q_back * scales[buf][2 * sb + g], 1.1754944e-38f), 1.7014118e38f);
                add[g] = scales[buf][NB + 2 * sb + g];
            } else {
                by[g] = q_back;
                add[g] = 0.f;
            }
            most[g] = c[EACH * g];
#pragma unroll
            for (int i = 1; i < EACH; ++i) most[g] = fmaxf(most[g], c[EACH * g + i]);
            top = fmaxf(top, fmaf(most[g], by[g], add[g]));
        }
        top = max_lanes<RW>(top);
        const float low = fminf(add[0], add[1]);
        float less = m; /* what the scores are taken relative to below */
        if (apart || __any(top > limit || (SCALED && rm - low > kApart))) {
            float to, fade;
            if (SCALED) {
                to = fmaxf(m, ceilf(max_lanes<RW>(fmaxf(most[0] * by[0], most[1] * by[1]))));
                const float now = rm + (m - to);
                float next = top > limit ? ceilf(top) - to : now;
                apart = apart || __any(next - low > kApart || (fabsf(to) > 4194304.f && to > kNothing));
                if (apart) {
                    const float best = max_lanes<RW>(only ? most[1] * by[1] : most[0] * by[0]);
                    const float own = ceilf(best) - to + (only ? add[1] : add[0]);
                    const float high = fmaxf(fmaxf(*peak + (m - to), now), own);
                    *peak = high;
                    /* now: the row attends no key of the block */
                    next = best == -INFINITY ? now : fmaxf(own, high - kReach);
                    /* A block below the reach: its weights are kept large enough
                     * for the sum, and are zero as f16. */
                    const float lift = fminf(fmaxf(next - kReach - own, 0.f), 400.f);
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
#pragma unroll
                        for (int i = EACH * g; i < EACH * (g + 1); ++i) c[i] = g == only ? fmaf(c[i], by[g], -to) : -INFINITY;
                        by[g] = 1.f;
                        add[g] += lift;
                    }
                    less = 0.f;
                } else {
                    less = to;
                }
                fade = __builtin_amdgcn_exp2f(now - next); /* at most 2^kReach */
                rm = next;
            } else {
                to = top > limit ? top : m;
                fade = __builtin_amdgcn_exp2f(m - to);
                less = to;
            }
            l *= __builtin_amdgcn_exp2f(m - to);
            m = to;
            limit = m + rm + kSlack;
#pragma unroll
            for (int i = 0; i < DB; ++i) o[i] *= fade;
        }
        h8_t phi[VS], plo[VS];
        float w[SCORES];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const float over = add[g] - rm, shift = (over + kShift) - less;
            float sum = 0.f;
#pragma unroll
            for (int i = EACH * g; i < EACH * (g + 1); ++i) {
                w[i] = __builtin_amdgcn_exp2f(fmaf(c[i], by[g], shift));
                sum += w[i];
            }
            l += SCALED ? __builtin_ldexpf(sum, -20 - (int)over) : sum; /* of zero weights zero */
        }
#pragma unroll
        for (int g = 0; g < VS; ++g) {
            limbs_of(w + 8 * g, &phi[g], &plo[g]);
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const h8_t v = v_frag(0, VS * sb + g, db);
                o[db] = P::run(v, phi[g], o[db]);
                o[db] = P::run(v, plo[g], o[db]);
                if (NL == 2) o[db] = P::run(v_frag(1, VS * sb + g, db), phi[g], o[db]);
            }
        }
    };
    auto compute = [&](int k0) {
#pragma unroll
        for (int sb = 0; sb < KT / 32; ++sb) {
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (SCALED) {
                int only = 0;
                do pass(k0, sb, only);
                while (apart && ++only < 2);
            } else {
                pass(k0, sb, 0);
            }
        }
    };

    if constexpr (IMAGE) {
        for (; k0 < end; k0 += STEP) {
            __builtin_amdgcn_s_waitcnt(0x0F70); /* vmcnt(0): this wave's part of the tile */
            lds_barrier();                      /* and the others'; the tile before has been read */
            if (k0 + STEP < end) fetch(k0 + STEP, buf ^ 1);
            if (scales[buf][3 * NB] != 0.f) { /* values that are not finite, zeros in the image */
                any_odd = 1;
                for (int i = tid; i < KT * dim; i += THREADS) {
                    const int j = k0 + i / dim, d = i % dim;
                    if (j >= it.n) break;
                    const float x = ((const float *)p.v)[(it.start + j) * p.v_stride + (int64_t)kvh * dim + d];
                    if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) atomicMin(&first_odd[d], j);
                }
            }
            if (works) compute(k0);
            buf ^= 1;
            tile = lds + buf * S::TILE;
        }
        lds_barrier();
    } else {
        for (int at = begin; at < end; at += STEP, k0 += STEP) {
            if (WR > 1) lds_barrier(); /* the last tile has been read */
            store(k0);
            if (at + STEP < end) load(next);
            next = place(k0 + 2 * STEP);
            if (WR > 1) lds_barrier();
            else asm volatile("" ::: "memory");
            if (k0 < end && works) compute(k0);
            if (WR == 1) asm volatile("" ::: "memory");
        }
    }
    l = sum_lanes<RW>(l);
    /* A row without weights: zeros if it attends nothing; if all its scores are
     * minus infinity NaN, as 0 / 0 is (of pieces their join says so). */
    const float nothing = pieces == 1 && pos >= 0 ? NAN : 0.f;
    /* O to the sums themselves, together with the factor 1 / l */
    const int back = SCALED ? (int)fminf(fmaxf(rm, -1000.f), 1000.f) - 20 : 0;
    auto scaled = [&](f4_t v, float f) {
        v *= f;
        if (SCALED)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __builtin_ldexpf(v[i], back);
        return v;
    };
    float *const part = p.partials + (int64_t)blockIdx.x * PARTIAL;

    if (WK == 1) {
        /* register 4 j + i of o[db]: element RW db + 8 j + 4 part_of + i of this lane's row */
        const int row_in_tile = wr * RW + col;
        float *to = pieces > 1 ? part + row_in_tile * DP
                               : p.out + (int64_t)(it.start + token) * p.out_stride + (int64_t)head * dim;
        const float by = l == 0.f ? nothing : 1.f / l;
        const int width = pieces > 1 ? DP : dim;
        if (any_odd) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < REGS; ++i)
                    if (pos >= first_odd[RW * db + 8 * (i >> 2) + 4 * part_of + (i & 3)]) o[db][i] = NAN;
        }
        if (!real) return;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int j = 0; j < REGS / 4; ++j) {
                const int d = RW * db + 8 * j + 4 * part_of;
                const f4_t v = {o[db][4 * j], o[db][4 * j + 1], o[db][4 * j + 2], o[db][4 * j + 3]};
                if (d < width) *(f4_t *)(to + d) = scaled(v, by);
            }
        if (pieces > 1 && part_of == 0) {
            const f2_t v = {m, l};
            *(f2_t *)(part + LAYOUT * DP + 2 * row_in_tile) = v;
        }
    } else {
        /* the waves' results meet in LDS */
        if (part_of == 0) {
            joined[wk][0][col] = m;
            joined[wk][1][col] = l;
        }
        lds_barrier(); /* tiles are done with, too */
        float top = joined[0][0][col];
#pragma unroll
        for (int w = 1; w < WK; ++w) top = fmaxf(top, joined[w][0][col]);
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) sum += joined[w][1][col] * __builtin_amdgcn_exp2f(joined[w][0][col] - top);
        float *mine = (float *)lds + wk * RW * DP;
        const float share = sum == 0.f ? nothing : __builtin_amdgcn_exp2f(m - top) / sum;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int j = 0; j < REGS / 4; ++j) {
                const int d4 = RW / 4 * db + 2 * j + part_of;
                const f4_t v = {o[db][4 * j], o[db][4 * j + 1], o[db][4 * j + 2], o[db][4 * j + 3]};
                *(f4_t *)(mine + col * DP + ((d4 ^ (col & 7)) << 2)) = scaled(v, share);
            }
        lds_barrier();
        const int rows = min(it.n * group - it.tile * S::ROWS, S::ROWS);
        for (int e = tid; e < rows * (DP / 4); e += THREADS) {
            const int rr = e / (DP / 4), d4 = e % (DP / 4);
            f4_t v = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < WK; ++w) v += *(const f4_t *)((const float *)lds + w * RW * DP + rr * DP + ((d4 ^ (rr & 7)) << 2));
            const int tile_row = it.tile * S::ROWS + rr, tk = tile_row / group;
            if (any_odd) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (it.first + tk >= first_odd[4 * d4 + i]) v[i] = NAN;
            }
            if (pieces == 1) {
                float *out = p.out + (int64_t)(it.start + tk) * p.out_stride + (int64_t)(kvh * group + tile_row - tk * group) * dim;
                if (4 * d4 < dim) *(f4_t *)(out + 4 * d4) = v;
            } else {
                *(f4_t *)(part + rr * DP + 4 * d4) = v;
                if (d4 == 0) {
                    float all = joined[0][0][rr], sum = 0.f;
#pragma unroll
                    for (int w = 1; w < WK; ++w) all = fmaxf(all, joined[w][0][rr]);
#pragma unroll
                    for (int w = 0; w < WK; ++w) sum += joined[w][1][rr] * __builtin_amdgcn_exp2f(joined[w][0][rr] - all);
                    const f2_t st = {all, sum};
                    *(f2_t *)(part + LAYOUT * DP + 2 * rr) = st;
                }
            }
        }
    }
}

/* From 32 rows on two waves a SIMD, except of fp32 with 128 elements, whose
 * tiles in LDS leave room for one workgroup (of 4 waves at 32 and 128 rows). Spilled,
 * of 128 elements: 23 registers of fp32 at 256 rows, 9 of bf16 and 6 of f16 at 32
 * (with one wave a SIMD none, but 149 us for 4 tokens each over 64 sequences of 4000
 * f16 keys, 112 with two), and 3 into accumulation registers of fp32 at 16 and 128.
 * At 16 and 32 rows the 4 waves have a tile each in their own LDS and need no
 * barrier. */
template <int TYPE, int DP, int RW, int WR, int WK>
__global__ __launch_bounds__(64 * WR * WK, WR == 8 || (RW == 32 && (TYPE != QMV_KV_F32 || DP == 64)) ? 2 : 1)
void attention_kernel(AttnParams p)
{
    using S = AttnShape<TYPE, DP, RW, WR, WK>;
    using Few = AttnShape<TYPE, DP, 16, 1, 4>;
    using Shared = AttnShared<S, DP, RW, WK>;
    using FewShared = AttnShared<Few, DP, 16, 4>;
    constexpr bool MIXED = S::ROWS >= 128 && !S::IMAGE;
    constexpr size_t BYTES = MIXED && sizeof(FewShared) > sizeof(Shared) ? sizeof(FewShared) : sizeof(Shared);
    __shared__ __attribute__((aligned(16))) unsigned char memory[BYTES];

    const AttnTokens &a = p.t;
    const int kvh = blockIdx.x % a.kv_heads, item = blockIdx.x / a.kv_heads;
    AttnItem it;
    int tiles_all;
    const bool found = find_item<S::ROWS, S::KT * WK>(p, item, threadIdx.x & 63, &it, &tiles_all);
    if (blockIdx.x == 0 && p.target && threadIdx.x == 0) p.joins[0].n = tiles_all;
    if (!found) return;
    /* A decoding sequence among longer ones: its one tile as the 16-row kernel
     * takes it (512 tokens and 15 decoding sequences of 8000 keys 106 us without, 71
     * with, 2048 and 8 of 6000 182 and 133; 28 and 4 heads of 128, f16). That has its
     * place in LDS beside the workgroups that run at once. */
    if constexpr (MIXED) {
        if (it.n * (a.heads / a.kv_heads) <= 16) {
            if (threadIdx.x >= 256) return; /* a barrier waits for the waves that are left */
            attend_piece<TYPE, DP, 16, 1, 4, S::ROWS>(p, it, item, kvh, *(FewShared *)memory);
            return;
        }
    }
    attend_piece<TYPE, DP, RW, WR, WK, S::ROWS>(p, it, item, kvh, *(Shared *)memory);
}

/* Joins the pieces of rows whose keys were cut, in their order within each of
 * GROUPS groups of threads and then in the groups' order: each is the average of
 * its values, with its weights' reference and sum, and the join averages those
 * by the sums. A second kernel:
 * joined by the last workgroup of a tile, the 128 pieces of one row tile at
 * 32749 keys took 17 us of one compute unit. */
template <int DP, int ROWS, int GROUPS>
__global__ __launch_bounds__(256) void attention_join_kernel(AttnParams p, int slices)
{
    constexpr int D4 = DP / 4, EACH = 256 / (D4 * GROUPS); /* rows of a workgroup */
    constexpr int AT_ONCE = GROUPS > 1 ? 8 : 16;
    constexpr int PARTIAL = ROWS * DP + 2 * ROWS;
    __shared__ f4_t sums[GROUPS > 1 ? GROUPS : 1][EACH][D4];
    __shared__ f2_t states[GROUPS > 1 ? GROUPS : 1][EACH];
    const AttnTokens &a = p.t;
    const int group = a.heads / a.kv_heads;
    const int slice = blockIdx.x % slices, rest = blockIdx.x / slices, kvh = rest % a.kv_heads, tile_at = rest / a.kv_heads;
    const int tiles = p.joins[0].n;
    const AttnJoin j = p.joins[1 + tile_at]; /* of no meaning past `tiles` */
    if (tile_at >= tiles || j.pieces == 0) return;
    const int d4 = threadIdx.x % D4, set = threadIdx.x / D4 % GROUPS, each = threadIdx.x / (D4 * GROUPS);
    const float *from = p.partials + ((int64_t)j.item * a.kv_heads + kvh) * PARTIAL;
    const int64_t apart = (int64_t)j.apart * a.kv_heads * PARTIAL;
    const int mine = (j.pieces + GROUPS - 1) / GROUPS, i_end = min((set + 1) * mine, j.pieces);
    const int rows = min(ROWS, j.n * group - j.tile * ROWS);
    for (int r0 = slice * EACH; r0 < rows; r0 += slices * EACH) {
        const int rr = r0 + each, row = j.tile * ROWS + rr, token = row / group;
        const bool real = rr < rows;
        float all = kNothing, sum = 0.f;
        f4_t v = {0, 0, 0, 0};
        if (real) {
            /* N pieces, whose loads are in flight together */
            auto take = [&](auto number, int i0) {
                constexpr int N = decltype(number)::value;
                f2_t st[N];
                f4_t x[N];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float *at = from + min(i0 + i, i_end - 1) * apart;
                    st[i] = *(const f2_t *)(at + ROWS * DP + 2 * rr);
                    x[i] = *(const f4_t *)(at + rr * DP + 4 * d4);
                }
                float top = all;
#pragma unroll
                for (int i = 0; i < N; ++i) top = fmaxf(top, st[i][0]);
                const float before = sum * __builtin_amdgcn_exp2f(all - top);
                float g[N];
                all = top;
                sum = before;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    g[i] = i0 + i < i_end ? st[i][1] * __builtin_amdgcn_exp2f(st[i][0] - all) : 0.f;
                    sum += g[i];
                }
                const float by = sum == 0.f ? 0.f : 1.f / sum;
                v *= before * by;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i0 + i < i_end) v += x[i] * (g[i] * by);
            };
            int i0 = set * mine;
            for (; i_end - i0 > 4; i0 += AT_ONCE) take(std::integral_constant<int, AT_ONCE>(), i0);
            if (i0 < i_end) take(std::integral_constant<int, 4>(), i0); /* the usual few without loads for nothing */
        }
        if (GROUPS > 1) {
            sums[set][each][d4] = v;
            if (d4 == 0) states[set][each] = f2_t{all, sum};
            __syncthreads();
            float top = states[0][each][0];
#pragma unroll
            for (int i = 1; i < GROUPS; ++i) top = fmaxf(top, states[i][each][0]);
            float g[GROUPS];
            sum = 0.f;
#pragma unroll
            for (int i = 0; i < GROUPS; ++i) {
                g[i] = states[i][each][1] * __builtin_amdgcn_exp2f(states[i][each][0] - top);
                sum += g[i];
            }
            const float by = sum == 0.f ? 0.f : 1.f / sum;
            v = f4_t{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < GROUPS; ++i) v += sums[i][each][d4] * (g[i] * by);
            __syncthreads();
        }
        if (real && set == 0 && 4 * d4 < a.dim) {
            float *out = p.out + (int64_t)(j.start + token) * p.out_stride + (int64_t)(kvh * group + row - token * group) * a.dim;
            const float nothing = sum == 0.f && j.first + token >= 0 ? NAN : 0.f; /* as in attend_piece; added, as a branch took 1 us more */
            *(f4_t *)(out + 4 * d4) = v + nothing;
        }
    }
}

/* Rows per workgroup, by what was measured (us; 28 and 4 heads of 128, f16
 * cache unless said, 16 / 128 / 256 rows):
 *   16, where no sequence fills more, or where all tiles of 16 are one round of
 *   the 256 compute units and the keys are few enough that reading them for
 *   each tile costs less than the larger tiles' start: prompt of 37 tokens 10.9 /
 *   13.2 / 16.4, of 128 11.5 / 18.4 / 21.7, of 256 28.8 / 25.4 / 28.9; 32 tokens
 *   over 512 15.7 / 19.1 / 22.4, over 4096 32.8 / 28.0 / 30.2.
 *   32, over a cache, where sequences have 17 to 32 rows, a few tokens that are
 *   checked at once: 4 tokens over 4000 keys in 64 sequences 180 / (32 rows) 113 /
 *   (128 rows) 214, over 500 in 256 148 / 88 / 99; of fp32 420 / 242 / 380. Two
 *   tiles of 32 read keys twice: 8 tokens over 16000 in 16 sequences 238, 165 at
 *   128. Prompts of 24 rows do better at 128 (64 of them 21 and 17).
 *   256, one workgroup of 8 waves per compute unit, where a sequence has more
 *   rows than a few tiles: 512 tokens over 4096 in 4 sequences 269 at 128, 253 at
 *   256; 128 tokens in 4 sequences 90 and 104. Keys of fp32 fill LDS and the
 *   registers at 128 already, so that the larger tile shares more sooner: 32
 *   tokens over 4096 in 8 sequences 124 and 88. Heads of up to 64 are half as
 *   much work per key, and two workgroups of 128 hide more: 8 prompts of 2502
 *   tokens, 14 and 2 heads, 38 and 41.
 * The average is over all sequences of the call, idle ones too: a chunk beside
 * many decoding sequences, or in a batch of mostly idle ones, gets the tiles of
 * those, and a long prompt packed with short ones no images.
 * Pieces (target): as many as run at once, two workgroups a compute unit at
 * 32 and 128 rows (of fp32 keys with more than 64 elements only one does, and the
 * pieces are two rounds) and one at 256 (prompts of 2048, 7B: 134 with 256 pieces, 152
 * with 512); of 16 rows twice that, because sequences that decode differ in length
 * most (64 of 1 to 8191 keys: 110 with 1024, 123 with 512), except over fp32,
 * whose tiles leave room for one workgroup. Also twice over a cache where tiles
 * of 128 or 256 alone are more than half of them, unless lengths and new tokens are alike
 * (which the device sees): 512 tokens and 63 decoding sequences of 4000 keys 170 and 223, 6
 * tokens each over 10 to 6310 keys in 64 sequences 150 and 206, 1024 tokens
 * and 40 of 1 to 7801 keys of fp32 299 and 380, but 64 tokens each over 1000 in 16
 * sequences 75 and 64.
 * Images: 5 us for their kernel, against splitting a key once per row tile: 1024
 * tokens per prompt are 28 tiles (7B), where both take the same time. */
AttnPlan plan_attention(const AttnTokens &t, int type)
{
    constexpr int64_t kUnits = 256;
    AttnPlan plan = {};
    const int64_t heads = t.kv_heads, group = t.heads / t.kv_heads, busy = t.count < t.tokens ? t.count : t.tokens;
    const int64_t rows = t.tokens * group, each = rows / t.count;
    const int64_t room = t.page_size ? (int64_t)t.table_stride * t.page_size : t.tokens; /* keys at most */
    const int64_t small = (rows / 16 + busy) * heads;
    if (each <= 16 || (small <= kUnits && small * room <= kUnits * 512)) plan.rows = 16;
    else if (each <= 32 && t.page_size) plan.rows = 32;
    else if (each <= (t.dim <= 64 ? 4096 : type == QMV_KV_F32 ? 128 : 1024)) plan.rows = 128;
    else plan.rows = 256;
    const int64_t tiles = rows / plan.rows + busy;
    plan.tiles = (int)tiles;

    plan.target = (int)(plan.rows == 256 ? kUnits : plan.rows != 16 || type == QMV_KV_F32 ? 2 * kUnits : 4 * kUnits);
    plan.alike = plan.target;
    if (plan.rows >= 128 && t.page_size && 2 * tiles * heads > plan.target) plan.target *= 2;
    plan.slots = plan.rows <= 32 && t.page_size && type != QMV_KV_F32 ? (int)(2 * kUnits) : 0;
    plan.least = plan.rows <= 32 && type != QMV_KV_F32 ? 256 : 128; /* keys, 64 KB of 128 elements */
    /* None where the tiles are enough (a cache's sequences may still differ in
     * length), or where no sequence can have more than one. */
    if (tiles * heads >= (t.page_size ? 16 * kUnits : plan.target) || room <= plan.least) plan.target = 0;

    /* find_item's chunks cut all of the lengths' sum (of prompts, which attend
     * half: half of it) into max(pieces - tiles, pieces / 2), and each tile has a
     * last piece. Workgroups that find none cost their start, with the LDS of the
     * others: 8 us of 21 where there were twice as many. */
    const int64_t pieces = plan.target / heads;
    const int64_t items = plan.target == 0   ? tiles
                          : t.page_size == 0 ? max(2 * pieces, pieces + tiles) + 1
                                             : max(pieces, pieces / 2 + tiles) + 1;
    plan.grid = items * heads;
    plan.items = (int)items;
    /* A list where every workgroup would read more than 256 sequences' lengths: 512
     * of 1000 keys 243 us without, 2048 of 500 854. */
    if (t.count > 256) plan.lists = sizeof(AttnLists) + (size_t)t.count * sizeof(int2) + (size_t)items * sizeof(int) + 16;
    const int dp = t.dim <= 64 ? 64 : 128;
    if (plan.target) {
        plan.joins = (1 + (size_t)tiles) * sizeof(AttnJoin);
        plan.partials = (size_t)plan.grid * (plan.rows * (dp + 2));
    }
    if (plan.rows == 256 && t.page_size == 0 && t.tokens / t.count >= 1024) {
        plan.images = ((int64_t)t.tokens / kImageKeys + t.count) * heads;
        plan.image_bytes = (size_t)(plan.images * image_bytes(dp));
    }
    return plan;
}

template <int DP, int ROWS, int GROUPS> static hipError_t launch_join(const AttnParams &p, const AttnPlan &plan, hipStream_t s)
{
    constexpr int EACH = 256 / (DP / 4 * GROUPS); /* rows of a workgroup */
    /* workgroups of a tile for the rows that a sequence has on average */
    const int64_t each = ((int64_t)p.t.tokens * (p.t.heads / p.t.kv_heads) + p.t.count - 1) / p.t.count;
    const int slices = (int)(((each < ROWS ? each : ROWS) + EACH - 1) / EACH);
    const unsigned grid = (unsigned)(plan.tiles * p.t.kv_heads * slices);
    attention_join_kernel<DP, ROWS, GROUPS><<<dim3(grid), 256, 0, s>>>(p, slices);
    return hipGetLastError();
}

/* Each kernel reads what the one before it wrote, and is launched only after it
 * has been. */
template <int TYPE, int DP, int RW, int WR, int WK> static hipError_t launch_shape(const AttnParams &p, const AttnPlan &plan, hipStream_t s)
{
    using S = AttnShape<TYPE, DP, RW, WR, WK>;
    if (plan.lists) {
        attention_list_kernel<S::ROWS, S::KT * WK><<<1, 1024, 0, s>>>(p);
        if (const hipError_t e = hipGetLastError()) return e;
    }
    attention_kernel<TYPE, DP, RW, WR, WK><<<dim3((unsigned)plan.grid), 64 * WR * WK, 0, s>>>(p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || plan.target == 0) return e;
    /* Groups of threads where a tile has many pieces (the tiles counted here are an
     * upper bound): 4 tokens over 32000 keys 31 us, 48 with one group; 64 sequences
     * of 1000 keys 34 with groups, 32 with one. */
    if (plan.target >= 8 * plan.tiles * p.t.kv_heads) return launch_join<DP, S::ROWS, 8>(p, plan, s);
    return launch_join<DP, S::ROWS, 1>(p, plan, s);
}

template <int TYPE, int DP> static hipError_t launch_rows(const AttnParams &p, const AttnPlan &plan, hipStream_t s)
{
    if (plan.rows == 16) return launch_shape<TYPE, DP, 16, 1, 4>(p, plan, s);
    if (plan.rows == 32) return launch_shape<TYPE, DP, 32, 1, 4>(p, plan, s);
    if (plan.rows == 128) return launch_shape<TYPE, DP, 32, 4, 1>(p, plan, s);
    return launch_shape<TYPE, DP, 32, 8, 1>(p, plan, s);
}

/* A prompt's rows of fp32, through images of their tiles. */
template <int DP> static hipError_t launch_images(const AttnParams &p, const AttnPlan &plan, hipStream_t s)
{
    attention_image_kernel<DP><<<dim3((unsigned)plan.images), 256, 0, s>>>(p);
    if (const hipError_t e = hipGetLastError()) return e;
    return launch_shape<QMV_KV_IMAGE, DP, 32, 8, 1>(p, plan, s);
}

template <int TYPE> static hipError_t launch_dim(const AttnParams &p, const AttnPlan &plan, hipStream_t s)
{
    return p.t.dim <= 64 ? launch_rows<TYPE, 64>(p, plan, s) : launch_rows<TYPE, 128>(p, plan, s);
}

hipError_t launch_attention(const AttnParams &p, const AttnPlan &plan, int type, hipStream_t s)
{
    if (plan.images) return p.t.dim <= 64 ? launch_images<64>(p, plan, s) : launch_images<128>(p, plan, s);
    if (type == QMV_KV_F32) return launch_dim<QMV_KV_F32>(p, plan, s);
    return type == QMV_KV_F16 ? launch_dim<QMV_KV_F16>(p, plan, s) : launch_dim<QMV_KV_BF16>(p, plan, s);
}

/* A workgroup per token: the pairs' sines once in LDS, then all heads. Bound by
 * memory on prompts (4096 tokens, 28 and 4 heads of 128, bf16 cache: 151 MB in 27
 * us, 5.6 TB/s), by the launch on decode steps (3 us alone, 7 for 64 tokens).
 * The angle p * freq is a product in 64 bits, brought
 * to [-pi, pi] there: at position 10^6 an fp32 angle is off by up to 0.03.
 * What is left is rounded to fp32 once (2^-24 relative, so at most 2^-22.3
 * absolute) before the sine. */
template <int TYPE> __global__ __launch_bounds__(256) void rope_kernel(RopeParams p)
{
    __shared__ float cs[64], sn[64];
    const AttnTokens &a = p.t;
    const int t = blockIdx.x, half = p.rotary / 2, dim = a.dim;
    const int s = sequence_of(a, t);
    if (s < 0) return;
    const int start = max(a.starts[s], 0), n = min(a.starts[s + 1], a.tokens) - start; /* start <= t < tokens */
    const int pos = (a.lengths ? a.lengths[s] - n : 0) + t - start;
    for (int i = threadIdx.x; i < half; i += 256) {
        const double angle = (double)pos * p.freq[i];
        const double turns = rint(angle * 0.15915494309189535);
        const double rest = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586, angle));
        sincosf((float)rest, &sn[i], &cs[i]);
    }
    __syncthreads();
    int64_t at = -1;
    if (a.page_size && pos >= 0) {
        at = key_at(a, s, pos, 0);
        if (at < 0 && a.status && threadIdx.x == 0) *a.status = 0;
    }
    /* element pairs: (i, i + half) or (2 i, 2 i + 1), then what is not turned */
    const int pairs = dim / 2, rows = a.heads + a.kv_heads;
    for (int w = threadIdx.x; w < rows * pairs; w += 256) {
        const int h = w / pairs, i = w % pairs;
        const bool key = h >= a.heads;
        const int head = key ? h - a.heads : h;
        const int e0 = i >= half ? 2 * i : p.interleaved ? 2 * i : i;
        const int e1 = i >= half ? 2 * i + 1 : p.interleaved ? 2 * i + 1 : i + half;
        const float *in = (key ? p.k + (int64_t)t * p.k_stride : p.q + (int64_t)t * p.q_stride) + (int64_t)head * dim;
        const float x = in[e0], y = in[e1];
        const float c = i < half ? cs[i] : 1.f, z = i < half ? sn[i] : 0.f;
        const float u = i < half ? x * c - y * z : x, v = i < half ? x * z + y * c : y;
        float *out = key ? p.k_out : p.q_out;
        if (out) {
            out += (int64_t)t * (key ? p.k_stride : p.q_stride) + (int64_t)head * dim;
            out[e0] = u;
            out[e1] = v;
        }
        if (key && at >= 0) {
            const int64_t to = at + (int64_t)head * a.head_stride;
            store_kv<TYPE>(p.keys, to + e0, u);
            store_kv<TYPE>(p.keys, to + e1, v);
        }
    }
    if (at < 0) return;
    for (int w = threadIdx.x; w < a.kv_heads * dim; w += 256) {
        const int head = w / dim, e = w % dim;
        store_kv<TYPE>(p.values, at + (int64_t)head * a.head_stride + e, p.v[(int64_t)t * p.v_stride + w]);
    }
}

hipError_t launch_rope(const RopeParams &p, int type, hipStream_t s)
{
    const dim3 grid((unsigned)p.t.tokens);
    if (type == QMV_KV_F32) rope_kernel<QMV_KV_F32><<<grid, 256, 0, s>>>(p);
    else if (type == QMV_KV_F16) rope_kernel<QMV_KV_F16><<<grid, 256, 0, s>>>(p);
    else rope_kernel<QMV_KV_BF16><<<grid, 256, 0, s>>>(p);
    return hipGetLastError();
}

} // namespace qmv
