/*
 * Host side of the attention entry points of include/qmv_hip.h: every rule for
 * arguments runs before any HIP call, so an invalid call returns 0 without
 * touching the GPU.
 */
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <exception>
#include <mutex>
#include <numeric>

#include "qmv_hip.h"
#include "qmv_kernels.h"
#include "qmv_shim.h"

#define QMV_API extern "C" __attribute__((visibility("default")))

namespace {

using qmv::overlap;
using qmv::set_error;

/* Bytes of `rows` rows of `width` floats that are `stride` apart. */
size_t rows_bytes(int rows, int64_t stride, int64_t width)
{
    return ((size_t)(rows - 1) * (size_t)stride + (size_t)width) * sizeof(float);
}

/* Whether `rows` rows of wa floats, sa apart, and of wb floats, sb apart, share
 * any: two rows lie the difference of the first ones and a multiple of the
 * strides' common divisor apart. (Of unlike strides rows may be said to meet that
 * are too few to.) */
bool rows_meet(const float *a, int64_t sa, int64_t wa, const float *b, int64_t sb, int64_t wb, int rows)
{
    if (!overlap(a, rows_bytes(rows, sa, wa), b, rows_bytes(rows, sb, wb))) return false;
    const int64_t g = std::gcd(sa, sb), apart = ((int64_t)((uintptr_t)b - (uintptr_t)a) / 4 % g + g) % g;
    return apart < wa || apart + wb > g;
}

bool aligned16(const void *p)
{
    return ((uintptr_t)p & 15) == 0;
}

/* A row stride in floats (0: the heads alone) of `heads` heads, and the
 * pointer it belongs to. Strides end at 2^31, so that no offset of the at most
 * 2^22 tokens overflows. */
bool row_stride_ok(const void *ptr, int64_t *stride, int heads, int dim, const char *what)
{
    const int64_t width = (int64_t)heads * dim;
    if (*stride == 0) *stride = width;
    if (ptr == nullptr || !aligned16(ptr) || *stride < width || *stride % 4 != 0 || *stride > INT_MAX) {
        set_error("%s: a null or unaligned pointer, or a stride that is no multiple of 4 or below the row", what);
        return false;
    }
    return true;
}

constexpr int kMaxTokens = 1 << 22;

bool heads_ok(int tokens, int q_heads, int kv_heads, int head_dim)
{
    if (tokens <= 0 || tokens > kMaxTokens || q_heads <= 0 || kv_heads <= 0 || q_heads > 65535 ||
        q_heads % kv_heads != 0) {
        set_error("invalid token or head counts (%d tokens, %d and %d heads)", tokens, q_heads, kv_heads);
        return false;
    }
    if ((int64_t)tokens * q_heads > 1 << 30) {
        set_error("more than 2^30 rows of tokens and heads");
        return false;
    }
    if (head_dim < 8 || head_dim > 128 || head_dim % 8 != 0) {
        set_error("head_dim must be a multiple of 8 from 8 to 128 (got %d)", head_dim);
        return false;
    }
    return true;
}

/* Arrays of ints at addresses of ints: scalar loads drop the bits below. */
bool aligned4(const void *p)
{
    return ((uintptr_t)p & 3) == 0;
}

bool sequences_ok(const QmvSequences *q, bool paged, const int *status)
{
    if (q == nullptr || q->starts == nullptr || q->count <= 0 || q->count > 65535) {
        set_error("invalid sequences (null, or not 1 to 65535 of them)");
        return false;
    }
    if (paged && (q->lengths == nullptr || q->pages == nullptr || q->table_stride <= 0)) {
        set_error("sequences over a cache need lengths and pages");
        return false;
    }
    if (!aligned4(q->starts) || !aligned4(q->lengths) || (paged && !aligned4(q->pages)) || !aligned4(status)) {
        set_error("unaligned sequences or status");
        return false;
    }
    return true;
}

bool cache_ok(const QmvPagedCache *c, const QmvSequences *q, int *type)
{
    if (c == nullptr || c->keys == nullptr || c->values == nullptr || !aligned16(c->keys) || !aligned16(c->values)) {
        set_error("null or unaligned cache");
        return false;
    }
    if (c->type != QMV_TYPE_F32 && c->type != QMV_TYPE_F16 && c->type != QMV_TYPE_BF16) {
        set_error("unsupported cache type %u (need F32, F16 or BF16)", c->type);
        return false;
    }
    if (c->kv_heads <= 0 || c->kv_heads > 65535 || c->head_dim < 8 || c->head_dim > 128 || c->head_dim % 8 != 0) {
        set_error("invalid heads of the cache (%d of %d)", c->kv_heads, c->head_dim);
        return false;
    }
    if (c->pages <= 0 || c->page_size <= 0 || (int64_t)q->table_stride * c->page_size > 1 << 30) {
        set_error("invalid pages (%d of %d tokens, %d per sequence)", c->pages, c->page_size, q->table_stride);
        return false;
    }
    const int64_t strides[3] = {c->page_stride, c->head_stride, c->token_stride};
    const int64_t counts[3] = {c->pages, c->kv_heads, c->page_size};
    int64_t room = INT64_MAX / 8; /* elements: bytes then fit too */
    for (int i = 0; i < 3; ++i) {
        if (strides[i] < c->head_dim || strides[i] % 8 != 0 || strides[i] > room / counts[i]) {
            set_error("cache strides must be multiples of 8, at least head_dim, and in range");
            return false;
        }
        room -= strides[i] * counts[i];
    }
    *type = c->type == QMV_TYPE_F32 ? QMV_KV_F32 : c->type == QMV_TYPE_F16 ? QMV_KV_F16 : QMV_KV_BF16;
    return true;
}

/* Bytes from the first to the last element of a cache's keys or values. */
size_t cache_bytes(const QmvPagedCache &c)
{
    const int64_t last = (c.pages - 1) * c.page_stride + (c.kv_heads - 1) * c.head_stride +
                         (int64_t)(c.page_size - 1) * c.token_stride + c.head_dim;
    return (size_t)last * (c.type == QMV_TYPE_F32 ? 4 : 2);
}

qmv::AttnTokens attn_tokens(const QmvSequences &q, int tokens, int heads, int kv_heads, int dim,
                            const QmvPagedCache *c, int *status)
{
    qmv::AttnTokens t = {};
    t.starts = q.starts;
    t.lengths = q.lengths;
    t.table = q.pages;
    t.count = q.count;
    t.table_stride = q.table_stride;
    t.tokens = tokens;
    t.heads = heads;
    t.kv_heads = kv_heads;
    t.dim = dim;
    t.status = status;
    if (c != nullptr) {
        t.page_size = c->page_size;
        t.pages = c->pages;
        t.page_stride = c->page_stride;
        t.head_stride = c->head_stride;
        t.token_stride = c->token_stride;
    }
    return t;
}

int attend(qmv::AttnParams &p, int type, hipStream_t stream)
try {
    const qmv::AttnPlan plan = qmv::plan_attention(p.t, type);
    /* a launch has less than 2^32 threads */
    if (plan.grid * qmv::attention_threads(plan) > UINT32_MAX || plan.images * 256 > UINT32_MAX) {
        set_error("too many tokens, sequences and heads for one call");
        return 0;
    }
    const int device = qmv::shim_device();
    HIP_TRY(hipSetDevice(device));
    unsigned char *at = nullptr;
    std::unique_lock<std::mutex> lock; /* until the launches are made */
    const size_t partial_bytes = plan.partials * sizeof(float), joins = (plan.joins + 15) / 16 * 16;
    const size_t counts = (size_t)p.t.count * sizeof(int2);
    if (!qmv::shim_scratch(device, stream, plan.image_bytes + partial_bytes + joins + plan.lists, &at, &lock)) return 0;
    p.target = plan.target;
    p.alike = plan.alike;
    p.least = plan.least;
    p.slots = plan.slots;
    p.image = at;
    p.partials = (float *)(at += plan.image_bytes);
    p.joins = (qmv::AttnJoin *)(at += partial_bytes);
    at += joins;
    if (plan.lists) { /* the head takes 16 bytes */
        p.lists = (qmv::AttnLists *)at;
        p.before = (int2 *)(at + 16);
        p.sequence_of_item = (int *)(at + 16 + counts);
        p.most_items = plan.items;
    }
    HIP_TRY(qmv::launch_attention(p, plan, type, stream));
    return 1;
} catch (const std::exception &e) { /* out of host memory */
    set_error("%s", e.what());
    return 0;
}

} // namespace

QMV_API int qmv_device_rope_append_f32(const float *d_q, int64_t q_stride, int q_heads, const float *d_k,
                                       int64_t k_stride, const float *d_v, int64_t v_stride, int kv_heads,
                                       int head_dim, int tokens, const double *d_frequencies, int rotary_dims,
                                       int interleaved, const QmvSequences *sequences, float *d_q_out, float *d_k_out,
                                       const QmvPagedCache *cache, int *d_status, void *stream)
{
    int type = QMV_KV_F32;
    if (!heads_ok(tokens, q_heads, kv_heads, head_dim) || !sequences_ok(sequences, cache != nullptr, d_status)) return 0;
    if (!row_stride_ok(d_q, &q_stride, q_heads, head_dim, "q") ||
        !row_stride_ok(d_k, &k_stride, kv_heads, head_dim, "k") ||
        (cache != nullptr && !row_stride_ok(d_v, &v_stride, kv_heads, head_dim, "v")))
        return 0;
    if (rotary_dims < 0 || rotary_dims > head_dim || rotary_dims % 8 != 0 ||
        (rotary_dims > 0 && (d_frequencies == nullptr || ((uintptr_t)d_frequencies & 7) != 0))) {
        set_error("rotary_dims must be a multiple of 8 up to head_dim, with frequencies");
        return 0;
    }
    if (d_q_out == nullptr || !aligned16(d_q_out) || !aligned16(d_k_out) ||
        (d_k_out == nullptr && cache == nullptr)) {
        set_error("null or unaligned rotary outputs");
        return 0;
    }
    if (cache != nullptr) {
        if (!cache_ok(cache, sequences, &type)) return 0;
        if (cache->kv_heads != kv_heads || cache->head_dim != head_dim) {
            set_error("the cache has other heads (%d of %d) than the keys (%d of %d)", cache->kv_heads,
                      cache->head_dim, kv_heads, head_dim);
            return 0;
        }
    }
    /* Heads of rows may lie between those of others (one buffer for q, k and
     * v), and an output may be its own input; otherwise no rows share floats. */
    const int64_t qw = (int64_t)q_heads * head_dim, kw = (int64_t)kv_heads * head_dim;
    const size_t qb = rows_bytes(tokens, q_stride, qw), kb = rows_bytes(tokens, k_stride, kw);
    const size_t vb = cache != nullptr ? rows_bytes(tokens, v_stride, kw) : 0;
    const auto meets_v = [&](const float *out, int64_t stride, int64_t width) {
        return cache != nullptr && rows_meet(out, stride, width, d_v, v_stride, kw, tokens);
    };
    if ((d_q_out != d_q && rows_meet(d_q_out, q_stride, qw, d_q, q_stride, qw, tokens)) ||
        rows_meet(d_q_out, q_stride, qw, d_k, k_stride, kw, tokens) || meets_v(d_q_out, q_stride, qw) ||
        (d_k_out != nullptr &&
         ((d_k_out != d_k && rows_meet(d_k_out, k_stride, kw, d_k, k_stride, kw, tokens)) ||
          rows_meet(d_k_out, k_stride, kw, d_q, q_stride, qw, tokens) || meets_v(d_k_out, k_stride, kw) ||
          rows_meet(d_q_out, q_stride, qw, d_k_out, k_stride, kw, tokens)))) {
        set_error("a rotary output overlaps rows other than its own input's");
        return 0;
    }
    if (cache != nullptr) {
        const size_t cb = cache_bytes(*cache);
        if (cache->keys == cache->values) {
            set_error("keys and values would be stored in one place");
            return 0;
        }
        for (const void *c : {cache->keys, cache->values})
            if (overlap(c, cb, d_q_out, qb) || overlap(c, cb, d_q, qb) || overlap(c, cb, d_k, kb) ||
                overlap(c, cb, d_v, vb) || (d_k_out != nullptr && overlap(c, cb, d_k_out, kb))) {
                set_error("the cache overlaps q, k, v or an output");
                return 0;
            }
    }
    HIP_TRY(hipSetDevice(qmv::shim_device()));
    qmv::RopeParams p = {};
    p.t = attn_tokens(*sequences, tokens, q_heads, kv_heads, head_dim, cache, d_status);
    p.q = d_q;
    p.k = d_k;
    p.v = d_v;
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.freq = d_frequencies;
    p.rotary = rotary_dims;
    p.interleaved = interleaved != 0;
    p.q_out = d_q_out;
    p.k_out = d_k_out;
    p.keys = cache != nullptr ? cache->keys : nullptr;
    p.values = cache != nullptr ? cache->values : nullptr;
    HIP_TRY(qmv::launch_rope(p, type, (hipStream_t)stream));
    return 1;
}

QMV_API int qmv_device_attention_prompt_f32(const float *d_q, int64_t q_stride, const float *d_k, int64_t k_stride,
                                            const float *d_v, int64_t v_stride, int tokens, int q_heads,
                                            int kv_heads, int head_dim, float scale, const QmvSequences *sequences,
                                            float *d_out, int64_t out_stride, void *stream)
{
    if (!heads_ok(tokens, q_heads, kv_heads, head_dim) || !sequences_ok(sequences, false, nullptr)) return 0;
    if (!row_stride_ok(d_q, &q_stride, q_heads, head_dim, "q") ||
        !row_stride_ok(d_k, &k_stride, kv_heads, head_dim, "k") ||
        !row_stride_ok(d_v, &v_stride, kv_heads, head_dim, "v") ||
        !row_stride_ok(d_out, &out_stride, q_heads, head_dim, "out"))
        return 0;
    if (!(std::fabs(scale) <= 1e38f)) { /* times log2(e) it has to be finite as well */
        set_error("scale must be finite and at most 1e38");
        return 0;
    }
    const size_t ob = rows_bytes(tokens, out_stride, (int64_t)q_heads * head_dim);
    if (overlap(d_out, ob, d_q, rows_bytes(tokens, q_stride, (int64_t)q_heads * head_dim)) ||
        overlap(d_out, ob, d_k, rows_bytes(tokens, k_stride, (int64_t)kv_heads * head_dim)) ||
        overlap(d_out, ob, d_v, rows_bytes(tokens, v_stride, (int64_t)kv_heads * head_dim))) {
        set_error("the attention output overlaps an input");
        return 0;
    }
    qmv::AttnParams p = {};
    p.t = attn_tokens(*sequences, tokens, q_heads, kv_heads, head_dim, nullptr, nullptr);
    p.t.lengths = nullptr;
    p.t.table = nullptr;
    p.q = d_q;
    p.k = d_k;
    p.v = d_v;
    p.out = d_out;
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.out_stride = out_stride;
    p.scale = scale;
    return attend(p, QMV_KV_F32, (hipStream_t)stream);
}

QMV_API int qmv_device_attention_paged_f32(const float *d_q, int64_t q_stride, int tokens, int q_heads, float scale,
                                           const QmvSequences *sequences, const QmvPagedCache *cache, float *d_out,
                                           int64_t out_stride, int *d_status, void *stream)
{
    int type = QMV_KV_F32;
    if (cache == nullptr) {
        set_error("null or unaligned cache");
        return 0;
    }
    const int kv_heads = cache->kv_heads, head_dim = cache->head_dim;
    if (!heads_ok(tokens, q_heads, kv_heads, head_dim) || !sequences_ok(sequences, true, d_status) ||
        !cache_ok(cache, sequences, &type))
        return 0;
    if (!row_stride_ok(d_q, &q_stride, q_heads, head_dim, "q") ||
        !row_stride_ok(d_out, &out_stride, q_heads, head_dim, "out"))
        return 0;
    if (!(std::fabs(scale) <= 1e38f)) { /* times log2(e) it has to be finite as well */
        set_error("scale must be finite and at most 1e38");
        return 0;
    }
    const size_t ob = rows_bytes(tokens, out_stride, (int64_t)q_heads * head_dim), cb = cache_bytes(*cache);
    if (overlap(d_out, ob, d_q, rows_bytes(tokens, q_stride, (int64_t)q_heads * head_dim)) ||
        overlap(d_out, ob, cache->keys, cb) || overlap(d_out, ob, cache->values, cb)) {
        set_error("the attention output overlaps q or the cache");
        return 0;
    }
    qmv::AttnParams p = {};
    p.t = attn_tokens(*sequences, tokens, q_heads, kv_heads, head_dim, cache, d_status);
    p.q = d_q;
    p.k = cache->keys;
    p.v = cache->values;
    p.out = d_out;
    p.q_stride = q_stride;
    p.out_stride = out_stride;
    p.scale = scale;
    return attend(p, type, (hipStream_t)stream);
}
