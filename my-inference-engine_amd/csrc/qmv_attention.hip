/*
 * gfx950 kernels between the q/k/v projections and the output projection:
 * rotary embedding with the write into a paged cache, and causal attention
 * over packed prompts and over a paged cache.
 */
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qmv_kernels.h"

namespace qmv {

typedef float f4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float from_bf16(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }

/* Nearest, ties to even; NaN stays NaN. */
__device__ __forceinline__ uint16_t to_bf16(float v)
{
    const uint32_t u = __float_as_uint(v);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)(u >> 16 | 0x40u);
    return (uint16_t)((u + 0x7fffu + (u >> 16 & 1u)) >> 16);
}

template <int TYPE> __device__ __forceinline__ float load_kv(const void *base, int64_t i)
{
    if (TYPE == QMV_KV_F32) return ((const float *)base)[i];
    if (TYPE == QMV_KV_F16) return (float)((const _Float16 *)base)[i];
    return from_bf16(((const uint16_t *)base)[i]);
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

/* Where key `j` of sequence s (its first token is `start`) and of head h
 * begins, -1 if its page is outside the cache or the table. */
__device__ __forceinline__ int64_t key_at(const AttnTokens &a, int s, int start, int j, int h)
{
    if (a.page_size == 0) return (int64_t)(start + j) * a.token_stride + (int64_t)h * a.head_stride;
    const int page = j / a.page_size;
    if (page >= a.table_stride) return -1;
    const int at = a.table[(int64_t)s * a.table_stride + page];
    if (at < 0 || at >= a.pages) return -1;
    return (int64_t)at * a.page_stride + (int64_t)h * a.head_stride + (int64_t)(j - page * a.page_size) * a.token_stride;
}

/* A wave per token and head: lanes over keys for the scores, over the head's
 * elements for the values; the running maximum and sum of the softmax. */
template <int TYPE> __global__ __launch_bounds__(256) void attention_kernel(AttnParams p)
{
    const AttnTokens &a = p.t;
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (item >= (int64_t)a.tokens * a.heads) return;
    const int t = (int)(item / a.heads), head = (int)(item % a.heads), kvh = head / (a.heads / a.kv_heads);
    const int s = sequence_of(a, t);
    if (s < 0) return;
    const int start = a.starts[s], n = min(a.starts[s + 1], a.tokens) - start;
    const int pos = (a.lengths ? a.lengths[s] - n : 0) + t - start;
    const float *q = p.q + (int64_t)t * p.q_stride + (int64_t)head * a.dim;
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int j0 = 0; j0 <= pos; j0 += 64) {
        const int j = j0 + lane;
        const int64_t at = j <= pos ? key_at(a, s, start, j, kvh) : 0;
        if (at < 0 && a.status) *a.status = 0;
        float score = 0.f;
        if (j <= pos && at >= 0)
            for (int d = 0; d < a.dim; ++d) score = fmaf(q[d], load_kv<TYPE>(p.k, at + d), score);
        score = j > pos ? -INFINITY : at < 0 ? NAN : score * p.scale;
        float top = score;
        bool nan = score != score;
        for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
        top = __any(nan) ? NAN : fmaxf(m, top);
        const float fade = m == -INFINITY ? 0.f : __expf(m - top);
        float w = j > pos ? 0.f : __expf(score - top);
        m = top;
        l *= fade;
        o0 *= fade;
        o1 *= fade;
        const int keys = pos - j0 < 63 ? pos - j0 + 1 : 64;
        for (int i = 0; i < keys; ++i) {
            const float wi = __shfl(w, i);
            const int64_t ai = __shfl(at, i);
            l += wi;
            if (ai < 0) continue;
            if (lane < a.dim) o0 = fmaf(wi, load_kv<TYPE>(p.v, ai + lane), o0);
            if (lane + 64 < a.dim) o1 = fmaf(wi, load_kv<TYPE>(p.v, ai + lane + 64), o1);
        }
    }
    float *out = p.out + (int64_t)t * p.out_stride + (int64_t)head * a.dim;
    if (lane < a.dim) out[lane] = pos < 0 ? 0.f : o0 / l;
    if (lane + 64 < a.dim) out[lane + 64] = pos < 0 ? 0.f : o1 / l;
}

hipError_t launch_attention(const AttnParams &p, int type, hipStream_t s)
{
    const int64_t items = (int64_t)p.t.tokens * p.t.heads;
    const dim3 grid((unsigned)((items + 3) / 4));
    if (type == QMV_KV_F32) attention_kernel<QMV_KV_F32><<<grid, 256, 0, s>>>(p);
    else if (type == QMV_KV_F16) attention_kernel<QMV_KV_F16><<<grid, 256, 0, s>>>(p);
    else attention_kernel<QMV_KV_BF16><<<grid, 256, 0, s>>>(p);
    return hipGetLastError();
}

/* A workgroup per token. The angle p * freq is a product in 64 bits, brought
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
    const int start = a.starts[s], n = min(a.starts[s + 1], a.tokens) - start;
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
        at = key_at(a, s, start, pos, 0);
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
