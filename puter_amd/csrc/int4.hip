// Attention over a paged cache held in 4 bits: one or a few query tokens per sequence, grouped
// heads (the reference gathers the pages and runs MultiHeadAttention: execution/page_intrinsic.go:
// 217-352, device/cpu/attention/typed_compute.go:142-237).  A cached value is scale * n + offset
// with the 4-bit code n in [-8, 7] and the (scale, offset) pair of its token, kv head and group of
// dims.  Query i of a sequence of `context` cached tokens and m queries sees the tokens up to
// context - m + i.
#include "common.hpp"

#include <algorithm>

namespace puter {

struct Int4Args {
    const uint16_t *q;
    const uint8_t *kp, *vp;
    const uint32_t *kpar, *vpar;
    const int32_t *table, *ctx;
    uint16_t *out;
    int64_t batch, max_pages, page_size, num_pages, max_context;
    int query_len, heads, kv_heads, dim, group;
    float scale;
};

__device__ __forceinline__ float int4_value(uint32_t w, int k, uint32_t pair) {
    const float s = (float)__builtin_bit_cast(_Float16, (uint16_t)(pair & 0xFFFFu));
    const float o = (float)__builtin_bit_cast(_Float16, (uint16_t)(pair >> 16));
    return (float)((int32_t)(w << (28 - 4 * k)) >> 28) * s + o;
}

// A wave per query token and head: lanes take 64 tokens at a time, then the head dims.
template <int DT>
__global__ __launch_bounds__(64) void int4_row_kernel(Int4Args a) {
    __shared__ float qrow[256];
    __shared__ float pk[64];
    __shared__ int64_t rows[64];
    const int lane = threadIdx.x, h = blockIdx.x % a.heads, qi = blockIdx.x / a.heads;
    const int64_t b = blockIdx.y;
    const int kvh = h / (a.heads / a.kv_heads), D = a.dim;
    const int64_t at = ((b * a.query_len + qi) * a.heads + h) * D;
    for (int d = lane; d < D; d += 64) qrow[d] = Elem<DT>::load(a.q[at + d]);
    __syncthreads();
    const int64_t ctx = min((int64_t)a.ctx[b], a.max_context);
    const int64_t hi = ctx - a.query_len + qi + 1;
    float m = -INFINITY, l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t c0 = 0; c0 < hi; c0 += 64) {
        const int64_t tok = c0 + lane;
        float s = -INFINITY;
        int64_t row = -1;   // (pool row, kv head); -1: hidden, past the context or a bad page id
        if (tok < hi) {
            const int32_t page = a.table[b * a.max_pages + tok / a.page_size];
            if (page >= 0 && page < a.num_pages) row = (page * a.page_size + tok % a.page_size) * a.kv_heads + kvh;
        }
        if (row >= 0) {
            float dot = 0.0f;
            for (int u = 0; u < D / 8; ++u) {
                const uint32_t w = reinterpret_cast<const uint32_t *>(a.kp)[row * (D / 8) + u];
                const uint32_t pair = a.kpar[row * (D / a.group) + 8 * u / a.group];
                for (int k = 0; k < 8; ++k) dot += qrow[8 * u + k] * int4_value(w, k, pair);
            }
            s = dot * a.scale;
        }
        const float mn = fmaxf(m, wave_max(s));
        const float mref = mn == -INFINITY ? 0.0f : mn;
        const float p = row >= 0 ? expf(s - mref) : 0.0f;
        const float alpha = m == -INFINITY ? 0.0f : expf(m - mref);
        l = l * alpha + wave_sum(p);
        m = mn;
        __syncthreads();
        pk[lane] = p;
        rows[lane] = row;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = lane + 64 * j;
            if (d >= D) break;
            float t = 0.0f;
            for (int i = 0; i < 64; ++i) {
                const int64_t r = rows[i];
                if (r < 0) continue;
                const uint32_t w = reinterpret_cast<const uint32_t *>(a.vp)[r * (D / 8) + d / 8];
                t += pk[i] * int4_value(w, d & 7, a.vpar[r * (D / a.group) + d / a.group]);
            }
            acc[j] = acc[j] * alpha + t;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (lane + 64 * j < D) a.out[at + lane + 64 * j] = Elem<DT>::store(l == 0.0f ? 0.0f : acc[j] / l);
}

}  // namespace puter

using namespace puter;

extern "C" {

size_t puter_hip_paged_int4_workspace_bytes(int64_t batch, int64_t query_len, int64_t num_heads, int64_t kv_heads,
                                            int64_t head_dim, int64_t max_context) {
    if (batch <= 0 || query_len <= 0 || num_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_context <= 0) return 0;
    return 16;
}

int puter_hip_paged_int4_attention(const void *query, const void *key_pages, const void *value_pages,
                                   const void *key_params, const void *value_params, const int32_t *page_table,
                                   const int32_t *context_lens, int64_t batch, int64_t query_len,
                                   int64_t max_pages_per_seq, int64_t page_size, int64_t num_pages, int64_t num_heads,
                                   int64_t kv_heads, int64_t head_dim, int64_t group, int64_t max_context, int dtype,
                                   void *output, void *workspace, size_t workspace_bytes, void *stream) {
    if (batch < 0 || query_len < 0 || max_pages_per_seq < 0 || page_size <= 0 || num_pages < 0 || num_heads <= 0 || kv_heads <= 0)
        return fail(PUTER_ERR_INVALID, "paged int4: invalid shape");
    if (dtype != PUTER_BF16 && dtype != PUTER_F16) return fail(PUTER_ERR_INVALID, "paged int4: dtype %d unsupported (bf16, f16)", dtype);
    if (!((head_dim == 64 || head_dim == 128 || head_dim == 256) && (group == 32 || group == 64 || group == 128) && group <= head_dim))
        return fail(PUTER_ERR_INVALID, "paged int4: head dims of 64, 128 or 256 in groups of 32, 64 or 128 dims");
    if (num_heads % kv_heads != 0) return fail(PUTER_ERR_INVALID, "paged int4: heads not divisible by kv heads");
    if (batch > 65535 || query_len > 65535 || num_heads > 65535) return fail(PUTER_ERR_INVALID, "paged int4: batch, query_len and heads up to 65535");
    if (page_size > 0x7FFFFFFF || num_pages > 0x7FFFFFFF / page_size || max_pages_per_seq > 0x7FFFFFFF / page_size)
        return fail(PUTER_ERR_INVALID, "paged int4: pool rows (num_pages * page_size) must stay below 2^31");
    if (batch == 0 || query_len == 0) return PUTER_OK;
    if (max_context <= 0 || max_context > max_pages_per_seq * page_size)
        return fail(PUTER_ERR_INVALID, "paged int4: max_context must be in [1, max_pages_per_seq*page_size]");
    if (!query || !output || !page_table || !context_lens || !workspace ||
        (num_pages > 0 && (!key_pages || !value_pages || !key_params || !value_params)))
        return fail(PUTER_ERR_NIL, "paged int4: nil buffer");
    if (!aligned16(query) || !aligned16(key_pages) || !aligned16(value_pages) || !aligned16(key_params) ||
        !aligned16(value_params) || !aligned16(output) || !aligned16(workspace))
        return fail(PUTER_ERR_INVALID, "paged int4: query, output, pools, pairs and workspace must be 16-byte aligned");
    const size_t need = puter_hip_paged_int4_workspace_bytes(batch, query_len, num_heads, kv_heads, head_dim, max_context);
    if (workspace_bytes < need) return fail(PUTER_ERR_INVALID, "paged int4: workspace %zu < %zu bytes", workspace_bytes, need);
    Int4Args a{static_cast<const uint16_t *>(query), static_cast<const uint8_t *>(key_pages),
               static_cast<const uint8_t *>(value_pages), static_cast<const uint32_t *>(key_params),
               static_cast<const uint32_t *>(value_params), page_table, context_lens, static_cast<uint16_t *>(output),
               batch, max_pages_per_seq, page_size, num_pages, max_context, (int)query_len, (int)num_heads, (int)kv_heads,
               (int)head_dim, (int)group, (float)(1.0 / sqrt((double)head_dim))};
    hipStream_t s = as_stream(stream);
    const dim3 grid((unsigned)(num_heads * query_len), (unsigned)batch);
    if (dtype == PUTER_BF16) int4_row_kernel<PUTER_BF16><<<grid, 64, 0, s>>>(a);
    else int4_row_kernel<PUTER_F16><<<grid, 64, 0, s>>>(a);
    return check_launch("paged int4");
}

}  // extern "C"
