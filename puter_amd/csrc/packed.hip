// MultiHeadAttention over packed sequences of different lengths (extension: the reference runs
// one MultiHeadAttention per sequence, device/cpu/attention/typed_compute.go:142-237).  Rows of
// all sequences stand back to back; the offsets that part them are read on the device, so a
// batch of other lengths needs no host synchronisation.  Per sequence the masks are
// MultiHeadAttention's: key k is visible to query q iff k <= q + seqK - seqQ (causal) and
// q - k < window, scores scaled by 1/sqrt(D), ALiBi added; a query that sees no key is zero.
#include "attention.hpp"

#include <algorithm>

namespace puter {

struct PackedMha {
    const void *q, *k, *v;
    void *o;
    const int32_t *qoff, *koff;
    int64_t batch, total_q, total_k, heads, kv_heads, dim;
    int causal;
    int64_t window;
    float alibi, scale;
    int32_t *status;
};

// Sequence b's rows [start, end) of a total, whatever the offsets hold: no access leaves the tensors.
__device__ __forceinline__ void packed_range(const int32_t *off, int64_t b, int64_t total, int64_t &start, int64_t &end) {
    start = min(max((int64_t)off[b], (int64_t)0), total);
    end = min(max((int64_t)off[b + 1], start), total);
}

// Offsets that fall, are negative or pass the total are reported, as bad page ids are.
__device__ __forceinline__ void packed_check(const int32_t *off, int64_t batch, int64_t total, int32_t *status) {
    if (!status) return;
    for (int64_t i = threadIdx.x; i < batch; i += blockDim.x)
        if (off[i] < 0 || off[i + 1] < off[i] || off[i + 1] > total) *status = PUTER_ERR_INVALID;
}

// Any dtype, head dim up to 256 and alignment: a wave per query row and head.  Lanes take 64
// keys at a time (online softmax, scores and sums in f32), then the head dims (up to four a lane).
template <int DT>
__global__ __launch_bounds__(64) void mha_packed_row_kernel(PackedMha a) {
    using T = typename Elem<DT>::T;
    __shared__ float qrow[256];
    __shared__ float pk[64];
    const int64_t row = blockIdx.x, h = blockIdx.y;
    const int lane = threadIdx.x;
    if (row == 0 && h == 0) {
        packed_check(a.qoff, a.batch, a.total_q, a.status);
        packed_check(a.koff, a.batch, a.total_k, a.status);
    }
    int64_t b = 0, past = a.batch;   // the last sequence that starts at or before the row
    while (past - b > 1) {
        const int64_t mid = (b + past) >> 1;
        if (a.qoff[mid] <= row) b = mid;
        else past = mid;
    }
    int64_t q0, q1, k0, k1;
    packed_range(a.qoff, b, a.total_q, q0, q1);
    packed_range(a.koff, b, a.total_k, k0, k1);
    if (row < q0 || row >= q1) return;   // between or behind the sequences: left as it is
    const int64_t qi = row - q0, seq_k = k1 - k0, D = a.dim;
    const int64_t ks = a.kv_heads * D, kvh = h / (a.heads / a.kv_heads);
    const T *Q = reinterpret_cast<const T *>(a.q) + (row * a.heads + h) * D;
    const T *K = reinterpret_cast<const T *>(a.k) + k0 * ks + kvh * D;
    const T *V = reinterpret_cast<const T *>(a.v) + k0 * ks + kvh * D;
    T *O = reinterpret_cast<T *>(a.o) + (row * a.heads + h) * D;
    for (int64_t d = lane; d < D; d += 64) qrow[d] = Elem<DT>::load(Q[d]);
    __syncthreads();
    int64_t hi = seq_k, lo = 0;
    if (a.causal) hi = min(hi, qi + seq_k - (q1 - q0) + 1);
    if (a.window > 0) lo = max(lo, qi - a.window + 1);
    float m = -INFINITY, l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t c0 = lo; c0 < hi; c0 += 64) {
        const int64_t k = c0 + lane;
        float s = -INFINITY;
        if (k < hi) {
            const T *kr = K + k * ks;
            float dot = 0.0f;
            for (int64_t d = 0; d < D; ++d) dot += qrow[d] * Elem<DT>::load(kr[d]);
            s = dot * a.scale;
            if (a.alibi != 0.0f) s += a.alibi * (float)(k - qi);
        }
        const float mn = fmaxf(m, wave_max(s));
        const float mref = mn == -INFINITY ? 0.0f : mn;
        const float p = k < hi ? expf(s - mref) : 0.0f;
        const float alpha = m == -INFINITY ? 0.0f : expf(m - mref);
        l = l * alpha + wave_sum(p);
        m = mn;
        __syncthreads();
        pk[lane] = p;
        __syncthreads();
        const int n = (int)min((int64_t)64, hi - c0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t d = lane + 64 * j;
            if (d >= D) break;
            float t = 0.0f;
            for (int i = 0; i < n; ++i) t += pk[i] * Elem<DT>::load(V[(c0 + i) * ks + d]);
            acc[j] = acc[j] * alpha + t;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (lane + 64 * j < D) O[lane + 64 * j] = Elem<DT>::store(l == 0.0f ? 0.0f : acc[j] / l);
}

}  // namespace puter

using namespace puter;

extern "C" int puter_hip_multi_head_attention_packed(const puter_mha_config *config, const void *query, const void *key,
                                                     const void *value, void *output, const int32_t *query_offsets,
                                                     const int32_t *key_offsets, int64_t batch, int64_t total_q,
                                                     int64_t total_k, int dtype, int32_t *status, void *stream) {
    if (!config) return fail(PUTER_ERR_NIL, "mha packed: nil config");
    if (!is_norm_dtype(dtype)) return fail(PUTER_ERR_INVALID, "mha packed: unsupported dtype %d", dtype);
    if (batch < 0 || total_q < 0 || total_k < 0) return fail(PUTER_ERR_INVALID, "mha packed: negative shape");
    const int64_t H = config->num_heads, D = config->head_dim;
    const int64_t kvh = config->kv_head_count > 0 ? config->kv_head_count : H;
    if (H <= 0 || D <= 0) return fail(PUTER_ERR_INVALID, "mha packed: heads and head_dim must be positive");
    if (H % kvh != 0)
        return fail(PUTER_ERR_INVALID, "mha packed: %lld heads not divisible by %lld kv heads", (long long)H, (long long)kvh);
    if (D > 256) return fail(PUTER_ERR_INVALID, "mha packed: head_dim %lld > 256 unsupported", (long long)D);
    if (config->window_size < 0) return fail(PUTER_ERR_INVALID, "mha packed: negative window");
    if (H > 65535 || total_q > 0x3FFFFFFF || total_k > 0x3FFFFFFF || batch > 0x3FFFFFFF)
        return fail(PUTER_ERR_INVALID, "mha packed: too many heads, rows or sequences");
    if (batch == 0 || total_q == 0) return PUTER_OK;
    if (!query || !output || !query_offsets || (total_k > 0 && (!key || !value))) return fail(PUTER_ERR_NIL, "mha packed: nil buffer");
    if (reinterpret_cast<uintptr_t>(status) & 3) return fail(PUTER_ERR_INVALID, "mha packed: misaligned status word");
    // no key offsets: every sequence's keys are its own rows
    if (!key_offsets && total_k != total_q) return fail(PUTER_ERR_INVALID, "mha packed: without key offsets the key rows are the query rows");
    PackedMha a{query, key, value, output, query_offsets, key_offsets ? key_offsets : query_offsets, batch, total_q, total_k,
                H, kvh, D, config->causal ? 1 : 0, config->window_size, config->alibi_slope,
                (float)(1.0 / sqrt((double)D)), status};
    hipStream_t s = as_stream(stream);
    const dim3 grid((unsigned)total_q, (unsigned)H);
    switch (dtype) {
    case PUTER_F32: mha_packed_row_kernel<PUTER_F32><<<grid, 64, 0, s>>>(a); break;
    case PUTER_BF16: mha_packed_row_kernel<PUTER_BF16><<<grid, 64, 0, s>>>(a); break;
    case PUTER_F16: mha_packed_row_kernel<PUTER_F16><<<grid, 64, 0, s>>>(a); break;
    }
    return check_launch("mha packed");
}
