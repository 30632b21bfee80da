// MultiHeadAttention over packed sequences of different lengths (extension: the reference runs
// one MultiHeadAttention per sequence, device/cpu/attention/typed_compute.go:142-237).  Rows of
// all sequences stand back to back; the offsets that part them are read on the device, so a
// batch of other lengths needs no host synchronisation.  Per sequence the masks are
// MultiHeadAttention's: key k is visible to query q iff k <= q + seqK - seqQ (causal) and
// q - k < window, scores scaled by 1/sqrt(D), ALiBi added; a query that sees no key is zero.
#include "prefill.hpp"

#include <algorithm>
#include <cmath>
#include <optional>

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

// The MFMA prefill kernels (prefill.hpp) over packed sequences: PrefillArgs whose map finds the
// block's sequence and sets the arguments to that sequence.
struct PackedArgs : PrefillArgs {
    const int32_t *qoff, *koff;
    int32_t *status;
    int total_q, total_k, elem;   // elem: bytes of an element
    int row0;                     // the sequence's first query row (set by the map)
    // the partials' row of query qi of the sequence in this block's split of the keys
    __device__ __forceinline__ int64_t part_row(int qi) const { return (int64_t)blockIdx.y * total_q + row0 + qi; }
};

constexpr int kPackedLanes = 256;   // sequences that a wave ranks by length, four a lane

__device__ __forceinline__ int packed_wave_sum(int v) {   // in every lane
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8: sums of 16
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);   // row_bcast 15, 31: of 32, of 64
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return __builtin_amdgcn_readlane(v, 63);
}

// The rank-th query tile of the call and its sequence.  Up to 256 sequences the tiles are ranked
// by how far down their sequence's keys they reach (their level: under a causal mask, their work),
// the longest first, as the batched kernel starts its heaviest blocks first: F(t), the tiles of
// level t or more, is one pass over the lanes, and the level where F passes the rank is found by
// bisection.  More sequences go in their order: sequence i's tiles start at slot
// floor(offset / 128) + i, which leaves room for each one's last tile.
__device__ __forceinline__ bool packed_tile(const PackedArgs &a, int rank, int &seq, int &tile) {
    const int lane = threadIdx.x & 63;
    if (a.batch > kPackedLanes) {
        int lo = 0, hi = a.batch;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (min(max(a.qoff[mid], 0), a.total_q) / fa::BM + mid <= rank) lo = mid;
            else hi = mid;
        }
        const int start = min(max(a.qoff[lo], 0), a.total_q);
        seq = lo;
        tile = rank - (start / fa::BM + lo);
        return tile >= 0;
    }
    int base[4], n[4], top = 0;   // per sequence: the level of its first tile, its tiles
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        base[c] = n[c] = 0;
        const int i = 64 * c + lane;
        if (64 * c >= a.batch) continue;
        if (i < a.batch) {
            int64_t q0, q1, k0, k1;
            packed_range(a.qoff, i, a.total_q, q0, q1);
            packed_range(a.koff, i, a.total_k, k0, k1);
            n[c] = (int)((q1 - q0 + fa::BM - 1) / fa::BM);
            base[c] = (int)max((int64_t)0, (k1 - k0) - (q1 - q0)) / fa::BM;
        }
        top = max(top, base[c] + n[c]);
    }
    for (int o = 32; o >= 1; o >>= 1) top = max(top, __shfl_xor(top, o, 64));
    top = __builtin_amdgcn_readfirstlane(top);
    auto from_level = [&](int t) __attribute__((always_inline)) {
        int f = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (64 * c < a.batch) f += min(max(base[c] + n[c] - t, 0), n[c]);
        return packed_wave_sum(f);
    };
    if (rank >= from_level(0)) return false;
    int lo = 0, hi = top;   // F(lo) > rank >= F(hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (from_level(mid) > rank) lo = mid;
        else hi = mid;
    }
    int j = rank - from_level(lo + 1);   // the j-th sequence with a tile of this level
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint64_t have = __ballot(lo >= base[c] && lo < base[c] + n[c]);
        const int count = __builtin_popcountll(have);
        if (j < count) {
            const int before = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(have >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)have, 0u));
            const uint64_t mine = __ballot(((have >> lane) & 1) && before == j);
            const int at = __builtin_ctzll(mine);
            seq = 64 * c + at;
            tile = lo - __builtin_amdgcn_readlane(base[c], at);
            return true;
        }
        j -= count;
    }
    return false;   // (offsets that fall: fewer tiles than they seemed)
}

// Block -> (tile, kv head, head of its group): eight (tile, kv head) pairs at a time, one to an
// XCD, the group's heads one after another there, so a sequence's keys of one kv head are read by
// one XCD (by few, with fewer kv heads than XCDs).
__device__ __forceinline__ bool prefill_map(PackedArgs &a, int &qt, int &b, int &h) {
    const int id = blockIdx.x, G = a.heads / a.kv_heads;
    if (id == 0) {
        packed_check(a.qoff, a.batch, a.total_q, a.status);
        packed_check(a.koff, a.batch, a.total_k, a.status);
    }
    const int pair = (id / (8 * G)) * 8 + (id & 7), slot = (id >> 3) % G;
    int seq = 0;
    if (!packed_tile(a, pair / a.kv_heads, seq, qt)) return false;
    seq = __builtin_amdgcn_readfirstlane(seq);
    qt = __builtin_amdgcn_readfirstlane(qt);
    h = (pair % a.kv_heads) * G + slot;
    b = 0;
    int64_t q0, q1, k0, k1;
    packed_range(a.qoff, seq, a.total_q, q0, q1);
    packed_range(a.koff, seq, a.total_k, k0, k1);
    q0 = __builtin_amdgcn_readfirstlane((int)q0), q1 = __builtin_amdgcn_readfirstlane((int)q1);
    k0 = __builtin_amdgcn_readfirstlane((int)k0), k1 = __builtin_amdgcn_readfirstlane((int)k1);
    a.seq_q = (int)(q1 - q0);
    a.seq_k = (int)(k1 - k0);
    if (qt >= (a.seq_q + fa::BM - 1) / fa::BM) return false;
    a.shift = a.seq_k - a.seq_q;
    a.row0 = (int)q0;
    const int64_t qrow = (int64_t)a.heads * a.dim * a.elem, krow = (int64_t)a.kv_heads * a.dim * a.elem;
    a.q = reinterpret_cast<const uint16_t *>(reinterpret_cast<const char *>(a.q) + q0 * qrow);
    a.o = reinterpret_cast<uint16_t *>(reinterpret_cast<char *>(a.o) + q0 * qrow);
    a.k = reinterpret_cast<const uint16_t *>(reinterpret_cast<const char *>(a.k) + k0 * krow);
    a.v = reinterpret_cast<const uint16_t *>(reinterpret_cast<const char *>(a.v) + k0 * krow);
    return true;
}

// The key splits of the f32 kernel: a thread per four dims of a row and head folds them in order with
// weights exp2(m_s - M), the loads of four splits at a time.  A split without tiles, or whose keys
// are all hidden, has m = -inf and adds its sum alone (0, or the NaN of scores that are NaN); its
// outputs may not have been written and are not used.  Rows outside every sequence have no partials
// and stay.
__global__ __launch_bounds__(256) void packed_f32_combine_kernel(PackedArgs a, int splits) {
    const uint32_t quads = a.dim / 4, id = blockIdx.x * 256 + threadIdx.x, at = id / quads, d = (id - at * quads) * 4;
    const int64_t rows = (int64_t)a.total_q * a.heads;
    if (at >= rows) return;
    const int row = (int)(at / (uint32_t)a.heads);
    if (row < a.qoff[0] || row >= a.qoff[a.batch]) return;
    float M = -INFINITY, sum = 0.0f;
    f32x4 acc = {};
    for (int s0 = 0; s0 < splits; s0 += 4) {
        float2 ml[4];
        f32x4 o[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int s = min(s0 + u, splits - 1);
            ml[u] = a.part_ml[s * rows + at];
            o[u] = *reinterpret_cast<const f32x4 *>(a.part_o + (s * rows + at) * a.dim + d);
        }
        float top = M;
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (s0 + u < splits) top = fmaxf(top, ml[u].x);
        const float keep = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - top);
        if (M != -INFINITY) {   // (a NaN or 0 alone has no weight to change)
            sum *= keep;
            acc *= keep;
        }
        M = top;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (s0 + u >= splits) break;
            if (ml[u].x == -INFINITY) {
                sum += ml[u].y;
            } else {
                const float w = __builtin_amdgcn_exp2f(ml[u].x - M);
                sum += w * ml[u].y;
                acc += w * o[u];
            }
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<f32x4 *>(reinterpret_cast<float *>(a.o) + (int64_t)at * a.dim + d) = acc * inv;
}

// 16-bit head dims of 8 n and f32 head dims of 4 n, 16-byte aligned; false: the row kernel's.
static bool launch_packed_mfma(const PackedMha &m, int dtype, hipStream_t s, int *status) {
    const bool f32 = dtype == PUTER_F32;
    if (m.dim % (f32 ? 4 : 8)) return false;
    if (m.kv_heads * m.dim > (f32 ? 32768 : 65536) * 128) return false;   // a K/V tile spans < 2^30 bytes
    if (!aligned16(m.q) || !aligned16(m.k) || !aligned16(m.v) || !aligned16(m.o)) return false;
    if (m.total_k >= ((int64_t)1 << 30)) return false;
    // ranks: every sequence's last tile may be a part of one
    const int64_t tiles = m.total_q / fa::BM + std::min(m.batch, m.total_q), G = m.heads / m.kv_heads;
    const int64_t ranks = m.batch > kPackedLanes ? m.total_q / fa::BM + m.batch : tiles;
    const int64_t blocks = (ranks * m.kv_heads + 7) / 8 * 8 * G;
    if (blocks > 0x7FFFFFFF) return false;
    PackedArgs a{};
    a.q = static_cast<const uint16_t *>(m.q);
    a.k = static_cast<const uint16_t *>(m.k);
    a.v = static_cast<const uint16_t *>(m.v);
    a.o = static_cast<uint16_t *>(m.o);
    a.batch = (int)m.batch;
    a.heads = (int)m.heads;
    a.kv_heads = (int)m.kv_heads;
    a.dim = (int)m.dim;
    a.nan_rows = 1;
    a.causal = m.causal;
    a.window = (int)std::min<int64_t>(m.window, 0x3FFFFFFF);
    a.alibi_s = m.alibi != 0.0f ? m.alibi / m.scale : 0.0f;
    a.scale_log2 = m.scale * 1.4426950408889634f;
    if (f32 && m.dim != 64 && m.dim != 128) {   // as launch_prefill_f32
        const double exact = (double)m.scale * 1.4426950408889634;
        a.scale_log2 = (float)exact;
        if ((double)a.scale_log2 >= exact) a.scale_log2 = std::nextafter(a.scale_log2, 0.0f);
        a.scale_log2_lo = (float)(exact - (double)a.scale_log2);
    }
    a.qoff = m.qoff, a.koff = m.koff, a.status = m.status;
    a.total_q = (int)m.total_q, a.total_k = (int)m.total_k, a.elem = f32 ? 4 : 2;
    const bool gen = a.window > 0 || a.alibi_s != 0.0f;
    // f32: a block's keys are split over blockIdx.y while there are fewer than two blocks a CU, up to
    // about two a CU, in runs of two key tiles or more; each block cuts its own tiles, whose number the
    // host does not know.  2331 rows of five sequences (8 heads of 80, a window of 512): 163 us unsplit,
    // 72 so, 85 at four splits in place of three, 90 at two; runs of one length for all
    // blocks, from the lengths on the device, 78; runs of 6 tiles or more lose where
    // sequences are short (300 rows, 8 heads of 64: 16 us against 24).  The partials lie in the
    // library's scratch, which cannot grow while a graph is recorded: there the keys stay together.
    int64_t splits = 1;
    const int64_t cus = device_cus(), rows = m.total_q * m.heads;
    if (f32 && blocks < 2 * cus && !scratch_capturing(s)) {
        const int64_t keys = m.window > 0 ? std::min(m.total_k, m.window + fa::BM) : m.total_k;
        splits = std::max<int64_t>(1, std::min<int64_t>((2 * cus + blocks - 1) / blocks, keys / 64));
    }
    const size_t part = (size_t)(splits * rows * m.dim) * sizeof(float), need = part + (size_t)(splits * rows) * sizeof(float2);
    std::optional<ScratchLease> lease;
    if (splits > 1) {
        lease.emplace(need, s, true);
        if (lease->status()) {
            lease.reset();   // no room: unsplit
            splits = 1;
        } else {   // outputs first: a multiple of 16 bytes
            a.part_o = static_cast<float *>(lease->ptr());
            a.part_ml = reinterpret_cast<float2 *>(static_cast<char *>(lease->ptr()) + part);
        }
    }
    const dim3 grid((unsigned)blocks, (unsigned)splits);
    with_head_dim(m.dim, [&](auto d) {
        if (f32) {
            if (gen) prefill_f32_kernel<d.D, true, d.PAD, PackedArgs><<<grid, 256, 0, s>>>(a);
            else prefill_f32_kernel<d.D, false, d.PAD, PackedArgs><<<grid, 256, 0, s>>>(a);
        } else if (dtype == PUTER_BF16) {
            if (gen) prefill_kernel<PUTER_BF16, d.D, true, d.PAD, PackedArgs><<<grid, 256, 0, s>>>(a);
            else prefill_kernel<PUTER_BF16, d.D, false, d.PAD, PackedArgs><<<grid, 256, 0, s>>>(a);
        } else {
            if (gen) prefill_kernel<PF_F16_DOT32, d.D, true, d.PAD, PackedArgs><<<grid, 256, 0, s>>>(a);
            else prefill_kernel<PF_F16_DOT32, d.D, false, d.PAD, PackedArgs><<<grid, 256, 0, s>>>(a);
        }
    });
    if (lease) packed_f32_combine_kernel<<<(unsigned)((rows * (m.dim / 4) + 255) / 256), 256, 0, s>>>(a, (int)splits);
    *status = check_launch("mha packed mfma");
    if (lease) {
        const int fin = lease->finish();
        if (!*status) *status = fin;
    }
    return true;
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
    int rc = PUTER_OK;
    if (launch_packed_mfma(a, dtype, s, &rc)) return rc;
    const dim3 grid((unsigned)total_q, (unsigned)H);
    switch (dtype) {
    case PUTER_F32: mha_packed_row_kernel<PUTER_F32><<<grid, 64, 0, s>>>(a); break;
    case PUTER_BF16: mha_packed_row_kernel<PUTER_BF16><<<grid, 64, 0, s>>>(a); break;
    case PUTER_F16: mha_packed_row_kernel<PUTER_F16><<<grid, 64, 0, s>>>(a); break;
    }
    return check_launch("mha packed");
}
