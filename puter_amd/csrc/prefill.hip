// The MFMA flash prefill kernels over batches of equal lengths (the block's work is in
// prefill.hpp) and the choice between them and the general kernel.
#include "prefill.hpp"

namespace puter {

// Merges the key splits of prefill_f32_kernel: one wave per (batch, query, head) row,
// lanes over the head dims; the splits are folded in order with weights
// exp2(m_s - M) (m in the scaled log2 domain), O = sum w_s O_s / sum w_s l_s; a row
// with no visible key (every m = -inf) is 0, as in the unsplit kernel.
template <int D, bool PAD>
__global__ __launch_bounds__(256) void prefill_f32_combine_kernel(PrefillArgs a, int splits, int64_t rows) {
    constexpr int J = (D + 63) / 64;
    const int dim = PAD ? a.dim : D;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int lane = threadIdx.x & 63;
    float M = -INFINITY;
    for (int s = 0; s < splits; ++s) M = fmaxf(M, a.part_ml[s * rows + row].x);
    float acc[J] = {}, lsum = 0.0f;   // dims lane, lane + 64, ..
    if (M != -INFINITY) {
        for (int s = 0; s < splits; ++s) {
            const float2 ml = a.part_ml[s * rows + row];
            const float w = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M);
            lsum += w * ml.y;
            const float *po = a.part_o + (s * rows + row) * dim;
#pragma unroll
            for (int j = 0; j < J; ++j)   // (past a padded row's end: its last dim, not stored)
                acc[j] += w * po[PAD ? min(64 * j + lane, dim - 1) : 64 * j + lane];
        }
    }
    const float inv = lsum > 0.0f ? 1.0f / lsum : 0.0f;
    // row = (batch, query, head): the output row of the same index, dim floats
    float *out = reinterpret_cast<float *>(a.o) + row * dim;
#pragma unroll
    for (int j = 0; j < J; ++j)
        if (!PAD || 64 * j + lane < dim) out[64 * j + lane] = acc[j] * inv;
}

// The general kernel or the padded one?  Estimates in us, fitted to 2900 bf16 and 1200 f32
// shapes (1 to 32 heads, 2 to 300 queries over 40 to 3000 keys, dims 16 to 256; 6% off for the padded
// kernels, 15% for the general one).  The general kernel has a block per query row and
// head: a row's keys in steps, 1.7 times slower where the heads that an XCD's rows see overflow
// its L2, or, once rows fill the chip, all rows' keys at a rate.  f16 needs no such rule: its
// general kernel widens in software and never wins.
static double general_us(const MhaArgs &m, bool f32) {
    const double rows = (double)m.batch * m.seq_q * m.heads, dim = (double)m.dim;
    double most = (double)m.seq_k, mean = most;   // keys that a row sees
    if (m.causal) mean = (double)m.shift + 0.5 * (double)(m.seq_q + 1);
    if (m.window > 0) most = std::min(most, (double)m.window);
    mean = std::min(std::max(mean, 1.0), most);
    const double heads = std::max(1.0, std::min((double)m.batch * m.kv_heads, rows / 8));
    const bool overflows = heads * (double)m.seq_k * dim * (f32 ? 8 : 4) > 4.2e6;
    const double steps = most * (f32 ? 0.0078 + 0.000162 * dim : 0.0082 + 0.000145 * dim) * (overflows ? 1.7 : 1.0);
    return (f32 ? 3.9 : 3.7) + std::hypot(steps, rows * mean * (f32 ? 1.3e-5 + 6.6e-7 * dim : 1.8e-5 + 4.4e-7 * dim));
}
// The padded kernels: the key tiles of the longest block, in rounds of blocks.
static double padded_us(const MhaArgs &m, int64_t blocks, int64_t tiles, int64_t splits, bool f32) {
    const int i = m.dim <= 64 ? 0 : m.dim <= 96 ? 1 : m.dim <= 128 ? 2 : 3;
    constexpr double base[2][4] = {{3.5, 4.2, 4.6, 7.4}, {3.7, 4.5, 6.2, 8.0}};
    constexpr double tile[2][4] = {{0.94, 1.14, 1.3, 2.85}, {2.5, 3.7, 6.3, 13.0}};
    const int64_t room = (int64_t)device_cus() * (m.dim > 128 ? 1 : 2), rounds = (blocks * splits + room - 1) / room;
    const double sums = splits > 1 ? 1.2 + 0.53 * (double)splits + 4.3e-6 * (double)(splits * m.batch * m.seq_q * m.heads * m.dim) : 0.0;
    return base[f32][i] + tile[f32][i] * (double)(tiles * rounds) + sums;
}
static int64_t prefill_tiles(const MhaArgs &m, int64_t bn) {   // key tiles of the longest block
    const int64_t keys = m.window > 0 ? std::min(m.seq_k, m.window + fa::BM + bn) : m.seq_k;
    return (keys + bn - 1) / bn;
}

// f32 MultiHeadAttention on prefill_f32_kernel: head dims of 4 n up to 256, at least 16 query
// rows, causal or not, with or without a sliding window and ALiBi.
static bool launch_prefill_f32(const MhaArgs &m, hipStream_t s, int *status) {
    if (m.dim % 4 || m.dim > 256) return false;
    if (m.seq_q < 16) return false;
    if (m.seq_q > 0x3FFFFFFF || m.seq_k > 0x3FFFFFFF || m.shift > 0x3FFFFFFF || m.shift < -0x3FFFFFFF) return false;
    if (m.kv_heads * m.dim > 32768 * 128) return false;   // a 32-row K/V tile spans < 2^30 bytes
    const uintptr_t mask = 15;
    if ((reinterpret_cast<uintptr_t>(m.q) | reinterpret_cast<uintptr_t>(m.k) |
         reinterpret_cast<uintptr_t>(m.v) | reinterpret_cast<uintptr_t>(m.o)) & mask)
        return false;
    PrefillArgs a;
    a.q = static_cast<const uint16_t *>(m.q);
    a.k = static_cast<const uint16_t *>(m.k);
    a.v = static_cast<const uint16_t *>(m.v);
    a.o = static_cast<uint16_t *>(m.o);
    a.batch = (int)m.batch;
    a.seq_q = (int)m.seq_q;
    a.seq_k = (int)m.seq_k;
    a.heads = (int)m.heads;
    a.kv_heads = (int)m.kv_heads;
    a.dim = (int)m.dim;
    a.nan_rows = m.nan_rows;
    a.qtiles = (int)((m.seq_q + fa::BM - 1) / fa::BM);
    a.causal = m.causal;
    a.shift = (int)m.shift;
    // a window of seq_q or more hides no key (a query's distance to a visible key is
    // below seq_q): run it as no window
    a.window = (m.window > 0 && m.window < m.seq_q) ? (int)m.window : 0;
    a.alibi_s = m.alibi != 0.0f ? m.alibi / m.scale : 0.0f;
    a.xcd_map = ((a.batch * a.kv_heads) % 8 == 0) ? 1 : 0;
    a.scale_log2 = m.scale * 1.4426950408889634f;
    if (m.dim != 64 && m.dim != 128) {
        // the padded kernels add the scale's low part; it is kept positive, so a masked
        // score's -inf stays -inf through both products
        const double exact = (double)m.scale * 1.4426950408889634;
        a.scale_log2 = (float)exact;
        if ((double)a.scale_log2 >= exact) a.scale_log2 = std::nextafter(a.scale_log2, 0.0f);
        a.scale_log2_lo = (float)(exact - (double)a.scale_log2);
    }
    const bool gen = a.window > 0 || a.alibi_s != 0.0f;   // the kernel with the window / ALiBi code
    const int64_t blocks = (int64_t)a.qtiles * a.batch * a.heads;
    if (blocks > 0x7FFFFFFF) return false;
    const int64_t cus = device_cus();
    const int64_t ktiles = (m.seq_k + 31) / 32;
    hipStreamCaptureStatus cst = hipStreamCaptureStatusNone;
    const bool capturing = hipStreamIsCapturing(s, &cst) != hipSuccess || cst != hipStreamCaptureStatusNone;
    // Grids of fewer than 24 blocks stay on the general kernel (one block per query
    // row and head) unless they are causal over at least 8 key tiles and can split
    // them (below): config 1's 128 queries x 8 heads of 64 (8 blocks) 9.2 us there
    // against 14.2 here even split; 256 x 8 x 128 (16 blocks) 33.1 against 24.1 split
    // (43 unsplit), 640 x 4 x 64 47.5 against 22.1.  From 24 blocks this kernel wins
    // unsplit too (384 x 8 x 64: 32.9 against 36.0, 4 x 128 x 8 x 64: 15.0 against 24.5)
    if (blocks < 24 && (!a.causal || ktiles < 8 || capturing)) return false;
    // other head dims than 64 and 128: from 2048 rows (batch x queries x heads) or 512 keys on
    // (2 x 21 x 12 rows over 173 keys of 96: 10.6 there against 24.9 here; 2 x 60 x 8 over 1500
    // keys of 256: 218 against 107, 2 x 200 x 16 over 200 keys of 40: 75 against 21), and there
    // by the estimates above (16 x 32 heads over 700 keys of 256: 77 there against 152)
    if (m.dim != 64 && m.dim != 128 && m.batch * m.seq_q * m.heads < 2048 && ktiles < 16) return false;
    // Small grids split each block's key range over blockIdx.y, partials in the
    // library's scratch: the longest block's key loop, the critical path, shrinks with
    // the split count.  Causal grids of under two blocks per CU aim at four blocks per
    // CU in runs of at least 8 key tiles (2 under 24 blocks) (the triangle leaves most
    // CUs idle while the last query tiles run: B1 S4096 8 x 64 causal 296 -> 221 us,
    // S2048 8 x 128 154 -> 146 us), other grids of under one block per CU at two, in
    // runs of at least 16 (B1 S2048 8 x 64, 150 -> 88 us; more splits lose there).  A
    // stream that is capturing a graph keeps the unsplit kernel (the scratch cannot
    // grow there)
    int64_t splits = 1;
    if (a.causal && blocks < 2 * cus)
        splits = std::max<int64_t>(1, std::min<int64_t>((4 * cus + blocks - 1) / blocks, ktiles / (blocks < 24 ? 2 : 8)));
    else if (!a.causal && blocks < cus)
        splits = std::max<int64_t>(1, std::min<int64_t>((2 * cus + blocks - 1) / blocks, ktiles / 16));
    if (capturing) splits = 1;
    if (m.dim != 64 && m.dim != 128 &&
        general_us(m, true) < padded_us(m, blocks, (prefill_tiles(m, 32) + splits - 1) / splits, splits, true))
        return false;
    auto launch = [&](dim3 grid) {
        with_head_dim(m.dim, [&](auto d) {
            if (gen) prefill_f32_kernel<d.D, true, d.PAD, PrefillArgs><<<grid, 256, 0, s>>>(a);
            else prefill_f32_kernel<d.D, false, d.PAD, PrefillArgs><<<grid, 256, 0, s>>>(a);
        });
    };
    if (splits > 1) {
        a.split_tiles = (int)((ktiles + splits - 1) / splits);
        splits = (ktiles + a.split_tiles - 1) / a.split_tiles;
        const int64_t rows = m.batch * m.seq_q * m.heads;
        const size_t need = (size_t)(splits * rows) * (sizeof(float2) + (size_t)m.dim * sizeof(float));
        ScratchLease lease(need, s, true);
        if (!lease.status()) {
            // outputs first: splits * rows * D floats keep the (max, sum) pairs 16-byte aligned
            a.part_o = static_cast<float *>(lease.ptr());
            a.part_ml = reinterpret_cast<float2 *>(a.part_o + splits * rows * m.dim);
            const dim3 grid((unsigned)blocks, (unsigned)splits);
            const unsigned cblocks = (unsigned)((rows + 3) / 4);
            launch(grid);
            with_head_dim(m.dim, [&](auto d) {
                prefill_f32_combine_kernel<d.D, d.PAD><<<cblocks, 256, 0, s>>>(a, (int)splits, rows);
            });
            const int rc = check_launch("prefill f32 mfma split");
            const int fin = lease.finish();
            *status = rc ? rc : fin;
            return true;
        }
        a.split_tiles = 0;   // no room: unsplit
    }
    launch(dim3((unsigned)blocks));
    *status = check_launch("prefill f32 mfma");
    return true;
}

bool launch_prefill_mfma(const MhaArgs &m, int dtype, hipStream_t s, int *status) {
    if (dtype == PUTER_F32) return launch_prefill_f32(m, s, status);
    if ((dtype != PUTER_BF16 && dtype != PUTER_F16) || m.dim % 8 || m.dim > 256) return false;
    if (m.dim != 128 && m.seq_q == 1) return false;   // one query row: the general kernel (no 127 padding rows)
    if (m.seq_q > 0x3FFFFFFF || m.seq_k > 0x3FFFFFFF || m.shift > 0x3FFFFFFF || m.shift < -0x3FFFFFFF)
        return false;
    // 32-bit buffer offsets: one 64-row tile of K/V must span at most 2^30 bytes
    if (m.kv_heads * m.dim > 65536 * 128) return false;
    const uintptr_t mask = 15;
    if ((reinterpret_cast<uintptr_t>(m.q) | reinterpret_cast<uintptr_t>(m.k) |
         reinterpret_cast<uintptr_t>(m.v) | reinterpret_cast<uintptr_t>(m.o)) & mask)
        return false;
    PrefillArgs a;
    a.q = static_cast<const uint16_t *>(m.q);
    a.k = static_cast<const uint16_t *>(m.k);
    a.v = static_cast<const uint16_t *>(m.v);
    a.o = static_cast<uint16_t *>(m.o);
    a.batch = (int)m.batch;
    a.seq_q = (int)m.seq_q;
    a.seq_k = (int)m.seq_k;
    a.heads = (int)m.heads;
    a.kv_heads = (int)m.kv_heads;
    a.dim = (int)m.dim;
    a.nan_rows = m.nan_rows;
    a.qtiles = (int)((m.seq_q + fa::BM - 1) / fa::BM);
    a.causal = m.causal;
    a.shift = (int)m.shift;
    // a window of seq_q or more hides no key (a query's distance to a visible key
    // is below seq_q): run it as no window
    a.window = (m.window > 0 && m.window < m.seq_q) ? (int)m.window : 0;
    a.alibi_s = m.alibi != 0.0f ? m.alibi / m.scale : 0.0f;
    a.xcd_map = ((a.batch * a.kv_heads) % 8 == 0) ? 1 : 0;
    a.scale_log2 = m.scale * 1.4426950408889634f;
    const int64_t blocks = (int64_t)a.qtiles * a.batch * a.heads;
    if (blocks > 0x7FFFFFFF) return false;
    const bool bf = dtype == PUTER_BF16, win = a.window > 0 || a.alibi_s != 0.0f;
    // few rows of other head dims, by the estimates above (8 x 8 heads over 200 keys of 256: 11.9
    // us on the general kernel against 18.4; one tile of keys is the padded kernel's up to 128
    // dims).  FlashAttention has another general kernel, slower than the padded one.
    if (bf && !m.nan_rows && m.dim != 64 && m.dim != 128 && (m.seq_k > 64 || m.dim > 128) &&
        general_us(m, false) < padded_us(m, blocks, prefill_tiles(m, 64), 1, false))
        return false;
    const dim3 grid((unsigned)blocks);
    with_head_dim(m.dim, [&](auto d) {
        if (win) {
            if (bf) prefill_kernel<PUTER_BF16, d.D, true, d.PAD, PrefillArgs><<<grid, 256, 0, s>>>(a);
            else prefill_kernel<PUTER_F16, d.D, true, d.PAD, PrefillArgs><<<grid, 256, 0, s>>>(a);
        } else {
            if (bf) prefill_kernel<PUTER_BF16, d.D, false, d.PAD, PrefillArgs><<<grid, 256, 0, s>>>(a);
            else prefill_kernel<PUTER_F16, d.D, false, d.PAD, PrefillArgs><<<grid, 256, 0, s>>>(a);
        }
    });
    *status = check_launch("prefill mfma");
    return true;
}

}  // namespace puter
