// Attention over a paged cache held in 4 bits: one or a few query tokens per sequence, grouped
// heads (the reference gathers the pages and runs MultiHeadAttention: execution/page_intrinsic.go:
// 217-352, device/cpu/attention/typed_compute.go:142-237).  A cached value is scale * n + offset
// with the 4-bit code n in [-8, 7] and the (scale, offset) pair of its token, kv head and group of
// dims.  Query i of a sequence of `context` cached tokens and m queries sees the tokens up to
// context - m + i.
//
// Split over the cache: a 256-thread block takes one kv head, `split` tokens of one sequence and up
// to 32 of the (query, head) rows that share the kv head; its four waves walk 64 tokens a step, each
// on its own, with a running maximum and sum, and join through LDS at the end.  A sequence of one
// split is stored at once; more leave (max, sum, row) partials that a second kernel joins.
//   loads: codes and pairs go from HBM straight to the wave's LDS (global_load_lds, no registers
//     between), whole rows to an instruction; a step's K codes are fetched under the softmax and
//     P.V of the step before, its V codes under its own scores.
//   scores: S^T[token, row] = K . Q^T on v_mfma_f32_16x16x32.  A code becomes a 16-bit operand in
//     two instructions for two codes: shifted to the mantissa's top and joined with the exponent of
//     16 it reads 24 + n, exactly; the accumulator starts at -24 sum(q), so the product is of n.
//     Scale and offset act on the f32 product of each group: s = sum_g scale C_g + offset sum_g(q).
//   values: O[row, dim] = P . V, V's columns read out of the row-major codes by ds_read_b64_tr_b4
//     (16 tokens of one dim to a lane), P scaled by the token's scale of the group before it is
//     rounded.  Offsets are summed in f32; the 24 that each code reads too much is taken off by one
//     more product of the same P with 24.
// P is rounded to bf16 once for bf16 outputs (half a step of the output's format, averaged over the
// tokens); for f16 outputs its rounding error is multiplied too (16 bits in all).
#include "common.hpp"

#include <algorithm>

namespace puter {

typedef __bf16 i4_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 i4_f16x8 __attribute__((ext_vector_type(8)));
typedef float i4_f32x4 __attribute__((ext_vector_type(4)));
typedef int i4_i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i4_i32x2 i4_lds_i32x2;
typedef __attribute__((address_space(3))) void i4_lds;
typedef const __attribute__((address_space(1))) void i4_global;

struct Int4Args {
    const uint16_t *q;
    const uint8_t *kp, *vp;
    const uint32_t *kpar, *vpar;
    const int32_t *table, *ctx;
    uint16_t *out;
    float *part_o, *part_ml;
    int64_t max_pages;
    int batch, page_size, page_shift, num_pages, max_context;   // page_shift: log2 of a power of two, else -1
    int query_len, heads, kv_heads, split, max_splits, row_tiles;
    float scale_log2;
};

// a sequence's tokens and its splits (one at least: it stores the zeros of an empty cache)
__device__ __forceinline__ int int4_context(const Int4Args &a, int b) { return max(0, min(a.ctx[b], a.max_context)); }
__device__ __forceinline__ int int4_splits(const Int4Args &a, int ctx) { return max(1, (ctx + a.split - 1) / a.split); }

template <int N> __device__ __forceinline__ void int4_wait_loads() {   // all but the last N
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
__device__ __forceinline__ void int4_wait_lds() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Eight codes (nibble k = code k) as 16-bit values 24 + n in the order 0, 4, 1, 5, 2, 6, 3, 7.
template <bool BF> __device__ __forceinline__ uint4 int4_expand(uint32_t w) {
    if constexpr (BF)
        return make_uint4(((w << 3) & 0x00780078u) ^ 0x41C041C0u, ((w >> 1) & 0x00780078u) ^ 0x41C041C0u,
                          ((w >> 5) & 0x00780078u) ^ 0x41C041C0u, ((w >> 9) & 0x00780078u) ^ 0x41C041C0u);
    else
        return make_uint4(((w << 6) & 0x03C003C0u) ^ 0x4E004E00u, ((w << 2) & 0x03C003C0u) ^ 0x4E004E00u,
                          ((w >> 2) & 0x03C003C0u) ^ 0x4E004E00u, ((w >> 6) & 0x03C003C0u) ^ 0x4E004E00u);
}
template <bool BF> __device__ __forceinline__ i4_f32x4 int4_mfma(uint4 a, uint4 b, i4_f32x4 c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(i4_bf16x8, a), __builtin_bit_cast(i4_bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(i4_f16x8, a), __builtin_bit_cast(i4_f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ float int4_lo(uint32_t pair) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(pair & 0xFFFFu)); }
__device__ __forceinline__ float int4_hi(uint32_t pair) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(pair >> 16)); }
__device__ __forceinline__ uint32_t int4_of(const uint4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Lane groups and dwords of four transposed: lane group g's dword t becomes group t's dword g.
__device__ __forceinline__ uint4 int4_transpose(uint4 v) {
    auto a = __builtin_amdgcn_permlane32_swap(v.x, v.z, false, false);
    auto b = __builtin_amdgcn_permlane32_swap(v.y, v.w, false, false);
    auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return make_uint4(c[0], c[1], d[0], d[1]);
}

// NG: groups of a head; NT: tiles of 16 rows.  LDS rows of D / 2 bytes keep 16-byte chunk c of token
// t at c ^ kswz(t) (K) or c ^ vswz(t) (V), so that the tokens that an LDS cycle's lanes read fall on
// distinct banks.
template <int D> struct Int4Dim {
    static constexpr int RB = D / 2, CPR = RB / 16;   // row bytes, 16-byte chunks of a row
    static constexpr int RPI = 64 / CPR;              // rows of a copy instruction
    static constexpr int kswz(int t) { return D == 64 ? (t >> 4) & 1 : D == 128 ? (t >> 4) & 3 : ((t >> 1) & 1) | (((t >> 4) & 3) << 1); }
    static constexpr int vswz(int t) { return D == 64 ? (t >> 3) & 1 : D == 128 ? (t >> 2) & 3 : (t >> 1) & 7; }
};

template <int DT, int D, int NG, int NT>
__global__ __launch_bounds__(256, NT == 1 && D <= 128 ? 3 : 2) void int4_split_kernel(Int4Args a) {
    using L = Int4Dim<D>;
    constexpr bool BF = DT == PUTER_BF16;
    constexpr int RB = L::RB, KS = D / 32, DC = D / 16, GD = D / NG;
    constexpr int NV = L::CPR + NG;   // load instructions of a step's K, and of its V
    __shared__ __attribute__((aligned(1024))) char k_lds[4][64 * RB];
    __shared__ __attribute__((aligned(1024))) char v_lds[4][64 * RB];
    __shared__ __attribute__((aligned(16))) uint32_t kp_lds[4][NG * 64];
    __shared__ __attribute__((aligned(16))) uint32_t vp_lds[4][NG * 64];

    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Block order: consecutive ids go round-robin over the 8 XCDs; one XCD runs all kv heads (and
    // row tiles) of a chunk of tokens back to back, whose rows share its L2's lines.
    const int G = a.heads / a.kv_heads, R = G * a.query_len;
    const int KVR = a.kv_heads * a.row_tiles;
    const int id = blockIdx.x, kvr = (id >> 3) % KVR;
    const int kvh = kvr % a.kv_heads, row0 = (kvr / a.kv_heads) * 16 * NT;
    int64_t chunk = (int64_t)(id / (8 * KVR)) * 8 + (id & 7);
    int b = -1, split = 0;
    if (a.batch <= 256) {
        // the chunk-th (sequence, split) pair, the sequences in order: a prefix sum of their splits
        int64_t base = 0;
        for (int j0 = 0; j0 < a.batch; j0 += 64) {
            const int j = j0 + lane;
            const int ns = j < a.batch ? int4_splits(a, int4_context(a, j)) : 0;
            int incl = ns;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int t = __shfl_up(incl, o, 64);
                if (lane >= o) incl += t;
            }
            const int total = __shfl(incl, 63, 64);
            if (chunk < base + total) {
                const int lj = __builtin_ctzll(__ballot(base + incl > chunk));
                b = j0 + lj;
                split = (int)(chunk - base) - (__shfl(incl, lj, 64) - __shfl(ns, lj, 64));
                break;
            }
            base += total;
        }
    } else {
        b = (int)min(chunk / a.max_splits, (int64_t)a.batch);
        split = (int)(chunk % a.max_splits);
        if (b >= a.batch || split >= int4_splits(a, int4_context(a, b))) b = -1;
    }
    if (b < 0) return;   // the whole block
    b = __builtin_amdgcn_readfirstlane(b);
    split = __builtin_amdgcn_readfirstlane(split);
    const int ctx = __builtin_amdgcn_readfirstlane(int4_context(a, b));
    const int nsplit = int4_splits(a, ctx);
    const int t0 = split * a.split, t1 = min(ctx, t0 + a.split);

    // Q^T operands, dims in the order of the expanded codes; sums of q per group
    uint4 qb[NT][KS];
    float qsum[NT][NG];
    int lim[NT];   // the row's last visible token
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int row = row0 + 16 * nt + l16;
        const bool in = row < R;
        const int qi = in ? row / G : 0, g = in ? row - qi * G : 0;
        lim[nt] = ctx - a.query_len + qi;
        const uint16_t *q = a.q + (((int64_t)b * a.query_len + qi) * a.heads + (int64_t)kvh * G + g) * D;
#pragma unroll
        for (int g2 = 0; g2 < NG; ++g2) qsum[nt][g2] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            // the lane's eight dims of the step: with one group whole runs of its dims, else 8 of each 32
            const int d0 = NG == 1 ? (D / 4) * grp + 8 * ks : 32 * ks + 8 * grp;
            uint4 u = make_uint4(0, 0, 0, 0);
            if (in) u = *reinterpret_cast<const uint4 *>(q + d0);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
            float t = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t e = (w[k >> 1] >> (16 * (k & 1))) & 0xFFFFu;
                t += BF ? bf16_to_f32(e) : int4_lo(e);
            }
            qsum[nt][NG == 1 ? 0 : 32 * ks / GD] += t;
            // 0, 4, 1, 5, 2, 6, 3, 7
            qb[nt][ks] = make_uint4((w[0] & 0xFFFFu) | (w[2] << 16), (w[0] >> 16) | (w[2] & 0xFFFF0000u),
                                    (w[1] & 0xFFFFu) | (w[3] << 16), (w[1] >> 16) | (w[3] & 0xFFFF0000u));
        }
#pragma unroll
        for (int g2 = 0; g2 < NG; ++g2) {
            qsum[nt][g2] += __shfl_xor(qsum[nt][g2], 16, 64);
            qsum[nt][g2] += __shfl_xor(qsum[nt][g2], 32, 64);
        }
    }

    i4_f32x4 acc[NT][DC], bias[NT][NG];   // O[row 4 grp + r][16 c + l16] as sums of P (24 + n); sums of P 24
    float m[NT], l[NT], osum[NT][NG];     // row l16: reference maximum (log2), this lane's sums of p and p * offset
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt] = -INFINITY;
        l[nt] = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; ++g) osum[nt][g] = 0.0f, bias[nt][g] = (i4_f32x4){};
#pragma unroll
        for (int c = 0; c < DC; ++c) acc[nt][c] = (i4_f32x4){};
    }

    // step n of this wave: tokens t0 + 64 (wave + 4 n) .. + 63
    const int steps = (t1 - t0 + 63) / 64;
    const int mine = steps > wave ? (steps - wave + 3) / 4 : 0;
    auto first = [&](int n) __attribute__((always_inline)) { return t0 + 64 * (wave + 4 * n); };
    // the page of the lane's token (past the context: the last token's, not used), always one load
    auto page_of = [&](int n) __attribute__((always_inline)) {
        const int tok = min(first(n) + lane, ctx - 1);
        const int p = a.page_shift >= 0 ? tok >> a.page_shift : tok / a.page_size;
        return a.table[(int64_t)b * a.max_pages + p];
    };
    // the pool row of the lane's token; -1: past the context or a bad page id
    auto row_of = [&](int n, int page) __attribute__((always_inline)) {
        const int tok = first(n) + lane;
        const int p = a.page_shift >= 0 ? tok >> a.page_shift : tok / a.page_size;
        return tok < ctx && page >= 0 && page < a.num_pages ? page * a.page_size + (tok - p * a.page_size) : -1;
    };
    // a step's codes and pairs into the wave's LDS (hidden tokens read pool row 0)
    auto fetch = [&](const uint8_t *codes, const uint32_t *pairs, int row, char *dst, uint32_t *pdst, bool key) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < L::CPR; ++k) {
            const int t = L::RPI * k + lane / L::CPR;
            const int r = max(__shfl(row, t, 64), 0);
            const int chunk = (lane % L::CPR) ^ (key ? L::kswz(t) : L::vswz(t));
            __builtin_amdgcn_global_load_lds((i4_global *)(codes + ((int64_t)r * a.kv_heads + kvh) * RB + 16 * chunk),
                                             (i4_lds *)(dst + 1024 * k), 16, 0, 0);
        }
        const int64_t at = ((int64_t)max(row, 0) * a.kv_heads + kvh) * NG;
#pragma unroll
        for (int g = 0; g < NG; ++g)
            __builtin_amdgcn_global_load_lds((i4_global *)(pairs + at + g), (i4_lds *)(pdst + 64 * g), 4, 0, 0);
    };
    char *const kt = k_lds[wave], *const vt = v_lds[wave];
    uint32_t *const kpt = kp_lds[wave], *const vpt = vp_lds[wave];

    if (mine > 0) {
        int row = row_of(0, page_of(0));
        int next_page = page_of(1);
        fetch(a.kp, a.kpar, row, kt, kpt, true);
        fetch(a.vp, a.vpar, row, vt, vpt, false);
        for (int n = 0; n < mine; ++n) {
            const bool more = n + 1 < mine;
            int4_wait_loads<NV>();   // K is there
            const int page2 = page_of(n + 2);
            const uint64_t live = __ballot(row >= 0);
            const int tw0 = first(n);
            // token 16 grp + 4 i + r of the step stands at row 4 grp + r of score tile i
            i4_f32x4 s[NT][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int t = 16 * (l16 >> 2) + 4 * i + (l16 & 3);
                uint32_t kw[KS];
                if constexpr (D == 64 && NG == 1) {
                    const uint2 u = *reinterpret_cast<const uint2 *>(kt + t * RB + (((grp >> 1) ^ L::kswz(t)) << 4) + 8 * (grp & 1));
                    kw[0] = u.x, kw[1] = u.y;
                } else if constexpr (D == 64) {
#pragma unroll
                    for (int ks = 0; ks < 2; ++ks)
                        kw[ks] = *reinterpret_cast<const uint32_t *>(kt + t * RB + ((ks ^ L::kswz(t)) << 4) + 4 * grp);
                } else {
#pragma unroll
                    for (int h = 0; h < D / 128; ++h) {
                        uint4 u = *reinterpret_cast<const uint4 *>(kt + t * RB + (((4 * h + grp) ^ L::kswz(t)) << 4));
                        if constexpr (NG > 1) u = int4_transpose(u);
                        kw[4 * h] = u.x, kw[4 * h + 1] = u.y, kw[4 * h + 2] = u.z, kw[4 * h + 3] = u.w;
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][i] = (i4_f32x4){};
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint4 pr = *reinterpret_cast<const uint4 *>(kpt + 64 * g + 16 * grp + 4 * i);
                    uint4 kf[KS / NG];
#pragma unroll
                    for (int k = 0; k < KS / NG; ++k) kf[k] = int4_expand<BF>(kw[g * (KS / NG) + k]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float c0 = -24.0f * qsum[nt][g];
                        i4_f32x4 c = (i4_f32x4){c0, c0, c0, c0};
#pragma unroll
                        for (int k = 0; k < KS / NG; ++k) c = int4_mfma<BF>(kf[k], qb[nt][g * (KS / NG) + k], c);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const uint32_t p = int4_of(pr, r);
                            s[nt][i][r] = __builtin_fmaf(int4_lo(p), c[r], __builtin_fmaf(int4_hi(p), qsum[nt][g], s[nt][i][r]));
                        }
                    }
                    if constexpr (NG > 1) __builtin_amdgcn_sched_barrier(0);   // one group's pairs and codes live at a time
                }
            }
            int4_wait_lds();   // K's LDS is read
            int next_row = -1;
            if (more) {
                next_row = row_of(n + 1, next_page);
                fetch(a.kp, a.kpar, next_row, kt, kpt, true);
            }
            const bool full = live == ~0ull && tw0 + 63 <= ctx - a.query_len;
            const uint32_t lg = (uint32_t)(live >> (16 * grp)) & 0xFFFFu;
            uint32_t vis[NT];   // bit 4 i + r
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                vis[nt] = 0xFFFFu;
                if (!full) {
                    const int last = lim[nt] - tw0 - 16 * grp;   // relative to the lane's first token
                    vis[nt] = last < 0 ? 0u : last >= 15 ? lg : lg & ((2u << last) - 1u);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (!((vis[nt] >> (4 * i + r)) & 1)) s[nt][i][r] = -INFINITY;
                }
                float mx = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[nt][i][r]);
                mx *= a.scale_log2;
                // a reference stands until a score passes it by 2^8 (p stays below 256)
                if (__any(mx > m[nt] + 8.0f)) {
                    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                    const float mn = fmaxf(m[nt], mx);
                    const float alpha = m[nt] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[nt] - mn);
                    m[nt] = mn;
                    l[nt] *= alpha;
#pragma unroll
                    for (int g = 0; g < NG; ++g) osum[nt][g] *= alpha;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float f = __shfl(alpha, 4 * grp + r, 64);
#pragma unroll
                        for (int c = 0; c < DC; ++c) acc[nt][c][r] *= f;
#pragma unroll
                        for (int g = 0; g < NG; ++g) bias[nt][g][r] *= f;
                    }
                }
                const float mref = m[nt] == -INFINITY ? 0.0f : m[nt];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nt][i][r], a.scale_log2, -mref));
                        l[nt] += p;
                        s[nt][i][r] = p;
                    }
            }
            if (more) int4_wait_loads<NV>();   // V is there
            else int4_wait_loads<0>();
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint4 pr[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) pr[i] = *reinterpret_cast<const uint4 *>(vpt + 64 * g + 16 * grp + 4 * i);
                i4_bf16x8 ph[NT][2], pl[NT][2];   // slot order as the codes': tokens 0, 4, 1, 5, ..
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            uint32_t p = int4_of(pr[i], r);
                            if (!full) p = ((vis[nt] >> (4 * i + r)) & 1) ? p : 0u;   // what is hidden may hold anything
                            const float w = s[nt][i][r] * int4_lo(p);
                            osum[nt][g] = __builtin_fmaf(s[nt][i][r], int4_hi(p), osum[nt][g]);
                            const __bf16 hi = (__bf16)w;
                            ph[nt][i >> 1][2 * r + (i & 1)] = hi;
                            if constexpr (!BF) pl[nt][i >> 1][2 * r + (i & 1)] = (__bf16)(w - (float)hi);
                        }
                const uint4 b24 = make_uint4(0x41C041C0u, 0x41C041C0u, 0x41C041C0u, 0x41C041C0u);
                auto product = [&](int nt, int st, uint4 vf, i4_f32x4 c) __attribute__((always_inline)) {
                    c = int4_mfma<true>(__builtin_bit_cast(uint4, ph[nt][st]), vf, c);
                    if constexpr (!BF) c = int4_mfma<true>(__builtin_bit_cast(uint4, pl[nt][st]), vf, c);
                    return c;
                };
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int st = 0; st < 2; ++st) bias[nt][g] = product(nt, st, b24, bias[nt][g]);
#pragma unroll
                for (int c = g * (GD / 16); c < (g + 1) * (GD / 16); ++c) {
                    const int t = 16 * grp + l16;
                    const i4_i32x2 v = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
                        (i4_lds_i32x2 *)(vt + t * RB + (((c >> 1) ^ L::vswz(t)) << 4) + 8 * (c & 1)));
#pragma unroll
                    for (int st = 0; st < 2; ++st) {
                        const uint4 vf = int4_expand<true>((uint32_t)v[st]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) acc[nt][c] = product(nt, st, vf, acc[nt][c]);
                    }
                }
                if constexpr (NG > 1) __builtin_amdgcn_sched_barrier(0);
            }
            if (more) {
                int4_wait_lds();   // V's LDS is read
                fetch(a.vp, a.vpar, next_row, vt, vpt, false);
            }
            row = next_row;
            next_page = page2;
        }
    }

    // sums over the lane groups; O of the plain codes, offsets added
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        l[nt] += __shfl_xor(l[nt], 16, 64);
        l[nt] += __shfl_xor(l[nt], 32, 64);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            osum[nt][g] += __shfl_xor(osum[nt][g], 16, 64);
            osum[nt][g] += __shfl_xor(osum[nt][g], 32, 64);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float o = __shfl(osum[nt][g], 4 * grp + r, 64) - bias[nt][g][r];
#pragma unroll
                for (int c = g * (GD / 16); c < (g + 1) * (GD / 16); ++c) acc[nt][c][r] += o;
            }
    }
    // the four waves joined: 1 into 0 and 3 into 2, then 2 into 0 (each lane the same lane's values)
    __shared__ float ml_lds[4][NT][16][2];
    __syncthreads();
    if (grp == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            ml_lds[wave][nt][l16][0] = m[nt];
            ml_lds[wave][nt][l16][1] = l[nt];
        }
    }
    __syncthreads();
    float M[NT][4], Lsum[NT][4];   // of row 4 grp + r
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 4 * grp + r;
            float mm = -INFINITY, ll = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ml_lds[w][nt][row][0]);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float mw = ml_lds[w][nt][row][0];
                if (mw != -INFINITY) ll += ml_lds[w][nt][row][1] * __builtin_amdgcn_exp2f(mw - mm);
            }
            const float own = ml_lds[wave][nt][row][0];
            const float f = own == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(own - mm);
            M[nt][r] = mm;
            Lsum[nt][r] = ll;
#pragma unroll
            for (int c = 0; c < DC; ++c) acc[nt][c][r] = own == -INFINITY ? 0.0f : acc[nt][c][r] * f;
        }
    float *const buf = reinterpret_cast<float *>(wave < 2 ? &k_lds[0][0] : &v_lds[0][0]);
    auto put = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < DC; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) buf[((nt * DC + c) * 4 + r) * 64 + lane] = acc[nt][c][r];
    };
    auto add = [&](const float *from) __attribute__((always_inline)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < DC; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[nt][c][r] += from[((nt * DC + c) * 4 + r) * 64 + lane];
    };
    if (wave & 1) put();
    __syncthreads();
    if (!(wave & 1)) add(buf);
    __syncthreads();
    if (wave == 2) put();
    __syncthreads();
    if (wave != 0) return;
    add(reinterpret_cast<const float *>(&v_lds[0][0]));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = row0 + 16 * nt + 4 * grp + r;
            if (row >= R) continue;
            const int qi = row / G;
            const int64_t at = ((int64_t)b * a.query_len + qi) * a.heads + (int64_t)kvh * G + (row - qi * G);
            if (nsplit == 1) {
                const float inv = Lsum[nt][r] == 0.0f ? 0.0f : 1.0f / Lsum[nt][r];
#pragma unroll
                for (int c = 0; c < DC; ++c) a.out[at * D + 16 * c + l16] = Elem<DT>::store(acc[nt][c][r] * inv);
            } else {
                const int64_t slot = at * a.max_splits + split;
#pragma unroll
                for (int c = 0; c < DC; ++c) a.part_o[slot * D + 16 * c + l16] = acc[nt][c][r];
                if (l16 == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * slot) = make_float2(M[nt][r], Lsum[nt][r]);
            }
        }
}

// Joins the splits of a row, in order: a block per row, a thread per dim, eight splits' loads at a time.
template <int DT, int D>
__global__ __launch_bounds__(D) void int4_join_kernel(Int4Args a) {
    const int64_t at = blockIdx.x;
    const int b = (int)(at / ((int64_t)a.query_len * a.heads)), d = threadIdx.x;
    const int nsplit = int4_splits(a, int4_context(a, b));
    if (nsplit == 1) return;   // stored already
    const float2 *ml = reinterpret_cast<const float2 *>(a.part_ml) + at * a.max_splits;
    const float *po = a.part_o + at * a.max_splits * D + d;
    float M = -INFINITY, Ls = 0.0f, O = 0.0f;
    for (int s0 = 0; s0 < nsplit; s0 += 8) {
        float2 mv[8];
        float ov[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const bool in = s0 + u < nsplit;
            mv[u] = in ? ml[s0 + u] : make_float2(-INFINITY, 0.0f);
            ov[u] = in ? po[(int64_t)(s0 + u) * D] : 0.0f;
        }
        float mb = M;
#pragma unroll
        for (int u = 0; u < 8; ++u) mb = fmaxf(mb, mv[u].x);
        if (mb == -INFINITY) {   // no score so far (or NaN alone)
#pragma unroll
            for (int u = 0; u < 8; ++u) Ls += mv[u].y, O += ov[u];
            continue;
        }
        const float fo = M == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - mb);
        Ls *= fo;
        O *= fo;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const float f = mv[u].x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mv[u].x - mb);
            Ls += mv[u].y * f;
            O += ov[u] * f;
        }
        M = mb;
    }
    a.out[at * D + d] = Elem<DT>::store(Ls == 0.0f ? 0.0f : O / Ls);
}

// Tokens of a split: enough of them that the blocks fill the chip's CUs several times over, and
// no more, since each split's partials are written and read back.
static int int4_split_tokens(int64_t batch, int64_t row_tiles, int64_t kv_heads, int64_t max_context) {
    const int64_t blocks = batch * row_tiles * kv_heads * ((max_context + 255) / 256);
    return (int)(256 * std::max<int64_t>(1, std::min<int64_t>(blocks / 4096, 16)));
}
// 16 rows a tile, two tiles a block where there are more (at 256 dims the second's registers would spill)
static int64_t int4_row_tiles(int64_t rows, int64_t dim) { return rows <= 16 || dim > 128 ? (rows + 15) / 16 : (rows + 31) / 32; }

template <int DT, int D, int NG> static void launch_int4(const Int4Args &a, int64_t blocks, hipStream_t s) {
    if (D > 128 || a.query_len * (a.heads / a.kv_heads) <= 16) int4_split_kernel<DT, D, NG, 1><<<(unsigned)blocks, 256, 0, s>>>(a);
    else int4_split_kernel<DT, D, NG, D <= 128 ? 2 : 1><<<(unsigned)blocks, 256, 0, s>>>(a);
    if (a.max_splits > 1)
        int4_join_kernel<DT, D><<<(unsigned)((int64_t)a.batch * a.query_len * a.heads), D, 0, s>>>(a);
}
template <int DT> static void launch_int4_dim(const Int4Args &a, int dim, int group, int64_t blocks, hipStream_t s) {
    switch (1000 * dim + group) {
    case 64064: launch_int4<DT, 64, 1>(a, blocks, s); break;
    case 64032: launch_int4<DT, 64, 2>(a, blocks, s); break;
    case 128128: launch_int4<DT, 128, 1>(a, blocks, s); break;
    case 128064: launch_int4<DT, 128, 2>(a, blocks, s); break;
    case 128032: launch_int4<DT, 128, 4>(a, blocks, s); break;
    case 256128: launch_int4<DT, 256, 2>(a, blocks, s); break;
    case 256064: launch_int4<DT, 256, 4>(a, blocks, s); break;
    case 256032: launch_int4<DT, 256, 8>(a, blocks, s); break;
    }
}

}  // namespace puter

using namespace puter;

extern "C" {

size_t puter_hip_paged_int4_workspace_bytes(int64_t batch, int64_t query_len, int64_t num_heads, int64_t kv_heads,
                                            int64_t head_dim, int64_t max_context) {
    if (batch <= 0 || query_len <= 0 || num_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_context <= 0) return 0;
    const int64_t tiles = int4_row_tiles(num_heads / kv_heads * query_len, head_dim);
    const int64_t split = int4_split_tokens(batch, tiles, kv_heads, max_context), splits = (max_context + split - 1) / split;
    return splits > 1 ? (size_t)(batch * query_len * num_heads * splits * (head_dim + 2)) * sizeof(float) : 16;
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
    const int64_t G = num_heads / kv_heads, tiles = int4_row_tiles(G * query_len, head_dim);
    Int4Args a{};
    a.q = static_cast<const uint16_t *>(query);
    a.kp = static_cast<const uint8_t *>(key_pages), a.vp = static_cast<const uint8_t *>(value_pages);
    a.kpar = static_cast<const uint32_t *>(key_params), a.vpar = static_cast<const uint32_t *>(value_params);
    a.table = page_table, a.ctx = context_lens, a.out = static_cast<uint16_t *>(output);
    a.split = int4_split_tokens(batch, tiles, kv_heads, max_context);
    a.max_splits = (int)((max_context + a.split - 1) / a.split);
    a.part_o = static_cast<float *>(workspace);
    a.part_ml = a.part_o + batch * query_len * num_heads * a.max_splits * head_dim;
    a.max_pages = max_pages_per_seq;
    a.batch = (int)batch, a.page_size = (int)page_size, a.num_pages = (int)num_pages;
    a.max_context = num_pages > 0 ? (int)max_context : 0;   // an empty pool: every sequence is empty
    a.page_shift = -1;
    if ((page_size & (page_size - 1)) == 0) a.page_shift = __builtin_ctzll((unsigned long long)page_size);
    a.query_len = (int)query_len, a.heads = (int)num_heads, a.kv_heads = (int)kv_heads, a.row_tiles = (int)tiles;
    a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)head_dim));
    const int64_t chunks = (batch * a.max_splits + 7) / 8 * 8, blocks = chunks * kv_heads * tiles;
    if (blocks > 0x7FFFFFFF || batch * query_len * num_heads > 0x7FFFFFFF) return fail(PUTER_ERR_INVALID, "paged int4: grid too large");
    hipStream_t s = as_stream(stream);
    if (dtype == PUTER_BF16) launch_int4_dim<PUTER_BF16>(a, (int)head_dim, (int)group, blocks, s);
    else launch_int4_dim<PUTER_F16>(a, (int)head_dim, (int)group, blocks, s);
    return check_launch("paged int4");
}

}  // extern "C"
