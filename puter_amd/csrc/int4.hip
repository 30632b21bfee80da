// Attention over a paged cache held in 4 bits: one or a few query tokens per sequence, grouped
// heads (the reference gathers the pages and runs MultiHeadAttention: execution/page_intrinsic.go:
// 217-352, device/cpu/attention/typed_compute.go:142-237).  A cached value is scale * n + offset
// with the 4-bit code n in [-8, 7] and the (scale, offset) pair of its token, kv head and group of
// dims.  Query i of a sequence of `context` cached tokens and m queries sees the tokens up to
// context - m + i.
//
// Work: a sequence's cache is walked in steps of 64 tokens, once per kv head and tile of up to 16 of
// the (query, head) rows that share the kv head.  All steps of the call stand in one line ([sequence]
// [row tile][head group][step]) that is cut evenly among the workers of a grid that just fills the
// chip, whatever the sequences' lengths.  A worker is 1, 2 or 4 neighbouring waves, one to a kv head
// of the head group, so the heads' short rows (32 to 128 bytes) are read as whole cache lines; each
// wave keeps a running maximum and sum of its own, and reads no other's LDS.  A sequence that lies
// in one worker is stored at once; the others leave (max, sum, row) partials, two a wave at most,
// that a second kernel joins.
//   loads: codes, pairs and page ids go from HBM straight to the wave's LDS, whole rows to an
//     instruction, into a ring of three tiles (K, V, K, ..): while one is computed on, the next two
//     are under way.  The copies are written in assembly, and waited for by count: of the compiler's
//     own LDS copies each LDS read waited for all, next tiles included.
//   scores: S^T[token, row] = K . Q^T on v_mfma_f32_16x16x32.  A code becomes a 16-bit operand in
//     two instructions for two codes: shifted to the mantissa's top and joined with the exponent of
//     16 it reads 24 + n, exactly; the accumulator starts at -24 sum(q), so the product is of n.
//     Scale and offset act on the f32 product of each group: s = sum_g scale C_g + offset sum_g(q).
//   values: O[row, dim] = P . V, V's columns read out of the row-major codes by ds_read_b64_tr_b4
//     (16 tokens of one dim to a lane), P scaled by the token's scale of the group before it is
//     rounded.  Offsets are summed in f32; the 24 that each code reads too much is taken off by one
//     more product of the same P with 24.
// What bounds it, and what it measured (8 kv heads of 128 dims, groups of 128, bf16): 64 tokens over 512
// to 8192 each, 303 MB of cache, 73 us in all, the walk 68 (4.5 TB/s): the stream, beside 550 vector instructions a step, half of which widen
// codes; the copies alone took 67 before the heads were kept in step.  By the clock of its waves: first codes
// 5 us after the start (contexts, table, codes: one behind the other), then a step at the stream's rate.  Three waves a SIMD (168 registers)
// where one group of 128 dims or heads of 64 allow it, else two (one at 256 dims).  Few steps a wave leave the chain of table, codes,
// scores and partials: 10.6 us for one token over 777.
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
typedef __attribute__((address_space(3))) char i4_lds;

struct Int4Args {
    const uint16_t *q;
    const uint8_t *kp, *vp;
    const uint32_t *kpar, *vpar;
    const int32_t *table, *ctx;
    uint16_t *out;
    float *part_o, *part_ml;
    int2 *starts;   // per sequence: where its steps begin in the line of all, how many; then the line's length
    int64_t max_pages;
    int batch, page_size, page_shift, num_pages, max_context;   // page_shift: log2 of a power of two, else -1
    int query_len, heads, kv_heads, row_tiles, head_group, workers, part_rows;   // part_rows: rows of a wave's partial
    float scale_log2;
};

// a sequence's tokens and its steps (one at least: it stores the zeros of an empty cache)
__device__ __forceinline__ int int4_context(const Int4Args &a, int b) { return max(0, min(a.ctx[b], a.max_context)); }
__device__ __forceinline__ int int4_steps(int ctx) { return max(1, (ctx + 63) / 64); }

// The line of all steps (`per` of them for each step of a sequence's walk), and where in it a
// sequence or a step lies.  One sequence to a lane, 64 at a time.
struct Int4Line {
    int ctx, n, incl;   // this lane's sequence: tokens, steps, steps up to and with it
    int total;          // the line's length
    __device__ __forceinline__ void scan(const Int4Args &a, int j0) {
        const int j = j0 + (int)(threadIdx.x & 63);
        ctx = j < a.batch ? int4_context(a, j) : 0;
        n = j < a.batch ? int4_steps(ctx) : 0;
        incl = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(incl, o, 64);
            if ((int)(threadIdx.x & 63) >= o) incl += t;
        }
    }
    __device__ __forceinline__ Int4Line(const Int4Args &a, int per) {
        scan(a, 0);
        total = __shfl(incl, 63, 64);
        if (a.batch > 64) {   // (the lanes keep the last 64: find() scans again)
            for (int j0 = 64; j0 < a.batch; j0 += 64) {
                scan(a, j0);
                total += __shfl(incl, 63, 64);
            }
        }
        total = __builtin_amdgcn_readfirstlane(total * per);
    }
    // the sequence of step u and its tokens; the line's steps before it
    __device__ __forceinline__ int find(const Int4Args &a, int per, int u, int &seq, int &tokens) {
        const int lane = threadIdx.x & 63;
        int before = 0;
        for (int j0 = 0; j0 < a.batch; j0 += 64) {
            if (a.batch > 64) scan(a, j0);
            const uint64_t here = __ballot(j0 + lane < a.batch && (before + incl) * per > u);
            if (here) {
                const int at = __builtin_ctzll(here);
                seq = __builtin_amdgcn_readfirstlane(j0 + at);
                tokens = __builtin_amdgcn_readlane(ctx, at);
                return (before + __builtin_amdgcn_readlane(incl, at) - __builtin_amdgcn_readlane(n, at)) * per;
            }
            before += __builtin_amdgcn_readlane(incl, 63);
        }
        seq = tokens = 0;
        return 0;
    }
    // for the join: every sequence's first step in the line and steps, and (at the batch's end) the total
    __device__ __forceinline__ void publish(const Int4Args &a, int per) {
        const int lane = threadIdx.x & 63;
        int before = 0;
        for (int j0 = 0; j0 < a.batch; j0 += 64) {
            if (a.batch > 64) scan(a, j0);
            if (j0 + lane < a.batch) a.starts[j0 + lane] = make_int2((before + incl - n) * per, n);
            before += __builtin_amdgcn_readlane(incl, 63);
        }
        if (lane == 0) a.starts[a.batch] = make_int2(total, 0);
    }
};
// The line cut among the workers: the first `more` take each + 1 steps, the others each.
struct Int4Cut {
    int workers, each, more;
    __device__ __forceinline__ Int4Cut(int limit, int total) : workers(min(limit, total)) {
        each = total / workers;
        more = total - each * workers;
    }
    __device__ __forceinline__ int start(int w) const { return w * each + min(w, more); }
    __device__ __forceinline__ int worker(int u) const {
        const int big = more * (each + 1);
        return u < big ? u / (each + 1) : more + (u - big) / each;
    }
};

// HBM -> LDS copies: 16 or 4 bytes a lane to lds + 16 or 4 bytes x lane.
__device__ __forceinline__ void int4_copy16(const void *from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds) : "memory");
}
__device__ __forceinline__ void int4_copy4(const void *from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(lds) : "memory");
}
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

__device__ __forceinline__ void int4_priority(int p) {   // wave-uniform, 0 to 2
    if (p == 0) __builtin_amdgcn_s_setprio(0);
    else if (p == 1) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(2);
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
__device__ __forceinline__ float int4_of(const float4 &v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Lane groups and dwords of four transposed: lane group g's dword t becomes group t's dword g.
__device__ __forceinline__ uint4 int4_transpose(uint4 v) {
    auto a = __builtin_amdgcn_permlane32_swap(v.x, v.z, false, false);
    auto b = __builtin_amdgcn_permlane32_swap(v.y, v.w, false, false);
    auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    return make_uint4(c[0], c[1], d[0], d[1]);
}

// LDS rows of D / 2 bytes, one a token, keep 16-byte chunk c of token t at c ^ swz(t): both the 16
// consecutive tokens of a score tile and the tokens 16 a + 4 g + b (a, b < 4) of a transposing read
// fall on distinct banks.
template <int D> struct Int4Dim {
    static constexpr int RB = D / 2, CPR = RB / 16;   // row bytes, 16-byte chunks of a row
    static constexpr int RPI = 64 / CPR;              // rows of a copy instruction
    static constexpr int swz(int t) {
        return D == 64 ? ((t >> 3) ^ (t >> 4) ^ (t >> 5)) & 1 : D == 128 ? ((t >> 2) ^ (t >> 4)) & 3
                                                                           : (((t >> 1) & 1) | ((((t >> 2) ^ (t >> 4)) & 3) << 1));
    }
};

// Blocks of the walk on a CU, by their registers and LDS.
constexpr int int4_blocks_per_cu(int dim, int groups) { return dim > 128 ? 1 : groups == 1 || dim == 64 ? 3 : 2; }

// NG: groups of a head.
template <int DT, int D, int NG>
__global__ __launch_bounds__(256, int4_blocks_per_cu(D, NG)) void int4_walk_kernel(Int4Args a) {
    using L = Int4Dim<D>;
    constexpr bool BF = DT == PUTER_BF16;
    // Row tiles a wave.  Two share the widening of the codes, but up to 100 of their registers spill and two
    // waves a SIMD are left: 16 x 5 queries of 4 heads over 3000 tokens of 128 dims 37, 43 and 57 us in
    // groups of 128, 64 and 32, one at a time 35, 37 and 40; over 6000 tokens 48 and 50, and at 128 rows over
    // 60000, the most that two gained, 52 and 59.
    constexpr int NT = 1;
    constexpr int RB = L::RB, KS = D / 32, DC = D / 16, GD = D / NG;
    constexpr int NP = NG >= 4 ? NG / 4 : NG, NV = L::CPR + NP;   // copies of a tile's pairs; of a tile
    constexpr int TILE = 64 * RB + 256 * NG;                      // codes, then pairs
    __shared__ __attribute__((aligned(1024))) char ring_lds[4][3 * TILE];
    // Up to two groups the pairs are read as they are, four tokens' of a group at once; more stand by
    // token, and are laid out as f32 [scale, offset][group][token] first
    constexpr bool WIDE = NG > 2;
    __shared__ __attribute__((aligned(16))) float pair_lds[WIDE ? 4 : 1][2][WIDE ? NG * 64 : 1];
    __shared__ __attribute__((aligned(16))) int32_t page_lds[4][64];

    const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, grp = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // The oldest of a SIMD's waves goes first, so of the blocks that share a CU the first to come was done
    // at 41 us and the third at 57 (12 steps each).  Their waves take turns at going first, a step at a
    // time, the youngest to begin with: 74.5 -> 73 us and 31.2 -> 30.4 (64 sequences, three long ones).
    constexpr int TURNS = int4_blocks_per_cu(D, NG);
    int turn = blockIdx.x >> 8;
    if constexpr (TURNS > 1) int4_priority(turn);
    const int G = a.heads / a.kv_heads, R = G * a.query_len;
    const int groups = a.kv_heads / a.head_group;   // head groups
    const int worker = blockIdx.x * (4 / a.head_group) + wave / a.head_group, member = wave % a.head_group;
    const int pairs = groups * a.row_tiles;         // (row tile, head group) pairs of a sequence

    int seq;
    Int4Line line(a, pairs);
    const Int4Cut cut(a.workers, line.total);
    if (worker >= cut.workers) return;
    // Four neighbouring heads' waves share the lines of a token's row (64 bytes of 128 each at D 128), but
    // the copies in flight are several times the L1: apart by a step, each fetches the line for itself.
    // Of one worker, they walk the same steps, so a barrier can keep them together.  64 sequences of 512 to 8192
    // tokens, 8 kv heads: 79 -> 74 us; runs of a step or two lose 1 %, and go without.
    const bool together = a.head_group == 4 && cut.each >= 4;
    const int line0 = cut.start(worker);
    int left = cut.start(worker + 1) - line0;
    int ctx;
    const int base = line.find(a, pairs, line0, seq, ctx);
    if (worker == 0 && member == 0) line.publish(a, pairs);
    int nsteps = int4_steps(ctx);
    int pair = (line0 - base) / nsteps;
    int step0 = (line0 - base) - pair * nsteps;
    int slot = 0;   // of a partial: 0 for a piece at the start of the worker's run, else 1

    char *const ring = ring_lds[wave];
    const uint32_t ring_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(i4_lds *)ring);
    const uint32_t page_at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(i4_lds *)&page_lds[wave][0]);
    float *const sct = pair_lds[WIDE ? wave : 0][0], *const oft = pair_lds[WIDE ? wave : 0][1];
    for (;;) {
        const int step1 = min(nsteps, step0 + left);
        const int kvh = (pair % groups) * a.head_group + member, row0 = (pair / groups) * 16 * NT;

        // Q^T operands: loaded here; under the first copies put in the order of the expanded codes'
        // dims and summed per group
        uint4 qb[NT][KS];
        float qsum[NT][NG];
        int lim[NT];   // the row's last visible token
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int row = row0 + 16 * nt + l16;
            const bool in = row < R;
            const int qi = in ? row / G : 0, g = in ? row - qi * G : 0;
            lim[nt] = ctx - a.query_len + qi;
            const uint16_t *q = a.q + (((int64_t)seq * a.query_len + qi) * a.heads + (int64_t)kvh * G + g) * D;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                // the lane's eight dims of the step: with one group whole runs of its dims, else 8 of each 32
                const int d0 = NG == 1 ? (D / 4) * grp + 8 * ks : 32 * ks + 8 * grp;
                qb[nt][ks] = make_uint4(0, 0, 0, 0);
                if (in) qb[nt][ks] = *reinterpret_cast<const uint4 *>(q + d0);
            }
        }
        auto prepare_q = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int g = 0; g < NG; ++g) qsum[nt][g] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const uint32_t w[4] = {qb[nt][ks].x, qb[nt][ks].y, qb[nt][ks].z, qb[nt][ks].w};
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
                for (int g = 0; g < NG; ++g) {
                    qsum[nt][g] += __shfl_xor(qsum[nt][g], 16, 64);
                    qsum[nt][g] += __shfl_xor(qsum[nt][g], 32, 64);
                }
            }
        };

        // O[row 4 grp + r][16 c + l16] as sums of P (24 + n); sums of P 24 of group l16
        i4_f32x4 acc[NT][DC], bias[NT];
        float m[NT], l[NT], osum[NT][NG];     // row l16: reference maximum (log2), this lane's sums of p and p * offset
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt] = -INFINITY;
            l[nt] = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; ++g) osum[nt][g] = 0.0f;
            bias[nt] = (i4_f32x4){};
#pragma unroll
            for (int c = 0; c < DC; ++c) acc[nt][c] = (i4_f32x4){};
        }

        // the table entry of the lane's token of a step (past the context: the last token's, not used)
        auto entry_of = [&](int step) __attribute__((always_inline)) {
            const int tok = min(64 * step + lane, ctx - 1);
            const int p = a.page_shift >= 0 ? tok >> a.page_shift : tok / a.page_size;
            return a.table + (seq * a.max_pages + p);
        };
        // the pool row of the lane's token; -1: past the context or a bad page id
        auto row_of = [&](int step, int page) __attribute__((always_inline)) {
            const int tok = 64 * step + lane;
            const int in_page = a.page_shift >= 0 ? tok & (a.page_size - 1) : tok % a.page_size;
            return tok < ctx && page >= 0 && page < a.num_pages ? page * a.page_size + in_page : -1;
        };
        // a step's codes and pairs into a tile of the ring (hidden tokens read pool row 0)
        auto fetch = [&](const uint8_t *codes, const uint32_t *prs, int row, uint32_t tile) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < L::CPR; ++k) {
                const int t = L::RPI * k + lane / L::CPR;
                const uint32_t r = (uint32_t)max(__shfl(row, t, 64), 0);
                const uint64_t off = (uint64_t)r * (uint32_t)(a.kv_heads * RB) + (uint32_t)(kvh * RB + 16 * ((lane % L::CPR) ^ L::swz(t)));
                int4_copy16(codes + off, ring_at + tile + 1024 * k);
            }
            const uint32_t *p = prs + (uint64_t)(uint32_t)max(row, 0) * (uint32_t)(a.kv_heads * NG) + (uint32_t)(kvh * NG);
#pragma unroll
            for (int k = 0; k < NP; ++k) {
                if constexpr (NG >= 4) int4_copy16(p + 4 * k, ring_at + tile + 64 * RB + 1024 * k);   // [k][token][4]
                else int4_copy4(p + k, ring_at + tile + 64 * RB + 256 * k);                          // [group][token]
            }
        };
        auto pairs_of = [&](const char *tile, uint32_t (&pr)[NG]) __attribute__((always_inline)) {   // of the lane's token
            const uint32_t *p = reinterpret_cast<const uint32_t *>(tile + 64 * RB);
            if constexpr (NG >= 4) {
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(p + 256 * k + 4 * lane);
                    pr[4 * k] = v.x, pr[4 * k + 1] = v.y, pr[4 * k + 2] = v.z, pr[4 * k + 3] = v.w;
                }
            } else {
#pragma unroll
                for (int k = 0; k < NP; ++k) pr[k] = p[64 * k + lane];
            }
        };

        if (ctx > 0) {
            int row = row_of(step0, *entry_of(step0));
            int row1 = row_of(step0 + 1, *entry_of(step0 + 1));
            // Order of the copies, for the counts below: the table entries of step n + 3 and K of
            // n + 2 at the end of step n; V of n + 1 after the scores of n
            int4_wait_lds();       // (the segment before has read its last)
            int4_wait_loads<0>();
            uint32_t tk = 0, tv = TILE, tn = 2 * TILE;   // tiles of K and V of this step, and of K of the next
            fetch(a.kp, a.kpar, row, tk);
            fetch(a.vp, a.vpar, row, tv);
            if (step0 + 1 < step1) {
                int4_copy4(entry_of(step0 + 2), page_at);
                fetch(a.kp, a.kpar, row1, tn);
            }
            prepare_q();
            for (int step = step0; step < step1; ++step) {
                const bool more = step + 1 < step1;
                if constexpr (TURNS > 1) {
                    turn = turn == 0 ? TURNS - 1 : turn - 1;
                    int4_priority(turn);
                }
                if (more) int4_wait_loads<2 * NV + 1>();   // K is there
                else int4_wait_loads<NV>();
                const char *const kt = ring + tk, *const vt = ring + tv;
                const uint64_t live = __ballot(row >= 0);
                if constexpr (WIDE) {
                    uint32_t pr[NG];
                    pairs_of(kt, pr);
#pragma unroll
                    for (int g = 0; g < NG; ++g) {   // (the offset less what the 24 of the codes adds)
                        sct[64 * g + lane] = int4_lo(pr[g]);
                        oft[64 * g + lane] = __builtin_fmaf(-24.0f, int4_lo(pr[g]), int4_hi(pr[g]));
                    }
                }
                // Token 16 i + 4 grp + r of the step stands at row 4 grp + r of score tile i.  A tile's and
                // group's products are scaled and summed under the next one's; summed there and then (the
                // empty asm), since put off they would all stay live, and spill.
                i4_f32x4 s[NT][4], prod[2][NT];
                float4 sc[2], of[2];
                uint4 pr[2];
                auto scaled = [&](int i, int g, int u) __attribute__((always_inline)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float c = prod[u][nt][r], before = g == 0 ? 0.0f : s[nt][i][r];
                            if constexpr (WIDE)
                                s[nt][i][r] = __builtin_fmaf(int4_of(sc[u], r), c, __builtin_fmaf(int4_of(of[u], r), qsum[nt][g], before));
                            else
                                s[nt][i][r] = __builtin_fmaf(int4_lo(int4_of(pr[u], r)), c, __builtin_fmaf(int4_hi(int4_of(pr[u], r)), qsum[nt][g], before));
                        }
                        asm volatile("" : "+v"(s[nt][i]));
                    }
                };
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = 16 * i + l16;
                    uint32_t kw[KS];
                    if constexpr (D == 64 && NG == 1) {
                        const uint2 u = *reinterpret_cast<const uint2 *>(kt + t * RB + (((grp >> 1) ^ L::swz(t)) << 4) + 8 * (grp & 1));
                        kw[0] = u.x, kw[1] = u.y;
                    } else if constexpr (D == 64) {
#pragma unroll
                        for (int ks = 0; ks < 2; ++ks)
                            kw[ks] = *reinterpret_cast<const uint32_t *>(kt + t * RB + ((ks ^ L::swz(t)) << 4) + 4 * grp);
                    } else {
#pragma unroll
                        for (int h = 0; h < D / 128; ++h) {
                            uint4 u = *reinterpret_cast<const uint4 *>(kt + t * RB + (((4 * h + grp) ^ L::swz(t)) << 4));
                            if constexpr (NG > 1) u = int4_transpose(u);
                            kw[4 * h] = u.x, kw[4 * h + 1] = u.y, kw[4 * h + 2] = u.z, kw[4 * h + 3] = u.w;
                        }
                    }
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const int u = (i * NG + g) & 1;
                        if constexpr (WIDE) {
                            sc[u] = *reinterpret_cast<const float4 *>(sct + 64 * g + 16 * i + 4 * grp);
                            of[u] = *reinterpret_cast<const float4 *>(oft + 64 * g + 16 * i + 4 * grp);
                        } else {
                            pr[u] = *reinterpret_cast<const uint4 *>(kt + 64 * RB + 256 * g + 64 * i + 16 * grp);
                        }
                        uint4 kf[KS / NG];
#pragma unroll
                        for (int k = 0; k < KS / NG; ++k) kf[k] = int4_expand<BF>(kw[g * (KS / NG) + k]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float c0 = WIDE ? 0.0f : -24.0f * qsum[nt][g];
                            prod[u][nt] = (i4_f32x4){c0, c0, c0, c0};
#pragma unroll
                            for (int k = 0; k < KS / NG; ++k) prod[u][nt] = int4_mfma<BF>(kf[k], qb[nt][g * (KS / NG) + k], prod[u][nt]);
                        }
                        if (i + g > 0) scaled(g ? i : i - 1, g ? g - 1 : NG - 1, u ^ 1);
                    }
                }
                scaled(3, NG - 1, (4 * NG - 1) & 1);
                int4_wait_lds();   // K's LDS is read
                if (together) __builtin_amdgcn_s_barrier();
                if (more) fetch(a.vp, a.vpar, row1, tk);   // V of the next step into K's tile
                const bool full = live == ~0ull && 64 * step + 63 <= ctx - a.query_len;
                uint32_t vis[NT];   // bit 4 i + r: the row sees the token
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    vis[nt] = 0xFFFFu;
                    if (!full) {
                        asm volatile("; masked step");   // (a branch: as selects it would cost every step)
                        const uint64_t lg = live >> (4 * grp);
                        const int last = lim[nt] - 64 * step - 4 * grp;   // relative to the lane's first token
                        vis[nt] = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const bool v = ((lg >> (16 * i + r)) & 1) && 16 * i + r <= last;
                                vis[nt] |= (uint32_t)v << (4 * i + r);
                                s[nt][i][r] = v ? s[nt][i][r] : -INFINITY;
                            }
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
                            bias[nt][r] *= f;
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
                if (more) int4_wait_loads<2 * NV>();   // V is there, and the table entries of step n + 2
                else int4_wait_loads<0>();
                uint32_t vpr[NG];
                pairs_of(vt, vpr);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    // a pair that is not finite, or of no token: zeros, whose products with any P are zero;
                    // the rows that see such a token get their NaN with the offsets
                    const bool fine = row >= 0 && (vpr[g] & 0x7C00u) != 0x7C00u && (vpr[g] >> 16 & 0x7C00u) != 0x7C00u;
                    if constexpr (WIDE) {
                        sct[64 * g + lane] = fine ? int4_lo(vpr[g]) : 0.0f;
                        oft[64 * g + lane] = fine ? int4_hi(vpr[g]) : 0.0f;
                    } else if (__any(!fine)) {
                        *reinterpret_cast<uint32_t *>(ring + tv + 64 * RB + 256 * g + 4 * lane) = fine ? vpr[g] : 0u;
                    }
                    const uint64_t odd = __ballot(row >= 0 && !fine);
                    if (odd) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if ((odd >> (16 * i + 4 * grp) & 15u) & (vis[nt] >> (4 * i))) osum[nt][g] = NAN;
                    }
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    // P in the codes' slot order 0, 4, 1, 5, .. of the lane group's tokens (i, r), product st: i = 2 st and 2 st + 1
                    i4_bf16x8 ph[NT][2], pl[NT][2];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float4 sc, of;
                        uint4 pr;
                        if constexpr (WIDE) {
                            sc = *reinterpret_cast<const float4 *>(sct + 64 * g + 16 * i + 4 * grp);
                            of = *reinterpret_cast<const float4 *>(oft + 64 * g + 16 * i + 4 * grp);
                        } else {
                            pr = *reinterpret_cast<const uint4 *>(vt + 64 * RB + 256 * g + 64 * i + 16 * grp);
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                float w;
                                if constexpr (WIDE) {
                                    w = s[nt][i][r] * int4_of(sc, r);
                                    osum[nt][g] = __builtin_fmaf(s[nt][i][r], int4_of(of, r), osum[nt][g]);
                                } else {
                                    w = __builtin_fmaf(s[nt][i][r], int4_lo(int4_of(pr, r)), 0.0f);
                                    osum[nt][g] = __builtin_fmaf(s[nt][i][r], int4_hi(int4_of(pr, r)), osum[nt][g]);
                                }
                                const __bf16 hi = (__bf16)w;
                                ph[nt][i >> 1][2 * r + (i & 1)] = hi;
                                if constexpr (!BF) pl[nt][i >> 1][2 * r + (i & 1)] = (__bf16)(w - (float)hi);
                            }
                    }
                    const uint32_t w24 = NG == 1 || l16 == g ? 0x41C041C0u : 0u;   // 24 in the group's column
                    const uint4 b24 = make_uint4(w24, w24, w24, w24);
                    auto product = [&](int nt, int st, uint4 vf, i4_f32x4 c) __attribute__((always_inline)) {
                        c = int4_mfma<true>(__builtin_bit_cast(uint4, ph[nt][st]), vf, c);
                        if constexpr (!BF) c = int4_mfma<true>(__builtin_bit_cast(uint4, pl[nt][st]), vf, c);
                        return c;
                    };
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int st = 0; st < 2; ++st) bias[nt] = product(nt, st, b24, bias[nt]);
#pragma unroll
                    for (int c = g * (GD / 16); c < (g + 1) * (GD / 16); ++c) {
                        // 16 tokens of dim 16 c + l16: lane i of the group addresses token 16 (i / 4) + 4 grp + i % 4
                        const int t = 16 * (l16 >> 2) + 4 * grp + (l16 & 3);
                        const i4_i32x2 v = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
                            (i4_lds_i32x2 *)(vt + t * RB + (((c >> 1) ^ L::swz(t)) << 4) + 8 * (c & 1)));
#pragma unroll
                        for (int st = 0; st < 2; ++st) {
                            const uint4 vf = int4_expand<true>((uint32_t)v[st]);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) acc[nt][c] = product(nt, st, vf, acc[nt][c]);
                        }
                    }
                    if constexpr (NG > 1) __builtin_amdgcn_sched_barrier(0);
                }
                int row2 = -1;
                if (step + 2 < step1) {
                    int4_wait_lds();   // V's LDS is read
                    row2 = row_of(step + 2, page_lds[wave][lane]);
                    int4_wait_lds();
                    int4_copy4(entry_of(step + 3), page_at);
                    fetch(a.kp, a.kpar, row2, tv);   // K of the step after next into V's tile
                }
                row = row1, row1 = row2;
                const uint32_t t = tk;
                tk = tn, tn = tv, tv = t;
            }
        }

        // sums over the lane groups; O of the plain codes, offsets added; then out
        const bool whole = step0 == 0 && step1 == nsteps;
        const int64_t part = ((int64_t)(worker * 2 + slot) * a.head_group + member) * a.part_rows;
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
            for (int r = 0; r < 4; ++r) {
                const int in_tile = 16 * nt + 4 * grp + r, row = row0 + in_tile;
                const float ls = __shfl(l[nt], 4 * grp + r, 64), ms = __shfl(m[nt], 4 * grp + r, 64);
                float o[NG];
#pragma unroll
                for (int g = 0; g < NG; ++g) o[g] = __shfl(osum[nt][g], 4 * grp + r, 64) - __shfl(bias[nt][r], 16 * grp + g, 64);
                if (row >= R) continue;
                if (whole) {
                    const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
                    const int qi = row / G;
                    typename Elem<DT>::T *out = a.out + (((int64_t)seq * a.query_len + qi) * a.heads + (int64_t)kvh * G + (row - qi * G)) * D;
#pragma unroll
                    for (int c = 0; c < DC; ++c) out[16 * c + l16] = Elem<DT>::store((acc[nt][c][r] + o[16 * c / GD]) * inv);
                } else {
                    float *out = a.part_o + (part + in_tile) * D;
#pragma unroll
                    for (int c = 0; c < DC; ++c) out[16 * c + l16] = acc[nt][c][r] + o[16 * c / GD];
                    if (l16 == 0) *reinterpret_cast<float2 *>(a.part_ml + 2 * (part + in_tile)) = make_float2(ms, ls);
                }
            }
        }
        left -= step1 - step0;
        if (left <= 0) return;
        slot = 1;
        step0 = 0;
        if (++pair == pairs) {
            pair = 0;
            ++seq;
            ctx = __builtin_amdgcn_readfirstlane(int4_context(a, seq));
            nsteps = int4_steps(ctx);
        }
    }
}

// Joins a row's pieces: T threads to a piece, 16 bytes each, the pieces dealt out to the block's groups
// of T threads, eight loads of each in flight; a wave's groups meet by shuffles, the waves in LDS, both in
// one order.  T = D / 4 in one wave where there are few pieces a row.  Where there are many (three contexts
// of 50 to 120 thousand tokens leave 340 a row, 174 KB, for 48 rows), one CU cannot read them fast enough:
// a block for every 32 dims, with eight waves of eight groups, takes 5.6 us, whole rows by eight waves 9.4.
template <int DT, int D, int WAVES, int T>
__global__ __launch_bounds__(64 * WAVES) void int4_join_kernel(Int4Args a) {
    constexpr int CUTS = D / 4 / T, PG = 64 * WAVES / T, U = 8;   // blocks of a row, groups, loads
    __shared__ float2 ml[WAVES];
    __shared__ float4 os[WAVES][T];
    const int h = blockIdx.x / CUTS, cut_at = blockIdx.x % CUTS * T, qi = blockIdx.y, b = blockIdx.z;
    const int2 start = a.starts[b];
    const Int4Cut cut(a.workers, a.starts[a.batch].x);
    const int G = a.heads / a.kv_heads, kvh = h / G, row = qi * G + (h - kvh * G);
    const int u0 = start.x + (row / 16 * (a.kv_heads / a.head_group) + kvh / a.head_group) * start.y;
    const int first = cut.worker(u0), last = cut.worker(u0 + start.y - 1);
    if (first == last) return;   // one worker's: stored already
    const int slot = cut.start(first) == u0 ? 0 : 1;
    const int g = threadIdx.x / T, t = threadIdx.x % T, wave = threadIdx.x / 64;
    const int64_t row_at = (int64_t)(kvh % a.head_group) * a.part_rows + row % 16, worker = 2 * (int64_t)a.head_group * a.part_rows;
    float M = -INFINITY, Ls = 0.0f;
    float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto fold = [&](float pm, float pls, float4 po) __attribute__((always_inline)) {
        const float mn = fmaxf(M, pm), ref = mn == -INFINITY ? 0.0f : mn;
        // (a piece without a maximum has seen nothing, or NaN alone, which stays)
        const float fo = M == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - ref), fp = pm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(pm - ref);
        Ls = Ls * fo + pls * fp;
        O = make_float4(O.x * fo + po.x * fp, O.y * fo + po.y * fp, O.z * fo + po.z * fp, O.w * fo + po.w * fp);
        M = mn;
    };
    for (int w0 = first + g; w0 <= last; w0 += U * PG) {
        float2 mv[U];
        float4 ov[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (w0 + u * PG <= last) {
                const int w = w0 + u * PG;
                const int64_t p = w * worker + (w == first ? slot : 0) * (worker / 2) + row_at;
                mv[u] = reinterpret_cast<const float2 *>(a.part_ml)[p];
                ov[u] = reinterpret_cast<const float4 *>(a.part_o)[p * (D / 4) + cut_at + t];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (w0 + u * PG <= last) fold(mv[u].x, mv[u].y, ov[u]);
    }
#pragma unroll
    for (int o = T; o < 64; o <<= 1)   // the wave's groups
        fold(__shfl_xor(M, o, 64), __shfl_xor(Ls, o, 64),
             make_float4(__shfl_xor(O.x, o, 64), __shfl_xor(O.y, o, 64), __shfl_xor(O.z, o, 64), __shfl_xor(O.w, o, 64)));
    if constexpr (WAVES > 1) {
        if (threadIdx.x % 64 < T) {
            if (t == 0) ml[wave] = make_float2(M, Ls);
            os[wave][t] = O;
        }
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int k = 1; k < WAVES; ++k) fold(ml[k].x, ml[k].y, os[k][t]);
    }
    if (g != 0) return;
    const float inv = Ls == 0.0f ? 0.0f : 1.0f / Ls;
    typename Elem<DT>::T v[4] = {Elem<DT>::store(O.x * inv), Elem<DT>::store(O.y * inv), Elem<DT>::store(O.z * inv), Elem<DT>::store(O.w * inv)};
    __builtin_memcpy(a.out + (((int64_t)b * a.query_len + qi) * a.heads + h) * D + 4 * (cut_at + t), v, 8);
}

// The grid: blocks that fill the chip (by their LDS and registers), fewer where there are fewer steps.
struct Int4Grid {
    int64_t head_group, row_tiles, blocks, part_rows, steps;
    Int4Grid(int64_t batch, int64_t query_len, int64_t heads, int64_t kv_heads, int64_t dim, int64_t group, int64_t max_context) {
        const int64_t rows = heads / kv_heads * query_len;
        head_group = kv_heads % 4 == 0 ? 4 : kv_heads % 2 == 0 ? 2 : 1;
        row_tiles = (rows + 15) / 16;
        part_rows = std::min<int64_t>(rows, 16);
        steps = batch * row_tiles * (kv_heads / head_group) * ((max_context + 63) / 64);
        blocks = std::min<int64_t>(256 * int4_blocks_per_cu((int)dim, (int)(dim / group)), (steps * head_group + 3) / 4);
    }
};

template <int DT, int D, int NG> static void launch_int4(const Int4Args &a, const Int4Grid &g, bool join, hipStream_t s) {
    int4_walk_kernel<DT, D, NG><<<(unsigned)g.blocks, 256, 0, s>>>(a);
    if (!join) return;
    // a row cut in many pieces has eight waves for every 32 dims to join them, else one for all
    const int64_t walks = (int64_t)a.batch * a.row_tiles * (a.kv_heads / a.head_group);
    const dim3 rows((unsigned)a.heads, (unsigned)a.query_len, (unsigned)a.batch);
    if (walks * 16 < a.workers)
        int4_join_kernel<DT, D, 8, 8><<<dim3(rows.x * (D / 32), rows.y, rows.z), 512, 0, s>>>(a);
    else
        int4_join_kernel<DT, D, 1, D / 4><<<rows, 64, 0, s>>>(a);
}
template <int DT> static void launch_int4_dim(const Int4Args &a, int dim, int group, const Int4Grid &g, bool join, hipStream_t s) {
    switch (1000 * dim + group) {
    case 64064: launch_int4<DT, 64, 1>(a, g, join, s); break;
    case 64032: launch_int4<DT, 64, 2>(a, g, join, s); break;
    case 128128: launch_int4<DT, 128, 1>(a, g, join, s); break;
    case 128064: launch_int4<DT, 128, 2>(a, g, join, s); break;
    case 128032: launch_int4<DT, 128, 4>(a, g, join, s); break;
    case 256128: launch_int4<DT, 256, 2>(a, g, join, s); break;
    case 256064: launch_int4<DT, 256, 4>(a, g, join, s); break;
    case 256032: launch_int4<DT, 256, 8>(a, g, join, s); break;
    }
}

}  // namespace puter

using namespace puter;

extern "C" {

size_t puter_hip_paged_int4_workspace_bytes(int64_t batch, int64_t query_len, int64_t num_heads, int64_t kv_heads,
                                            int64_t head_dim, int64_t max_context) {
    if (batch <= 0 || query_len <= 0 || num_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || max_context <= 0) return 0;
    const Int4Grid g(batch, query_len, num_heads, kv_heads, head_dim, head_dim, max_context);   // (one group: the largest grid)
    return (size_t)(g.blocks * 4 * 2 * g.part_rows * (head_dim + 2)) * sizeof(float) + (size_t)(batch + 1) * sizeof(int2);
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
    const Int4Grid g(batch, query_len, num_heads, kv_heads, head_dim, group, max_context);
    if (batch * query_len * num_heads > 0x7FFFFFFF || g.steps > 0x3FFFFFFF)
        return fail(PUTER_ERR_INVALID, "paged int4: too many query rows or tokens");
    Int4Args a{};
    a.q = static_cast<const uint16_t *>(query);
    a.kp = static_cast<const uint8_t *>(key_pages), a.vp = static_cast<const uint8_t *>(value_pages);
    a.kpar = static_cast<const uint32_t *>(key_params), a.vpar = static_cast<const uint32_t *>(value_params);
    a.table = page_table, a.ctx = context_lens, a.out = static_cast<uint16_t *>(output);
    a.part_o = static_cast<float *>(workspace);
    a.part_ml = a.part_o + g.blocks * 4 * 2 * g.part_rows * head_dim;
    a.starts = reinterpret_cast<int2 *>(a.part_ml + g.blocks * 4 * 2 * g.part_rows * 2);
    a.max_pages = max_pages_per_seq;
    a.batch = (int)batch, a.page_size = (int)page_size, a.num_pages = (int)num_pages;
    a.max_context = num_pages > 0 ? (int)max_context : 0;   // an empty pool: every sequence is empty
    a.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctzll((unsigned long long)page_size) : -1;
    a.query_len = (int)query_len, a.heads = (int)num_heads, a.kv_heads = (int)kv_heads;
    a.row_tiles = (int)g.row_tiles, a.head_group = (int)g.head_group, a.part_rows = (int)g.part_rows;
    a.workers = (int)(g.blocks * 4 / g.head_group);
    a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)head_dim));
    const bool join = max_context > 64;   // one step is never cut
    hipStream_t s = as_stream(stream);
    if (dtype == PUTER_BF16) launch_int4_dim<PUTER_BF16>(a, (int)head_dim, (int)group, g, join, s);
    else launch_int4_dim<PUTER_F16>(a, (int)head_dim, (int)group, g, join, s);
    return check_launch("paged int4");
}

}  // extern "C"
