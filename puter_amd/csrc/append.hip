// KV append: new rows of Q, K and V rotated at their own positions, Q written out, K and V stored
// in a paged cache (the reference runs RoPE on Q and on K, then KVPageWrite twice:
// device/cpu/rope/compute.go:55-126, execution/page_intrinsic.go:135-215).  The cache holds the
// rows' own format, fp8-E4M3 with a scale per kv head, or 4 bits with a scale and an offset per
// group of dims; and the gather that reads 4-bit pages back as values.
//
//   angle(r, i) = (start + positions[r]) * invfreq(i) in float64, cos and sin rounded to f32
//   (x, y) -> (x c - y s, x s + y c) in f32, each operation rounded; rounded once to the stored format
//   4 bits, per group of G dims: lo, hi = least and greatest value (kept to +-65504, f16's range),
//     scale = f16((hi - lo) / 15), offset = f16((lo + hi) / 2 + scale / 2),
//     n = rint((x - offset) * (1 / scale)) in [-8, 7]; the value is scale n + offset.
//     A NaN in a group makes its scale and offset NaN.
//
// Page ids and slots are checked as KVPageWrite's (a bad one is flagged and its rows of K and V not
// stored), and among rows of one (page, slot) the last is the one stored.
#include "page.hpp"

#include <algorithm>
#include <cmath>

namespace puter {

struct AppendArgs {
    const void *q, *k, *v;
    void *qo;
    uint8_t *kp, *vp;
    void *kpar, *vpar;   // fp8: float scales per kv head; 4 bits: (scale, offset) pairs
    const int32_t *pos, *ids, *offs;
    int64_t rows, q_stride, k_stride, v_stride, page_count, page_size, rows_per_block;
    int q_heads, kv_heads, dim, group, table_bits, table_rows, rotate, mode, chunk_rows;
    int slots_at, angles_at;   // LDS bytes before the rows' slots and the angles
    int64_t start;
    double log_base, factor, low, high, orig_ctx;
    int scaling;
    int32_t *status;
};

enum { CACHE_SAME = 0, CACHE_FP8 = 1, CACHE_I4 = 2 };

__device__ __forceinline__ double append_inv_freq(const AppendArgs &a, int pair) {
    // ropeInverseFrequency compute.go:98-107 (base^x as exp(x log base)), llama3ScaledInverseFrequency :109-126
    const double inv = exp(-(double)(2 * pair) / (double)a.dim * a.log_base);
    if (a.scaling != 1) return inv;
    const double wavelength = (2.0 * M_PI) / inv;
    if (wavelength > a.orig_ctx / a.low) return inv / a.factor;
    if (wavelength < a.orig_ctx / a.high) return inv;
    const double smooth = (a.orig_ctx / wavelength - a.low) / (a.high - a.low);
    return (1.0 - smooth) * (inv / a.factor) + smooth * inv;
}

// cos and sin of a float64 angle, to f32: reduced by multiples of pi / 2 in two parts (Cody and
// Waite; the products are exact in the FMA), then the Taylor sums to r^13 and r^14, whose next terms
// are below 2^-45 for |r| <= pi / 4: far inside f32's rounding.  (A library sincos in float64 takes
// several times as many instructions, for angles and digits that are not needed here.)
__device__ __forceinline__ float2 append_cos_sin(double theta) {
    const double n = rint(theta * 0.63661977236758134308);
    double r = fma(-n, 1.5707963267948965580, theta);
    r = fma(-n, 6.1232339957367658e-17, r);
    const double z = r * r;
    double sn = 1.0 / 6227020800.0, cn = -1.0 / 87178291200.0;
    sn = fma(sn, z, -1.0 / 39916800.0), cn = fma(cn, z, 1.0 / 479001600.0);
    sn = fma(sn, z, 1.0 / 362880.0), cn = fma(cn, z, -1.0 / 3628800.0);
    sn = fma(sn, z, -1.0 / 5040.0), cn = fma(cn, z, 1.0 / 40320.0);
    sn = fma(sn, z, 1.0 / 120.0), cn = fma(cn, z, -1.0 / 720.0);
    sn = fma(sn, z, -1.0 / 6.0), cn = fma(cn, z, 1.0 / 24.0);
    sn = fma(sn * z, r, r), cn = fma(fma(cn, z, -0.5), z, 1.0);
    const int q = (int)(int64_t)n & 3;
    const float s = (float)(q & 1 ? cn : sn), c = (float)(q & 1 ? sn : cn);
    return make_float2(q == 1 || q == 2 ? -c : c, q >= 2 ? -s : s);
}

// 16 bytes at any alignment of elements.  STREAM: rows that are read or written once pass by the
// caches' retention.
typedef uint32_t append_u32x4 __attribute__((ext_vector_type(4), aligned(2)));
template <bool STREAM> __device__ __forceinline__ uint4 append_ld(const void *p) {
    const append_u32x4 *q = reinterpret_cast<const append_u32x4 *>(p);
    append_u32x4 v;
    if constexpr (STREAM) v = __builtin_nontemporal_load(q);
    else v = *q;
    return make_uint4(v.x, v.y, v.z, v.w);
}
template <bool STREAM> __device__ __forceinline__ void append_st(void *p, const uint4 &v) {
    const append_u32x4 t = {v.x, v.y, v.z, v.w};
    append_u32x4 *q = reinterpret_cast<append_u32x4 *>(p);
    if constexpr (STREAM) __builtin_nontemporal_store(t, q);
    else *q = t;
}
// eight consecutive elements: one or two such vectors
template <int DT> struct Eight {
    static constexpr int N = Vec<DT>::N, NV = 8 / N;
    using T = typename Elem<DT>::T;
    uint4 v[NV];
    template <bool STREAM> __device__ __forceinline__ void load(const void *base, int64_t at) {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = append_ld<STREAM>(reinterpret_cast<const T *>(base) + at + j * N);
    }
    __device__ __forceinline__ void values(float (&f)[8]) const {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            float t[N];
            unpack_value<DT>(v[j], t);
#pragma unroll
            for (int i = 0; i < N; ++i) f[j * N + i] = t[i];
        }
    }
};
template <int DT, bool STREAM> __device__ __forceinline__ void store8(void *base, int64_t at, const float (&f)[8]) {
    constexpr int N = Vec<DT>::N;
    typename Elem<DT>::T *p = reinterpret_cast<typename Elem<DT>::T *>(base) + at;
#pragma unroll
    for (int j = 0; j < 8 / N; ++j) {
        float t[N];
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = f[j * N + i];
        append_st<STREAM>(p + j * N, pack_vec<DT>(t));
    }
}

// Eight values as E4M3(value / s), r the rounded 1 / s: the quotient's own remainder corrects it to the
// rounded division's (an estimate past 2^100, infinite or NaN stays: it saturates, or is NaN), and
// v_cvt_pk_fp8_f32 rounds as f32_to_e4m3 once its range is kept.  Where s lies in 2^+-60, a quotient
// that does not round to zero has a remainder far above the least float, so that the correction is
// exact; other scales, and eights that hold a NaN (whose sign the instruction drops), take the division
// itself.
__device__ __forceinline__ void store_fp8x8(uint8_t *p, const float (&f)[8], float s, float r) {
    int w[2] = {0, 0};
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float q[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float e = f[i + u] * r, c = __builtin_fmaf(__builtin_fmaf(-e, s, f[i + u]), r, e);
            const float d = __builtin_fabsf(e) < 0x1p100f ? c : e;
            q[u] = __builtin_fabsf(d) > 448.0f ? __builtin_copysignf(448.0f, d) : d;
            sum += q[u];
        }
        w[i >> 2] = (i & 2) ? __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], w[i >> 2], true)
                            : __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], w[i >> 2], false);
    }
    if (__builtin_fabsf(s) >= 0x1p-60f && __builtin_fabsf(s) <= 0x1p60f && sum == sum) {
        __builtin_memcpy(p, w, 8);
    } else {
        for (int i = 0; i < 8; ++i) p[i] = (uint8_t)f32_to_e4m3(__fdiv_rn(f[i], s));
    }
}

// A group's scale and offset from its least and greatest value.
struct Int4Group {
    float scale, offset, inverse;
    uint32_t pair;   // f16 scale | f16 offset << 16
    __device__ __forceinline__ Int4Group(float lo, float hi, bool nan) {
        const float kMax = 65504.0f;
        lo = fminf(fmaxf(lo, -kMax), kMax);
        hi = fminf(fmaxf(hi, -kMax), kMax);
        uint32_t s = f32_to_f16(__fdiv_rn(hi - lo, 15.0f));
        scale = (float)__builtin_bit_cast(_Float16, (uint16_t)s);
        uint32_t o = f32_to_f16((0.5f * lo + 0.5f * hi) + 0.5f * scale);
        offset = (float)__builtin_bit_cast(_Float16, (uint16_t)o);
        inverse = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
        if (nan) s = o = 0x7E00u;
        pair = s | (o << 16);
    }
    __device__ __forceinline__ uint32_t codes(const float (&f)[8]) const {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float n = fminf(fmaxf(rintf((f[i] - offset) * inverse), -8.0f), 7.0f);
            w |= ((uint32_t)(int)n & 15u) << (4 * i);
        }
        return w;
    }
};

// A block takes a run of rows.  An item is 8 dims of a head's first half and the 8 of its second half
// that stand D/2 further on, so that it holds whole pairs in either mode; the D/16 items of a head are
// neighbouring lanes, which find a 4-bit group's range by shuffles.  A wave takes 64 items of one row
// at a time, so that the row's addresses are scalar, and asks for its next before it works on one.
//
// FEW (up to 4096 rows, 1 to 4 a block): latency is all.  Every thread has its first item's loads, its
// share of the angles and of the later rows' keys (compared with the block's own, one by one) under
// way at once, and one barrier stands between them and the items.  64 rows of 32 + 8 heads of 128, of
// a fused QKV row, to bf16 pages: 4.2 us in a graph, most of it one chain of loads and the launch (6.4
// the other way; 1024 rows 8.0 and 11.0, 4096 rows 20 and 24, 8 + 2 heads of 64 to fp8 pages 11.3 and 11.7; at
// 8192 such rows 22 and 15, as every block reads all later rows' keys).
//
// Else the rows that store are settled as the page write settles them (page.hpp), then taken
// chunk_rows at a time with a table of (cos, sin) for the chunk's positions in LDS.  The rows are
// cut evenly into as many blocks as are resident at once: 332 blocks of 32 rows left a third of the
// card idle, 87 us against 69.  What it reads and writes bounds it: 10.6 K rows of 32 + 8 heads of 128
// into fp8 pages take 62 us, 5.0 TB/s, the rate of a large copy; into 4-bit pages 8 K rows take 40 us,
// 4.6 TB/s, as finding the ranges costs instructions (the vector units are busy half the time).
// Rows pass the caches by (non-temporal loads 5 us, stores 7 us of the 62).
// by value: a conditional between members would choose an address and load through it
template <class P> __device__ __forceinline__ P append_pick(bool first, P a, P b) { return first ? a : b; }

constexpr int kAppendThreads = 512;
// blocks a CU, all resident at once: three where an item's 80 registers allow it; two of f32 rows
constexpr int append_blocks_per_cu(int dt) { return dt == PUTER_F32 ? 2 : 3; }
constexpr int kFewAppendRows = 4096;
template <int DT, int CACHE, bool FEW>
__global__ __launch_bounds__(kAppendThreads, FEW ? 4 : 2 * append_blocks_per_cu(DT)) void kv_append_kernel(AppendArgs a) {
#pragma clang fp contract(off)
    extern __shared__ __align__(16) char lds[];
    constexpr int THREADS = kAppendThreads;
    constexpr bool STREAM = !FEW;
    using T = typename Elem<DT>::T;
    const int tid = threadIdx.x;
    const int64_t row0 = (int64_t)blockIdx.x * a.rows_per_block;
    const int nrows = (int)min(a.rows_per_block, a.rows - row0);
    const int half = a.dim / 2, per_head = a.dim / 16, per_row = (a.q_heads + 2 * a.kv_heads) * per_head;
    int64_t *const slots = reinterpret_cast<int64_t *>(lds + a.slots_at);   // the row's pool row; -1: not stored
    double *const invf = reinterpret_cast<double *>(lds + a.angles_at);
    float2 *const cs = reinterpret_cast<float2 *>(FEW ? invf : invf + half);

    // A wave's unit: up to 64 items of one row, so that the row's addresses are scalar.
    constexpr int WAVES = THREADS / kWave;
    const int lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int chunks = (per_row + kWave - 1) / kWave, step_r = WAVES / chunks, step_c = WAVES - step_r * chunks;
    const int head_shift = (per_head & (per_head - 1)) == 0 ? 31 - __clz(per_head) : -1;
    struct Item {
        int r, c;         // the unit: row of the chunk, and which of the row's runs of 64 items
        int kind, h, j;   // Q, K, V or past the row (3), its head, the items before it in the head
        float scale;      // fp8 pages: its head's
        Eight<DT> x, y;
    };
    auto load = [&](Item &it, int64_t first) __attribute__((always_inline)) {
        const int in_row = it.c * kWave + lane, hd = head_shift >= 0 ? in_row >> head_shift : in_row / per_head;
        it.j = in_row - hd * per_head;
        it.kind = hd < a.q_heads ? 0 : hd < a.q_heads + a.kv_heads ? 1 : in_row < per_row ? 2 : 3;
        it.h = hd - (it.kind == 0 ? 0 : it.kind == 1 ? a.q_heads : a.q_heads + a.kv_heads);
        if (it.kind == 3) return;
        const T *const qr = reinterpret_cast<const T *>(a.q) + (first + it.r) * a.q_stride;
        const T *const kr = reinterpret_cast<const T *>(a.k) + (first + it.r) * a.k_stride;
        const T *const vr = reinterpret_cast<const T *>(a.v) + (first + it.r) * a.v_stride;
        const T *const src = (it.kind == 0 ? qr : it.kind == 1 ? kr : vr) + (it.h * a.dim + 8 * it.j);
        it.x.template load<STREAM>(src, 0);
        it.y.template load<STREAM>(src, half);
        if (CACHE == CACHE_FP8 && it.kind > 0) it.scale = reinterpret_cast<const float *>(append_pick(it.kind == 1, a.kpar, a.vpar))[it.h];
    };
    auto finish = [&](const Item &it, int64_t first, const float2 *c, int64_t slot) __attribute__((always_inline)) {
        float x[8], y[8];
        it.x.values(x);
        it.y.values(y);
        const int j = it.j;
        if (it.kind == 3) return;
        if (a.rotate && it.kind < 2) {
            if (a.mode == 1) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float2 p = c[8 * j + i];
                    const float e = x[i], o = y[i];
                    x[i] = e * p.x - o * p.y;
                    y[i] = e * p.y + o * p.x;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 p = c[4 * j + i], p2 = c[half / 2 + 4 * j + i];
                    float e = x[2 * i], o = x[2 * i + 1];
                    x[2 * i] = e * p.x - o * p.y;
                    x[2 * i + 1] = e * p.y + o * p.x;
                    e = y[2 * i], o = y[2 * i + 1];
                    y[2 * i] = e * p2.x - o * p2.y;
                    y[2 * i + 1] = e * p2.y + o * p2.x;
                }
            }
        }
        if (it.kind == 0) {
            const int64_t out = ((first + it.r) * a.q_heads + it.h) * (int64_t)a.dim;
            store8<DT, STREAM>(a.qo, out + 8 * j, x);
            store8<DT, STREAM>(a.qo, out + half + 8 * j, y);
            return;
        }
        uint8_t *const pool = append_pick(it.kind == 1, a.kp, a.vp);
        const int64_t out = (slot * a.kv_heads + it.h) * (int64_t)a.dim;
        if constexpr (CACHE == CACHE_SAME) {
            if (slot < 0) return;
            store8<DT, STREAM>(pool, out + 8 * j, x);
            store8<DT, STREAM>(pool, out + half + 8 * j, y);
        } else if constexpr (CACHE == CACHE_FP8) {
            if (slot < 0) return;
            const float s = it.scale, r = __fdiv_rn(1.0f, s);
            store_fp8x8(pool + out + 8 * j, x, s, r);
            store_fp8x8(pool + out + half + 8 * j, y, s, r);
        } else {
            // the ranges of x's group and y's (one and the same if a group is the whole head)
            float lo[2], hi[2];
            int nan[2] = {0, 0};
            lo[0] = hi[0] = x[0];
            lo[1] = hi[1] = y[0];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                lo[0] = fminf(lo[0], x[i]), hi[0] = fmaxf(hi[0], x[i]), nan[0] |= x[i] != x[i];
                lo[1] = fminf(lo[1], y[i]), hi[1] = fmaxf(hi[1], y[i]), nan[1] |= y[i] != y[i];
            }
            if (a.group == a.dim) {
                lo[0] = lo[1] = fminf(lo[0], lo[1]);
                hi[0] = hi[1] = fmaxf(hi[0], hi[1]);
                nan[0] = nan[1] = nan[0] | nan[1];
            }
            const int width = min(a.group / 8, per_head);   // lanes of a group
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                for (int o = 1; o < width; o <<= 1) {
                    lo[u] = fminf(lo[u], __shfl_xor(lo[u], o, kWave));
                    hi[u] = fmaxf(hi[u], __shfl_xor(hi[u], o, kWave));
                    nan[u] |= __shfl_xor(nan[u], o, kWave);
                }
            }
            if (slot < 0) return;
            const Int4Group gx(lo[0], hi[0], nan[0]), gy(lo[1], hi[1], nan[1]);
            const int dx = 8 * j, dy = half + 8 * j;
            *reinterpret_cast<uint32_t *>(pool + ((out + dx) >> 1)) = gx.codes(x);
            *reinterpret_cast<uint32_t *>(pool + ((out + dy) >> 1)) = gy.codes(y);
            uint32_t *par = reinterpret_cast<uint32_t *>(append_pick(it.kind == 1, a.kpar, a.vpar)) + out / a.group;
            if (dx % a.group == 0) par[dx / a.group] = gx.pair;
            if (dy % a.group == 0) par[dy / a.group] = gy.pair;
        }
    };
    // units of nr rows from `first` on, whose angles stand in cs and places slot(row) gives; the first
    // is under way, and each is asked for before the one ahead of it is finished
    auto units = [&](Item &it, int64_t first, int nr, auto slot) __attribute__((always_inline)) {
        while (it.r < nr) {
            Item ahead;
            ahead.r = it.r + step_r;
            ahead.c = it.c + step_c;
            if (ahead.c >= chunks) ahead.c -= chunks, ++ahead.r;
            if (ahead.r < nr) load(ahead, first);
            finish(it, first, cs + it.r * half, slot(it.r));
            it = ahead;
        }
    };
    Item it;
    auto begin = [&](int64_t first, int nr) __attribute__((always_inline)) {
        it.r = wave / chunks;
        it.c = wave - it.r * chunks;
        if (it.r < nr) load(it, first);
    };
    if constexpr (FEW) {
        begin(row0, nrows);
        // the block's keys, and whether a later row has one of them
        int32_t id[4], off[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            id[i] = i < nrows ? a.ids[row0 + i] : -1;
            off[i] = i < nrows ? a.offs[row0 + i] : -1;
        }
        if (a.rotate)
            for (int e = tid; e < nrows * half; e += THREADS) {
                const int r = e / half, i = e - r * half;
                cs[e] = append_cos_sin((double)(a.start + a.pos[row0 + r]) * append_inv_freq(a, i));
            }
        uint32_t seen = 0;
        for (int64_t r = row0 + 1 + tid; r < a.rows; r += THREADS) {
            const int32_t rid = a.ids[r], roff = a.offs[r];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (r > row0 + i && rid == id[i] && roff == off[i]) seen |= 1u << i;
        }
        uint32_t *const found = reinterpret_cast<uint32_t *>(lds);   // per wave
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (__ballot(seen >> i & 1)) mine |= 1u << i;
        if (tid % kWave == 0) found[tid / kWave] = mine;
        __syncthreads();
        const uint32_t lost = found[0] | found[1] | found[2] | found[3] | found[4] | found[5] | found[6] | found[7];
        const int32_t pc = (int32_t)min(a.page_count, (int64_t)0x7FFFFFFF), ps = (int32_t)min(a.page_size, (int64_t)0x7FFFFFFF);
        int64_t at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool valid = write_valid(id[i], off[i], pc, ps);
            if (!valid && i < nrows && tid == 0) flag_invalid(a.status);
            at[i] = valid && !(lost >> i & 1) ? (int64_t)id[i] * a.page_size + off[i] : -1;
        }
        units(it, row0, nrows, [&](int r) { return r == 0 ? at[0] : r == 1 ? at[1] : r == 2 ? at[2] : at[3]; });
    } else {
        const WriteTable t = write_table(lds, a.table_rows, a.table_bits);
        int32_t my_id = -1, my_off = -1;
        if (tid < nrows) {
            my_id = a.ids[row0 + tid];
            my_off = a.offs[row0 + tid];
        }
        if (a.rotate)
            for (int i = tid; i < half; i += THREADS) invf[i] = append_inv_freq(a, i);
        begin(row0, min(a.chunk_rows, nrows));
        ScanChunk c0;
        scan_load<THREADS>(c0, a.ids, a.offs, row0 + nrows, a.rows);
        write_winners<THREADS>(t, my_id, my_off, c0, a.ids, a.offs, row0, nrows, a.rows, a.page_count, a.page_size, a.status);
        if (tid < nrows) slots[tid] = write_wins(t, tid) ? write_slot(t, tid, a.page_size) : -1;
        for (int r0 = 0; r0 < nrows; r0 += a.chunk_rows) {
            const int nr = min(a.chunk_rows, nrows - r0);
            if (r0) begin(row0 + r0, nr);
            __syncthreads();   // the slots are there; the previous chunk's angles are free
            if (a.rotate)
                for (int e = tid; e < nr * half; e += THREADS) {
                    const int r = e / half, i = e - r * half;
                    cs[e] = append_cos_sin((double)(a.start + a.pos[row0 + r0 + r]) * invf[i]);
                }
            __syncthreads();
            units(it, row0 + r0, nr, [&](int r) { return slots[r0 + r]; });
        }
    }
}

// Head dims that are no multiple of 16: a block of 256 threads, an item is one pair.
template <int DT, int CACHE>
__global__ __launch_bounds__(256) void kv_append_pair_kernel(AppendArgs a) {
#pragma clang fp contract(off)
    extern __shared__ __align__(16) char lds[];
    constexpr int THREADS = 256;
    const int tid = threadIdx.x;
    const int64_t row0 = (int64_t)blockIdx.x * a.rows_per_block;
    const int nrows = (int)min(a.rows_per_block, a.rows - row0);
    const WriteTable t = write_table(lds, a.table_rows, a.table_bits);
    const int half = a.dim / 2;
    double *const invf = reinterpret_cast<double *>(lds + a.angles_at);
    float2 *const cs = reinterpret_cast<float2 *>(invf + half);
    int32_t my_id = -1, my_off = -1;
    if (tid < nrows) {
        my_id = a.ids[row0 + tid];
        my_off = a.offs[row0 + tid];
    }
    if (a.rotate)
        for (int i = tid; i < half; i += THREADS) invf[i] = append_inv_freq(a, i);
    ScanChunk c0;
    scan_load<THREADS>(c0, a.ids, a.offs, row0 + nrows, a.rows);
    write_winners<THREADS>(t, my_id, my_off, c0, a.ids, a.offs, row0, nrows, a.rows, a.page_count, a.page_size, a.status);
    const int per_row = (a.q_heads + 2 * a.kv_heads) * half;
    for (int r0 = 0; r0 < nrows; r0 += a.chunk_rows) {
        const int nr = min(a.chunk_rows, nrows - r0);
        if (a.rotate) {
            __syncthreads();   // the previous chunk's angles are free
            for (int e = tid; e < nr * half; e += THREADS) {
                const int r = e / half, i = e - r * half;
                cs[e] = append_cos_sin((double)(a.start + a.pos[row0 + r0 + r]) * invf[i]);
            }
            __syncthreads();
        }
        for (int w = tid; w < nr * per_row; w += THREADS) {
            const int r = w / per_row, hd = (w - r * per_row) / half, j = w - r * per_row - hd * half;
            const int64_t row = row0 + r0 + r;
            const int kind = hd < a.q_heads ? 0 : hd < a.q_heads + a.kv_heads ? 1 : 2;   // Q, K or V
            const int h = kind == 0 ? hd : hd - a.q_heads - (kind == 2 ? a.kv_heads : 0);
            if (kind != 0 && !write_wins(t, r0 + r)) continue;
            const void *src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
            const int64_t at = row * (kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride) + (int64_t)h * a.dim;
            const int64_t out = kind == 0 ? (row * a.q_heads + h) * (int64_t)a.dim
                                          : (write_slot(t, r0 + r, a.page_size) * a.kv_heads + h) * (int64_t)a.dim;
            const int i0 = a.mode == 1 ? j : 2 * j, i1 = a.mode == 1 ? half + j : 2 * j + 1;
            const typename Elem<DT>::T *p = reinterpret_cast<const typename Elem<DT>::T *>(src) + at;
            float x = Elem<DT>::load(p[i0]), y = Elem<DT>::load(p[i1]);
            if (a.rotate && kind < 2) {
                const float2 c = cs[r * half + j];
                const float e = x, o = y;
                x = e * c.x - o * c.y;
                y = e * c.y + o * c.x;
            }
            uint8_t *const pool = kind == 1 ? a.kp : a.vp;
            if (CACHE == CACHE_SAME || kind == 0) {
                typename Elem<DT>::T *d = reinterpret_cast<typename Elem<DT>::T *>(kind == 0 ? a.qo : pool) + out;
                d[i0] = Elem<DT>::store(x), d[i1] = Elem<DT>::store(y);
            } else {
                const float s = reinterpret_cast<const float *>(kind == 1 ? a.kpar : a.vpar)[h];
                pool[out + i0] = (uint8_t)f32_to_e4m3(__fdiv_rn(x, s));
                pool[out + i1] = (uint8_t)f32_to_e4m3(__fdiv_rn(y, s));
            }
        }
    }
}

// Rows of 4-bit pages as values: a thread takes eight dims (four bytes of codes, one pair) four times,
// the loads of all four first.  Rows are numbered in 32 bits, so that a row's page costs a 32-bit
// division; the places in the pool take 64.
template <int DT>
__global__ __launch_bounds__(256) void int4_gather_kernel(const uint32_t *__restrict__ pages, const uint32_t *__restrict__ pairs,
                                                          const int32_t *__restrict__ table, void *__restrict__ out,
                                                          int64_t page_count, uint32_t page_size, uint32_t units, int pair_shift,
                                                          uint32_t rows, uint32_t rows_per_block, int32_t *status) {
    constexpr int U = 4;
    for (int64_t row0 = (int64_t)blockIdx.x * rows_per_block; row0 < rows; row0 += (int64_t)gridDim.x * rows_per_block) {
        const uint32_t total = min(rows_per_block, (uint32_t)(rows - row0)) * units;
        for (uint32_t e0 = threadIdx.x; e0 < total; e0 += 256 * U) {
            uint32_t w[U] = {}, pair[U] = {};
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const uint32_t e = e0 + 256 * k;
                if (e >= total) break;
                const uint32_t r = e / units, row = (uint32_t)row0 + r, page = row / page_size;
                const int32_t id = table[page];
                if (id < 0 || id >= page_count) {
                    flag_invalid(status);
                } else {
                    const int64_t at = ((int64_t)id * page_size + (row - page * page_size)) * units + (e - r * units);
                    w[k] = pages[at], pair[k] = pairs[at >> pair_shift];
                }
            }
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const uint32_t e = e0 + 256 * k;
                if (e >= total) break;
                const float s = (float)__builtin_bit_cast(_Float16, (uint16_t)(pair[k] & 0xFFFFu));
                const float o = (float)__builtin_bit_cast(_Float16, (uint16_t)(pair[k] >> 16));
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = (float)((int32_t)(w[k] << (28 - 4 * i)) >> 28) * s + o;
                store8<DT, false>(out, (row0 * units + e) * 8, f);
            }
        }
    }
}

static bool int4_shape(int64_t dim, int64_t group) {
    return (dim == 64 || dim == 128 || dim == 256) && (group == 32 || group == 64 || group == 128) && group <= dim;
}


template <int DT>
static void launch_append(AppendArgs a, int cache, hipStream_t s) {
    const int64_t half = a.dim / 2;
    auto align = [](size_t n) { return (int)((n + 15) & ~(size_t)15); };
    auto go = [&](auto kernel, int threads, size_t lds) {
        kernel<<<(unsigned)((a.rows + a.rows_per_block - 1) / a.rows_per_block), threads, lds, s>>>(a);
    };
    // rows a block and what it holds of LDS: the winners' table (a power of two of rows), the rows'
    // places, frequencies and a chunk's angles
    auto spread = [&](int64_t blocks, int64_t most) {
        a.rows_per_block = std::min(most, (a.rows + blocks - 1) / blocks);
        a.table_rows = 2, a.table_bits = 2;
        while (a.table_rows < a.rows_per_block) a.table_rows *= 2, ++a.table_bits;
        a.chunk_rows = (int)std::min(a.rows_per_block, std::max<int64_t>(1, 2048 / half));
        a.slots_at = align(write_lds_bytes(a.table_rows));
        a.angles_at = align((size_t)a.slots_at + (size_t)a.rows_per_block * 8);
        return (size_t)a.angles_at + (size_t)half * 8 * (1 + a.chunk_rows);
    };
    if (a.dim % 16 != 0) {
        const size_t lds = spread(512, 256);
        if (cache == CACHE_SAME) go(kv_append_pair_kernel<DT, CACHE_SAME>, 256, lds);
        else go(kv_append_pair_kernel<DT, CACHE_FP8>, 256, lds);
        return;
    }
    const bool few = a.rows <= kFewAppendRows;
    size_t lds;
    if (few) {
        a.rows_per_block = a.rows <= 256 ? 1 : a.rows <= 512 ? 2 : 4;
        a.angles_at = 32;
        lds = 32 + (size_t)(a.rows_per_block * half) * 8;
    } else {
        lds = spread(256 * append_blocks_per_cu(DT), 512);
    }
#define PUTER_APPEND(C)                                                        \
    if (few) go(kv_append_kernel<DT, C, true>, kAppendThreads, lds);                      \
    else go(kv_append_kernel<DT, C, false>, kAppendThreads, lds);
    if (cache == CACHE_SAME) { PUTER_APPEND(CACHE_SAME) }
    else if (cache == CACHE_FP8) { PUTER_APPEND(CACHE_FP8) }
    else { PUTER_APPEND(CACHE_I4) }
#undef PUTER_APPEND
}

}  // namespace puter

using namespace puter;

extern "C" {

int puter_hip_kv_page_append_rope(const puter_rope_config *config, const void *query, const void *key, const void *value,
                                  const int32_t *positions, const int32_t *page_ids, const int32_t *offsets,
                                  void *query_out, void *key_pages, void *value_pages, void *key_params,
                                  void *value_params, int64_t rows, int64_t query_heads, int64_t kv_heads,
                                  int64_t head_dim, int64_t query_stride, int64_t key_stride, int64_t value_stride,
                                  int64_t page_count, int64_t page_size, int64_t group, int dtype, int cache_dtype,
                                  int32_t *status, void *stream) {
    if (!is_norm_dtype(dtype)) return fail(PUTER_ERR_INVALID, "kv append: unsupported dtype %d", dtype);
    if (cache_dtype != dtype && cache_dtype != PUTER_F8E4M3 && cache_dtype != PUTER_I4)
        return fail(PUTER_ERR_INVALID, "kv append: cache dtype %d unsupported for rows of dtype %d", cache_dtype, dtype);
    if (rows < 0 || query_heads < 0 || kv_heads <= 0 || head_dim <= 0 || page_count < 0 || page_size <= 0)
        return fail(PUTER_ERR_INVALID, "kv append: invalid shape");
    if (head_dim % 2 != 0 || head_dim > 1024) return fail(PUTER_ERR_INVALID, "kv append: head_dim %lld unsupported (even, at most 1024)", (long long)head_dim);
    if (query_heads > 65536 || kv_heads > 65536) return fail(PUTER_ERR_INVALID, "kv append: too many heads");
    if (query_stride < query_heads * head_dim || key_stride < kv_heads * head_dim || value_stride < kv_heads * head_dim)
        return fail(PUTER_ERR_INVALID, "kv append: a row stride is less than its row");
    if (cache_dtype == PUTER_I4 && !int4_shape(head_dim, group))
        return fail(PUTER_ERR_INVALID, "kv append: 4-bit pages take head dims of 64, 128 or 256 in groups of 32, 64 or 128 dims");
    if (config) {
        // RoPEConfig.Validate device/config.go:215-258
        const puter_rope_config &c = *config;
        if (!(c.base_freq > 0) || !std::isfinite(c.base_freq)) return fail(PUTER_ERR_INVALID, "kv append: base frequency must be positive, got %g", c.base_freq);
        if (c.mode != 0 && c.mode != 1) return fail(PUTER_ERR_INVALID, "kv append: unsupported mode %d", c.mode);
        if (c.scaling != 0 && c.scaling != 1) return fail(PUTER_ERR_INVALID, "kv append: unsupported scaling %d", c.scaling);
        if (c.scaling == 1 && (!(c.scaling_factor > 0) || !(c.low_freq_factor > 0) ||
                               !(c.high_freq_factor > c.low_freq_factor) || c.original_context <= 0))
            return fail(PUTER_ERR_INVALID, "kv append: invalid Llama-3 scaling");
        // the kernel's reduction of angles holds to 2^45; int32 positions add up to 2^31 to the start
        const double fastest = std::max(1.0, std::pow(c.base_freq, 2.0 / (double)head_dim - 1.0)) *
                               (c.scaling == 1 ? std::max(1.0, 1.0 / c.scaling_factor) : 1.0);
        if (!((std::fabs((double)c.start_position) + 0x1p31) * fastest <= 0x1p45))
            return fail(PUTER_ERR_INVALID, "kv append: angles past 2^45 radians");
    }
    if (rows == 0) return PUTER_OK;
    if (!key || !value || !page_ids || !offsets || !key_pages || !value_pages || (config && !positions) ||
        (query_heads > 0 && (!query || !query_out)))
        return fail(PUTER_ERR_NIL, "kv append: nil buffer");
    if (cache_dtype != dtype && (!key_params || !value_params)) return fail(PUTER_ERR_NIL, "kv append: fp8 and 4-bit pages need their scales");
    if (reinterpret_cast<uintptr_t>(status) & 3) return fail(PUTER_ERR_INVALID, "kv append: misaligned status word");
    if (cache_dtype == PUTER_I4 && ((reinterpret_cast<uintptr_t>(key_pages) | reinterpret_cast<uintptr_t>(value_pages)) & 15))
        return fail(PUTER_ERR_INVALID, "kv append: 4-bit pools must be 16-byte aligned");
    if (cache_dtype != dtype && ((reinterpret_cast<uintptr_t>(key_params) | reinterpret_cast<uintptr_t>(value_params)) & 3))
        return fail(PUTER_ERR_INVALID, "kv append: misaligned scales");
    AppendArgs a{};
    a.q = query, a.k = key, a.v = value, a.qo = query_out;
    a.kp = static_cast<uint8_t *>(key_pages), a.vp = static_cast<uint8_t *>(value_pages);
    a.kpar = key_params, a.vpar = value_params;
    a.pos = positions, a.ids = page_ids, a.offs = offsets;
    a.rows = rows, a.q_stride = query_stride, a.k_stride = key_stride, a.v_stride = value_stride;
    a.page_count = page_count, a.page_size = page_size;
    a.q_heads = (int)query_heads, a.kv_heads = (int)kv_heads, a.dim = (int)head_dim, a.group = (int)group;
    a.rotate = config != nullptr;
    if (config) {
        a.mode = config->mode, a.start = config->start_position, a.log_base = std::log(config->base_freq), a.scaling = config->scaling;
        a.factor = config->scaling_factor, a.low = config->low_freq_factor, a.high = config->high_freq_factor;
        a.orig_ctx = (double)config->original_context;
    } else {
        a.mode = 1;
    }
    a.status = status;
    if (rows > 0x3FFFFFFFFll) return fail(PUTER_ERR_INVALID, "kv append: too many rows");
    const int cache = cache_dtype == dtype ? CACHE_SAME : cache_dtype == PUTER_F8E4M3 ? CACHE_FP8 : CACHE_I4;
    hipStream_t s = as_stream(stream);
    switch (dtype) {
    case PUTER_F32: launch_append<PUTER_F32>(a, cache, s); break;
    case PUTER_BF16: launch_append<PUTER_BF16>(a, cache, s); break;
    case PUTER_F16: launch_append<PUTER_F16>(a, cache, s); break;
    }
    return check_launch("kv append");
}

int puter_hip_kv_page_gather_int4(const void *pages, const void *params, const int32_t *page_table, void *output,
                                  int64_t page_count, int64_t page_size, int64_t kv_heads, int64_t head_dim, int64_t group,
                                  int64_t out_rows, int dtype, int32_t *status, void *stream) {
    if (!is_norm_dtype(dtype)) return fail(PUTER_ERR_INVALID, "kv gather int4: unsupported dtype %d", dtype);
    if (page_count < 0 || page_size <= 0 || kv_heads <= 0 || out_rows < 0) return fail(PUTER_ERR_INVALID, "kv gather int4: invalid shape");
    if (!int4_shape(head_dim, group))
        return fail(PUTER_ERR_INVALID, "kv gather int4: head dims of 64, 128 or 256 in groups of 32, 64 or 128 dims");
    if (out_rows == 0) return PUTER_OK;
    if (!pages || !params || !page_table || !output) return fail(PUTER_ERR_NIL, "kv gather int4: nil buffer");
    if ((reinterpret_cast<uintptr_t>(status) | reinterpret_cast<uintptr_t>(pages) | reinterpret_cast<uintptr_t>(params)) & 3)
        return fail(PUTER_ERR_INVALID, "kv gather int4: misaligned status word, pages or scales");
    if (kv_heads > 65536 || out_rows > 0x7FFFFFFF || page_size > 0x7FFFFFFF) return fail(PUTER_ERR_INVALID, "kv gather int4: too many rows or heads");
    const int64_t units = kv_heads * head_dim / 8, most = std::max<int64_t>(1, 1024 / units);
    // an item a thread up to 1024 blocks of rows, then up to four
    const int64_t per_block = std::min(most, std::max((256 + units - 1) / units, out_rows / 1024));
    const unsigned blocks = (unsigned)std::min<int64_t>((out_rows + per_block - 1) / per_block, 1 << 20);
    hipStream_t s = as_stream(stream);
    const uint32_t *p = static_cast<const uint32_t *>(pages), *q = static_cast<const uint32_t *>(params);
    const int shift = group == 32 ? 2 : group == 64 ? 3 : 4;
    const uint32_t ps = (uint32_t)page_size;
#define PUTER_GATHER(DT)                                                                                                       \
    case DT:                                                                                                                   \
        int4_gather_kernel<DT><<<blocks, 256, 0, s>>>(p, q, page_table, output, page_count, ps, (uint32_t)units, shift,        \
                                                      (uint32_t)out_rows, (uint32_t)per_block, status);                        \
        break;
    switch (dtype) {
        PUTER_GATHER(PUTER_F32)
        PUTER_GATHER(PUTER_BF16)
        PUTER_GATHER(PUTER_F16)
    }
#undef PUTER_GATHER
    return check_launch("kv gather int4");
}

}  // extern "C"
