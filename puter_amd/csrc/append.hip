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
    int q_heads, kv_heads, dim, group, table_bits, rotate, mode, chunk_rows, angles_at;   // angles_at: LDS bytes before the angles
    int64_t start;
    double base, factor, low, high, orig_ctx;
    int scaling;
    int32_t *status;
};

enum { CACHE_SAME = 0, CACHE_FP8 = 1, CACHE_I4 = 2 };

__device__ __forceinline__ double append_inv_freq(const AppendArgs &a, int pair) {
    // ropeInverseFrequency compute.go:98-107, llama3ScaledInverseFrequency :109-126
    const double inv = pow(a.base, -(double)(2 * pair) / (double)a.dim);
    if (a.scaling != 1) return inv;
    const double wavelength = (2.0 * M_PI) / inv;
    if (wavelength > a.orig_ctx / a.low) return inv / a.factor;
    if (wavelength < a.orig_ctx / a.high) return inv;
    const double smooth = (a.orig_ctx / wavelength - a.low) / (a.high - a.low);
    return (1.0 - smooth) * (inv / a.factor) + smooth * inv;
}

// eight consecutive elements at any element alignment
template <int DT> __device__ __forceinline__ void load8(const void *base, int64_t at, float (&f)[8]) {
    constexpr int N = Vec<DT>::N;
    const typename Elem<DT>::T *p = reinterpret_cast<const typename Elem<DT>::T *>(base) + at;
#pragma unroll
    for (int j = 0; j < 8 / N; ++j) {
        uint4 v;
        __builtin_memcpy(&v, p + j * N, 16);
        float t[N];
        unpack_value<DT>(v, t);
#pragma unroll
        for (int i = 0; i < N; ++i) f[j * N + i] = t[i];
    }
}
template <int DT> __device__ __forceinline__ void store8(void *base, int64_t at, const float (&f)[8]) {
    constexpr int N = Vec<DT>::N;
    typename Elem<DT>::T *p = reinterpret_cast<typename Elem<DT>::T *>(base) + at;
#pragma unroll
    for (int j = 0; j < 8 / N; ++j) {
        float t[N];
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = f[j * N + i];
        const uint4 v = pack_vec<DT>(t);
        __builtin_memcpy(p + j * N, &v, 16);
    }
}

__device__ __forceinline__ void store_fp8x8(uint8_t *p, const float (&f)[8], float s) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 2] |= f32_to_e4m3(__fdiv_rn(f[i], s)) << (8 * (i & 3));
    __builtin_memcpy(p, w, 8);
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

// One block per run of rows (rows_per_block): which of them store is settled first (page.hpp), then
// they are taken chunk_rows at a time: a table of (cos, sin) for the chunk's positions in LDS, then
// every head's items.  VEC: an item is 8 dims of the head's first half and the 8 of the second half
// that stand D/2 further on, so that it holds whole pairs in either mode, and the D/16 items of a
// head are neighbouring lanes, which find a 4-bit group's range by shuffles.  Else (head dims that
// are no multiple of 16) an item is one pair.
template <int DT, int CACHE, bool VEC>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
#pragma clang fp contract(off)
    extern __shared__ __align__(16) char lds[];
    constexpr int THREADS = 256;
    const int tid = threadIdx.x;
    const int64_t row0 = (int64_t)blockIdx.x * a.rows_per_block;
    const int nrows = (int)min(a.rows_per_block, a.rows - row0);
    const WriteTable t = write_table(lds, a.rows_per_block, a.table_bits);
    const int half = a.dim / 2;
    double *invf = reinterpret_cast<double *>(lds + a.angles_at);
    float2 *cs = reinterpret_cast<float2 *>(invf + half);
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
    const int heads = a.q_heads + 2 * a.kv_heads;
    const int per_head = VEC ? a.dim / 16 : half;
    const int per_row = heads * per_head;
    for (int r0 = 0; r0 < nrows; r0 += a.chunk_rows) {
        const int nr = min(a.chunk_rows, nrows - r0);
        if (a.rotate) {
            __syncthreads();   // the previous chunk's table is free
            for (int e = tid; e < nr * half; e += THREADS) {
                const int r = e / half, i = e - r * half;
                const double theta = (double)(a.start + a.pos[row0 + r0 + r]) * invf[i];
                double sn, cn;
                sincos(theta, &sn, &cn);
                cs[e] = make_float2((float)cn, (float)sn);
            }
            __syncthreads();
        }
        for (int w = tid; w < nr * per_row; w += THREADS) {
            const int r = w / per_row, in_row = w - r * per_row;
            const int hd = in_row / per_head, j = in_row - hd * per_head;
            const int64_t row = row0 + r0 + r;
            const int kind = hd < a.q_heads ? 0 : hd < a.q_heads + a.kv_heads ? 1 : 2;   // Q, K or V
            const int h = kind == 0 ? hd : hd - a.q_heads - (kind == 2 ? a.kv_heads : 0);
            const void *src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
            const int64_t at = row * (kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride) + (int64_t)h * a.dim;
            const bool turn = a.rotate && kind < 2;
            const bool stores = kind == 0 || write_wins(t, r0 + r);
            const int64_t slot = kind != 0 && stores ? write_slot(t, r0 + r, a.page_size) : 0;
            const int64_t out = kind == 0 ? (row * a.q_heads + h) * (int64_t)a.dim : (slot * a.kv_heads + h) * (int64_t)a.dim;
            uint8_t *const pool = kind == 1 ? a.kp : a.vp;
            const float2 *c = cs + r * half;
            if constexpr (VEC) {
                float x[8], y[8];
                load8<DT>(src, at + 8 * j, x);
                load8<DT>(src, at + half + 8 * j, y);
                if (turn) {
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
                if (kind == 0) {
                    store8<DT>(a.qo, out + 8 * j, x);
                    store8<DT>(a.qo, out + half + 8 * j, y);
                } else if constexpr (CACHE == CACHE_SAME) {
                    if (stores) {
                        store8<DT>(pool, out + 8 * j, x);
                        store8<DT>(pool, out + half + 8 * j, y);
                    }
                } else if constexpr (CACHE == CACHE_FP8) {
                    if (stores) {
                        const float s = reinterpret_cast<const float *>(kind == 1 ? a.kpar : a.vpar)[h];
                        store_fp8x8(pool + out + 8 * j, x, s);
                        store_fp8x8(pool + out + half + 8 * j, y, s);
                    }
                } else {
                    // the ranges of x's group and y's (one and the same if a group is the whole head)
                    float lo[2], hi[2];
                    bool nan[2] = {false, false};
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
                        int bad = nan[u];
                        for (int o = 1; o < width; o <<= 1) {
                            lo[u] = fminf(lo[u], __shfl_xor(lo[u], o, kWave));
                            hi[u] = fmaxf(hi[u], __shfl_xor(hi[u], o, kWave));
                            bad |= __shfl_xor(bad, o, kWave);
                        }
                        nan[u] = bad;
                    }
                    if (stores) {
                        const Int4Group gx(lo[0], hi[0], nan[0]), gy(lo[1], hi[1], nan[1]);
                        const int dx = 8 * j, dy = half + 8 * j;
                        *reinterpret_cast<uint32_t *>(pool + ((out + dx) >> 1)) = gx.codes(x);
                        *reinterpret_cast<uint32_t *>(pool + ((out + dy) >> 1)) = gy.codes(y);
                        uint32_t *par = reinterpret_cast<uint32_t *>(kind == 1 ? a.kpar : a.vpar) + out / a.group;
                        if (dx % a.group == 0) par[dx / a.group] = gx.pair;
                        if (dy % a.group == 0) par[dy / a.group] = gy.pair;
                    }
                }
            } else {
                const int i0 = a.mode == 1 ? j : 2 * j, i1 = a.mode == 1 ? half + j : 2 * j + 1;
                const typename Elem<DT>::T *p = reinterpret_cast<const typename Elem<DT>::T *>(src) + at;
                float x = Elem<DT>::load(p[i0]), y = Elem<DT>::load(p[i1]);
                if (turn) {
                    const float e = x, o = y;
                    x = e * c[j].x - o * c[j].y;
                    y = e * c[j].y + o * c[j].x;
                }
                if (CACHE == CACHE_SAME || kind == 0) {
                    typename Elem<DT>::T *d = reinterpret_cast<typename Elem<DT>::T *>(kind == 0 ? a.qo : pool) + out;
                    if (stores) d[i0] = Elem<DT>::store(x), d[i1] = Elem<DT>::store(y);
                } else if (stores) {
                    const float s = reinterpret_cast<const float *>(kind == 1 ? a.kpar : a.vpar)[h];
                    pool[out + i0] = (uint8_t)f32_to_e4m3(__fdiv_rn(x, s));
                    pool[out + i1] = (uint8_t)f32_to_e4m3(__fdiv_rn(y, s));
                }
            }
        }
    }
}

// Rows of 4-bit pages as values: a thread per eight dims (four bytes of codes, one pair).
template <int DT>
__global__ __launch_bounds__(256) void int4_gather_kernel(const uint32_t *__restrict__ pages, const uint32_t *__restrict__ pairs,
                                                          const int32_t *__restrict__ table, void *__restrict__ out,
                                                          int64_t page_count, int64_t page_size, int64_t units, int group8,
                                                          int64_t total, int32_t *status) {
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / units, u = i - row * units;
        const int32_t id = table[row / page_size];
        float f[8] = {};
        if (id < 0 || id >= page_count) {
            flag_invalid(status);
        } else {
            const int64_t at = ((int64_t)id * page_size + row % page_size) * units + u;
            const uint32_t w = pages[at], pair = pairs[at / group8];
            const float s = (float)__builtin_bit_cast(_Float16, (uint16_t)(pair & 0xFFFFu));
            const float o = (float)__builtin_bit_cast(_Float16, (uint16_t)(pair >> 16));
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = (float)((int32_t)(w << (28 - 4 * k)) >> 28) * s + o;
        }
        store8<DT>(out, i * 8, f);
    }
}

static bool int4_shape(int64_t dim, int64_t group) {
    return (dim == 64 || dim == 128 || dim == 256) && (group == 32 || group == 64 || group == 128) && group <= dim;
}

template <int DT>
static void launch_append(const AppendArgs &a, int cache, unsigned blocks, size_t lds, hipStream_t s) {
    const bool vec = a.dim % 16 == 0;
#define PUTER_APPEND(C)                                                        \
    if (vec) kv_append_kernel<DT, C, true><<<blocks, 256, lds, s>>>(a);        \
    else kv_append_kernel<DT, C, false><<<blocks, 256, lds, s>>>(a);
    if (cache == CACHE_SAME) { PUTER_APPEND(CACHE_SAME) }
    else if (cache == CACHE_FP8) { PUTER_APPEND(CACHE_FP8) }
    else kv_append_kernel<DT, CACHE_I4, true><<<blocks, 256, lds, s>>>(a);
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
        if (!(c.base_freq > 0)) return fail(PUTER_ERR_INVALID, "kv append: base frequency must be positive, got %g", c.base_freq);
        if (c.mode != 0 && c.mode != 1) return fail(PUTER_ERR_INVALID, "kv append: unsupported mode %d", c.mode);
        if (c.scaling != 0 && c.scaling != 1) return fail(PUTER_ERR_INVALID, "kv append: unsupported scaling %d", c.scaling);
        if (c.scaling == 1 && (!(c.scaling_factor > 0) || !(c.low_freq_factor > 0) ||
                               !(c.high_freq_factor > c.low_freq_factor) || c.original_context <= 0))
            return fail(PUTER_ERR_INVALID, "kv append: invalid Llama-3 scaling");
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
        a.mode = config->mode, a.start = config->start_position, a.base = config->base_freq, a.scaling = config->scaling;
        a.factor = config->scaling_factor, a.low = config->low_freq_factor, a.high = config->high_freq_factor;
        a.orig_ctx = (double)config->original_context;
    } else {
        a.mode = 1;
    }
    a.status = status;
    a.rows_per_block = write_rows_per_block(rows, rows <= 1024, &a.table_bits);
    if (a.rows_per_block > 256) {   // a thread brings each of the block's rows
        a.rows_per_block = 256;
        a.table_bits = 9;
    }
    const int64_t blocks = (rows + a.rows_per_block - 1) / a.rows_per_block;
    if (blocks > 0x7FFFFFFF) return fail(PUTER_ERR_INVALID, "kv append: too many rows");
    a.chunk_rows = (int)std::min<int64_t>(a.rows_per_block, std::max<int64_t>(1, 2048 / (head_dim / 2)));
    a.angles_at = (int)((write_lds_bytes(a.rows_per_block) + 15) & ~(size_t)15);
    const size_t lds = (size_t)a.angles_at + (size_t)(head_dim / 2) * 8 * (size_t)(1 + a.chunk_rows);
    const int cache = cache_dtype == dtype ? CACHE_SAME : cache_dtype == PUTER_F8E4M3 ? CACHE_FP8 : CACHE_I4;
    hipStream_t s = as_stream(stream);
    switch (dtype) {
    case PUTER_F32: launch_append<PUTER_F32>(a, cache, (unsigned)blocks, lds, s); break;
    case PUTER_BF16: launch_append<PUTER_BF16>(a, cache, (unsigned)blocks, lds, s); break;
    case PUTER_F16: launch_append<PUTER_F16>(a, cache, (unsigned)blocks, lds, s); break;
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
    if (kv_heads > 65536 || out_rows > 0x7FFFFFFFFFFFll / (kv_heads * head_dim))
        return fail(PUTER_ERR_INVALID, "kv gather int4: too many rows or heads");
    const int64_t units = kv_heads * head_dim / 8, total = out_rows * units;
    const unsigned blocks = (unsigned)std::min<int64_t>((total + 255) / 256, 1 << 20);
    hipStream_t s = as_stream(stream);
    const uint32_t *p = static_cast<const uint32_t *>(pages), *q = static_cast<const uint32_t *>(params);
    const int g8 = (int)(group / 8);
    switch (dtype) {
    case PUTER_F32: int4_gather_kernel<PUTER_F32><<<blocks, 256, 0, s>>>(p, q, page_table, output, page_count, page_size, units, g8, total, status); break;
    case PUTER_BF16: int4_gather_kernel<PUTER_BF16><<<blocks, 256, 0, s>>>(p, q, page_table, output, page_count, page_size, units, g8, total, status); break;
    case PUTER_F16: int4_gather_kernel<PUTER_F16><<<blocks, 256, 0, s>>>(p, q, page_table, output, page_count, page_size, units, g8, total, status); break;
    }
    return check_launch("kv gather int4");
}

}  // extern "C"
