// What the kernels that write page rows share: the device checks of page ids and slots, and
// which row of a call stores where several target one (page, slot): the last.
#pragma once

#include "common.hpp"

namespace puter {

__device__ __forceinline__ void flag_invalid(int32_t *status) {
    if (status) *status = PUTER_ERR_INVALID;
}

constexpr int kWriteMaxRows = 1024;  // rows per write block, at most
// threads per write block: 256 up to kSmallWriteRows rows, else 1024
constexpr int kSmallWriteRows = 8192;
constexpr int kScanKeys = 16;        // later-row keys per thread per scan step
constexpr uint64_t kNoKey = ~(uint64_t)0;
constexpr int kBufWord3 = 0x00020000;  // buffer resource word 3: raw buffer, dword access

// The block's share of LDS for the last-row-wins table (dynamic shared memory,
// write_lds_bytes(R)): a 65536-bit filter with one bit set per block key (a
// later row whose bit is clear cannot match: one LDS read per streamed key, no
// probe chain), T = 2R entries of (key, highest local row, hit flag), and per
// local row its entry (-1: the row is out of range and stores nothing).
constexpr int kFilterWords = 2048;  // 65536 bits
struct WriteTable {
    uint32_t *filter;
    uint64_t *key;
    int *last;
    int *hit;
    int *entry;
    int bits;  // log2 T
};
static inline size_t write_lds_bytes(int64_t r) {
    return (size_t)kFilterWords * 4 + (size_t)r * 2 * (8 + 4 + 4) + (size_t)r * 4;
}

__device__ __forceinline__ WriteTable write_table(char *lds, int64_t r, int bits) {
    WriteTable t;
    t.filter = reinterpret_cast<uint32_t *>(lds);
    t.key = reinterpret_cast<uint64_t *>(t.filter + kFilterWords);
    t.last = reinterpret_cast<int *>(t.key + 2 * r);
    t.hit = t.last + 2 * r;
    t.entry = t.hit + 2 * r;
    t.bits = bits;
    return t;
}

// key of a (page id, slot) pair and its table position, in 32-bit arithmetic
__device__ __forceinline__ uint64_t write_key(int32_t id, int32_t off) {
    return ((uint64_t)(uint32_t)id << 32) | (uint32_t)off;
}
__device__ __forceinline__ uint32_t write_mix(int32_t id, int32_t off) {
    return (uint32_t)id * 0x9E3779B1u + (uint32_t)off * 0x85EBCA77u;
}
__device__ __forceinline__ uint32_t write_hash(int32_t id, int32_t off, int bits) {
    return write_mix(id, off) >> (32 - bits);
}
// id in [0, page_count) and off in [0, page_size), both bounds clamped to int32
// (ids and slots are int32)
__device__ __forceinline__ bool write_valid(int32_t id, int32_t off, int32_t pc, int32_t ps) {
    return id >= 0 && id < pc && off >= 0 && off < ps;
}

// Keys of the later rows [jb, jb + kScanKeys * THREADS): unconditional
// buffer loads that share one VGPR offset (the thread's) and step by an SGPR
// offset, so they hold no addresses of their own; the resources end at the last
// row and lanes past it read zeros (skipped by index in scan_probe).
struct ScanChunk {
    int32_t id[kScanKeys], off[kScanKeys];
};
template <int THREADS>
__device__ __forceinline__ void scan_load(ScanChunk &c, const int32_t *__restrict__ ids,
                                          const int32_t *__restrict__ offsets, int64_t jb, int64_t value_rows) {
    const int tid = threadIdx.x;
    const int64_t stride = (int64_t)THREADS * kScanKeys;
    const int bytes = (int)(max((int64_t)0, min(value_rows - jb, stride)) * 4);
    const __amdgpu_buffer_rsrc_t ir = __builtin_amdgcn_make_buffer_rsrc((void *)(ids + jb), (short)0, bytes, kBufWord3);
    const __amdgpu_buffer_rsrc_t orc =
        __builtin_amdgcn_make_buffer_rsrc((void *)(offsets + jb), (short)0, bytes, kBufWord3);
#pragma unroll
    for (int u = 0; u < kScanKeys; ++u) {
        c.id[u] = (int32_t)__builtin_amdgcn_raw_buffer_load_b32(ir, tid * 4, u * THREADS * 4, 0);
        c.off[u] = (int32_t)__builtin_amdgcn_raw_buffer_load_b32(orc, tid * 4, u * THREADS * 4, 0);
    }
}
// Marks the table entries that the chunk's keys hit (`left` = rows from the
// chunk's first row to the last row): a key whose filter bit is clear matches
// no block key; the few that pass take the exact lookup.
template <int THREADS>
__device__ __forceinline__ void scan_probe(const WriteTable &t, const ScanChunk &c, int64_t left, int32_t pc,
                                           int32_t ps) {
    const int tid = threadIdx.x, T = 1 << t.bits;
    uint32_t maybe = 0;  // bit u: key u's filter bit is set
#pragma unroll
    for (int u = 0; u < kScanKeys; ++u) {
        const uint32_t f = write_mix(c.id[u], c.off[u]) & 0xFFFFu;
        maybe |= ((t.filter[f >> 5] >> (f & 31)) & 1u) << u;
    }
    while (maybe) {
        const int u = __builtin_ctz(maybe);
        maybe &= maybe - 1;
        int32_t kid = c.id[0], koff = c.off[0];
#pragma unroll
        for (int w = 1; w < kScanKeys; ++w)
            if (w == u) kid = c.id[w], koff = c.off[w];
        if (tid + u * THREADS >= left || !write_valid(kid, koff, pc, ps)) continue;
        const uint64_t k = write_key(kid, koff);
        uint32_t h = write_hash(kid, koff, t.bits);
        // the table holds at most T / 2 keys: an empty entry ends every probe
        for (uint64_t cur = t.key[h]; cur != kNoKey; cur = t.key[h]) {
            if (cur == k) {
                t.hit[h] = 1;
                break;
            }
            h = (h + 1) & (uint32_t)(T - 1);
        }
    }
}

// (The write kernels take their block size as the template constant THREADS,
// not blockDim.x, which is read from the dispatch packet by a load whose wait
// would drain every load issued before it.)
//
// Which of the block's rows [row0, row0 + nrows) store (after the call, every
// thread of the block sees t.entry / t.last / t.hit): out-of-range ids or slots
// flag the status word and store nothing; among the rows of one slot only the
// highest stores.  Thread i < nrows brings local row i's (id, slot), and every
// thread the keys of its share of the first chunk of later rows (c0, from row
// row0 + nrows), both loaded by the caller at the kernel's start so that they
// and its other loads share one round trip (nrows <= the block's threads).
// Later chunks (16 x THREADS rows each: 16K for a 1024-thread block) are loaded
// here.  Ends with a barrier.
template <int THREADS>
__device__ void write_winners(const WriteTable &t, int32_t my_id, int32_t my_off, const ScanChunk &c0,
                              const int32_t *__restrict__ ids, const int32_t *__restrict__ offsets,
                              int64_t row0, int nrows, int64_t value_rows, int64_t page_count,
                              int64_t page_size, int32_t *status) {
    const int tid = threadIdx.x, T = 1 << t.bits;
    const int32_t pc = (int32_t)min(page_count, (int64_t)0x7FFFFFFF);
    const int32_t ps = (int32_t)min(page_size, (int64_t)0x7FFFFFFF);
    for (int e = tid; e < T; e += THREADS) {
        t.key[e] = kNoKey;
        t.last[e] = -1;
        t.hit[e] = 0;
    }
    for (int w = tid; w < kFilterWords; w += THREADS) t.filter[w] = 0;
    __syncthreads();
    if (tid < nrows) {
        if (!write_valid(my_id, my_off, pc, ps)) {
            flag_invalid(status);
            t.entry[tid] = -1;
        } else {
            const uint64_t k = write_key(my_id, my_off);
            uint32_t h = write_hash(my_id, my_off, t.bits);
            // at most nrows <= T / 2 keys: an empty entry is always reached
            for (;;) {
                const uint64_t prev = atomicCAS(reinterpret_cast<unsigned long long *>(&t.key[h]),
                                                (unsigned long long)kNoKey, (unsigned long long)k);
                if (prev == kNoKey || prev == k) break;
                h = (h + 1) & (uint32_t)(T - 1);
            }
            atomicMax(&t.last[h], tid);
            t.entry[tid] = (int)h;
            const uint32_t f = write_mix(my_id, my_off) & 0xFFFFu;
            atomicOr(&t.filter[f >> 5], 1u << (f & 31));
        }
    }
    __syncthreads();
    const int64_t first = row0 + nrows;
    const int64_t stride = (int64_t)THREADS * kScanKeys;
    if (first < value_rows) scan_probe<THREADS>(t, c0, value_rows - first, pc, ps);
    for (int64_t jb = first + stride; jb < value_rows; jb += stride) {
        ScanChunk c;
        scan_load<THREADS>(c, ids, offsets, jb, value_rows);
        scan_probe<THREADS>(t, c, value_rows - jb, pc, ps);
    }
    __syncthreads();
}

__device__ __forceinline__ bool write_wins(const WriteTable &t, int i) {
    const int e = t.entry[i];
    return e >= 0 && t.last[e] == i && t.hit[e] == 0;
}
// Unconditional loads of one V unit through a buffer resource (a unit past the
// resource's range reads as zero): with no branch around them the compiler's
// wait counts stay exact, so later waits need not drain these loads.
template <typename V> __device__ __forceinline__ V buf_load(__amdgpu_buffer_rsrc_t r, int vo, int so);
template <> __device__ __forceinline__ uint4 buf_load<uint4>(__amdgpu_buffer_rsrc_t r, int vo, int so) {
    const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, vo, so, 0);
    return make_uint4(v[0], v[1], v[2], v[3]);
}
template <> __device__ __forceinline__ uint32_t buf_load<uint32_t>(__amdgpu_buffer_rsrc_t r, int vo, int so) {
    return __builtin_amdgcn_raw_buffer_load_b32(r, vo, so, 0);
}
template <> __device__ __forceinline__ uint8_t buf_load<uint8_t>(__amdgpu_buffer_rsrc_t r, int vo, int so) {
    return __builtin_amdgcn_raw_buffer_load_b8(r, vo, so, 0);
}

// the pool row (page id * page_size + slot) of a local row that passed write_wins
__device__ __forceinline__ int64_t write_slot(const WriteTable &t, int i, int64_t page_size) {
    const uint64_t k = t.key[t.entry[i]];
    return (int64_t)(k >> 32) * page_size + (int64_t)(uint32_t)k;
}

// Rows per write block (a power of two, from 2, when the rows are to be spread, or 8 to 1024,
// about rows / 512; at most 16 for the 256-thread blocks of calls up to kSmallWriteRows
// rows, so R never exceeds the block's threads) and log2 of its table size (2R entries).
static inline int64_t write_rows_per_block(int64_t rows, bool spread, int *table_bits) {
    int64_t r = spread ? 2 : 8;
    while (r < kWriteMaxRows && r * 512 < rows) r <<= 1;
    int bits = 0;
    while (((int64_t)1 << bits) < 2 * r) ++bits;
    *table_bits = bits;
    return r;
}

}  // namespace puter
