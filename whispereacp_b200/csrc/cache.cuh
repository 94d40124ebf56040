// The paged key/value cache's device views and the pieces its kernels share
// (sm_100a): what include/wsp_cache.h describes, as kernels read it.
#pragma once

#include "common.cuh"

#include <cuda_fp8.h>

namespace wsp {

// The storage codes of wsp_cache.h.
constexpr int kCacheF16 = 1, kCacheBf16 = 2, kCacheE4m3 = 3, kCacheInt8 = 4;
__host__ __device__ constexpr bool cache_eight(int storage) { return storage >= kCacheE4m3; }
__host__ __device__ constexpr int cache_bytes(int storage) { return cache_eight(storage) ? 1 : 2; }

struct CacheView {
    unsigned char* keys;
    unsigned char* values;
    uint8_t* key_scales;    // [pages][heads][page_rows], null for 16-bit storage
    uint8_t* value_scales;
    long long page_bytes, head_bytes, row_bytes;  // strides of the pools
    int heads, pages, page_shift;                 // page_rows = 1 << page_shift
};

struct CacheBatchView {
    const int* table;
    const int* lengths;
    const int* starts;
    long long table_stride;
    int columns, sequences;
};

// One sequence of a batch: its first new row and how many it has, the position
// of the first, and the rows it holds that the table has places for.
struct CacheSequence {
    int first, rows, before, length;
};
__device__ __forceinline__ CacheSequence cache_sequence(const CacheView& c, const CacheBatchView& b, int s) {
    CacheSequence q;
    q.first = b.starts[s];
    q.rows = b.starts[s + 1] - q.first;
    const int length = b.lengths[s];
    q.before = length - q.rows;
    q.length = (int)max(0ll, min((long long)length, (long long)b.columns << c.page_shift));
    return q;
}

// The page of `position` of sequence s, -1 where there is none: behind the
// table's columns, before its first row, or an id outside the pool.
__device__ __forceinline__ int cache_page(const CacheView& c, const CacheBatchView& b, int s, int position) {
    if (position < 0) return -1;
    const int column = position >> c.page_shift;
    if (column >= b.columns) return -1;
    const int page = __ldg(b.table + s * b.table_stride + column);
    return (unsigned)page < (unsigned)c.pages ? page : -1;
}

// Bytes from a pool's base to a row of a page's head; offsets pass 32 bits.
__device__ __forceinline__ long long cache_offset(const CacheView& c, int page, int head, int row) {
    return page * c.page_bytes + head * c.head_bytes + row * c.row_bytes;
}
__device__ __forceinline__ long long cache_scale_index(const CacheView& c, int page, int head, int row) {
    return (((long long)page * c.heads + head) << c.page_shift) + row;
}

// What a scale byte stands for: 2^(b - 127), 0 for 0, NaN for 255.  The
// bits b << 23 are those of 2^(b - 127) for 1..254, of 0 for 0, and of
// infinity for 255, which the select makes a NaN.
__device__ __forceinline__ float cache_scale(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(byte << 23);
}

// Two held elements (their 16 or 2 x 16 bits) as floats, unscaled.
template <int S>
__device__ __forceinline__ float2 cache_pair(uint32_t bits) {
    if constexpr (S == kCacheF16) {
        return Half16<__half>::pair_to_float2(bits);
    } else if constexpr (S == kCacheBf16) {
        return Half16<__nv_bfloat16>::pair_to_float2(bits);
    } else if constexpr (S == kCacheE4m3) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)bits, __NV_E4M3);
        return __half22float2(__half2(h));
    } else {
        // 2^23 + (x + 128) has x + 128 in its low mantissa bits: no conversion,
        // of which an SM does 16 a cycle
        const uint32_t u = bits ^ 0x8080u;
        return make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7550)) - 8388736.f,
                           __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7551)) - 8388736.f);
    }
}

}  // namespace wsp
