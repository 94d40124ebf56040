// The attention of new rows over a paged cache (sm_100a): the kernel of few
// rows -- single tokens, chunks of a few -- and the join of its splits.
//
// o_i = sum_j p_ij v_j / sum_j p_ij, p_ij = 2^(s_ij - m_i), s_ij = scale log2(e)
// q_i . k_j, with the maximum m_i and both sums running over the keys.
//
// Few rows read every held key and value once and do little with them, so the
// kernel is bound by HBM: all that matters is that every SM keeps enough bytes
// in flight until the last key.  The work is the list of units (sequence, key
// head, 16-row tile, 64 keys), in that order, and every CTA takes an equal run
// of it, wherever items (sequence, head, tile) begin and end: ragged lengths
// cannot unbalance it.  An item cut by a run's border leaves partial results
// (m, sum, o) in the workspace, which cache_join_kernel adds in order, so the
// result has the same bits every time.
//
// In a CTA a producer warp copies units' keys and values into a ring of
// shared-memory stages (bulk tensor copies, a box a page), and four warps take
// 16 keys of each unit: scores by mma.sync m16n8k16 with the rows as A, one
// running softmax a warp, P (as two 16-bit halves, hi + lo: no rounding that
// shows) times the values.  A single token fills one of the tile's 16 rows;
// the tensor cores are idle enough.  The warps' results meet once per item.
//
// 8-bit keys and values become fp16 exactly (both types fit) and are
// multiplied unscaled.  A key's scale multiplies its score; a value's scale
// multiplies its probability, relative to the warp's largest so far, so that
// the product stays in fp16's range whatever the scales are.  bf16 queries
// become fp16 after a power of two a row brings them near 1.
#include "cache_device.cuh"
#include "host.h"

#include <algorithm>

namespace wsp {
namespace {

constexpr int kUnitKeys = 64;
constexpr int kTileRows = 16;
constexpr int kWorkers = 4;  // consumer warps, 16 keys of a unit each
constexpr int kTokenThreads = 32 * (kWorkers + 1);

enum CacheWait : int { kWaitFull = 1, kWaitFree = 2, kWaitDrain = 3 };

// Shared memory: the stages, the item join's rows, the warps' softmax rows,
// barriers and the abort flag.  More bytes of stages than about 64 KB a CTA
// and 128 KB an SM gained nothing.
template <int S, int D>
struct TokenLayout {
    static constexpr int row_bytes = D * cache_bytes(S);
    static constexpr int span = row_bytes < 128 ? row_bytes : 128;  // bytes of a box's row
    static constexpr int halves = row_bytes / span;
    static constexpr int pool_bytes = kUnitKeys * row_bytes;        // a unit's keys, or values
    static constexpr int scale_bytes = cache_eight(S) ? 128 : 0;    // 64 key bytes, 64 value bytes
    static constexpr int stages = pool_bytes <= 4096 ? 8 : pool_bytes <= 8192 ? 4 : 3;
    static constexpr int scale_at = stages * 2 * pool_bytes;
    static constexpr int join_at = scale_at + stages * scale_bytes;
    static constexpr int ml_at = join_at + 2 * kTileRows * D * 4;
    static constexpr int bar_at = ml_at + kWorkers * kTileRows * 2 * 4;
    static constexpr int bytes = bar_at + 2 * stages * 8 + 16;
    // CTAs that an SM's 228 KB hold, 1 KB each being the system's
    static constexpr int ctas = 233472 / (bytes + 1024);
};

// A run of the unit list.
struct Runs {
    long long units, per;  // units of the call, units of a CTA's run
};

// Workspace: a cut item's record for each CTA whose run begins inside one,
// then two partial results for each CTA: [0] of the item its run begins in,
// [1] of the item its run ends in.
struct CutItem {
    long long first_unit, units;  // the item's; units 0: the run begins with an item
    int sequence, head, tile, pad;
};
template <int D>
struct Partial {
    static constexpr int floats = kTileRows * (D + 2);  // o, then m, then sum
};

__device__ __forceinline__ int item_units(int length) { return max(1, (length + kUnitKeys - 1) / kUnitKeys); }

// The items of a sequence of one head: 16-row tiles of its n * group rows.
__device__ __forceinline__ int item_tiles(const CacheSequence& q, int group) {
    return q.rows > 0 ? (int)(((long long)q.rows * group + kTileRows - 1) / kTileRows) : 0;
}
__device__ __forceinline__ long long sequence_units(const CacheSequence& q, int group, int heads) {
    return (long long)item_tiles(q, group) * heads * item_units(q.length);
}

// Where a unit lies; every warp finds it for itself.
struct Place {
    int s;            // sequence
    CacheSequence q;
    int head, tile;
    int unit;         // of the item
    int units, tiles; // of the item; items of a head
};

__device__ __forceinline__ long long warp_scan(long long v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
    }
    return v;
}

__device__ long long all_units(const CacheBatchView& b, int group, int heads, int lane) {
    long long sum = 0;
    for (int s = lane; s < b.sequences; s += 32) sum += sequence_units(cache_sequence(b, s), group, heads);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// The place of unit u (below all_units); a warp.
__device__ Place find_unit(const CacheBatchView& b, int group, int heads, long long u, int lane) {
    Place p{};
    for (int base = 0; base < b.sequences; base += 32) {
        const int s = base + lane;
        CacheSequence q{};
        if (s < b.sequences) q = cache_sequence(b, s);
        const long long mine = s < b.sequences ? sequence_units(q, group, heads) : 0;
        const long long upto = warp_scan(mine, lane);
        const unsigned holds = __ballot_sync(0xffffffffu, u < upto);
        if (holds) {
            const int at = __ffs(holds) - 1;
            const long long inside = __shfl_sync(0xffffffffu, u - (upto - mine), at);
            p.s = base + at;
            p.q.first = __shfl_sync(0xffffffffu, q.first, at);
            p.q.rows = __shfl_sync(0xffffffffu, q.rows, at);
            p.q.length = __shfl_sync(0xffffffffu, q.length, at);
            p.units = item_units(p.q.length);
            p.tiles = item_tiles(p.q, group);
            const long long item = inside / p.units;
            p.unit = (int)(inside - item * p.units);
            p.head = (int)(item / p.tiles);
            p.tile = (int)(item - (long long)p.head * p.tiles);
            return p;
        }
        u -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return p;
}

// The next item's first unit.
__device__ __forceinline__ void next_item(Place& p, const CacheBatchView& b, int group, int heads) {
    p.unit = 0;
    if (++p.tile < p.tiles) return;
    p.tile = 0;
    if (++p.head < heads) return;
    p.head = 0;
    while (++p.s < b.sequences) {
        p.q = cache_sequence(b, p.s);
        p.tiles = item_tiles(p.q, group);
        if (p.tiles > 0) break;
    }
    p.units = item_units(p.q.length);
}

// ------------------------------------------------------------ tensor pieces

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(address)
                 : "memory");
}

// Bytes {i0, i1} of four held 8-bit values as two fp16, exact.
template <int S>
__device__ __forceinline__ void widen4(uint32_t bytes, bool interleaved, uint32_t& lo, uint32_t& hi) {
    if constexpr (S == kCacheE4m3) {
        const uint32_t b = interleaved ? __byte_perm(bytes, 0, 0x3120) : bytes;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"((uint16_t)(b & 0xffffu)));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"((uint16_t)(b >> 16)));
    } else {
        // 1024 + (x + 128) has x + 128 in its low mantissa bits
        const uint32_t u = bytes ^ 0x80808080u;
        lo = __byte_perm(u, 0x64646464u, interleaved ? 0x4240 : 0x4140);
        hi = __byte_perm(u, 0x64646464u, interleaved ? 0x4341 : 0x4342);
        const __half2 base = __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));  // 1152
        __half2 a = __hsub2(*reinterpret_cast<__half2*>(&lo), base), b = __hsub2(*reinterpret_cast<__half2*>(&hi), base);
        lo = *reinterpret_cast<uint32_t*>(&a);
        hi = *reinterpret_cast<uint32_t*>(&b);
    }
}

// The byte offset of 16-byte piece c of row r in a swizzled box of `span`
// byte rows: the copy engine's 128- or 64-byte pattern.
template <int kSpan>
__device__ __forceinline__ uint32_t swizzled(int r, int c) {
    if constexpr (kSpan == 128) return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
    else return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// --------------------------------------------------------------- the kernel

template <typename T, int S, int D>
__global__ void __launch_bounds__(kTokenThreads, TokenLayout<S, D>::ctas)
    cache_tokens_kernel(const __grid_constant__ CacheAttendArgs a, const __grid_constant__ CacheMaps maps) {
    using Layout = TokenLayout<S, D>;
    using MT = typename std::conditional<cache_eight(S), __half, T>::type;  // the products' type
    constexpr bool kEight = cache_eight(S);
    constexpr int kSteps = D / 16;   // k16 steps of a score, 16-wide groups of values
    extern __shared__ __align__(1024) unsigned char smem[];  // the swizzle counts from 1024-byte borders
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Layout::bar_at);
    uint64_t* empty = full + Layout::stages;
    volatile int* abort = reinterpret_cast<volatile int*>(empty + Layout::stages);
    int* redo = reinterpret_cast<int*>(empty + Layout::stages) + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int heads = a.cache.heads;

    if (threadIdx.x == 0) {
        for (int i = 0; i < Layout::stages; ++i) {
            cache_barrier_init(full + i, 1);
            cache_barrier_init(empty + i, kWorkers);
        }
        *abort = 0;
        *redo = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const long long total = all_units(a.batch, a.group, heads, lane);
    const long long per = max(1ll, (total + gridDim.x - 1) / gridDim.x);
    const long long begin = min(total, blockIdx.x * per), end = min(total, begin + per);
    CutItem* cuts = reinterpret_cast<CutItem*>(a.workspace);
    float* partials = reinterpret_cast<float*>(a.workspace + ((sizeof(CutItem) * gridDim.x + 255) / 256) * 256);
    Place p = begin < end ? find_unit(a.batch, a.group, heads, begin, lane) : Place{};
    if (threadIdx.x == 0) {
        CutItem cut{};
        if (begin < end && p.unit > 0) cut = {begin - p.unit, p.units, p.s, p.head, p.tile, 0};
        cuts[blockIdx.x] = cut;
    }
    __syncthreads();

    if (warp == kWorkers) {
        // ------------------------------------------------------- producer
        const int box_shift = cache_box_shift(a.cache.page_shift);
        const int boxes = kUnitKeys >> box_shift;  // of a unit: 1, 2 or 4
        int table_s = -1, table_base = 0, entry = -1;
        unsigned long long n = 0;
        for (long long u = begin; u < end;) {
            const int last = (int)min((long long)p.units, p.unit + (end - u));
            for (int t = p.unit; t < last; ++t, ++u, ++n) {
                const int stage = (int)(n % Layout::stages);
                if (n >= Layout::stages &&
                    !cache_wait(empty + stage, (uint32_t)((n / Layout::stages - 1) & 1), abort, a.status, kWaitFree))
                    break;
                if (*abort) break;
                // 32 table entries at a time, a lane an entry
                const int column = (t * kUnitKeys) >> a.cache.page_shift;
                if (p.s != table_s || column < table_base || column + boxes > table_base + 32) {
                    table_s = p.s;
                    table_base = column;
                    entry = cache_page(a.cache, a.batch, p.s, (int)min((long long)(column + lane) << a.cache.page_shift, 0x7fffffffll));
                }
                const int b = min(lane, boxes - 1);
                const int position = t * kUnitKeys + (b << box_shift);
                const int page = __shfl_sync(0xffffffffu, entry, (position >> a.cache.page_shift) - table_base);
                const bool mine = lane < boxes && position < p.q.length;
                unsigned char* keys = smem + stage * 2 * Layout::pool_bytes;
                unsigned char* values = keys + Layout::pool_bytes;
                uint8_t* scales = smem + Layout::scale_at + stage * Layout::scale_bytes;
                const int box_rows = 1 << box_shift;
                const int row = position & ((1 << a.cache.page_shift) - 1);
                const unsigned live = __ballot_sync(0xffffffffu, mine);
                uint32_t bytes = (uint32_t)__popc(live) * 2u * (uint32_t)(box_rows * Layout::row_bytes);
                if (kEight) {
                    const unsigned paged = __ballot_sync(0xffffffffu, mine && page >= 0);
                    bytes += (uint32_t)__popc(paged) * 2u * (uint32_t)box_rows;
                    if (mine && page < 0)
                        for (int i = 0; i < box_rows; i += 4) {
                            *reinterpret_cast<uint32_t*>(scales + b * box_rows + i) = 0;
                            *reinterpret_cast<uint32_t*>(scales + 64 + b * box_rows + i) = 0;
                        }
                    if (mine && page < 0) cache_proxy_fence();
                    __syncwarp();
                }
                if (lane == 0) cache_arrive_expect(full + stage, bytes);
                __syncwarp();
                if (mine) {
                    const int at = page >= 0 ? page : a.cache.pages;  // outside: zeros
#pragma unroll
                    for (int h = 0; h < Layout::halves; ++h) {
                        const int to = h * kUnitKeys * Layout::span + b * box_rows * Layout::span;
                        cache_copy_box(keys + to, &maps.keys, h * 64, row, p.head, at, full + stage);
                        cache_copy_box(values + to, &maps.values, h * 64, row, p.head, at, full + stage);
                    }
                    if (kEight && page >= 0) {
                        const long long si = cache_scale_index(a.cache, page, p.head, row);
                        cache_copy_bytes(scales + b * box_rows, a.cache.key_scales + si, box_rows, full + stage);
                        cache_copy_bytes(scales + 64 + b * box_rows, a.cache.value_scales + si, box_rows, full + stage);
                    }
                }
            }
            if (*abort) break;
            next_item(p, a.batch, a.group, heads);
        }
        if (*abort)  // the copies in flight land before the CTA's memory is given up
            for (unsigned long long i = n > Layout::stages ? n - Layout::stages : 0; i < n; ++i) {
                const unsigned long long start = cache_clock_ns();
                while (!cache_phase_done(full + i % Layout::stages, (uint32_t)((i / Layout::stages) & 1)) &&
                       cache_clock_ns() - start < kCacheTimeoutNs) {
                }
            }
        return;
    }

    // ----------------------------------------------------------- consumers
    const int g = lane >> 2, t4 = lane & 3;
    float* join = reinterpret_cast<float*>(smem + Layout::join_at);
    float* ml = reinterpret_cast<float*>(smem + Layout::ml_at);
    unsigned long long n = 0;
    for (long long u = begin; u < end;) {
        const int last = (int)min((long long)p.units, p.unit + (end - u));
        const TileRow rows[2] = {tile_row(a, p.q, p.head, p.tile * kTileRows + g),
                                 tile_row(a, p.q, p.head, p.tile * kTileRows + g + 8)};
        // The rows' fragments.  16-bit: element pairs 2t, 2t + 1 and 2t + 8, 2t
        // + 9 of each 16.  8-bit: 4t .. 4t + 3, the order in which a lane's
        // four bytes of a key come.
        uint32_t qf[kSteps][4];
        float unscale[2] = {1.f, 1.f};
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const unsigned char* qp =
                a.queries + ((long long)p.q.first + rows[r].token) * a.q_row + rows[r].head * a.q_head;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                qf[k][r] = qf[k][r + 2] = 0;
                if (rows[r].valid) {
                    if (kEight) {
                        const uint2 v = *reinterpret_cast<const uint2*>(qp + k * 32 + t4 * 8);
                        qf[k][r] = v.x;
                        qf[k][r + 2] = v.y;
                    } else {
                        qf[k][r] = *reinterpret_cast<const uint32_t*>(qp + k * 32 + t4 * 4);
                        qf[k][r + 2] = *reinterpret_cast<const uint32_t*>(qp + k * 32 + t4 * 4 + 16);
                    }
                }
            }
            if constexpr (kEight && std::is_same<T, __nv_bfloat16>::value) {
                // fp16 holds a bf16 exactly between 2^-14 and 2^15: bring the
                // row's largest to 2^8.. and keep the power of two.
                float top = 0.f;
#pragma unroll
                for (int k = 0; k < kSteps; ++k)
#pragma unroll
                    for (int h = 0; h < 4; h += 2) {
                        const float2 f = Half16<T>::pair_to_float2(qf[k][r + h]);
                        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e = (int)(__float_as_uint(top) >> 23);  // biased; 255: not finite
                const bool fine = e < 255 && e > 20;
                const float down = fine ? __uint_as_float((uint32_t)max(1, 262 - e) << 23) : 1.f;  // 2^(135 - e)
                unscale[r] = fine ? __uint_as_float((uint32_t)max(1, e - 8) << 23) : 1.f;          // 2^(e - 135)
#pragma unroll
                for (int k = 0; k < kSteps; ++k)
#pragma unroll
                    for (int h = 0; h < 4; h += 2) {
                        const float2 f = Half16<T>::pair_to_float2(qf[k][r + h]);
                        qf[k][r + h] = Half16<__half>::pack2(f.x * down, f.y * down);
                    }
            }
        }
        const float to_log2[2] = {a.scale * kLog2e * unscale[0], a.scale * kLog2e * unscale[1]};
        float o[kSteps][8];  // 16 values' columns: two n8 tiles of 4
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) o[k][e] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
        int largest = 0;  // the value scales' largest byte so far
        // Keys below `clear` are seen by every row of the tile that counts.
        int clear = p.q.length;
        if (a.causal) clear = tile_row(a, p.q, p.head, p.tile * kTileRows).seen;

        for (int t = p.unit; t < last; ++t, ++u, ++n) {
            const int stage = (int)(n % Layout::stages);
            cache_wait(full + stage, (uint32_t)((n / Layout::stages) & 1), abort, a.status, kWaitFull);
            unsigned char* keys = smem + stage * 2 * Layout::pool_bytes;
            unsigned char* values = keys + Layout::pool_bytes;
            const uint8_t* scales = smem + Layout::scale_at + stage * Layout::scale_bytes;
            const int key0 = t * kUnitKeys + warp * 16;
            if (key0 < p.q.length) {
                if (key0 + 16 > p.q.length) {
                    // What lies behind the last row may be anything, and 0
                    // times a NaN is one.
                    constexpr int kPieces = Layout::row_bytes / 16;
                    for (int i = lane; i < 16 * kPieces; i += 32) {
                        const int r = i / kPieces, c = i % kPieces;
                        if (key0 + r >= p.q.length)
                            *reinterpret_cast<uint4*>(values + (c / (Layout::span / 16)) * kUnitKeys * Layout::span +
                                                      swizzled<Layout::span>(warp * 16 + r, c % (Layout::span / 16))) =
                                make_uint4(0, 0, 0, 0);
                    }
                    cache_proxy_fence();
                    __syncwarp();
                }
                float s[2][4] = {};
                const uint32_t key_base = smem_address(keys), value_base = smem_address(values);
                if constexpr (!kEight) {
                    const int r = warp * 16 + (lane >> 4) * 8 + (lane & 7), c = (lane >> 3) & 1;
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        uint32_t b[4];
                        ldmatrix4(b, key_base + (k / 4) * kUnitKeys * 128 + swizzled<128>(r, (k % 4) * 2 + c));
                        mma_16816<MT>(s[0], qf[k], b);
                        mma_16816<MT>(s[1], qf[k], b + 2);
                    }
                } else {
                    const int r = warp * 16 + (lane >> 4) * 8 + (lane & 7), c = (lane >> 3) & 1;
#pragma unroll
                    for (int k = 0; k < kSteps; k += 2) {
                        uint32_t b[4], w[2];
                        ldmatrix4(b, key_base + swizzled<Layout::span>(r, k + c));
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            widen4<S>(b[h], false, w[0], w[1]);
                            mma_16816<MT>(s[0], qf[k + h], w);
                            widen4<S>(b[2 + h], false, w[0], w[1]);
                            mma_16816<MT>(s[1], qf[k + h], w);
                        }
                    }
                }
                // Scores in log2, masked where a row does not see the key.
                float factor[2][2];
                if constexpr (kEight) {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t kb = *reinterpret_cast<const uint16_t*>(scales + warp * 16 + j * 8 + t4 * 2);
                        const float k0 = cache_scale(kb & 255u), k1 = cache_scale(kb >> 8);
                        s[j][0] *= k0 * to_log2[0], s[j][1] *= k1 * to_log2[0];
                        s[j][2] *= k0 * to_log2[1], s[j][3] *= k1 * to_log2[1];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        s[j][0] *= to_log2[0], s[j][1] *= to_log2[0];
                        s[j][2] *= to_log2[1], s[j][3] *= to_log2[1];
                    }
                }
                const bool masked = key0 + 16 > clear;
                if (masked)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (key0 + j * 8 + t4 * 2 + (e & 1) >= rows[e >> 1].seen) s[j][e] = -INFINITY;
                float alpha[2];
                bool grew = false;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float top = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    top = fmaxf(top, m[r]);
                    const float from = top == -INFINITY ? 0.f : top;
                    grew |= top > m[r];
                    alpha[r] = exp2_fast(m[r] - from);
                    m[r] = top;
                    float part = 0.f;
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 2 * r; e < 2 * r + 2; ++e) {
                            s[j][e] = exp2_fast(s[j][e] - from);
                            part += s[j][e];
                        }
                    sum[r] = sum[r] * alpha[r] + part;
                }
                float relative = 1.f;
                if constexpr (kEight) {
                    // The values' scale bytes, those behind the last row as 0.
                    uint32_t byte[2][2];
                    int top = largest;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t vb = *reinterpret_cast<const uint16_t*>(scales + 64 + warp * 16 + j * 8 + t4 * 2);
                        byte[j][0] = vb & 255u;
                        byte[j][1] = vb >> 8;
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            if (key0 + j * 8 + t4 * 2 + e >= p.q.length) byte[j][e] = 0;
                            if (byte[j][e] < 255u) top = max(top, (int)byte[j][e]);
                        }
                    }
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    if (top > largest) {
                        const int drop = largest == 0 ? 127 : top - largest;
                        relative = drop < 127 ? __uint_as_float((uint32_t)(127 - drop) << 23) : 0.f;
                        largest = top;
                        grew = true;
                    }
                    // 2^15 for the largest: hi + lo in fp16 then reaches 2^-40 of it
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int x = (int)byte[j][e] - largest + 142;
                            factor[j][e] = byte[j][e] == 255u ? cache_scale(255u)
                                           : byte[j][e] == 0u || x <= 0 ? 0.f
                                                                        : __uint_as_float((uint32_t)x << 23);
                        }
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool unseen = masked && key0 + j * 8 + t4 * 2 + (e & 1) >= rows[e >> 1].seen;
                            s[j][e] = unseen ? 0.f : s[j][e] * factor[j][e & 1];
                        }
                }
                if (__any_sync(0xffffffffu, grew)) {
                    const float a0 = alpha[0] * relative, a1 = alpha[1] * relative;
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        o[k][0] *= a0, o[k][1] *= a0, o[k][4] *= a0, o[k][5] *= a0;
                        o[k][2] *= a1, o[k][3] *= a1, o[k][6] *= a1, o[k][7] *= a1;
                    }
                }
                uint32_t hi[4], lo[4];
                split_pair<MT>(s[0][0], s[0][1], hi[0], lo[0]);
                split_pair<MT>(s[0][2], s[0][3], hi[1], lo[1]);
                split_pair<MT>(s[1][0], s[1][1], hi[2], lo[2]);
                split_pair<MT>(s[1][2], s[1][3], hi[3], lo[3]);
                const int r = warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), c = lane >> 4;
                if constexpr (!kEight) {
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        uint32_t b[4];
                        ldmatrix4_t(b, value_base + (k / 4) * kUnitKeys * 128 + swizzled<128>(r, (k % 4) * 2 + c));
                        mma_16816<MT>(o[k], hi, b);
                        mma_16816<MT>(o[k] + 4, hi, b + 2);
                        mma_16816<MT>(o[k], lo, b);
                        mma_16816<MT>(o[k] + 4, lo, b + 2);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < kSteps; k += 2) {
                        uint32_t b[4];
                        ldmatrix4_t(b, value_base + swizzled<Layout::span>(r, k + c));
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t even[2], odd[2];
                            widen4<S>(b[2 * h], true, even[0], odd[0]);
                            widen4<S>(b[2 * h + 1], true, even[1], odd[1]);
                            mma_16816<MT>(o[k + h], hi, even);
                            mma_16816<MT>(o[k + h] + 4, hi, odd);
                            mma_16816<MT>(o[k + h], lo, even);
                            mma_16816<MT>(o[k + h] + 4, lo, odd);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) cache_arrive(empty + stage);
        }

        // ------------------------------------------- the warps' results meet
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
            sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
            if (t4 == 0) {
                ml[(warp * kTileRows + g + 8 * r) * 2] = m[r];
                ml[(warp * kTileRows + g + 8 * r) * 2 + 1] = sum[r];
            }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        float top[2], all[2], mine[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            top[r] = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWorkers; ++w) top[r] = fmaxf(top[r], ml[(w * kTileRows + g + 8 * r) * 2]);
            const float from = top[r] == -INFINITY ? 0.f : top[r];
            all[r] = 0.f;
#pragma unroll
            for (int w = 0; w < kWorkers; ++w)
                all[r] += ml[(w * kTileRows + g + 8 * r) * 2 + 1] * exp2_fast(ml[(w * kTileRows + g + 8 * r) * 2] - from);
            mine[r] = exp2_fast(m[r] - from);
        }
        if constexpr (kEight) {
            // o is in units of 2^(largest - 127 - 15)
            const float unit = cache_scale((uint32_t)largest);
            mine[0] = mine[0] * unit * 0x1p-15f;
            mine[1] = mine[1] * unit * 0x1p-15f;
        }
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) o[k][e] *= mine[(e >> 1) & 1];
        // A lane's column pairs of step k: 16-bit, 8 columns apart; 8-bit, the
        // even and the odd columns of four neighbours.
        const bool both = (long long)p.q.rows * a.group - p.tile * kTileRows > 8;
        const auto exchange = [&](float* to, bool add) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if (r && !both) break;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    float4* at = reinterpret_cast<float4*>(to + ((r * kSteps + k) * 32 + lane) * 4);
                    if (add) {
                        const float4 v = *at;
                        o[k][2 * r] += v.x, o[k][2 * r + 1] += v.y, o[k][4 + 2 * r] += v.z, o[k][5 + 2 * r] += v.w;
                    } else {
                        *at = make_float4(o[k][2 * r], o[k][2 * r + 1], o[k][4 + 2 * r], o[k][5 + 2 * r]);
                    }
                }
            }
        };
        if (warp >= 2) exchange(join + (warp - 2) * kTileRows * D, false);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (warp < 2) exchange(join + warp * kTileRows * D, true);
        if (warp == 1) exchange(join + kTileRows * D, false);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const bool whole = p.unit == 0 && last == p.units;
        if (warp == 0) {
            exchange(join + kTileRows * D, true);
            const long long slot = (long long)blockIdx.x * 2 + (p.unit > 0 ? 0 : 1);
            float* part = partials + slot * Partial<D>::floats;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if (!rows[r].valid) continue;
                const int row = g + 8 * r;
                const long long at = (long long)p.q.first + rows[r].token;
                if (whole) {
                    const float inverse = rows[r].seen > 0 ? 1.f / all[r] : 0.f;
                    unsigned char* op = a.out + at * a.o_row + rows[r].head * a.o_head;
                    bool fine = true;
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        const float x0 = o[k][2 * r] * inverse, x1 = o[k][2 * r + 1] * inverse;
                        const float y0 = o[k][4 + 2 * r] * inverse, y1 = o[k][5 + 2 * r] * inverse;
                        fine = fine && fabsf(x0) + fabsf(x1) + fabsf(y0) + fabsf(y1) < INFINITY;
                        if constexpr (kEight) {
                            *reinterpret_cast<uint2*>(op + k * 32 + t4 * 8) =
                                make_uint2(Half16<T>::pack2(x0, y0), Half16<T>::pack2(x1, y1));
                        } else {
                            *reinterpret_cast<uint32_t*>(op + k * 32 + t4 * 4) = Half16<T>::pack2(x0, x1);
                            *reinterpret_cast<uint32_t*>(op + k * 32 + t4 * 4 + 16) = Half16<T>::pack2(y0, y1);
                        }
                    }
                    if (a.lse && t4 == 0)
                        a.lse[at * a.query_heads + rows[r].head] =
                            rows[r].seen > 0 ? (top[r] + log2f(all[r])) * kLn2 : -INFINITY;
                    if (!fine && rows[r].seen < p.q.length && rows[r].seen > 0) atomicOr(redo, 1 << row);
                } else {
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        if constexpr (kEight) {
                            *reinterpret_cast<float4*>(part + row * D + k * 16 + t4 * 4) =
                                make_float4(o[k][2 * r], o[k][4 + 2 * r], o[k][2 * r + 1], o[k][5 + 2 * r]);
                        } else {
                            *reinterpret_cast<float2*>(part + row * D + k * 16 + t4 * 2) = make_float2(o[k][2 * r], o[k][2 * r + 1]);
                            *reinterpret_cast<float2*>(part + row * D + k * 16 + t4 * 2 + 8) =
                                make_float2(o[k][4 + 2 * r], o[k][5 + 2 * r]);
                        }
                    }
                    if (t4 == 0) {
                        part[kTileRows * D + row] = top[r];
                        part[kTileRows * (D + 1) + row] = all[r];
                    }
                }
            }
        }
        if (a.causal && p.q.rows > 1 && whole) {
            asm volatile("bar.sync 1, 128;" ::: "memory");
            const int again = *reinterpret_cast<volatile int*>(redo);
            if (again) {
                for (int row = warp; row < kTileRows; row += kWorkers)
                    if (again >> row & 1) {
                        const TileRow r = tile_row(a, p.q, p.head, p.tile * kTileRows + row);
                        attend_row<T, S, D>(a, p.s, p.q.first, p.q.rows, p.q.length, r.token, r.head);
                    }
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (threadIdx.x == 0) *redo = 0;
            }
        }
        next_item(p, a.batch, a.group, heads);
    }
}

// ----------------------------------------------------------------- the join

constexpr int kJoinThreads = 512;
constexpr int kJoinRows = 4;

// Block (c, y) joins rows 4 y .. of the item that the border between the runs
// of CTAs c and c + 1 cuts, if no earlier border does.  Its 16 warps share out
// the rows and each row's partial results, in an order that the sizes fix.
template <typename T, int S, int D>
__global__ void __launch_bounds__(kJoinThreads) cache_join_kernel(const __grid_constant__ CacheAttendArgs a, int grid) {
    constexpr int kPer = D / 32;
    constexpr int kJoinWarps = kJoinThreads / 32;
    __shared__ float shared_o[kJoinWarps][D];
    __shared__ float shared_ml[kJoinWarps][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const CutItem* cuts = reinterpret_cast<const CutItem*>(a.workspace);
    const int c = blockIdx.x + 1;
    const CutItem cut = cuts[c];
    if (cut.units == 0) return;
    const long long total = all_units(a.batch, a.group, a.cache.heads, lane);
    const long long per = max(1ll, (total + grid - 1) / grid);
    if (cut.first_unit / per != c - 1) return;
    const int lastc = (int)((cut.first_unit + cut.units - 1) / per);
    const int parts = lastc - (c - 1) + 1;
    const float* partials = reinterpret_cast<const float*>(a.workspace + ((sizeof(CutItem) * grid + 255) / 256) * 256);
    const CacheSequence q = cache_sequence(a.batch, cut.sequence);
    const int rows = (int)min((long long)kJoinRows,
                              (long long)q.rows * a.group - cut.tile * kTileRows - (int)blockIdx.y * kJoinRows);
    if (rows <= 0) return;
    int share = 1;  // warps of a row
    while (share * 2 * rows <= kJoinWarps && share < parts) share *= 2;
    const int local = warp / share, sub = warp % share;
    const int row = (int)blockIdx.y * kJoinRows + local;
    const bool active = local < rows;
    float m = -INFINITY, sum = 0.f, o[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = 0.f;
    if (active) {
        const int from = (int)((long long)parts * sub / share), to = (int)((long long)parts * (sub + 1) / share);
#pragma unroll 4
        for (int i = from; i < to; ++i) {
            const float* part = partials + ((long long)(c - 1 + i) * 2 + (i == 0 ? 1 : 0)) * Partial<D>::floats;
            const float pm = part[kTileRows * D + row], ps = part[kTileRows * (D + 1) + row];
            float v[kPer];
#pragma unroll
            for (int e = 0; e < kPer; ++e) v[e] = part[row * D + lane * kPer + e];
            const float top = fmaxf(m, pm), ref = top == -INFINITY ? 0.f : top;
            const float keep = exp2_fast(m - ref), add = exp2_fast(pm - ref);
            sum = sum * keep + ps * add;
#pragma unroll
            for (int e = 0; e < kPer; ++e) o[e] = o[e] * keep + v[e] * add;
            m = top;
        }
    }
    if (share > 1) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kPer; ++e) shared_o[warp][lane * kPer + e] = o[e];
        if (lane == 0) {
            shared_ml[warp][0] = m;
            shared_ml[warp][1] = sum;
        }
        __syncthreads();
        if (sub == 0)
            for (int w = warp + 1; w < warp + share; ++w) {
                const float pm = shared_ml[w][0], top = fmaxf(m, pm), ref = top == -INFINITY ? 0.f : top;
                const float keep = exp2_fast(m - ref), add = exp2_fast(pm - ref);
                sum = sum * keep + shared_ml[w][1] * add;
#pragma unroll
                for (int e = 0; e < kPer; ++e) o[e] = o[e] * keep + shared_o[w][lane * kPer + e] * add;
                m = top;
            }
    }
    if (!active || sub != 0) return;
    const TileRow r = tile_row(a, q, cut.head, cut.tile * kTileRows + row);
    if (!r.valid) return;
    const float inverse = r.seen > 0 ? 1.f / sum : 0.f;
    const long long at = (long long)q.first + r.token;
    unsigned char* op = a.out + at * a.o_row + r.head * a.o_head + lane * (kPer * 2);
    bool fine = true;
#pragma unroll
    for (int e = 0; e < kPer; e += 2) {
        const float x = o[e] * inverse, y = o[e + 1] * inverse;
        fine = fine && fabsf(x) + fabsf(y) < INFINITY;
        *reinterpret_cast<uint32_t*>(op + e * 2) = Half16<T>::pack2(x, y);
    }
    if (a.lse && lane == 0)
        a.lse[at * a.query_heads + r.head] = r.seen > 0 ? (m + log2f(sum)) * kLn2 : -INFINITY;
    if (__any_sync(0xffffffffu, !fine) && r.seen < q.length && r.seen > 0)
        attend_row<T, S, D>(a, cut.sequence, q.first, q.rows, q.length, r.token, r.head);
}

// ------------------------------------------------------------------- launch

// CTAs of the few-row kernel: all that the SMs hold, or as many as there can
// be units (the table bounds a sequence's, the rows the tiles).
long long token_ctas(int storage, int width) {
    if (cache_eight(storage)) return width == 64 ? TokenLayout<kCacheInt8, 64>::ctas : TokenLayout<kCacheInt8, 128>::ctas;
    return width == 64 ? TokenLayout<kCacheF16, 64>::ctas : TokenLayout<kCacheF16, 128>::ctas;
}
size_t token_workspace(long long grid, int width) {
    return (sizeof(CutItem) * grid + 255) / 256 * 256 + grid * 2 * kTileRows * (width + 2) * 4;
}

template <typename T, int S, int D>
void launch_tokens(const CacheAttendArgs& a, const CacheMaps& maps, int sms, cudaStream_t stream) {
    const long long tiles = (long long)a.rows * a.group / kTileRows + a.batch.sequences;
    const long long units = (((long long)a.batch.columns << a.cache.page_shift) + kUnitKeys - 1) / kUnitKeys;
    const long long held = (long long)sms * TokenLayout<S, D>::ctas;
    const int grid = (int)std::min((double)held, (double)tiles * a.cache.heads * std::max(1ll, units));
    cache_tokens_kernel<T, S, D><<<grid, kTokenThreads, TokenLayout<S, D>::bytes, stream>>>(a, maps);
    CUDA_CHECK(cudaGetLastError());
    if (grid == 1) return;
    // The join's launch overlaps the end of the kernel it waits for.
    const int rows = (int)std::min<long long>((long long)a.rows * a.group, kTileRows);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(grid - 1, (rows + kJoinRows - 1) / kJoinRows);
    config.blockDim = dim3(kJoinThreads);
    config.stream = stream;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    CUDA_CHECK(cudaLaunchKernelEx(&config, cache_join_kernel<T, S, D>, a, grid));
}

template <typename F>
void with_types(int storage, bool bf16, int width, F&& f) {
    const auto typed = [&](auto t, auto s) {
        if (width == 64) f(t, s, std::integral_constant<int, 64>{});
        else f(t, s, std::integral_constant<int, 128>{});
    };
    if (storage == kCacheF16) typed(__half{}, std::integral_constant<int, kCacheF16>{});
    else if (storage == kCacheBf16) typed(__nv_bfloat16{}, std::integral_constant<int, kCacheBf16>{});
    else if (storage == kCacheE4m3 && bf16) typed(__nv_bfloat16{}, std::integral_constant<int, kCacheE4m3>{});
    else if (storage == kCacheE4m3) typed(__half{}, std::integral_constant<int, kCacheE4m3>{});
    else if (bf16) typed(__nv_bfloat16{}, std::integral_constant<int, kCacheInt8>{});
    else typed(__half{}, std::integral_constant<int, kCacheInt8>{});
}

}  // namespace

size_t cache_attend_workspace(const CacheAttendShape& shape, int) {
    return token_workspace(shape.sms * token_ctas(shape.storage, shape.width), shape.width);
}

void prepare_cache_attend(int storage, int width) {
    for (bool bf16 : {false, true})
        with_types(storage, bf16, width, [&](auto t, auto s, auto d) {
            using T = decltype(t);
            CUDA_CHECK(cudaFuncSetAttribute(cache_tokens_kernel<T, s.value, d.value>,
                                            cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            TokenLayout<s.value, d.value>::bytes));
        });
}

void launch_cache_attend(const CacheAttendArgs& a, const CacheMaps& maps, const CacheAttendShape& shape,
                         cudaStream_t stream) {
    with_types(shape.storage, shape.bf16, shape.width, [&](auto t, auto s, auto d) {
        launch_tokens<decltype(t), s.value, d.value>(a, maps, shape.sms, stream);
    });
}

}  // namespace wsp
