// The attention of new rows over a paged cache (sm_100a): the kernel of few
// rows -- single tokens, chunks of a few -- and the join of its splits.
//
// o_i = sum_j p_ij v_j / sum_j p_ij, p_ij = 2^(s_ij - m_i), s_ij = scale log2(e)
// q_i . k_j, with the maximum m_i and both sums running over the keys.
//
// Few rows read every held key and value once and do little with them, so the
// kernel is bound by HBM: all that matters is that every SM keeps enough bytes
// in flight until the last key, and that what is done with them stays small.
// The work is the list of units (sequence, key head, tile of 8 or 16 rows, 64
// or 128 keys), in that order, and every CTA takes an equal run of it,
// wherever items (sequence, head, tile) begin and end: ragged lengths cannot
// unbalance it.  An item cut by a run's border leaves partial results (m, sum,
// o) in the workspace, which cache_join_kernel adds in an order that the sizes
// fix, so the result has the same bits every time.  Short items go whole to a
// CTA, and nothing is joined.
//
// In a CTA a producer warp copies units' keys and values into a ring of
// shared-memory stages (bulk tensor copies, a box a page), and four warps take
// a quarter of each unit: scores by mma.sync m16n8k16 with 16 keys as A and 8
// rows as B, so a single token costs an eighth of the products, not a
// sixteenth, and 16 scores of a lane's two rows are its whole softmax; then o^T
// by 16 value columns as A and P as B, P as two 16-bit halves, hi + lo: no
// rounding that shows down to 2^-32 of the largest (fp16 starts at 2^7 for that).
// The running maximum moves only when a score is more
// than 2^8 above it, which a vote finds: P may reach 2^8, and the shuffles and
// the rescaling of o are rare.  The warps' results meet once per item.
//
// 8-bit keys and values become fp16 exactly (both types fit) and are
// multiplied unscaled.  A key's scale multiplies its score, a value's scale its
// P, and the reference of a row's exponentials follows the largest of these
// products, over the keys that the row sees: one that it does not see, or that
// weighs nothing, leaves it alone whatever its scale.  P is one fp16 here,
// rounded by 2^-11 at most down to 2^-21 of the row's largest and by 2^-32 of
// that below (a hi + lo cost 3 us of 56 on 64 windows over int8 cross rows).
// bf16 queries become fp16 after a power of two a row brings them near 1.
//
// Measured (6.54 TB/s is a copy's rate): one token of 12 sequences of up to
// 32768 bf16 rows, 128 wide, 148 us for 967 MB, 6.5 TB/s; of 64 windows x 20
// heads over 1500 int8 rows 52 us for 250 MB, 4.8 TB/s, where no unit is full
// (DRAM 61 %, issue slots 58 %) and a warp waits as long for its own last
// instruction as for the copies; of 64 windows over up to 448 bf16 rows 18 us for
// 66 MB, of which the launch, the search of the list and an item's 2500 cycles
// are the most; of one window 5.8 us, all latency.  Rows that are computed again
// alone take a warp each and cost far more: if every row of 64 tokens x 20 heads
// over 1500 fp16 rows sees an infinity, 1360 us for 84; one token of 8 heads over
// 32768 int8 rows 3.8 ms for 15 us.
#include "cache_join.cuh"

#include <algorithm>

namespace wsp {
namespace {

constexpr int kWorkers = 4;  // consumer warps
constexpr int kTokenThreads = 32 * (kWorkers + 1);
constexpr float kLazy = 8.f;  // how far a score may pass the running maximum, in log2

enum CacheWait : int { kWaitFull = 1, kWaitFree = 2 };

// Shared memory: the stages, the item join's rows, the warps' softmax rows,
// barriers and the abort flag.  A stage is 16 KB (32 KB for 128-wide 16-bit
// heads), and an SM holds as many as fit with two or three CTAs: latency is
// hidden by CTAs at different points more than by deeper rings.
template <int S, int D, int NT>
struct TokenLayout {
    static constexpr int row_bytes = D * cache_bytes(S);
    static constexpr int keys = row_bytes == 64 ? 128 : 64;         // of a unit
    static constexpr int span = row_bytes < 128 ? row_bytes : 128;  // bytes of a box's row
    static constexpr int halves = row_bytes / span;
    static constexpr int pool_bytes = keys * row_bytes;             // a unit's keys, or values
    static constexpr int scale_bytes = cache_eight(S) ? 2 * keys : 0;
    static constexpr int rows = 8 * NT;                             // of a tile
    static constexpr int join_row = D + 4;                          // floats: rows fall in other banks
    static constexpr int join_bytes = kWorkers * rows * join_row * 4;
    static constexpr int ctas = D == 64 && NT == 1 ? 3 : 2;
    static constexpr int other = join_bytes + kWorkers * rows * 2 * 4 + 256;
    static constexpr int stages = (233472 / ctas - 1024 - other) / (2 * pool_bytes + scale_bytes);
    static constexpr int scale_at = stages * 2 * pool_bytes;
    static constexpr int join_at = scale_at + stages * scale_bytes;
    static constexpr int ml_at = join_at + join_bytes;
    static constexpr int bar_at = ml_at + kWorkers * rows * 2 * 4;
    static constexpr int bytes = bar_at + 2 * stages * 8 + kBarrierWords * 4;
    static_assert(stages >= 2 && stages <= 14, "a ring");
};

template <int kKeys>
__device__ __forceinline__ int item_units(int length) {
    return max(1, (length + kKeys - 1) / kKeys);
}
// What an item costs beside its units (its queries, the warps' meeting, its
// results: 2500 cycles), in units (700 to 900): the list that the CTAs share
// out counts it in front of the item's first unit (64 ragged windows: 26.3 us
// without, 20.5 with).
template <int kKeys>
constexpr int item_cost() {
    return kKeys == 64 ? 3 : 2;
}

// The items of a sequence of one head: tiles of its n * group rows, none where
// those are more than this kernel is to take.
template <int kRows>
__device__ __forceinline__ int item_tiles(const CacheSequence& q, const CacheAttendArgs& a) {
    const long long rows = (long long)q.rows * a.group;
    return rows > 0 && rows <= a.few ? (int)((rows + kRows - 1) / kRows) : 0;
}
template <int kKeys, int kRows>
__device__ __forceinline__ long long sequence_units(const CacheSequence& q, const CacheAttendArgs& a) {
    return (long long)item_tiles<kRows>(q, a) * a.cache.heads * (item_units<kKeys>(q.length) + item_cost<kKeys>());
}

// Where a unit lies; every warp finds it for itself.
struct Place {
    int s;            // sequence
    CacheSequence q;
    int head, tile;
    int unit;         // of the item
    int units, tiles; // of the item; items of a head
};

// A lane's sequences of the first 64 and their units, kept for find_unit.
struct FirstSequences {
    CacheSequence q[2];
    long long units[2];
};

template <int kKeys, int kRows>
__device__ __forceinline__ long long all_units(const CacheAttendArgs& a, int lane, FirstSequences& kept) {
    kept = FirstSequences{};
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (32 * i + lane < a.batch.sequences) kept.q[i] = attend_sequence(a, 32 * i + lane);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (32 * i + lane < a.batch.sequences) kept.units[i] = sequence_units<kKeys, kRows>(kept.q[i], a);
    long long sum = kept.units[0] + kept.units[1];
    for (int s = lane + 64; s < a.batch.sequences; s += 32) sum += sequence_units<kKeys, kRows>(attend_sequence(a, s), a);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// The place of unit u (below all_units) of the list, and where in its item it
// lies, the item's cost counted (below 0: in it).
template <int kKeys, int kRows>
__device__ __forceinline__ Place find_unit(const CacheAttendArgs& a, long long u, int lane, const FirstSequences& kept) {
    Place p{};
    for (int base = 0; base < a.batch.sequences; base += 32) {
        CacheSequence q = base == 0 ? kept.q[0] : kept.q[1];
        long long mine = base == 0 ? kept.units[0] : kept.units[1];
        if (base > 32) {
            mine = 0;
            if (base + lane < a.batch.sequences) {
                q = attend_sequence(a, base + lane);
                mine = sequence_units<kKeys, kRows>(q, a);
            }
        }
        const long long upto = warp_scan(mine, lane);
        const unsigned holds = __ballot_sync(0xffffffffu, u < upto);
        if (holds) {
            const int at = __ffs(holds) - 1;
            const long long inside = __shfl_sync(0xffffffffu, u - (upto - mine), at);
            p.s = base + at;
            p.q.first = __shfl_sync(0xffffffffu, q.first, at);
            p.q.rows = __shfl_sync(0xffffffffu, q.rows, at);
            p.q.before = __shfl_sync(0xffffffffu, q.before, at);
            p.q.length = __shfl_sync(0xffffffffu, q.length, at);
            p.units = item_units<kKeys>(p.q.length);
            p.tiles = item_tiles<kRows>(p.q, a);
            const int each = p.units + item_cost<kKeys>();
            // 32-bit division where it will do
            const long long item = inside < 0x7fffffff ? (long long)((unsigned)inside / (unsigned)each) : inside / each;
            p.unit = (int)(inside - item * each) - item_cost<kKeys>();
            p.head = p.tiles == 1 ? (int)item : (int)(item / p.tiles);
            p.tile = (int)(item - (long long)p.head * p.tiles);
            return p;
        }
        u -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return p;
}

// The next item's first unit.
template <int kKeys, int kRows>
__device__ __forceinline__ void next_item(Place& p, const CacheAttendArgs& a) {
    p.unit = -item_cost<kKeys>();
    if (++p.tile < p.tiles) return;
    p.tile = 0;
    if (++p.head < a.cache.heads) return;
    p.head = 0;
    while (++p.s < a.batch.sequences) {
        p.q = attend_sequence(a, p.s);
        p.tiles = item_tiles<kRows>(p.q, a);
        if (p.tiles > 0) break;
    }
    p.units = item_units<kKeys>(p.q.length);
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

// The byte offset of 16-byte piece c of row r in a swizzled box of `span`
// byte rows: the copy engine's 128- or 64-byte pattern.
template <int kSpan>
__device__ __forceinline__ uint32_t swizzled(int r, int c) {
    if constexpr (kSpan == 128) return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
    else return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

// --------------------------------------------------------------- the kernel

// A 8 x 8 matrix of 16-bit pairs, transposed across the warp.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// A tile's queries as B fragments: row g of each 8, element pairs 2t, 2t + 1
// and 2t + 8, 2t + 9 of each 16 (16-bit keys), or 4t .. 4t + 3, the order in
// which a lane's four bytes of an 8-bit key come.
template <typename T, int S, int D, int NT>
__device__ __forceinline__ void load_queries(const CacheAttendArgs& a, const Place& p, uint32_t (&qf)[NT][D / 16][2],
                                             int lane) {
    const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const TileRow r = tile_row(a, p.q, p.head, p.tile * 8 * NT + 8 * j + g);
        const unsigned char* qp = a.queries + ((long long)p.q.first + r.token) * a.q_row + r.head * a.q_head;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            qf[j][k][0] = qf[j][k][1] = 0;
            if (r.valid) {
                if constexpr (cache_eight(S)) {
                    const uint2 v = *reinterpret_cast<const uint2*>(qp + k * 32 + t4 * 8);
                    qf[j][k][0] = v.x;
                    qf[j][k][1] = v.y;
                } else {
                    qf[j][k][0] = *reinterpret_cast<const uint32_t*>(qp + k * 32 + t4 * 4);
                    qf[j][k][1] = *reinterpret_cast<const uint32_t*>(qp + k * 32 + t4 * 4 + 16);
                }
            }
        }
    }
}

__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Over 8-bit values the reference of a row's exponentials is such that the
// largest product of P and a value's scale stands between 2^7 and 2^15, unless P
// itself would pass 2^kFar and 2^8 of it (rows of zeros have scales of next to
// nothing), which sums of 2^31 keys bear.
constexpr float kFar = 80.f;
// A row is computed again alone where that leaves its sum below kLeastSum, so
// that smaller P underflow, or where the row's sum times the least scale among
// its keys is below kLeastScaled, scales 2^13 apart at least, and a column shows
// it: where the values of large scales are zeros the small ones' are the
// result, and P's 2^-25 a key may be more than 2^-11 of that.
constexpr float kLeastSum = 0x1p-95f, kLeastScaled = 0x1p-6f;
template <int S> constexpr float kLeastColumn = (S == kCacheE4m3 ? 448.f : 128.f) * 0x1p-14f;

// bf16 queries of an 8-bit cache as fp16, which holds a bf16 exactly between
// 2^-14 and 2^15: a power of two brings the row's largest to 2^8.., and its
// inverse is returned.
template <int D>
__device__ __forceinline__ float narrow_queries(uint32_t (&qf)[D / 16][2]) {
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float2 f = Half16<__nv_bfloat16>::pair_to_float2(qf[k][h]);
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // Biased; 255: not finite; 9 is the least whose power of two is fp32's, and
    // brings a row below 2^-118 as near.
    const int e = max((int)(__float_as_uint(top) >> 23), 9);
    const bool fine = e < 255;
    const float down = fine ? __uint_as_float((uint32_t)(262 - e) << 23) : 1.f;  // 2^(135 - e)
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float2 f = Half16<__nv_bfloat16>::pair_to_float2(qf[k][h]);
            qf[k][h] = Half16<__half>::pack2(f.x * down, f.y * down);
        }
    return fine ? __uint_as_float((uint32_t)(e - 8) << 23) : 1.f;  // 2^(e - 135)
}

// The consumer warps' barrier; whether any of their threads says so.
__device__ __forceinline__ bool workers_any(bool v) {
    int any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.or.pred q, 1, 128, p;\n\tselp.s32 %0, 1, 0, q;\n\t}\n"
        : "=r"(any)
        : "r"((int)v)
        : "memory");
    return any != 0;
}

// A grid that was launched behind another, whose results it does not read,
// ends behind it all the same: who waits for this one waits for both.
__device__ __forceinline__ void ends_behind() { wait_for_kernel_before(); }

// The producer warp: every unit of the run into the ring.
template <int S, int D, int NT>
__device__ __forceinline__ void token_producer(const CacheAttendArgs& a, const CacheMaps& maps, unsigned char* smem,
                                               uint64_t* full, uint64_t* empty, volatile int* abort, Place p,
                                               int left, int lane) {
    using Layout = TokenLayout<S, D, NT>;
    const int box_shift = cache_box_shift(a.cache.page_shift);
    const int box_rows = 1 << box_shift;
    const int boxes = Layout::keys >> box_shift;  // of a unit: 1 to 8
    const int pages = max(1, Layout::keys >> a.cache.page_shift);
    int table_s = -1, table_base = 0, entry = -1;
    int stage = 0, n = 0;
    uint32_t parity = 1;  // of the stage's previous release
    for (; left > 0; next_item<Layout::keys, Layout::rows>(p, a)) {
        const int last = a.uncut ? p.units : min(p.units, p.unit + left);
        left -= last - p.unit;
        for (int t = max(p.unit, 0); t < last; ++t) {
            if (n >= Layout::stages && !cache_wait(empty + stage, parity, abort, a.status, kWaitFree)) break;
            if (*abort) break;
            // 32 table entries at a time, a lane an entry
            const int column = (int)(((long long)t * Layout::keys) >> a.cache.page_shift);
            if (p.s != table_s || column < table_base || column + pages > table_base + 32) {
                table_s = p.s;
                table_base = column;
                entry = cache_page(a.cache, a.batch, p.s,
                                   (int)min((long long)(column + lane) << a.cache.page_shift, 0x7fffffffll));
            }
            const int b = min(lane, boxes - 1);
            const int position = t * Layout::keys + (b << box_shift);
            const int page = __shfl_sync(0xffffffffu, entry, (position >> a.cache.page_shift) - table_base);
            const bool mine = lane < boxes && position < p.q.length;
            unsigned char* keys = smem + stage * 2 * Layout::pool_bytes;
            unsigned char* values = keys + Layout::pool_bytes;
            uint8_t* scales = smem + Layout::scale_at + stage * Layout::scale_bytes;
            const int row = position & ((1 << a.cache.page_shift) - 1);
            uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xffffffffu, mine)) * 2u * (uint32_t)(box_rows * Layout::row_bytes);
            if constexpr (cache_eight(S)) {
                bytes += (uint32_t)__popc(__ballot_sync(0xffffffffu, mine && page >= 0)) * 2u * (uint32_t)box_rows;
                if (mine && page < 0) {
                    for (int i = 0; i < box_rows; i += 4) {
                        *reinterpret_cast<uint32_t*>(scales + b * box_rows + i) = 0;
                        *reinterpret_cast<uint32_t*>(scales + Layout::keys + b * box_rows + i) = 0;
                    }
                    cache_proxy_fence();
                }
                __syncwarp();
            }
            if (lane == 0) cache_arrive_expect(full + stage, bytes);
            __syncwarp();
            if (mine) {
                const int at = page >= 0 ? page : a.cache.pages;  // outside: zeros
#pragma unroll
                for (int h = 0; h < Layout::halves; ++h) {
                    const int to = h * Layout::keys * Layout::span + b * box_rows * Layout::span;
                    cache_copy_box(keys + to, &maps.keys, h * 64, row, p.head, at, full + stage);
                    cache_copy_box(values + to, &maps.values, h * 64, row, p.head, at, full + stage);
                }
                if (cache_eight(S) && page >= 0) {
                    const long long si = cache_scale_index(a.cache, page, p.head, row);
                    cache_copy_bytes(scales + b * box_rows, a.cache.key_scales + si, box_rows, full + stage);
                    cache_copy_bytes(scales + Layout::keys + b * box_rows, a.cache.value_scales + si, box_rows, full + stage);
                }
            }
            ++n;
            if (++stage == Layout::stages) {
                stage = 0;
                parity ^= 1;
            }
        }
        if (*abort) break;
    }
    if (*abort)  // the copies in flight land before the CTA's memory is given up
        for (int i = max(0, n - Layout::stages); i < n; ++i) {
            const unsigned long long start = cache_clock_ns();
            while (!cache_phase_done(full + i % Layout::stages, (uint32_t)((i / Layout::stages) & 1)) &&
                   cache_clock_ns() - start < kCacheTimeoutNs) {
            }
        }
}

// With 128 registers a thread for three CTAs an SM, and 168 for two, only tiles of
// 16 rows spill: 260 bytes a thread at 128 wide over 16 bits, 340 to 450 over 8,
// 44 to 92 at 64 wide over 8.
template <typename T, int S, int D, int NT>
__global__ void __launch_bounds__(kTokenThreads, TokenLayout<S, D, NT>::ctas)
    cache_tokens_kernel(const __grid_constant__ CacheAttendArgs a, const __grid_constant__ CacheMaps maps) {
    using Layout = TokenLayout<S, D, NT>;
    using MT = typename std::conditional<cache_eight(S), __half, T>::type;  // the products' type
    constexpr bool kEight = cache_eight(S);
    constexpr bool kNarrow = kEight && std::is_same<T, __nv_bfloat16>::value;
    // fp16 P start at 2^7, so that the small ones keep their bits; over 8 bits the
    // values' scales are counted with it.
    constexpr float kRaise = !kEight && std::is_same<T, __half>::value ? 7.f : 0.f;
    constexpr int kSteps = D / 16;                       // k16 steps of a score, 16-wide groups of values
    constexpr int kWarpKeys = Layout::keys / kWorkers;   // of a unit
    constexpr int MK = kWarpKeys / 16;
    constexpr int kRows = Layout::rows;
    extern __shared__ __align__(1024) unsigned char smem[];  // the swizzle counts from 1024-byte borders
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Layout::bar_at);
    uint64_t* empty = full + Layout::stages;
    volatile int* abort = reinterpret_cast<volatile int*>(empty + Layout::stages);
    int* redo = reinterpret_cast<int*>(empty + Layout::stages) + kOwnWord;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int i = 0; i < Layout::stages; ++i) {
            cache_barrier_init(full + i, 1);
            cache_barrier_init(empty + i, kWorkers);
        }
        *abort = abort[kBeatWord] = 0;
        abort[kMarkWord] = a.mark;
        *redo = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (!a.behind) wait_for_kernel_before();
    FirstSequences kept;
    const long long total = all_units<Layout::keys, kRows>(a, lane, kept);
    const long long per = max(1ll, (total + gridDim.x - 1) / gridDim.x);
    const long long begin = min(total, blockIdx.x * per), end = min(total, begin + per);
    Place p = begin < end ? find_unit<Layout::keys, kRows>(a, begin, lane, kept) : Place{};
    int left = (int)(end - begin);
    if (a.uncut) {
        // Items that begin in the run, whole.
        if (left > 0 && p.unit > -item_cost<Layout::keys>()) {
            left -= p.units - p.unit;
            if (left > 0) next_item<Layout::keys, kRows>(p, a);
        }
    } else if (threadIdx.x == 0) {
        CutItem cut{};
        const long long first = begin - p.unit;  // the item's first unit
        if (begin < end && p.unit > 0 && first >= begin - per)
            cut = {(int)((first + p.units - 1) / per - blockIdx.x) + 2, p.s, p.head, p.tile, p.q};
        cut_items(a.workspace)[blockIdx.x] = cut;
    }
    __syncthreads();
    if (left <= 0) {
        ends_behind();
        return;
    }
    if (warp == kWorkers) {
        token_producer<S, D, NT>(a, maps, smem, full, empty, abort, p, left, lane);
        ends_behind();
        return;
    }

    // ----------------------------------------------------------- consumers
    float* partials = cut_partials(a.workspace, gridDim.x);
    const int g = lane >> 2, t4 = lane & 3;
    float* join = reinterpret_cast<float*>(smem + Layout::join_at);
    float* ml = reinterpret_cast<float*>(smem + Layout::ml_at);
    int stage = 0;
    uint32_t parity = 0;
    uint32_t qf[NT][kSteps][2];
    load_queries<T, S, D, NT>(a, p, qf, lane);
    while (left > 0) {
        const int last = a.uncut ? p.units : min(p.units, p.unit + left);
        left -= last - p.unit;
        p.unit = max(p.unit, 0);
        if (last <= 0) break;  // the run ends in an item's cost
        const int valid = (int)min((long long)kRows, (long long)p.q.rows * a.group - (long long)p.tile * kRows);
        // A lane's rows are columns 2t and 2t + 1 of each 8.
        int seen[NT][2];
        float to_log2[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            float unscale = 1.f;
            if constexpr (kNarrow) unscale = narrow_queries<D>(qf[j]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                seen[j][e] = tile_row(a, p.q, p.head, p.tile * kRows + 8 * j + 2 * t4 + e).seen;
                to_log2[j][e] = a.scale * kLog2e;
                if constexpr (kNarrow) to_log2[j][e] *= __shfl_sync(0xffffffffu, unscale, (2 * t4 + e) * 4);
            }
        }
        // Keys below `clear` are seen by every row of the tile.
        const int clear = a.causal ? tile_row(a, p.q, p.head, p.tile * kRows).seen : p.q.length;
        const int reach = tile_row(a, p.q, p.head, p.tile * kRows + valid - 1).seen;  // and below this by its last
        uint32_t qn[NT][kSteps][2];  // the next item's
        Place pn = p;
        if (!a.uncut && left <= item_cost<Layout::keys>()) left = 0;  // nothing behind this item but a cost
        if (left > 0) {
            next_item<Layout::keys, kRows>(pn, a);
            load_queries<T, S, D, NT>(a, pn, qn, lane);
        }
        float o[kSteps][NT][4];
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[k][j][e] = 0.f;
        // The reference of the exponentials (0 until a key is seen), how far
        // above it a score may be, and the sum of this lane's keys.  Over 8
        // bits, the least byte above 1 (rows of zeros), less 2, that a row of the tile met.
        float from[NT][2], limit[NT][2], sum[NT][2];
        uint32_t least = 0xffffffffu;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) from[j][e] = sum[j][e] = 0.f, limit[j][e] = -INFINITY;

        for (int t = p.unit; t < last; ++t) {
            cache_wait(full + stage, parity, abort, a.status, kWaitFull);
            unsigned char* keys = smem + stage * 2 * Layout::pool_bytes;
            unsigned char* values = keys + Layout::pool_bytes;
            const uint8_t* scales = smem + Layout::scale_at + stage * Layout::scale_bytes;
            const int key0 = t * Layout::keys + warp * kWarpKeys;
            if (key0 < p.q.length) {
                if (key0 + kWarpKeys > p.q.length) {
                    // What lies behind the last row may be anything, and 0
                    // times a NaN is one.
                    constexpr int kPieces = Layout::row_bytes / 16;
                    for (int i = lane; i < kWarpKeys * kPieces; i += 32) {
                        const int r = i / kPieces, c = i % kPieces;
                        if (key0 + r >= p.q.length)
                            *reinterpret_cast<uint4*>(values + (c / (Layout::span / 16)) * Layout::keys * Layout::span +
                                                      swizzled<Layout::span>(warp * kWarpKeys + r, c % (Layout::span / 16))) =
                                make_uint4(0, 0, 0, 0);
                    }
                    cache_proxy_fence();
                    __syncwarp();
                }
                float s[MK][NT][4], size[kEight ? MK : 1][2];  // 8-bit keys' scales
#pragma unroll
                for (int i = 0; i < MK; ++i) {
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[i][j][e] = 0.f;
                    const uint32_t base = smem_address(keys);
                    // 16 keys' rows; lanes 0-15 give the first piece, 16-31 the next
                    const int r = warp * kWarpKeys + i * 16 + (lane & 15), c = lane >> 4;
                    if constexpr (!kEight) {
#pragma unroll
                        for (int k = 0; k < kSteps; ++k) {
                            uint32_t f[4];
                            ldmatrix4(f, base + (k / 4) * Layout::keys * 128 + swizzled<128>(r, (k % 4) * 2 + c));
#pragma unroll
                            for (int j = 0; j < NT; ++j) mma_16816<MT>(s[i][j], f, qf[j][k]);
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < kSteps; k += 2) {
                            uint32_t b[4];
                            ldmatrix4(b, base + swizzled<Layout::span>(r, k + c));
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                uint32_t f[4];
                                widen4<S>(b[2 * h], false, f[0], f[2]);
                                widen4<S>(b[2 * h + 1], false, f[1], f[3]);
#pragma unroll
                                for (int j = 0; j < NT; ++j) mma_16816<MT>(s[i][j], f, qf[j][k + h]);
                            }
                        }
                        size[i][0] = cache_scale(scales[warp * kWarpKeys + i * 16 + g]);
                        size[i][1] = cache_scale(scales[warp * kWarpKeys + i * 16 + g + 8]);
                    }
                }
                // x = log2 of the probability, relative; s stays.
                float x[MK][NT][4], factor[MK][2];
                const bool masked = key0 + kWarpKeys > clear;
                // What a score counts beside: log2 of its value's scale less 7,
                // so that the largest P, scaled, is brought to 2^7; and P alone
                // to 2^kFar at most.
                float beside[kEight ? MK : 1][2];
                if constexpr (kEight)
#pragma unroll
                    for (int i = 0; i < MK; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t byte = scales[Layout::keys + warp * kWarpKeys + i * 16 + g + 8 * h];
                            factor[i][h] = __uint_as_float(byte << 23);  // infinity for 255
                            beside[i][h] = fmaxf(log2_fast(factor[i][h]) - 7.f, -kFar);
                            if (!masked || key0 + i * 16 + g + 8 * h < reach) least = min(least, byte - 2u);
                        }
                const auto counted = [&](float v, int i, int h) {
                    if constexpr (kEight) return v + beside[i][h];
                    else return v;
                };
                // The scales first: large keys may meet small queries.
                const auto score_factor = [&](int i, int j, int e) {
                    if constexpr (kEight) return size[i][e >> 1] * to_log2[j][e & 1];
                    else return to_log2[j][e & 1];
                };
                const auto relative = [&] {
#pragma unroll
                    for (int i = 0; i < MK; ++i)
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                x[i][j][e] = fmaf(s[i][j][e], score_factor(i, j, e), -from[j][e & 1]);
                    if (masked)
#pragma unroll
                        for (int i = 0; i < MK; ++i)
#pragma unroll
                            for (int j = 0; j < NT; ++j)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (key0 + i * 16 + g + (e >> 1) * 8 >= seen[j][e & 1]) x[i][j][e] = -INFINITY;
                };
                relative();
                bool above = false;
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(counted(x[0][j][e], 0, 0), counted(x[0][j][e + 2], 0, 1));
#pragma unroll
                        for (int i = 1; i < MK; ++i) top = fmaxf(top, fmaxf(counted(x[i][j][e], i, 0), counted(x[i][j][e + 2], i, 1)));
                        above |= top > limit[j][e];
                    }
                if (__any_sync(0xffffffffu, above)) {
                    if constexpr (kEight)  // a scale that stands for NaN makes its P one
#pragma unroll
                        for (int i = 0; i < MK; ++i)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                if (factor[i][h] == INFINITY) factor[i][h] = NAN, beside[i][h] = -kFar;
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float top = fmaxf(counted(x[0][j][e], 0, 0), counted(x[0][j][e + 2], 0, 1));
#pragma unroll
                            for (int i = 1; i < MK; ++i) top = fmaxf(top, fmaxf(counted(x[i][j][e], i, 0), counted(x[i][j][e + 2], i, 1)));
#pragma unroll
                            for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                            float keep = 1.f;
                            top -= kRaise;
                            if (top > (limit[j][e] == -INFINITY ? -INFINITY : 0.f)) {
                                const float higher = from[j][e] + top;
                                keep = limit[j][e] == -INFINITY ? 0.f : exp2_fast(-top);
                                from[j][e] = higher;
                                limit[j][e] = kLazy + kRaise;
                            }
                            sum[j][e] *= keep;
#pragma unroll
                            for (int k = 0; k < kSteps; ++k) o[k][j][e] *= keep, o[k][j][e + 2] *= keep;
                        }
                    relative();
                }
#pragma unroll
                for (int i = 0; i < MK; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[i][j][e] = exp2_fast(x[i][j][e]);
                        sum[j][0] += x[i][j][0] + x[i][j][2];
                        sum[j][1] += x[i][j][1] + x[i][j][3];
                    }
                if constexpr (kEight) {
#pragma unroll
                    for (int i = 0; i < MK; ++i) {
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            x[i][j][0] *= factor[i][0], x[i][j][1] *= factor[i][0];
                            x[i][j][2] *= factor[i][1], x[i][j][3] *= factor[i][1];
                            if (masked)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (key0 + i * 16 + g + (e >> 1) * 8 >= seen[j][e & 1]) x[i][j][e] = 0.f;
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < MK; ++i) {
                    uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if constexpr (kEight) {
                                hi[j][h] = transposed(Half16<MT>::pack2(x[i][j][2 * h], x[i][j][2 * h + 1]));
                            } else {
                                split_pair<MT>(x[i][j][2 * h], x[i][j][2 * h + 1], hi[j][h], lo[j][h]);
                                hi[j][h] = transposed(hi[j][h]);
                                lo[j][h] = transposed(lo[j][h]);
                            }
                        }
                    const uint32_t base = smem_address(values);
                    if constexpr (!kEight) {
                        // columns 0-7 and 8-15 of the first 8 keys, then of the next
                        const int r = warp * kWarpKeys + i * 16 + (lane >> 4) * 8 + (lane & 7), c = (lane >> 3) & 1;
#pragma unroll
                        for (int k = 0; k < kSteps; ++k) {
                            uint32_t f[4];
                            ldmatrix4_t(f, base + (k / 4) * Layout::keys * 128 + swizzled<128>(r, (k % 4) * 2 + c));
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                mma_16816<MT>(o[k][j], f, hi[j]);
                                mma_16816<MT>(o[k][j], f, lo[j]);
                            }
                        }
                    } else {
                        const int r = warp * kWarpKeys + i * 16 + (lane & 15), c = lane >> 4;
#pragma unroll
                        for (int k = 0; k < kSteps; k += 2) {
                            uint32_t b[4];
                            ldmatrix4_t(b, base + swizzled<Layout::span>(r, k + c));
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                // even columns are the tile's first 8 rows, odd ones the next
                                uint32_t f[4];
                                widen4<S>(b[2 * h], true, f[0], f[1]);
                                widen4<S>(b[2 * h + 1], true, f[2], f[3]);
#pragma unroll
                                for (int j = 0; j < NT; ++j) {
                                    mma_16816<MT>(o[k + h][j], f, hi[j]);
                                }
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) cache_arrive(empty + stage);
            if (++stage == Layout::stages) {
                stage = 0;
                parity ^= 1;
            }
        }

        // ------------------------------------------- the warps' results meet
        if constexpr (kEight) least = __reduce_min_sync(0xffffffffu, least);
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float all = sum[j][e];
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) all += __shfl_xor_sync(0xffffffffu, all, w);
                const int row = 8 * j + 2 * t4 + e;
                float unit = 1.f;
                if constexpr (kEight) {
                    // References carry scales: a power of two a row brings the
                    // sum to 1, so that those of the warps can meet.
                    const int power = min(max((int)(__float_as_uint(all) >> 23), 1), 253);
                    bool far = least < 253u && all * __uint_as_float((least + 2u) << 23) < kLeastScaled;
                    if (__any_sync(0xffffffffu, far)) {
                        float low = INFINITY;
#pragma unroll
                        for (int k = 0; k < kSteps; ++k) low = fminf(low, fminf(fabsf(o[k][j][e]), fabsf(o[k][j][e + 2])));
#pragma unroll
                        for (int w = 4; w < 32; w <<= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, w));
                        far = far && low < (float)((last - p.unit) * kWarpKeys) * kLeastColumn<S>;
                    }
                    far = far || all < kLeastSum;
                    if (limit[j][e] > -INFINITY) {
                        unit = __uint_as_float((uint32_t)(254 - power) << 23);
                        from[j][e] += (float)(power - 127);
                        all = far ? NAN : all * unit;
                    }
                }
                if (g == 0) {
                    ml[(warp * kRows + row) * 2] = limit[j][e] == -INFINITY ? -INFINITY : from[j][e];
                    ml[(warp * kRows + row) * 2 + 1] = all;
                }
                if (row >= valid) continue;
                float* to = join + (warp * kRows + row) * Layout::join_row;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                    if constexpr (kEight) {
                        *reinterpret_cast<float2*>(to + k * 16 + 2 * g) = make_float2(o[k][j][e] * unit, o[k][j][e + 2] * unit);
                    } else {
                        to[k * 16 + g] = o[k][j][e];
                        to[k * 16 + g + 8] = o[k][j][e + 2];
                    }
                }
            }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const bool whole = p.unit == 0 && last == p.units;
        constexpr int kRowThreads = D / 2;  // a thread two columns of a row
        bool broken = false;                // a result of this thread's is not finite
        float* part = partials + ((long long)blockIdx.x * 2 + (p.unit > 0 ? 0 : 1)) * partial_floats<D>(kRows);
        for (int row = threadIdx.x / kRowThreads; row < valid; row += 128 / kRowThreads) {
            const int d = (threadIdx.x % kRowThreads) * 2;
            float top = -INFINITY, all = *abort ? NAN : 0.f;
            float2 v = make_float2(0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWorkers; ++w) top = fmaxf(top, ml[(w * kRows + row) * 2]);
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < kWorkers; ++w) {
                const float f = exp2_fast(ml[(w * kRows + row) * 2] - base);
                const float2 x = *reinterpret_cast<const float2*>(join + (w * kRows + row) * Layout::join_row + d);
                all += ml[(w * kRows + row) * 2 + 1] * f;
                v.x += x.x * f;
                v.y += x.y * f;
            }
            if (!whole) {
                *reinterpret_cast<float2*>(part + row * D + d) = v;
                if (d == 0) {
                    part[kRows * D + row] = top;
                    part[kRows * (D + 1) + row] = all;
                }
                continue;
            }
            const TileRow r = tile_row(a, p.q, p.head, p.tile * kRows + row);
            if (!r.valid) continue;
            // A row without a key is zeros whatever the tile's other rows met.
            const float inverse = 1.f / all;
            const long long at = (long long)p.q.first + r.token;
            v.x = r.seen > 0 ? v.x * inverse : 0.f;
            v.y = r.seen > 0 ? v.y * inverse : 0.f;
            *reinterpret_cast<uint32_t*>(a.out + at * a.o_row + r.head * a.o_head + d * 2) = Half16<T>::pack2(v.x, v.y);
            if (a.lse && d == 0) a.lse[at * a.query_heads + r.head] = r.seen > 0 ? (top + log2f(all)) * kLn2 : -INFINITY;
            if (!(fabsf(v.x) + fabsf(v.y) < INFINITY) && r.seen > 0) {
                atomicOr(redo, 1 << row);
                broken = true;
            }
        }
        if (workers_any(broken)) {
            const int again = *reinterpret_cast<volatile int*>(redo);
            for (int row = warp; row < kRows; row += kWorkers)
                if (again >> row & 1) {
                    const TileRow r = tile_row(a, p.q, p.head, p.tile * kRows + row);
                    attend_row<T, S, D>(a, p.s, p.q.first, p.q.before, p.q.length, r.token, r.head, abort + kBeatWord);
                }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (threadIdx.x == 0) *redo = 0;
        }
        p = pn;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int k = 0; k < kSteps; ++k) qf[j][k][0] = qn[j][k][0], qf[j][k][1] = qn[j][k][1];
    }
    ends_behind();
}

// ------------------------------------------------------------------- launch

// CTAs of the few-row kernel: all that the SMs hold, or as many as there can
// be units (the table bounds a sequence's, the rows the tiles).
template <typename Layout>
long long token_grid(const CacheAttendArgs& a, int sms) {
    const long long tiles = (long long)a.rows * a.group / Layout::rows + a.batch.sequences;
    const long long units = (((long long)a.batch.columns << a.cache.page_shift) + Layout::keys - 1) / Layout::keys;
    return (long long)std::min((double)sms * Layout::ctas, (double)tiles * a.cache.heads * std::max(1ll, units));
}

// Where no item can hold more keys than this, whole items go to the CTAs
// instead of equal runs: no partial results and no second kernel, at the price
// of runs that end up to an item late.  Single tokens over fp16 64-wide heads,
// equal runs and whole items: 1 window x 16 heads of 512 keys 6.9 and 5.6 us,
// 64 windows 17.3 and 15.2; of 1024 keys 7.6 and 7.2, 64 windows 35.9 and 33.2,
// but 8-bit ones of 1024 keys 7.9 and 9.3 us, and 128-wide ones of 1536 keys in
// 8 windows 11.4 and 17.2.
constexpr long long kUncutKeys = 512;
bool token_uncut(const CacheAttendShape& shape, int group) {
    return (long long)shape.max_rows * group <= 8 && shape.held <= kUncutKeys;
}

template <typename T, int S, int D, int NT>
CutPart launch_tokens(const CacheAttendArgs& a, const CacheMaps& maps, int sms, cudaStream_t stream) {
    using Layout = TokenLayout<S, D, NT>;
    const int grid = (int)token_grid<Layout>(a, sms);
    CUDA_CHECK(launch_early(cache_tokens_kernel<T, S, D, NT>, dim3(grid), kTokenThreads, Layout::bytes, stream, a, maps));
    return {a.workspace, a.uncut ? 0 : grid, Layout::rows};
}

}  // namespace

// Rows of a key head up to which a call is the few-row kernel's alone, in tiles
// of 16: the chunk kernel's 128-row tiles cost the same for fewer, and its
// 8-bit blocks the widening besides.  16 x 1500 keys x 8 heads, few-row and
// chunk kernel: 32 fp16 rows 22 and 28 us (64 wide), 39 and 46 (128 wide, where
// 4 x 8192 keys take 57 and 51, and 4 x 32768 171 and 113); 48 fp16 rows 28.5 and
// 28.8 (4 x 8192 31.6 and 31.3); 64 int8 rows 35 and 48 (64 x 450 keys 51 and
// 61); 128 wide 48 int8 rows 48 and 66 (64 x 450 82 and 86), 64 of them 61 and
// 68 but 99 and 87.
static long long few_rows(const CacheAttendShape& shape) {
    if (cache_eight(shape.storage)) return shape.width == 64 ? 64 : 48;
    return shape.width == 64 ? 32 : 16;
}
// And up to which a sequence is the few-row kernel's, in tiles of 8, beside
// sequences of more.  One of 48 sequences of up to 1200 keys x 8 heads has 200
// rows, 11 have these, the others one, taken by the few-row and by the chunk
// kernel: 20 int8 rows 35.6 and 41.1 us (64 wide), 55 and 57 (128 wide), 32 of
// them 42.2 and 41.4, 57 and 57; 20 fp16 rows 34.7 and 31.1, 58 and 53.
static long long few_rows_beside(const CacheAttendShape& shape) { return cache_eight(shape.storage) ? 24 : 16; }
// Calls whose units, 16 rows each, come to this many for each of two CTAs an SM
// at most are the few-row kernel's too, whatever their rows: it starts sooner.
// Few-row and chunk kernel by units a CTA, 64 wide: 3.8 (one window's 224 rows
// over 450 keys x 20 heads) int8 11.7 and 23.3 us, 7.6 fp16 11.4 and 18.1, int8
// (two windows) 18.2 and 27.0, 15 fp16 21.3 and 22.8 but int8 35.0 and 29.8.
// 128 wide: 7 (128 rows over 4 x 450 keys x 8 heads) fp16 22.7 and 22.3, int8 22.3
// and 27.5, 9 (224 rows over 1500 keys x 8 heads) 23.7 and 24.0, 23.1 and 29.5, 12
// 31.5 and 26.5, 31.2 and 32.4, 15 35.6 and 28.2, 35.0 and 33.9.
constexpr int kSmallUnits = 10;
static bool few_alone(const CacheAttendArgs& a, const CacheAttendShape& shape) {
    if ((long long)shape.max_rows * a.group <= few_rows(shape)) return true;
    const int keys = shape.width * cache_bytes(shape.storage) == 64 ? 128 : 64;
    const double tiles = (double)((long long)a.rows * a.group / 16 + a.batch.sequences);
    return tiles * a.cache.heads * (double)((shape.held + keys - 1) / keys) <= (double)kSmallUnits * 2 * shape.sms;
}

static size_t token_workspace(const CacheAttendShape& shape) {
    // 3 CTAs of 8-row tiles, or 2 of 16-row tiles
    return std::max(cut_workspace(shape.sms * 3, shape.width, 8), cut_workspace(shape.sms * 2, shape.width, 16));
}

size_t cache_attend_workspace(const CacheAttendShape& shape, int group) {
    if (token_uncut(shape, group)) return 0;
    const bool chunks = (long long)shape.max_rows * group > few_rows(shape);
    return token_workspace(shape) + (chunks ? cache_chunk_workspace(shape) : 0);
}

void prepare_cache_attend(int storage, int width) {
    for (bool bf16 : {false, true})
        with_cache_types(storage, bf16, width, [&](auto t, auto s, auto d) {
            using T = decltype(t);
            constexpr int S = s.value, D = d.value;
            CUDA_CHECK(cudaFuncSetAttribute(cache_tokens_kernel<T, S, D, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            TokenLayout<S, D, 1>::bytes));
            CUDA_CHECK(cudaFuncSetAttribute(cache_tokens_kernel<T, S, D, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            TokenLayout<S, D, 2>::bytes));
        });
    prepare_cache_chunk(storage, width);
}

void launch_cache_attend(const CacheAttendArgs& args, const CacheMaps& maps, const CacheAttendShape& shape,
                         cudaStream_t stream) {
    CacheAttendArgs a = args;
    const long long most = (long long)shape.max_rows * a.group;
    a.few = 0x7fffffffffffll;
    CutPart chunks{};
    const bool alone = few_alone(a, shape);
    if (!alone) {
        // Sequences of many rows first; the others' kernel fills the SMs as
        // these leave them, and ends behind them.
        a.few = few_rows_beside(shape);
        CacheAttendArgs b = a;
        b.workspace += token_workspace(shape);
        chunks = launch_cache_chunk(b, maps, shape, stream);
        a.behind = 1;
    }
    a.uncut = token_uncut(shape, a.group);
    // Tiles of 16 rows where some sequence may have more than 8; beside chunks,
    // those that are left are mostly single tokens.
    with_cache_types(shape.storage, shape.bf16, shape.width, [&](auto t, auto s, auto d) {
        using T = decltype(t);
        constexpr int S = s.value, D = d.value;
        const CutPart tokens = alone && most > 8
                                   ? launch_tokens<T, S, D, 2>(a, maps, shape.sms, stream)
                                   : launch_tokens<T, S, D, 1>(a, maps, shape.sms, stream);
        launch_join<T, S, D>(a, tokens, chunks, stream);
    });
}

}  // namespace wsp
