// The attention of chunks of new rows over a paged cache, on the tcgen05 tensor
// cores (sm_100a).  The mathematics is cache_attend.cu's; here a key or value
// meets hundreds of rows, so the products and the exponentials bound it.
//
// An item is (sequence, key head, 256 packed rows): two tiles of 128 rows (the
// products' M) over the blocks of 128 keys that their last row sees.  A tile's
// 128 x 128 scores cost 128 x 128 exponentials, 1024 cycles of an SM's 16 a
// cycle, next to 4 x 128 x 128 x D flop, 512 (D 64) or 1024 cycles of the tensor
// cores: neither may wait for the other.  So two tiles take turns:
//
//   warps 0-3, 4-7  the softmax of tile 0 and of tile 1, a thread a row: read
//                   the scores from tensor memory, p = 2^(s - m), P as 16-bit
//                   values back into the scores' columns, half a block at a
//                   time (rounded once to the queries' type, which the
//                   products take: 2^-8 or 2^-11 of a probability, as much as
//                   the output's own rounding, and of either sign), the
//                   sum of p in a register.  m comes from the first block that
//                   the row sees; it moves, and the row of o in tensor memory
//                   is rescaled, only when a block's sum of P says so.
//   warp 8          issues the products: S_t = Q_t K^T (both from shared
//                   memory) and O_t += P_t V (P from tensor memory), those of
//                   one tile while the other's softmax runs.
//   warp 9          copies the blocks' keys and values into a ring, a box a
//                   page, as the 128-byte-swizzled tiles the products read:
//                   keys K-major, values MN-major, as they lie in the cache.
//   warps 9-15      over 8-bit caches instead: bring the blocks in as they are
//                   held and widen them into the ring.  A warp issues them at
//                   its own latency, so their number counts: 8 sequences of
//                   8192 int8 keys, 128 wide, 256 rows, took 231 us with three
//                   warps, 198 with four, 151 with seven (at 128 registers a
//                   thread, of which 64 to 104 bytes spill, where the softmax
//                   has no scores on their way; 155 under fp16 queries since
//                   their keys share a power of two).
//
// 16-bit 64-wide heads have items of one tile, and an SM two CTAs, which then
// are the two that take turns: ragged prompts of 32 windows 42 us against 47.
//
// Tensor memory: S_0, S_1 (128 columns each, P in the first 64), O_0, O_1 (D
// columns each).  The order of products on one issuing thread is the order of
// their execution, so S_t of the next block may follow P_t V in P_t's place,
// and the commit behind S_t also says that O_t stands still.
//
// The blocks of all items form one list, dealt evenly over the SMs as in
// cache_attend.cu; cut items leave partial results for the join.  What an item
// passes once (its queries, results, a rescaling) is kept in loops, not
// unrolled: the code then stays in the instruction caches, and the widening's
// loops likewise (64 x 450 int8 keys, 256 rows, 86 -> 71 us in all).
//
// Measured: two chunks of up to 1500 bf16 rows x 32 heads over up to 15.5k keys
// of 8 heads, 128 wide, 0.66 ms for 664 GFLOP, 1.0 PFLOP/s of a matrix product's 1.63: a
// block's scores, softmax and product follow one another, and two tiles in
// turn do not hide all of that.  Ragged prompts of 32 windows (fp16, 64 wide,
// 450 keys) 34.6 us, nearly all of it what an item and a launch cost; a mixed
// batch of 48 sequences over e4m3, the few-row kernel's share behind it, 72 us.
// Rows that are computed again alone take a warp each: if all of 256 rows x 8
// heads over 16 x 1500 keys are, 9.9 ms for 48 us (fp16, infinities among the
// values) or 7.8 ms for 60 (int8 values above 65504 under fp16 queries, which
// come to fp16 results above or near its largest).
#include "cache_join.cuh"

#include <algorithm>

namespace wsp {
namespace {

constexpr int kBlockKeys = 128;
constexpr int kTile = 128;               // rows of a tile
constexpr int kHalfBytes = kTile * 128;  // 128 rows of 64 16-bit columns

enum ChunkWait : int { kWaitBlock = 11, kWaitSlot = 12, kWaitScores = 13, kWaitP = 14, kWaitQueries = 15, kWaitO = 16,
                       kWaitDone = 17, kWaitFirst = 18, kWaitPower = 19 };

// Whether a block's keys, widened to the queries' type, share a power of two that
// the scores are multiplied by: fp16 would not hold all scaled keys.  bf16 does,
// each value exactly.
template <typename T, int S>
constexpr bool keys_share() {
    return cache_eight(S) && std::is_same<T, __half>::value;
}

template <int S, int D>
struct ChunkLayout {
    // Tiles of a CTA.  16-bit 64-wide heads: one, and two CTAs an SM, each at a
    // point of its own (their smaller blocks may cross from L2 twice).
    static constexpr int tiles = D == 64 && !cache_eight(S) ? 1 : 2;
    static constexpr int ctas = 3 - tiles;
    static constexpr int rows = tiles * kTile;  // of an item
    static constexpr int mma_warp = 4 * tiles;
    static constexpr int copy_warps = cache_eight(S) ? 7 : 1;
    static constexpr int threads = 32 * (mma_warp + 1 + copy_warps);
    static constexpr int columns = tiles == 1 ? 256 : 512;  // of tensor memory
    static constexpr int out_column = tiles * 128;
    static constexpr int halves = D / 64;
    static constexpr int tile_bytes = halves * kHalfBytes;  // of Q_t, or of a block's keys or values
    static constexpr int stages = D == 64 && tiles == 2 ? 8 : cache_eight(S) ? 3 : 5;
    static constexpr int ring_at = tiles * tile_bytes;
    // 8-bit storage: blocks as they are held, and their scale bytes.
    static constexpr int depth = cache_eight(S) ? 4 : 0;
    static constexpr int held_bytes = kBlockKeys * (D + 1) + 16;  // and how many of the keys are seen
    static constexpr int held_at = ring_at + stages * tile_bytes;
    static constexpr int bar_at = held_at + depth * held_bytes;
    // And the powers of two of as many blocks' keys as can have scores under way.
    static constexpr int powers = cache_eight(S) ? stages / 2 + 1 : 0;
    // full, empty; per tile: scores, P's halves, first half, queries, O; done;
    // powers
    static constexpr int bars = 2 * stages + 6 * tiles + 1 + powers;
    static constexpr int powers_at = bar_at + bars * 8 + kBarrierWords * 4;
    static constexpr int bytes = powers_at + powers * 4;
};

// ------------------------------------------------------------ the block list

struct ChunkPlace {
    int s;
    CacheSequence q;
    int head, item;
    int block, blocks;  // the item's first in this run; its blocks
    int items;          // of a head
};

template <int kRows>
__device__ __forceinline__ int chunk_items(const CacheSequence& q, const CacheAttendArgs& a) {
    const long long rows = (long long)q.rows * a.group;
    return rows > a.few ? (int)((rows + kRows - 1) / kRows) : 0;
}

// Keys that any of the first `rows` packed rows sees; rows * group of a call
// fit 31 bits.
__device__ __forceinline__ int chunk_seen(const CacheSequence& q, const CacheAttendArgs& a, int rows) {
    if (!a.causal) return q.length;
    const int token = min((rows - 1) / a.group, q.rows - 1);
    return max(0, min(q.before + token + 1, q.length));
}
template <int kRows>
__device__ __forceinline__ int chunk_blocks(const CacheSequence& q, const CacheAttendArgs& a, int item) {
    return max(1, (chunk_seen(q, a, (item + 1) * kRows) + kBlockKeys - 1) / kBlockKeys);
}
// What an item costs beside its blocks (queries, the first block's maximum,
// results), in blocks: the list that the CTAs share out counts it in front of
// the item's first block (ragged prompts of 32 windows: 42 us without, 35 with).
constexpr int kItemCost = 2;

// A sequence's blocks.
template <int kRows>
__device__ __forceinline__ long long chunk_units(const CacheSequence& q, const CacheAttendArgs& a) {
    const int items = chunk_items<kRows>(q, a);
    if (items == 0) return 0;
    long long sum = 0;
    if (!a.causal) sum = (long long)items * (chunk_blocks<kRows>(q, a, 0) + kItemCost);
    else
        for (int p = 0; p < items; ++p) sum += chunk_blocks<kRows>(q, a, p) + kItemCost;
    return sum * a.cache.heads;
}

// A lane's sequence of the first 32 and its blocks, kept for find_block.
struct FirstSequences {
    CacheSequence q;
    long long blocks;
};

template <int kRows>
__device__ __forceinline__ long long all_blocks(const CacheAttendArgs& a, int lane, FirstSequences& kept) {
    kept = FirstSequences{};
    if (lane < a.batch.sequences) {
        kept.q = attend_sequence(a, lane);
        kept.blocks = chunk_units<kRows>(kept.q, a);
    }
    long long sum = kept.blocks;
    for (int s = lane + 32; s < a.batch.sequences; s += 32) sum += chunk_units<kRows>(attend_sequence(a, s), a);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// The place of block u (below all_blocks) of the list, and where in its item
// it lies, the item's cost counted (below 0: in it).
template <int kRows>
__device__ __forceinline__ ChunkPlace find_block(const CacheAttendArgs& a, long long u, int lane,
                                                 const FirstSequences& kept) {
    ChunkPlace p{};
    for (int base = 0; base < a.batch.sequences; base += 32) {
        CacheSequence q = kept.q;
        long long mine = kept.blocks;
        if (base > 0) {
            mine = 0;
            if (base + lane < a.batch.sequences) {
                q = attend_sequence(a, base + lane);
                mine = chunk_units<kRows>(q, a);
            }
        }
        const long long upto = warp_scan(mine, lane);
        const unsigned holds = __ballot_sync(0xffffffffu, u < upto);
        if (holds) {
            const int at = __ffs(holds) - 1;
            long long inside = __shfl_sync(0xffffffffu, u - (upto - mine), at);
            p.s = base + at;
            p.q.first = __shfl_sync(0xffffffffu, q.first, at);
            p.q.rows = __shfl_sync(0xffffffffu, q.rows, at);
            p.q.before = __shfl_sync(0xffffffffu, q.before, at);
            p.q.length = __shfl_sync(0xffffffffu, q.length, at);
            p.items = chunk_items<kRows>(p.q, a);
            const long long all = __shfl_sync(0xffffffffu, mine, at);  // of every head
            const long long head = all < 0x7fffffff ? (long long)((unsigned)all / (unsigned)a.cache.heads) : all / a.cache.heads;
            // 32-bit division where it will do
            p.head = inside < 0x7fffffff && head < 0x7fffffff ? (int)((unsigned)inside / (unsigned)head) : (int)(inside / head);
            inside -= p.head * head;
            // 32 items at a time
            for (;; p.item += 32) {
                const int blocks = p.item + lane < p.items ? chunk_blocks<kRows>(p.q, a, p.item + lane) + kItemCost : 0;
                const long long to = warp_scan(blocks, lane);
                const unsigned in = __ballot_sync(0xffffffffu, inside < to);
                if (in) {
                    const int i = __ffs(in) - 1;
                    p.block = (int)__shfl_sync(0xffffffffu, inside - (to - blocks), i) - kItemCost;
                    p.blocks = __shfl_sync(0xffffffffu, blocks, i) - kItemCost;
                    p.item += i;
                    return p;
                }
                inside -= __shfl_sync(0xffffffffu, to, 31);
            }
        }
        u -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return p;
}

template <int kRows>
__device__ __forceinline__ void next_item(ChunkPlace& p, const CacheAttendArgs& a) {
    p.block = -kItemCost;
    if (++p.item >= p.items) {
        p.item = 0;
        if (++p.head >= a.cache.heads) {
            p.head = 0;
            while (++p.s < a.batch.sequences) {
                p.q = attend_sequence(a, p.s);
                p.items = chunk_items<kRows>(p.q, a);
                if (p.items > 0) break;
            }
        }
    }
    p.blocks = chunk_blocks<kRows>(p.q, a, p.item);
}

// Takes the item at p out of the run, of which `todo` is left: returns the end
// of the run's blocks of it (0 or less: the run ends in the item's cost).
__device__ __forceinline__ int take_item(ChunkPlace& p, int& todo) {
    const int last = min(p.blocks, p.block + todo);
    todo -= last - p.block;
    if (todo <= kItemCost) todo = 0;  // nothing behind this item but a cost
    p.block = max(p.block, 0);
    return last;
}

// The blocks of tile t of an item: 0 if it has no rows, else one at least.
template <int kRows>
__device__ __forceinline__ int tile_blocks(const ChunkPlace& p, const CacheAttendArgs& a, int t) {
    const int first = p.item * kRows + t * kTile;
    if (first >= p.q.rows * a.group) return 0;
    return max(1, (chunk_seen(p.q, a, first + kTile) + kBlockKeys - 1) / kBlockKeys);
}

// ------------------------------------------------------------ tensor pieces

// Shared-memory descriptors as two words: the upper one is fixed, and 16-byte
// steps in a tile add to the lower one.  Queries and keys, K-major, are
// umma_desc's tiles.  Values as they lie are MN-major: 128-byte rows of 64
// columns, 8 of them (keys) 1024 bytes apart from the next 8, the next 64
// columns a half on.
constexpr uint32_t kDescUpper = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t key_desc(uint32_t address) { return (address >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t value_desc(uint32_t address) {
    return (address >> 4) | ((uint32_t)(kHalfBytes >> 4) << 16);
}

// D[tmem] (+)= A . B of one k16 step, one thread: A from shared memory, or from
// tensor memory.
__device__ __forceinline__ void product_ss(uint32_t tmem, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}\n" ::"r"(tmem),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescUpper)
        : "memory");
}
__device__ __forceinline__ void product_ts(uint32_t tmem, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tmov.b64 y, {%2, %5};\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}\n" ::"r"(tmem),
        "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "n"(kDescUpper)
        : "memory");
}
// One lane of the warp, the same every time; the compiler then keeps what the
// products take in uniform registers.
__device__ __forceinline__ bool elected() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// 32 columns of this warp's lanes on their way into r; tmem_arrived waits for
// every such load so far, and r may be used behind it.
__device__ __forceinline__ void tmem_load32_begin(uint32_t address, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(address)
        : "memory");
}
__device__ __forceinline__ void tmem_arrived(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

__device__ __forceinline__ void tmem_store16(uint32_t address, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            address),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t address, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(address),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// Two fp32 values of a register pair, and arithmetic on both at once.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 pair_values(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ float2 exp2_pair(uint64_t v) {
    const float2 x = pair_values(v);
    return make_float2(exp2_fast(x.x), exp2_fast(x.y));
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// ---------------------------------------------------------------- the roles

struct ChunkBars {
    uint64_t *full, *empty, *scores, *p, *first, *queries, *o, *done, *powers;
};

template <int S, int D>
__device__ void chunk_copy(const CacheAttendArgs& a, const CacheMaps& maps, unsigned char* smem, const ChunkBars& bar,
                           volatile int* abort, ChunkPlace p, long long begin, long long end, int lane) {
    using Layout = ChunkLayout<S, D>;
    const int box_shift = cache_box_shift(a.cache.page_shift);
    const int box_rows = 1 << box_shift;
    const int boxes = kBlockKeys >> box_shift;
    int stage = 0, n = 0;
    uint32_t parity = 1;
    for (int todo = (int)(end - begin); todo > 0;) {
        const int last = take_item(p, todo);
        const int seen = chunk_seen(p.q, a, (p.item + 1) * Layout::rows);
        for (int j = p.block; j < last; ++j) {
            const int position = j * kBlockKeys + (min(lane, boxes - 1) << box_shift);
            const int row = position & ((1 << a.cache.page_shift) - 1);
            const bool mine = lane < boxes && position < seen;
            int page = mine ? cache_page(a.cache, a.batch, p.s, position) : -1;
            if (page < 0) page = a.cache.pages;  // outside: zeros
            const uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xffffffffu, mine)) * (uint32_t)(box_rows * D * 2);
            for (int v = 0; v < 2; ++v) {
                if (n >= Layout::stages && !cache_wait(bar.empty + stage, parity, abort, a.status, kWaitSlot)) break;
                if (*abort) break;
                unsigned char* to = smem + Layout::ring_at + stage * Layout::tile_bytes + lane * box_rows * 128;
                if (lane == 0) cache_arrive_expect(bar.full + stage, bytes);
                __syncwarp();
                if (mine)
#pragma unroll
                    for (int h = 0; h < Layout::halves; ++h)
                        cache_copy_box(to + h * kHalfBytes, v ? &maps.values : &maps.keys, h * 64, row, p.head, page,
                                       bar.full + stage);
                ++n;
                if (++stage == Layout::stages) {
                    stage = 0;
                    parity ^= 1;
                }
            }
            if (*abort) break;
        }
        if (*abort) break;
        next_item<Layout::rows>(p, a);
    }
    if (*abort)  // the copies in flight land before the CTA's memory is given up
        for (int i = max(0, n - Layout::stages); i < n; ++i) {
            const unsigned long long start = cache_clock_ns();
            while (!cache_phase_done(bar.full + i % Layout::stages, (uint32_t)((i / Layout::stages) & 1)) &&
                   cache_clock_ns() - start < kCacheTimeoutNs) {
            }
        }
}

// 16 held 8-bit values times their scale (byte `scale`), as 16-bit values.
template <typename T, int S>
__device__ __forceinline__ void widen_piece(const uint4& raw, uint32_t scale, uint32_t (&out)[8]) {
    const uint32_t in[4] = {raw.x, raw.y, raw.z, raw.w};
    if (std::is_same<T, __half>::value && scale - 113u < 30u) {
        // 2^-14 .. 2^15 is a number of fp16's: the product rounds as the
        // float's way does
        const unsigned short bits = (unsigned short)((scale - 112u) << 10);
        const __half2 by = __half2(__ushort_as_half(bits), __ushort_as_half(bits));
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            widen4<S>(in[h], false, out[2 * h], out[2 * h + 1]);
#pragma unroll
            for (int e = 2 * h; e < 2 * h + 2; ++e) {
                const __half2 x = __hmul2(*reinterpret_cast<__half2*>(&out[e]), by);
                out[e] = *reinterpret_cast<const uint32_t*>(&x);
            }
        }
    } else {
        const float by = cache_scale(scale);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float2 f = cache_pair<S>((in[e / 2] >> (16 * (e & 1))) & 0xffffu);
            out[e] = Half16<T>::pack2(f.x * by, f.y * by);
        }
    }
}

// What the scores of fp16 queries over a block of 8-bit keys are multiplied by,
// log2(e) and the keys' power of two in it; a masked score of -infinity stays
// one at a scale of 0.
__device__ __forceinline__ float scores_factor(float scale, uint32_t power) {
    return fmaxf(fabsf(scale) * kLog2e * __uint_as_float(power << 23), 0x1p-126f);
}

// The scale byte of a key relative to its block's power of two, which stands
// kUp below the block's largest byte: fp16 holds the largest scaled value (448 x
// 2^7, 128 x 2^8) then, and whole every value of a scale down to kDown below the
// power.  Values of keys further down (2^22 or 2^32 below the largest) are off by
// up to 2^-25, kKeyStep: a row whose queries make more than kScoreStep of a score
// of that is computed again alone, which takes scores of thousands.  Blocks whose
// bytes are all 112 to 127, rows whose largest lies between 2^-6 and 2^6 among
// them, need no power (it is 127, 2^0).
constexpr float kKeyStep = 0x1p-25f, kScoreStep = 0x1p-20f;
template <int S> constexpr uint32_t kUp = S == kCacheE4m3 ? 7 : 8;
template <int S> constexpr uint32_t kDown = S == kCacheE4m3 ? 15 : 24;
template <int S>
__device__ __forceinline__ uint32_t shared_scale(uint32_t byte, uint32_t power) {
    if (byte == 255u) return byte;
    return byte + 126u < power ? 0u : byte + 127u - power;
}

// The power of a block of `keys` keys, by every warp of the kThreads that widen
// it: kUp below the largest scale byte that stands for a number (25 at least),
// and kFarKeys if a key lies further below than kDown, rows of zeros aside.
// `four` are the lane's four bytes at `bytes`, in whose place the first warp puts
// them relative to the power.  Rare, and kept out of the loop's instructions.
constexpr uint32_t kFarKeys = 256;
template <int S, int kThreads>
__device__ __noinline__ uint32_t share_power(uint32_t* bytes, uint32_t four, int keys, int warp, int lane) {
    uint32_t most = 25, relative = 0;
    for (int i = 0; i < 4; ++i) {
        const uint32_t byte = (four >> (8 * i)) & 255u;
        if (lane * 4 + i < keys && byte != 255u) most = max(most, byte);
    }
    const uint32_t power = __reduce_max_sync(0xffffffffu, most) - kUp<S>;
    bool far = false;
    for (int i = 0; i < 4; ++i) {
        const uint32_t byte = (four >> (8 * i)) & 255u;
        relative |= (shared_scale<S>(byte, power) & 255u) << (8 * i);
        far |= lane * 4 + i < keys && byte > 1u && byte + kDown<S> < power;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
    if (warp == 0) bytes[lane] = relative;
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
    return power | (__any_sync(0xffffffffu, far) ? kFarKeys : 0u);
}

// The sum of the magnitudes of a row's queries as they lie in a tile; rare too.
template <int kHalves>
__device__ __noinline__ float queries_sum(const unsigned char* tile, int row) {
    float sum = 0.f;
    for (int i = 0; i < kHalves * 64; i += 2) {
        const float2 q = Half16<__half>::pair_to_float2(
            *reinterpret_cast<const uint32_t*>(tile + (i / 64) * kHalfBytes + row * 128 + (i % 64) * 2));
        sum += fabsf(q.x) + fabsf(q.y);
    }
    return sum;
}

// 8-bit caches: the warps bring the blocks in as they are held, four tiles
// (keys or values of a block) deep, and write them into the ring widened to the
// queries' type, each value times its scale (a power of two: exact in bf16; fp16
// rounds what it does not hold whole by as much as it rounds the results, and
// makes an infinity of what is above 65504: rows that meet one are computed
// again alone).  Keys for fp16 queries are taken relative to their block's power
// of two, which goes to the softmax.  Block n's lies in place n % powers: its
// keys' tile, number 2 n of the ring, is written when tile 2 n - stages is
// released, and so the values of block n - powers, which every tile's softmax
// has then passed.
template <typename T, int S, int D>
__device__ void chunk_widen(const CacheAttendArgs& a, unsigned char* smem, const ChunkBars& bar, volatile int* abort,
                            ChunkPlace p, long long begin, long long end, int warp, int lane) {
    using Layout = ChunkLayout<S, D>;
    constexpr int kThreads = 32 * Layout::copy_warps;
    constexpr int kPieces = kBlockKeys * D / 16;  // 16 values each
    constexpr int kDepth = Layout::depth;
    const int me = warp * 32 + lane;
    int todo = (int)(end - begin);
    int last = take_item(p, todo);
    if (last <= 0) return;
    int seen = chunk_seen(p.q, a, (p.item + 1) * Layout::rows), j = p.block;
    bool values = false, more = true;  // of the tile to ask for; there is one
    int asked = 0;
    // Asks for the next tile; what is not there, or not seen, comes as zeros.
    const auto ask = [&] {
        if (more) {
            unsigned char* held = smem + Layout::held_at + (asked % kDepth) * Layout::held_bytes;
            const unsigned char* pool = values ? a.cache.values : a.cache.keys;
            const uint8_t* scales = values ? a.cache.value_scales : a.cache.key_scales;
            // A lane a page, of 16 rows at least.
            const int pages = max(1, kBlockKeys >> a.cache.page_shift);
            const int first = j * kBlockKeys + (min(lane, pages - 1) << a.cache.page_shift);
            const int entry = first < seen ? cache_page(a.cache, a.batch, p.s, first) : -1;
            const auto copy16 = [&](unsigned char* to, const void* from, bool there) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_address(to)), "l"(from),
                             "r"(there ? 16 : 0)
                             : "memory");
            };
            if (me == 0) *reinterpret_cast<int*>(held + kPieces * 16 + kBlockKeys) = seen - j * kBlockKeys;
#pragma unroll 1
            for (int i = 0; i < (kPieces + 8 + kThreads - 1) / kThreads; ++i) {
                const int piece = me + i * kThreads;
                const bool scale = piece >= kPieces;  // 16 keys' scale bytes
                const int key = min(scale ? (piece - kPieces) * 16 : piece / (D / 16), kBlockKeys - 1);
                const int position = j * kBlockKeys + key;
                const int page = __shfl_sync(0xffffffffu, entry, min(key >> a.cache.page_shift, pages - 1));
                if (piece >= kPieces + 8) continue;
                const bool there = position < seen && page >= 0;
                const int slot = position & ((1 << a.cache.page_shift) - 1);
                if (scale)
                    copy16(held + kPieces * 16 + key,
                           there ? scales + cache_scale_index(a.cache, page, p.head, slot) : scales, there);
                else
                    copy16(held + piece * 16,
                           there ? pool + cache_offset(a.cache, page, p.head, slot) + (piece % (D / 16)) * 16 : pool, there);
            }
            ++asked;
            // keys of block 0, its values, keys of block 1, ...
            values = !values;
            if (!values && ++j >= last) {
                more = todo > 0;
                if (more) {
                    next_item<Layout::rows>(p, a);
                    last = take_item(p, todo);
                    seen = chunk_seen(p.q, a, (p.item + 1) * Layout::rows);
                    j = p.block;
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int i = 0; i < kDepth - 1; ++i) ask();
    int stage = 0;
    uint32_t parity = 1;
    for (int n = 0; n < asked; ++n) {
        // This tile's copies are in, everybody's, and the last tile's place is
        // read.
        asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 2) : "memory");
        asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
        ask();
        unsigned char* held = smem + Layout::held_at + (n % kDepth) * Layout::held_bytes;
        const int keys = *reinterpret_cast<const int*>(held + kPieces * 16 + kBlockKeys);  // seen; the others are zeros
        const uint32_t four = reinterpret_cast<const uint32_t*>(held + kPieces * 16)[lane];  // of the scale bytes
        if (n >= Layout::stages) cache_wait(bar.empty + stage, parity, abort, a.status, kWaitSlot);
        unsigned char* tile = smem + Layout::ring_at + stage * Layout::tile_bytes;
        if (keys_share<T, S>() && (n & 1) == 0) {
            uint32_t power = 127;
            if (__any_sync(0xffffffffu, lane * 4 < keys && (four & 0xf0f0f0f0u) != 0x70707070u))
                power = share_power<S, kThreads>(reinterpret_cast<uint32_t*>(held + kPieces * 16), four, keys, warp, lane);
            if (me == 0) {
                const int at = (n >> 1) % Layout::powers;
                const float factor = scores_factor(a.scale, power & 255u);
                reinterpret_cast<float*>(smem + Layout::powers_at)[at] = power & kFarKeys ? -factor : factor;
                cache_arrive(bar.powers + at);
            }
        }
#pragma unroll 1
        for (int piece = me; piece < kPieces; piece += kThreads) {
            const int key = piece / (D / 16), c = piece % (D / 16);
            uint32_t out[8];
            widen_piece<T, S>(*reinterpret_cast<const uint4*>(held + piece * 16), key < keys ? held[kPieces * 16 + key] : 0u, out);
            unsigned char* to = tile + (c / 4) * kHalfBytes + key * 128;
            const int at = (c % 4) * 2;
            *reinterpret_cast<uint4*>(to + ((at ^ (key & 7)) << 4)) = make_uint4(out[0], out[1], out[2], out[3]);
            *reinterpret_cast<uint4*>(to + (((at + 1) ^ (key & 7)) << 4)) = make_uint4(out[4], out[5], out[6], out[7]);
        }
        cache_proxy_fence();
        __syncwarp();
        if (lane == 0) cache_arrive(bar.full + stage);
        if (++stage == Layout::stages) {
            stage = 0;
            parity ^= 1;
        }
    }
}

template <typename T, int S, int D>
__device__ void chunk_products(const CacheAttendArgs& a, unsigned char* smem, const ChunkBars& bar, uint32_t tmem_base,
                               volatile int* abort, ChunkPlace p, long long begin, long long end, int lane) {
    using Layout = ChunkLayout<S, D>;
    const uint32_t score_desc = umma_idesc<T>(kBlockKeys), out_desc = umma_idesc<T>(D) | (1u << 16);
    const uint32_t tmem = (uint32_t)uniform((int)tmem_base);
    const uint32_t queries = key_desc(smem_address(smem)), ring = smem_address(smem + Layout::ring_at);
    int stage = 0;
    uint32_t parity = 0, p_parity[2] = {0, 0}, q_parity[2] = {0, 0};
    const auto advance = [&] {
        if (++stage == Layout::stages) {
            stage = 0;
            parity ^= 1;
        }
    };
    const auto scores = [&](int t, uint32_t keys) {
        if (elected()) {
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const uint32_t at = (uint32_t)((k / 4) * kHalfBytes + (k % 4) * 32) >> 4;
                product_ss(tmem + t * 128, queries + ((uint32_t)(t * Layout::tile_bytes) >> 4) + at, keys + at, score_desc,
                           k != 0);
            }
            umma_commit(bar.scores + t);
        }
        __syncwarp();
    };
    for (int todo = uniform((int)(end - begin)); todo > 0;) {
        const int last = uniform(take_item(p, todo)), first = uniform(p.block);
        todo = uniform(todo);
        if (last <= 0) break;
        int blocks[Layout::tiles];
#pragma unroll
        for (int t = 0; t < Layout::tiles; ++t) blocks[t] = uniform(min(last, tile_blocks<Layout::rows>(p, a, t)));
        const int seen = uniform(chunk_seen(p.q, a, (p.item + 1) * Layout::rows));
        // The first block's scores.
        cache_wait(bar.full + stage, parity, abort, a.status, kWaitBlock);
#pragma unroll
        for (int t = 0; t < Layout::tiles; ++t)
            if (first < blocks[t]) {
                cache_wait(bar.queries + t, q_parity[t], abort, a.status, kWaitQueries);
                q_parity[t] ^= 1;
                tmem_fence_after();
                scores(t, key_desc(ring + stage * Layout::tile_bytes));
            }
        if (elected()) umma_commit(bar.empty + stage);
        __syncwarp();
        advance();
        for (int j = first; j < last; ++j) {
            const int v_stage = stage;
            cache_wait(bar.full + stage, parity, abort, a.status, kWaitBlock);
            const uint32_t values = value_desc(ring + stage * Layout::tile_bytes);
            if (!cache_eight(S) && (j + 1) * kBlockKeys > seen) {
                // What lies behind the last row that the item sees was not
                // copied or may be anything, and 0 times a NaN is one.
                unsigned char* tile = smem + Layout::ring_at + stage * Layout::tile_bytes;
                const int from = max(0, seen - j * kBlockKeys);
                for (int h = 0; h < Layout::halves; ++h)
                    for (int i = from * 8 + lane; i < kBlockKeys * 8; i += 32)
                        *reinterpret_cast<uint4*>(tile + h * kHalfBytes + i * 16) = make_uint4(0, 0, 0, 0);
                cache_proxy_fence();
                __syncwarp();
            }
            advance();
            const int k_stage = stage;
            if (j + 1 < last) {
                cache_wait(bar.full + stage, parity, abort, a.status, kWaitBlock);
                advance();
            }
#pragma unroll
            for (int t = 0; t < Layout::tiles; ++t) {
                if (j >= blocks[t]) continue;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    cache_wait(bar.p + 2 * t + half, p_parity[t], abort, a.status, kWaitP);
                    tmem_fence_after();
                    if (elected()) {
#pragma unroll
                        for (int k = half * 4; k < half * 4 + 4; ++k)
                            product_ts(tmem + Layout::out_column + t * D, tmem + t * 128 + k * 8, values + k * (2048 >> 4), out_desc,
                                       k != 0 ? 1u : (uint32_t)(j > first));
                        if (half == 0) umma_commit(bar.first + t);
                        else if (j + 1 >= blocks[t]) umma_commit(bar.o + t);
                    }
                    __syncwarp();
                }
                p_parity[t] ^= 1;
                if (j + 1 < blocks[t]) scores(t, key_desc(ring + k_stage * Layout::tile_bytes));
            }
            if (elected()) {
                umma_commit(bar.empty + v_stage);
                if (j + 1 < last) umma_commit(bar.empty + k_stage);
            }
            __syncwarp();
        }
        next_item<Layout::rows>(p, a);
    }
    // Every product has completed before the tensor memory goes.
    if (elected()) {
        umma_commit(bar.done);
        const unsigned long long start = cache_clock_ns();
        while (!cache_phase_done(bar.done, 0))
            if (cache_clock_ns() - start > kCacheTimeoutNs) {
                atomicExch(a.status, a.mark | kWaitDone);
                break;
            }
    }
    __syncwarp();
}

template <typename T, int S, int D>
__device__ void chunk_softmax(const CacheAttendArgs& a, unsigned char* smem, const ChunkBars& bar, uint32_t tmem,
                              volatile int* abort, ChunkPlace p, long long begin, long long end, int t) {
    using Layout = ChunkLayout<S, D>;
    // The reference of a row's exponentials comes from the maximum of the first
    // block it sees and stays as long as a block's sum of P says that no P left
    // the 16-bit type's range: fp16 keeps 2^-14 .. 2^15 whole, so P starts at
    // 2^8 at most, and 64 of them sum up to 2^14; bf16 has fp32's range.
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr float kShift = kHalf ? 8.f : 0.f;
    constexpr float kMost = kHalf ? 32768.f : 0x1p60f;
    // The next 32 scores on their way while 32 are worked on, where the
    // registers reach for it; 8-bit caches' 512 threads have 128 each.
    constexpr bool kAhead = !cache_eight(S);
    const int lane = threadIdx.x & 31, row = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)(row & ~31) << 16;
    const uint32_t s_at = tmem + t * 128 + lanes, o_at = tmem + Layout::out_column + t * D + lanes;
    const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;  // the sign goes into the queries
    float to_log2 = scores_factor(a.scale, 127u);
    uint32_t s_parity = 0, o_parity = 0, h_parity = 0;
    int passed = 0;  // blocks of the run before the item
    // The row's queries, swizzled as the copy engine does it.
    const auto give_queries = [&](const ChunkPlace& p, const TileRow& r) {
        const unsigned char* qp = a.queries + ((long long)p.q.first + r.token) * a.q_row + r.head * a.q_head;
#pragma unroll 1
        for (int h = 0; h < Layout::halves; ++h) {
            uint4 v[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                v[c] = make_uint4(0, 0, 0, 0);
                if (r.valid) v[c] = *reinterpret_cast<const uint4*>(qp + h * 128 + c * 16);
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                v[c].x ^= flip, v[c].y ^= flip, v[c].z ^= flip, v[c].w ^= flip;
                *reinterpret_cast<uint4*>(smem + t * Layout::tile_bytes + h * kHalfBytes + row * 128 +
                                          ((c ^ (row & 7)) << 4)) = v[c];
            }
        }
        cache_proxy_fence();
        __syncwarp();
        if (lane == 0) cache_arrive(bar.queries + t);
    };
    int todo = (int)(end - begin);
    int last = take_item(p, todo);
    if (last <= 0) return;
    int blocks = min(last, tile_blocks<Layout::rows>(p, a, t));
    TileRow r = tile_row(a, p.q, p.head, p.item * Layout::rows + t * kTile + row);
    if (p.block < blocks) give_queries(p, r);
    while (true) {
        const int packed = p.item * Layout::rows + t * kTile;
        const bool active = p.block < blocks;
        const long long at = (long long)p.q.first + r.token;
        float from = 0.f, sum = 0.f;
        bool unset = true, ready = false;  // no key seen yet; every row of the warp has seen one
        if (active) {
            // Keys below `clear` are seen by every row of the tile.
            const int clear = tile_row(a, p.q, p.head, packed).seen;
            for (int j = p.block; j < blocks; ++j) {
                cache_wait(bar.scores + t, s_parity, abort, a.status, kWaitScores);
                s_parity ^= 1;
                tmem_fence_after();
                const bool masked = (j + 1) * kBlockKeys > clear;
                if constexpr (keys_share<T, S>()) {
                    // Behind the scores' wait: a tile that passes items by would
                    // take an older phase of the place for its own.
                    const int n = passed + j - p.block, at = n % Layout::powers;
                    cache_wait(bar.powers + at, (uint32_t)(n / Layout::powers) & 1u, abort, a.status, kWaitPower);
                    to_log2 = reinterpret_cast<const volatile float*>(smem + Layout::powers_at)[at];
                    if (to_log2 < 0.f) {  // there are keys far below the largest
                        to_log2 = -to_log2;
                        const float most = queries_sum<Layout::halves>(smem + t * Layout::tile_bytes, row) * kKeyStep;
                        if (j * kBlockKeys < r.seen && !(most * to_log2 < kScoreStep)) sum = NAN;
                    }
                }
                // 32 scores at a time, the next 32 on their way.  Half a block's
                // P goes out at a time, so that the products of the first 64
                // keys' run while the second 64 are computed; its check, its
                // store and the store's wait each stand behind later work.
                uint32_t s[2][32], w[2][16];
                float part[2];
                uint64_t sums[2];
                const auto take = [&](int c) {
                    tmem_arrived(s[c & 1]);
                    const int seen = r.seen - j * kBlockKeys - c * 32;
                    if (masked && __any_sync(0xffffffffu, seen < 32))
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (e >= seen) s[c & 1][e] = 0xff800000u;
                };
                const auto exponentials = [&](int c) {
                    const uint64_t scale2 = pair_of(to_log2, to_log2), from2 = pair_of(-from, -from);
                    if ((c & 1) == 0) sums[0] = sums[1] = 0;
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const uint64_t x = fma_pair(
                            pair_of(__uint_as_float(s[c & 1][e]), __uint_as_float(s[c & 1][e + 1])), scale2, from2);
                        const float2 p = exp2_pair(x);
                        sums[(e >> 1) & 1] = add_pair(sums[(e >> 1) & 1], pair_of(p.x, p.y));
                        w[c & 1][e / 2] = Half16<T>::pack2(p.x, p.y);
                    }
                    if (c & 1) {
                        const float2 v = pair_values(add_pair(sums[0], sums[1]));
                        part[c >> 1] = v.x + v.y;
                    }
                };
                // The half's rows get a reference from their maximum, and what
                // stands in o follows it.
                const auto refer = [&](int half) {
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 2 * half; c < 2 * half + 2; ++c) {
                        if (kAhead) tmem_arrived(s[c & 1]);  // whatever is on its way
                        tmem_load32_begin(s_at + c * 32, s[c & 1]);
                        take(c);
#pragma unroll
                        for (int e = 0; e < 32; ++e) top[e & 3] = fmaxf(top[e & 3], __uint_as_float(s[c & 1][e]));
                    }
                    const float higher = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * to_log2 - kShift;
                    float keep = 1.f;
                    if (higher > (unset ? -INFINITY : from)) {
                        keep = unset ? 0.f : exp2_fast(from - higher);
                        from = higher;
                        unset = false;
                        sum *= keep;
                    }
                    ready = !__any_sync(0xffffffffu, unset);
                    if ((j > p.block || half) && __any_sync(0xffffffffu, keep != 1.f)) {
                        // The products behind these scores are done; those of
                        // the first half's P have a barrier.
                        if (half) {
                            cache_wait(bar.first + t, h_parity, abort, a.status, kWaitFirst);
                            tmem_fence_after();
                        }
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[32];
                            tmem_load32(o_at + c * 32, o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tmem_store32(o_at + c * 32, o);
                        }
                    }
                    exponentials(2 * half);
                    exponentials(2 * half + 1);
                };
                const auto store = [&](int half) {
                    sum += part[half];
                    tmem_store16(s_at + half * 32, w[0]);
                    tmem_store16(s_at + half * 32 + 16, w[1]);
                };
                const auto hand_over = [&](int half) {
                    tmem_store_wait();
                    tmem_fence_before();
                    __syncwarp();
                    if (lane == 0) cache_arrive(bar.p + 2 * t + half);
                };
                tmem_load32_begin(s_at, s[0]);
                take(0);
                if (kAhead) tmem_load32_begin(s_at + 32, s[1]);
                if (ready) {
                    exponentials(0);
                    if (!kAhead) tmem_load32_begin(s_at + 32, s[1]);
                    take(1);
                    if (kAhead) tmem_load32_begin(s_at + 64, s[0]);
                    exponentials(1);
                } else {
                    part[0] = INFINITY;
                }
                if (__any_sync(0xffffffffu, !(part[0] <= kMost))) {
                    refer(0);
                    if (kAhead) tmem_load32_begin(s_at + 64, s[0]);
                }
                store(0);
                if (!kAhead) tmem_load32_begin(s_at + 64, s[0]);
                take(2);
                if (kAhead) tmem_load32_begin(s_at + 96, s[1]);
                exponentials(2);
                hand_over(0);
                if (!kAhead) tmem_load32_begin(s_at + 96, s[1]);
                take(3);
                exponentials(3);
                if (!ready || __any_sync(0xffffffffu, !(part[1] <= kMost))) refer(1);
                store(1);
                hand_over(1);
                h_parity ^= 1;
            }
        }
        // The next item's queries go out before this one's results, and its
        // first scores are made meanwhile.
        ChunkPlace pn = p;
        int last_n = 0, blocks_n = 0;
        TileRow rn = r;
        if (todo > 0) {
            next_item<Layout::rows>(pn, a);
            last_n = take_item(pn, todo);
            blocks_n = min(last_n, tile_blocks<Layout::rows>(pn, a, t));
            rn = tile_row(a, pn.q, pn.head, pn.item * Layout::rows + t * kTile + row);
            if (pn.block < blocks_n) give_queries(pn, rn);
        }
        if (active) {
            cache_wait(bar.o + t, o_parity, abort, a.status, kWaitO);
            o_parity ^= 1;
            tmem_fence_after();
        }
        const bool whole = p.block == 0 && last == p.blocks;
        if (*abort) sum = NAN;
        const bool some = r.seen > 0;  // a row without a key is zeros whatever the tile's other rows met
        const float inverse = 1.f / sum;
        const float log_sum = unset ? -INFINITY : from;
        float* part = cut_partials(a.workspace, gridDim.x) + ((long long)blockIdx.x * 2 + (p.block > 0 ? 0 : 1)) * partial_floats<D>(Layout::rows);
        bool fine = true;
        unsigned char* op = a.out + at * a.o_row + r.head * a.o_head;
        if (active || !whole) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                if (active) tmem_load32(o_at + c * 32, o);
                else
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0;
                if (!r.valid) continue;
                if (whole) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float x = some ? __uint_as_float(o[e + 2 * i]) * inverse : 0.f;
                            const float y = some ? __uint_as_float(o[e + 2 * i + 1]) * inverse : 0.f;
                            fine = fine && fabsf(x) + fabsf(y) < INFINITY;
                            w[i] = Half16<T>::pack2(x, y);
                        }
                        *reinterpret_cast<uint4*>(op + c * 64 + e * 2) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<uint4*>(part + (t * kTile + row) * D + c * 32 + e) =
                            make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
        }
        if (r.valid && whole && a.lse) a.lse[at * a.query_heads + r.head] = some ? (log_sum + log2f(sum)) * kLn2 : -INFINITY;
        if (r.valid && !whole) {
            part[Layout::rows * D + t * kTile + row] = log_sum;
            part[Layout::rows * (D + 1) + t * kTile + row] = sum;
        }
        // Rows that are no numbers (attend_row).
        unsigned again = __ballot_sync(0xffffffffu, whole && r.valid && !fine && some);
        while (again) {
            const int i = __ffs(again) - 1;
            again &= again - 1;
            const int token = __shfl_sync(0xffffffffu, r.token, i), head = __shfl_sync(0xffffffffu, r.head, i);
            __syncwarp();
            attend_row<T, S, D>(a, p.s, p.q.first, p.q.before, p.q.length, token, head, abort + kBeatWord);
        }
        tmem_fence_before();  // this tile's reads, before the products that the next arrival lets run
        if (last_n == 0) break;
        passed += last - p.block;
        p = pn;
        last = last_n;
        blocks = blocks_n;
        r = rn;
    }
}

template <typename T, int S, int D>
__global__ void __launch_bounds__(ChunkLayout<S, D>::threads, ChunkLayout<S, D>::ctas)
    cache_chunk_kernel(const __grid_constant__ CacheAttendArgs a, const __grid_constant__ CacheMaps maps) {
    using Layout = ChunkLayout<S, D>;
    extern __shared__ __align__(1024) unsigned char smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Layout::bar_at);
    uint64_t* tile_bars = bars + 2 * Layout::stages;
    constexpr int kTiles = Layout::tiles;
    const ChunkBars bar = {bars, bars + Layout::stages, tile_bars, tile_bars + kTiles, tile_bars + 3 * kTiles,
                           tile_bars + 4 * kTiles, tile_bars + 5 * kTiles, tile_bars + 6 * kTiles, tile_bars + 6 * kTiles + 1};
    volatile int* abort = reinterpret_cast<volatile int*>(bars + Layout::bars);
    uint32_t* slot = reinterpret_cast<uint32_t*>(bars + Layout::bars) + kOwnWord;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < Layout::stages; ++i) {
            cache_barrier_init(bar.full + i, Layout::copy_warps);
            cache_barrier_init(bar.empty + i, 1);
        }
        for (int t = 0; t < Layout::tiles; ++t) {
            cache_barrier_init(bar.scores + t, 1);
            cache_barrier_init(bar.p + 2 * t, kTile / 32);
            cache_barrier_init(bar.p + 2 * t + 1, kTile / 32);
            cache_barrier_init(bar.first + t, 1);
            cache_barrier_init(bar.queries + t, kTile / 32);
            cache_barrier_init(bar.o + t, 1);
        }
        cache_barrier_init(bar.done, 1);
        for (int i = 0; i < Layout::powers; ++i) cache_barrier_init(bar.powers + i, 1);
        *abort = abort[kBeatWord] = 0;
        abort[kMarkWord] = a.mark;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == Layout::mma_warp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(slot)),
                     "r"((uint32_t)Layout::columns));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    wait_for_kernel_before();
    // The few-row kernel behind this one may fill what SMs are left.
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    FirstSequences kept;
    const long long total = all_blocks<Layout::rows>(a, lane, kept);
    const long long per = max(1ll, (total + gridDim.x - 1) / gridDim.x);
    const long long begin = min(total, blockIdx.x * per), end = min(total, begin + per);
    const ChunkPlace p = begin < end ? find_block<Layout::rows>(a, begin, lane, kept) : ChunkPlace{};
    if (threadIdx.x == 0) {
        CutItem cut{};
        const long long first = begin - p.block;  // the item's first block
        if (begin < end && p.block > 0 && first >= begin - per)
            cut = {(int)((first + p.blocks - 1) / per - blockIdx.x) + 2, p.s, p.head, p.item, p.q};
        cut_items(a.workspace)[blockIdx.x] = cut;
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *slot;
    if (begin < end) {
        if (warp > Layout::mma_warp) {
            if constexpr (cache_eight(S))
                chunk_widen<T, S, D>(a, smem, bar, abort, p, begin, end, warp - Layout::mma_warp - 1, lane);
            else chunk_copy<S, D>(a, maps, smem, bar, abort, p, begin, end, lane);
        } else if (warp == Layout::mma_warp) chunk_products<T, S, D>(a, smem, bar, tmem, abort, p, begin, end, lane);
        else chunk_softmax<T, S, D>(a, smem, bar, tmem, abort, p, begin, end, warp >> 2);
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    if (warp == Layout::mma_warp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)Layout::columns));
}

// ------------------------------------------------------------------- launch

// As many CTAs as there can be blocks, those that the SMs hold at most.
template <int S, int D>
int chunk_grid(const CacheAttendArgs& a, int sms) {
    using Layout = ChunkLayout<S, D>;
    const long long items = (long long)a.rows * a.group / Layout::rows + a.batch.sequences;
    const long long blocks = (((long long)a.batch.columns << a.cache.page_shift) + kBlockKeys - 1) / kBlockKeys;
    return (int)std::min((double)sms * Layout::ctas, (double)items * a.cache.heads * std::max(1ll, blocks));
}

}  // namespace

size_t cache_chunk_workspace(const CacheAttendShape& shape) {
    // one CTA of two tiles an SM, or two of one
    return cut_workspace(shape.sms * 2, shape.width, kTile) + 256;
}

void prepare_cache_chunk(int storage, int width) {
    for (bool bf16 : {false, true})
        with_cache_types(storage, bf16, width, [&](auto t, auto s, auto d) {
            CUDA_CHECK(cudaFuncSetAttribute(cache_chunk_kernel<decltype(t), s.value, d.value>,
                                            cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            ChunkLayout<s.value, d.value>::bytes));
        });
}

CutPart launch_cache_chunk(const CacheAttendArgs& a, const CacheMaps& maps, const CacheAttendShape& shape,
                           cudaStream_t stream) {
    CutPart part{};
    with_cache_types(shape.storage, shape.bf16, shape.width, [&](auto t, auto s, auto d) {
        constexpr int S = s.value, D = d.value;
        using Layout = ChunkLayout<S, D>;
        const int grid = chunk_grid<S, D>(a, shape.sms);
        CUDA_CHECK(launch_early(cache_chunk_kernel<decltype(t), S, D>, dim3(grid), Layout::threads, Layout::bytes, stream,
                                a, maps));
        part = {a.workspace, grid, Layout::rows};
    });
    return part;
}

}  // namespace wsp
