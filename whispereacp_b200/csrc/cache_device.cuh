// Device pieces the cache's attention kernels share: bounded waits, bulk
// tensor copies, 8-bit widening, and the row that is computed alone.
#pragma once

#include "cache_attend.cuh"
#include "umma.cuh"

#include <type_traits>

namespace wsp {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// ------------------------------------------------------------------- waits

constexpr unsigned long long kCacheTimeoutNs = 2000000000ull;

__device__ __forceinline__ unsigned long long cache_clock_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

__device__ __forceinline__ bool cache_phase_done(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred P;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, P;\n\t}\n"
        : "=r"(done)
        : "r"(smem_address(bar)), "r"(parity)
        : "memory");
    return done != 0;
}

// The words behind a CTA's barriers: first whether a wait has given up (`abort`),
// then a word of the kernel's own, one that changes while a warp does a row
// alone, and the cache's mark.
constexpr int kOwnWord = 1, kBeatWord = 2, kMarkWord = 3, kBarrierWords = 4;

// Waits for the phase of `parity`.  After 2 s, or once another wait of the CTA
// has given up, it records `kind` and returns false, and so does every later
// wait at once: the roles then run through their loops without waiting, so
// all meet at the barriers between them, and the sums become NaN, so that the
// rows are computed again alone, which takes no waits.  A warp of
// the CTA that does rows alone may take longer over a long context; the 2 s
// count from its last sign (its loops end by themselves).
static __device__ __noinline__ bool cache_wait_slow(uint64_t* bar, uint32_t parity, volatile int* abort, int* status,
                                                    int kind) {
    unsigned long long start = cache_clock_ns();
    int beat = abort[kBeatWord];
    for (unsigned spin = 1;; ++spin) {
        if (cache_phase_done(bar, parity)) return true;
        if ((spin & 15) != 0) continue;
        if (*abort) return false;
        if (cache_clock_ns() - start > kCacheTimeoutNs) {
            const int now = abort[kBeatWord];
            if (now != beat) {
                beat = now;
                start = cache_clock_ns();
                continue;
            }
            atomicExch(status, abort[kMarkWord] | kind);
            *abort = 1;
            return false;
        }
    }
}
__device__ __forceinline__ bool cache_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* status, int kind) {
    if (cache_phase_done(bar, parity)) return true;
    return cache_wait_slow(bar, parity, abort, status, kind);
}

__device__ __forceinline__ void cache_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_address(bar)) : "memory");
}
__device__ __forceinline__ void cache_arrive_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_address(bar)), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void cache_barrier_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(smem_address(bar)), "r"(count) : "memory");
}

// ------------------------------------------------------------------- copies

// One box of a pool: columns x.., rows y.. of a head's page.  x is 0 or 64
// 16-bit columns, so the copy starts on 16 bytes; a page outside the pool
// reads as zeros.
__device__ __forceinline__ void cache_copy_box(void* to, const CUtensorMap* map, int x, int y, int head, int page,
                                               uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(smem_address(to)),
        "l"(map), "r"(x), "r"(y), "r"(head), "r"(page), "r"(smem_address(bar))
        : "memory");
}
__device__ __forceinline__ void cache_copy_bytes(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_address(to)),
                 "l"(from), "r"(bytes), "r"(smem_address(bar))
                 : "memory");
}
// Orders this thread's shared-memory accesses before later bulk copies and
// tensor-core reads of the same memory.
__device__ __forceinline__ void cache_proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ----------------------------------------------------------------- numbers

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Four held 8-bit values, unscaled, as two pairs of fp16, exact: 0 1 and 2 3, or
// (interleaved) 0 2 and 1 3.
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

// ------------------------------------------------- a row that is done alone

// One row of one query head by one warp: o = sum_j p_j v_j / sum_j p_j with p_j =
// exp(s_j - max), the maximum and both sums running, all in fp32.  Only keys the
// row sees are read.  The tiled kernels multiply whole tiles by P of 16 bits, or
// of two: an infinity or NaN among the values of a key behind the row (0 times
// it) makes the row NaN there, and so may a seen infinity (P's lower half is 0 or
// negative).  Rows whose results are not finite come here, with those whose
// scales the 16 bits do not reach, and have here what the definition says.
//
// 32 keys at a time: a lane scores a key, its 16-byte pieces one after another
// against queries handed round; then the lanes share out the columns and go over
// the keys, 8 values on their way.  Latency bounds it; how long a call takes in
// which many rows come here is told beside the kernels.  `beat` (null: nobody
// waits) changes every 32 keys.
template <typename T, int S, int D>
__device__ __noinline__ void attend_row(const CacheAttendArgs& a, int s, int first, int before, int length, int i,
                                        int head, volatile int* beat) {
    constexpr int kPer = D / 32;  // a lane's columns
    constexpr int kPiece = 16 / cache_bytes(S);  // values of 16 bytes
    constexpr int kAtOnce = 8;
    using Pair = typename std::conditional<cache_eight(S), uint16_t, uint32_t>::type;
    const int lane = threadIdx.x & 31;
    const int keys = a.causal ? min(before + i + 1, length) : length;
    const long long row = (long long)first + i;
    const int kv = head / a.group;
    float qv[kPer], o[kPer];
    const unsigned char* qp = a.queries + row * a.q_row + head * a.q_head + lane * (kPer * 2);
#pragma unroll
    for (int e = 0; e < kPer; e += 2) {
        const float2 f = Half16<T>::pair_to_float2(*reinterpret_cast<const uint32_t*>(qp + e * 2));
        qv[e] = f.x;
        qv[e + 1] = f.y;
        o[e] = o[e + 1] = 0.f;
    }
    float top = -INFINITY, total = 0.f;
    for (int j0 = 0; j0 < keys; j0 += 32) {
        if (beat && lane == 0) *beat = *beat + 1;
        const int j = j0 + lane, count = min(32, keys - j0);
        const int page = lane < count ? cache_page(a.cache, a.batch, s, j) : -1;
        long long at = -1;  // the key's row in the pools, -1: zeros
        float by = 1.f, score = 0.f;  // its value's scale
        if (page >= 0) {
            const int slot = j & ((1 << a.cache.page_shift) - 1);
            at = cache_offset(a.cache, page, kv, slot);
            if constexpr (cache_eight(S)) {
                const long long si = cache_scale_index(a.cache, page, kv, slot);
                score = cache_scale(a.cache.key_scales[si]);
                by = cache_scale(a.cache.value_scales[si]);
            } else {
                score = 1.f;
            }
        }
        float dot = 0.f;
#pragma unroll 2
        for (int c = 0; c < D / kPiece; ++c) {
            uint4 piece = make_uint4(0, 0, 0, 0);
            if (at >= 0) piece = *reinterpret_cast<const uint4*>(a.cache.keys + at + c * 16);
            const uint32_t words[4] = {piece.x, piece.y, piece.z, piece.w};
#pragma unroll
            for (int e = 0; e < kPiece; e += 2) {
                const uint32_t bits = cache_eight(S) ? (words[e / 4] >> (8 * (e & 2))) & 0xffffu : words[e / 2];
                const float2 f = cache_pair<S>(bits);
                const int from = (c * kPiece + e) / kPer;
                dot += __shfl_sync(0xffffffffu, qv[e % kPer], from) * f.x;
                dot += __shfl_sync(0xffffffffu, qv[e % kPer + 1], from) * f.y;
            }
        }
        score = lane < count ? dot * score * a.scale : -INFINITY;
        const float higher = fmaxf(top, warp_max(score));
        const float from = higher == -INFINITY ? 0.f : higher;
        const float keep = expf(top - from), p = expf(score - from);
        total = total * keep + warp_sum(p);
        if (!(total == total)) break;  // and so it stays, and every sum of it
        top = higher;
#pragma unroll
        for (int e = 0; e < kPer; ++e) o[e] *= keep;
        for (int n0 = 0; n0 < count; n0 += kAtOnce) {
            Pair v[kAtOnce][kPer / 2];
#pragma unroll
            for (int n = 0; n < kAtOnce; ++n) {
                const long long of = __shfl_sync(0xffffffffu, at, n0 + n);
#pragma unroll
                for (int e = 0; e < kPer / 2; ++e) {
                    v[n][e] = 0;
                    if (of >= 0)
                        v[n][e] = *reinterpret_cast<const Pair*>(a.cache.values + of +
                                                                 (lane * kPer + 2 * e) * cache_bytes(S));
                }
            }
#pragma unroll
            for (int n = 0; n < kAtOnce; ++n) {
                const float pn = __shfl_sync(0xffffffffu, p, n0 + n), bn = __shfl_sync(0xffffffffu, by, n0 + n);
#pragma unroll
                for (int e = 0; e < kPer / 2; ++e) {
                    const float2 f = cache_pair<S>(v[n][e]);
                    o[2 * e] += pn * (f.x * bn);
                    o[2 * e + 1] += pn * (f.y * bn);
                }
            }
        }
    }
    const float inverse = keys > 0 ? 1.f / total : 0.f;
    unsigned char* op = a.out + row * a.o_row + head * a.o_head + lane * (kPer * 2);
#pragma unroll
    for (int e = 0; e < kPer; e += 2)
        *reinterpret_cast<uint32_t*>(op + e * 2) = Half16<T>::pack2(o[e] * inverse, o[e + 1] * inverse);
    if (a.lse && lane == 0) a.lse[row * a.query_heads + head] = keys > 0 ? top + logf(total) : -INFINITY;
}

// ------------------------------------------------------------ a tile's rows

// A sequence as the attention takes it: none of its rows if any lies outside
// the call's arrays.
__device__ __forceinline__ CacheSequence attend_sequence(const CacheAttendArgs& a, int s) {
    CacheSequence q = cache_sequence(a.cache, a.batch, s);
    if (q.first < 0 || (long long)q.first + q.rows > a.rows) q.rows = 0;
    return q;
}

// Packed row R of a sequence's n * group rows of one key head is token R /
// group of query head R % group.
struct TileRow {
    int token, head, seen;  // seen: the keys it sees
    bool valid;
};
__device__ __forceinline__ TileRow tile_row(const CacheAttendArgs& a, const CacheSequence& q, int kv, int packed) {
    TileRow r;
    r.token = a.group == 1 ? packed : packed / a.group;
    r.head = kv * a.group + packed - r.token * a.group;
    r.valid = r.token < q.rows;
    r.seen = a.causal ? max(0, min(q.before + r.token + 1, q.length)) : q.length;
    return r;
}

}  // namespace wsp
