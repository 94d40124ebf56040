// The attention of new rows over a paged cache (sm_100a).
#include "cache_attend.cuh"

namespace wsp {
namespace {

// One row of one query head by one warp, key by key: o = sum_j p_j v_j / sum_j
// p_j with p_j = exp(s_j - max), the maximum and both sums running.  Only keys
// the row sees are read.
template <typename T, int S, int D>
__device__ void attend_row(const CacheAttendArgs& a, int s, const CacheSequence& q, int i, int head) {
    constexpr int kPer = D / 32;  // a lane's elements
    const int lane = threadIdx.x & 31;
    const int position = q.length - q.rows + i;
    const int keys = a.causal ? min(position + 1, q.length) : q.length;
    const long long row = (long long)q.first + i;
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
    for (int j = 0; j < keys; ++j) {
        const int page = cache_page(a.cache, a.batch, s, j);
        float k[kPer], v[kPer], ks = 1.f, vs = 1.f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) k[e] = v[e] = 0.f;
        if (page >= 0) {
            const int slot = j & ((1 << a.cache.page_shift) - 1);
            const long long at = cache_offset(a.cache, page, kv, slot) + lane * kPer * cache_bytes(S);
#pragma unroll
            for (int e = 0; e < kPer; e += 2) {
                using Pair = typename std::conditional<cache_eight(S), uint16_t, uint32_t>::type;
                const float2 fk = cache_pair<S>(*reinterpret_cast<const Pair*>(a.cache.keys + at + e * cache_bytes(S)));
                const float2 fv = cache_pair<S>(*reinterpret_cast<const Pair*>(a.cache.values + at + e * cache_bytes(S)));
                k[e] = fk.x, k[e + 1] = fk.y, v[e] = fv.x, v[e + 1] = fv.y;
            }
            if (cache_eight(S)) {
                const long long si = cache_scale_index(a.cache, page, kv, slot);
                ks = cache_scale(a.cache.key_scales[si]);
                vs = cache_scale(a.cache.value_scales[si]);
            }
        }
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < kPer; ++e) dot += qv[e] * k[e];
        const float score = warp_sum(dot) * ks * a.scale;
        const float higher = fmaxf(top, score);
        const float keep = expf(top - higher), p = expf(score - higher);
        total = total * keep + p;
#pragma unroll
        for (int e = 0; e < kPer; ++e) o[e] = o[e] * keep + p * (v[e] * vs);
        top = higher;
    }
    const float inverse = keys > 0 ? 1.f / total : 0.f;
    unsigned char* op = a.out + row * a.o_row + head * a.o_head + lane * (kPer * 2);
#pragma unroll
    for (int e = 0; e < kPer; e += 2)
        *reinterpret_cast<uint32_t*>(op + e * 2) = Half16<T>::pack2(o[e] * inverse, o[e + 1] * inverse);
    if (a.lse && lane == 0) a.lse[row * a.query_heads + head] = keys > 0 ? top + logf(total) : -INFINITY;
}

// The sequence that row r belongs to: the last s with starts[s] <= r, if r
// is below starts[s + 1]; -1 if none.
__device__ int sequence_of(const CacheBatchView& b, int r) {
    int low = 0, high = b.sequences;  // starts[low] <= r < starts[high], if it is anywhere
    if (r < b.starts[0] || r >= b.starts[high]) return -1;
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (b.starts[mid] <= r) low = mid;
        else high = mid;
    }
    return low;
}

template <typename T, int S, int D>
__global__ void __launch_bounds__(256) attend_rows_kernel(const CacheAttendArgs a) {
    const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= (long long)a.rows * a.query_heads) return;
    const int row = (int)(item / a.query_heads), head = (int)(item % a.query_heads);
    const int s = sequence_of(a.batch, row);
    if (s < 0) return;
    const CacheSequence q = cache_sequence(a.batch, s);
    attend_row<T, S, D>(a, s, q, row - q.first, head);
}

template <typename T, int S>
void launch_width(const CacheAttendArgs& a, int width, cudaStream_t stream) {
    const long long items = (long long)a.rows * a.query_heads;
    const unsigned grid = (unsigned)((items + 7) / 8);
    if (width == 64) attend_rows_kernel<T, S, 64><<<grid, 256, 0, stream>>>(a);
    else attend_rows_kernel<T, S, 128><<<grid, 256, 0, stream>>>(a);
}

}  // namespace

size_t cache_attend_workspace(int, int, int, int) { return 0; }

void launch_cache_attend(const CacheAttendArgs& a, int storage, bool bf16, int width, int, int, void*,
                         cudaStream_t stream) {
    if (storage == kCacheF16) launch_width<__half, kCacheF16>(a, width, stream);
    else if (storage == kCacheBf16) launch_width<__nv_bfloat16, kCacheBf16>(a, width, stream);
    else if (storage == kCacheE4m3 && bf16) launch_width<__nv_bfloat16, kCacheE4m3>(a, width, stream);
    else if (storage == kCacheE4m3) launch_width<__half, kCacheE4m3>(a, width, stream);
    else if (bf16) launch_width<__nv_bfloat16, kCacheInt8>(a, width, stream);
    else launch_width<__half, kCacheInt8>(a, width, stream);
}

}  // namespace wsp
