// Items of the cache's attention that the CTAs' runs cut: what a CTA leaves of
// them in the workspace, and the kernel that joins it.
#pragma once

#include "cache_device.cuh"
#include "host.h"

#include <algorithm>

namespace wsp {
namespace {

// Workspace: a record for each CTA whose run begins inside an item, then two
// partial results for each CTA: [0] of the item its run begins in, [1] of the
// item its run ends in.
struct CutItem {
    int parts;  // partial results of the item, if this CTA's is the second; else 0
    int sequence, head, tile;
    CacheSequence q;
};
// A partial result: o, then m, then sum.
template <int D>
__host__ __device__ constexpr int partial_floats(int rows) {
    return rows * (D + 2);
}
inline size_t cut_workspace(long long grid, int width, int rows) {
    return (sizeof(CutItem) * grid + 255) / 256 * 256 + (grid * 2 * rows * (width + 2) * 4 + 255) / 256 * 256;
}
__device__ __forceinline__ CutItem* cut_items(unsigned char* workspace) { return reinterpret_cast<CutItem*>(workspace); }
__device__ __forceinline__ float* cut_partials(unsigned char* workspace, int grid) {
    return reinterpret_cast<float*>(workspace + ((sizeof(CutItem) * grid + 255) / 256) * 256);
}

__device__ __forceinline__ long long warp_scan(long long v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
    }
    return v;
}

// ----------------------------------------------------------------- the join

// Block (c, y) of a part joins rows of the item that the border between the
// runs of CTAs c and c + 1 cuts, if no earlier border does.  Its warps share
// out the rows and each row's partial results.
template <typename T, int S, int D, int kThreads>
__global__ void __launch_bounds__(kThreads)
    cache_join_kernel(const __grid_constant__ CacheAttendArgs a, CutPart first, CutPart second) {
    constexpr int kPer = D / 32;
    constexpr int kJoinWarps = kThreads / 32;
    __shared__ float shared_o[kJoinWarps][D];
    __shared__ float shared_ml[kJoinWarps][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool late = (int)blockIdx.x >= first.blocks();
    const CutPart part_of = late ? second : first;
    const int block = (int)blockIdx.x - (late ? first.blocks() : 0);
    const int c = block / part_of.slices() + 1, slice = block % part_of.slices();
    wait_for_kernel_before();
    const CutItem* record = cut_items(part_of.workspace) + c;
    const int4 head_of = *reinterpret_cast<const int4*>(record), rest = *(reinterpret_cast<const int4*>(record) + 1);
    const CutItem cut = {head_of.x, head_of.y, head_of.z, head_of.w, {rest.x, rest.y, rest.z, rest.w}};
    if (cut.parts == 0) return;
    const float* partials = cut_partials(part_of.workspace, part_of.grid);
    const int tile_rows = part_of.rows, floats = partial_floats<D>(tile_rows);
    const CacheSequence q = cut.q;
    const int all_rows = (int)min((long long)tile_rows, (long long)q.rows * a.group - (long long)cut.tile * tile_rows);
    const int base = slice * kJoinRows, rows = min(kJoinRows, all_rows - base);
    if (rows <= 0) return;
    int share = 1;  // warps of a row
    while (share * 2 * rows <= kJoinWarps && share < cut.parts) share *= 2;
    const int local = warp / share, sub = warp % share, row = base + local;
    const bool active = local < rows;
    float m = -INFINITY, sum = 0.f, o[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) o[e] = 0.f;
    const auto add = [&](float pm, float ps, const float* v) {
        const float top = fmaxf(m, pm), from = top == -INFINITY ? 0.f : top;
        const float keep = exp2_fast(m - from), gain = exp2_fast(pm - from);
        sum = sum * keep + ps * gain;
#pragma unroll
        for (int e = 0; e < kPer; ++e) o[e] = o[e] * keep + v[e] * gain;
        m = top;
    };
    if (active) {
        const int from = (int)((long long)cut.parts * sub / share), to = (int)((long long)cut.parts * (sub + 1) / share);
#pragma unroll 4
        for (int i = from; i < to; ++i) {
            const float* part = partials + ((long long)(c - 1 + i) * 2 + (i == 0 ? 1 : 0)) * floats;
            float v[kPer];
#pragma unroll
            for (int e = 0; e < kPer; ++e) v[e] = part[row * D + lane * kPer + e];
            add(part[tile_rows * D + row], part[tile_rows * (D + 1) + row], v);
        }
    }
    if (share > 1) {
#pragma unroll
        for (int e = 0; e < kPer; ++e) shared_o[warp][lane * kPer + e] = o[e];
        if (lane == 0) {
            shared_ml[warp][0] = m;
            shared_ml[warp][1] = sum;
        }
        __syncthreads();
        if (sub == 0)
            for (int w = warp + 1; w < warp + share; ++w) add(shared_ml[w][0], shared_ml[w][1], &shared_o[w][lane * kPer]);
    }
    if (!active || sub != 0) return;
    const TileRow r = tile_row(a, q, cut.head, cut.tile * tile_rows + row);
    if (!r.valid) return;
    const bool some = r.seen > 0;  // a row without a key is zeros whatever the tile's other rows met
    const float inverse = 1.f / sum;
    const long long at = (long long)q.first + r.token;
    unsigned char* op = a.out + at * a.o_row + r.head * a.o_head + lane * (kPer * 2);
    bool fine = true;
#pragma unroll
    for (int e = 0; e < kPer; e += 2) {
        const float x = some ? o[e] * inverse : 0.f, y = some ? o[e + 1] * inverse : 0.f;
        fine = fine && fabsf(x) + fabsf(y) < INFINITY;
        *reinterpret_cast<uint32_t*>(op + e * 2) = Half16<T>::pack2(x, y);
    }
    if (a.lse && lane == 0) a.lse[at * a.query_heads + r.head] = some ? (m + log2f(sum)) * kLn2 : -INFINITY;
    if (__any_sync(0xffffffffu, !fine) && some)
        attend_row<T, S, D>(a, cut.sequence, q.first, q.before, q.length, r.token, r.head, nullptr);
}

// Joins the items that a call's kernels cut, the last of which it was launched
// behind: its launch overlaps that one's end.  Where items are far fewer than
// CTAs, 16 warps share a row's many parts: 32768 bf16 keys of one sequence, 8
// heads, 31.4 us against 36.9 with 8; 64 sequences of 1500 int8 keys, 16 heads,
// 46.7 against 43.5 (the rule's side).
template <typename T, int S, int D>
void launch_join(const CacheAttendArgs& a, const CutPart& first, const CutPart& second, cudaStream_t stream) {
    const int blocks = first.blocks() + second.blocks();
    if (blocks == 0) return;
    const long long items = std::max((long long)a.batch.sequences, (long long)a.rows * a.group / first.rows) * a.cache.heads;
    const bool many = first.grid > 8 * items;
    CUDA_CHECK(launch_early(many ? cache_join_kernel<T, S, D, 512> : cache_join_kernel<T, S, D, 256>, dim3(blocks),
                            many ? 512 : 256, 0, stream, a, first, second));
}

template <typename F>
void with_cache_types(int storage, bool bf16, int width, F&& f) {
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
}  // namespace wsp
