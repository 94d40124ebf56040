// The attention over a paged cache: arguments and launches.
#pragma once

#include "cache.cuh"

#include <cuda.h>

namespace wsp {

// Rows of the box a tensor map of a pool copies: a page's rows, or 64 of them.
__host__ __device__ constexpr int cache_box_shift(int page_shift) { return page_shift < 6 ? page_shift : 6; }

struct CacheAttendArgs {
    CacheView cache;
    CacheBatchView batch;
    const unsigned char* queries;  // 16-bit rows, strides in bytes
    long long q_row, q_head;
    unsigned char* out;
    long long o_row, o_head;
    float* lse;                    // [rows][query_heads], or null
    int rows, query_heads, group;  // group = query heads of a key head
    float scale;
    int causal;
    int uncut;                     // the few-row kernel's CTAs take whole items
    int behind;                    // the few-row kernel runs behind the chunks', which waited for what is before
    int mark;                      // the cache's, a multiple of 256: caches may share the status word
    long long few;                 // rows * group up to which a sequence is the few-row kernel's
    int* status;                   // where a wait that gives up is recorded: its kind, and the mark
    unsigned char* workspace;
};

// The pools as tensor maps: [pages][heads][page_rows][head_width], a box one
// page's (or 64) rows of up to 128 bytes, swizzled over as many.
struct CacheMaps {
    CUtensorMap keys, values;
};

// What a launch needs to know beside its arguments: the cache's storage, the
// type of queries and out, the heads' width, the bounds of a sequence's new
// and held rows.
struct CacheAttendShape {
    int storage;
    bool bf16;
    int width, max_rows;
    long long held;
    int sms;
};

// What a kernel leaves to be joined: its workspace, its CTAs, and the rows of
// its items.  The join takes 8 of an item's rows a block.
constexpr int kJoinRows = 8;
struct CutPart {
    unsigned char* workspace;
    int grid, rows;
    __host__ __device__ int slices() const { return rows / kJoinRows; }
    __host__ __device__ int blocks() const { return grid > 1 ? (grid - 1) * slices() : 0; }
};

// The kernel of many rows (cache_chunk.cu): sequences of more than `few` rows
// of a key head.
void prepare_cache_chunk(int storage, int width);
CutPart launch_cache_chunk(const CacheAttendArgs& args, const CacheMaps& maps, const CacheAttendShape& shape,
                           cudaStream_t stream);
size_t cache_chunk_workspace(const CacheAttendShape& shape);

// A launch that may begin while the kernel before it ends: the kernel's first
// act is to wait for that (griddepcontrol.wait), so that only its launch and
// what comes before the wait overlap.
template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, int threads, size_t shared, cudaStream_t stream,
                         const Args&... args) {
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args...);
}
__device__ __forceinline__ void wait_for_kernel_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Raises the kernels' limits of shared memory on the current device.
void prepare_cache_attend(int storage, int width);
void launch_cache_attend(const CacheAttendArgs& args, const CacheMaps& maps, const CacheAttendShape& shape,
                         cudaStream_t stream);
size_t cache_attend_workspace(const CacheAttendShape& shape, int group);

}  // namespace wsp
