/*
 * wsp_cache.hpp -- the C++ binding of the paged key/value cache, header only,
 * over the C ABI of wsp_cache.h: the cache ops of Net (appendLinear's cache
 * write and the attention over a Cache, Lib/WhisperEACP/Net/Net.h:110-171)
 * for windows that stand at their own tokens.  Status codes become the
 * exceptions of wsp_decoder.hpp.  All data pointers are device pointers; calls
 * queue on `stream` (a cudaStream_t) and return without waiting.
 */
#ifndef WSP_CACHE_HPP
#define WSP_CACHE_HPP

#include "wsp_cache.h"
#include "wsp_decoder.hpp"

#include <cstddef>
#include <utility>

namespace wsp {

using CacheShape = wsp_cache_shape;
using CacheMemory = wsp_cache_memory;
using CacheBatch = wsp_cache_batch;
using CacheRows = wsp_cache_rows;

class CudaCache {
public:
    /* Over the caller's memory, or (memory null) over zeroed memory of its own. */
    CudaCache(const CacheShape& shape, int device, const CacheMemory* memory = nullptr) : shape_(shape) {
        check(wsp_cache_create(&shape_, device, memory, &handle_));
    }
    ~CudaCache() { wsp_cache_destroy(handle_); }
    CudaCache(const CudaCache&) = delete;
    CudaCache& operator=(const CudaCache&) = delete;
    CudaCache(CudaCache&& other) noexcept : shape_(other.shape_), handle_(std::exchange(other.handle_, nullptr)) {}

    const CacheShape& shape() const { return shape_; }
    CacheMemory memory() const {
        CacheMemory m{};
        check(wsp_cache_get_memory(handle_, &m));
        return m;
    }

    /* A contiguous row array [rows, heads, head_width]. */
    CacheRows rows(void* data, int heads, wsp_dtype dtype) const {
        return {data, (int64_t)heads * shape_.head_width, shape_.head_width, dtype};
    }

    /* The sequences' new rows into the pages, rounded (8-bit: scaled) once. */
    void append(const CacheBatch& batch, int rows, const CacheRows& keys, const CacheRows& values,
                void* stream = nullptr) {
        check(wsp_cache_append(handle_, &batch, rows, &keys, &values, stream));
    }
    /* The sequences' last rows out of the pages. */
    void read(const CacheBatch& batch, int rows, const CacheRows& keys, const CacheRows& values,
              void* stream = nullptr) {
        check(wsp_cache_read(handle_, &batch, rows, &keys, &values, stream));
    }

    /* What attend's workspace holds, for this batch and any with the same
       max_rows and table_columns. */
    size_t attendWorkspace(const CacheBatch& batch, int rows, int queryHeads) const {
        size_t bytes = 0;
        check(wsp_cache_attend_workspace(handle_, &batch, rows, queryHeads, &bytes));
        return bytes;
    }
    /* out = softmax(scale q . k) v of the new rows over what their sequences
       hold; lse [rows, queryHeads] or null. */
    void attend(const CacheBatch& batch, int rows, int queryHeads, const CacheRows& queries, const CacheRows& out,
                float* lse, float scale, bool causal, void* workspace, size_t workspaceBytes, void* stream = nullptr) {
        check(wsp_cache_attend(handle_, &batch, rows, queryHeads, &queries, &out, lse, scale, causal ? 1 : 0, workspace,
                               workspaceBytes, stream));
    }

    /* Waits for the device; throws if a wait inside a kernel gave up. */
    void checkDevice() { check(wsp_cache_check(handle_)); }

private:
    CacheShape shape_;
    wsp_cache* handle_ = nullptr;
};

}  // namespace wsp

#endif
