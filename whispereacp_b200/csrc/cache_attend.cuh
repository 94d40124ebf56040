// The attention over a paged cache: arguments and launches (cache_attend.cu).
#pragma once

#include "cache.cuh"

namespace wsp {

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
};

// storage: the cache's; bf16: the type of queries and out; width: 64 or 128.
void launch_cache_attend(const CacheAttendArgs& args, int storage, bool bf16, int width, int max_rows, int sms,
                         void* workspace, cudaStream_t stream);
size_t cache_attend_workspace(int width, int max_rows, int group, int sms);

}  // namespace wsp
