// Waits of the paged cache's kernels that give up: a wait for a barrier that
// nothing completes ends after its limit, says so and lets every later one end at
// once; and caches that share a status word report their own waits only.
//
//   cache_wait_test      prints "ok", or the first failure and exits 1
#include "../../whispereacp_b200/csrc/cache.cu"
#include "../../whispereacp_b200/csrc/cache_device.cuh"

#include <cstdio>
#include <vector>

namespace {

int failures = 0;

void expect(bool fine, const char* text) {
    if (fine) return;
    std::printf("%s: %s\n", text, wsp_last_error());
    ++failures;
}

// said: whether each of three waits was met (the first is, the second never,
// the third would be), and the abort word.
__global__ void waits(int* status, int mark, int* said) {
    __shared__ uint64_t bars[2];
    __shared__ int words[wsp::kBarrierWords];
    if (threadIdx.x == 0) {
        wsp::cache_barrier_init(bars, 1);
        wsp::cache_barrier_init(bars + 1, 1);
        for (int i = 0; i < wsp::kBarrierWords; ++i) words[i] = 0;
        words[wsp::kMarkWord] = mark;
        wsp::cache_arrive(bars);
        volatile int* abort = words;
        said[0] = wsp::cache_wait(bars, 0, abort, status, 7);
        said[1] = wsp::cache_wait(bars + 1, 0, abort, status, 9);
        said[2] = wsp::cache_wait(bars + 1, 0, abort, status, 11);
        said[3] = words[0];
    }
}

int run() {
    const wsp_cache_shape shape{1, 64, 16, 1, WSP_CACHE_FLOAT16};
    void* pool = nullptr;
    int* said = nullptr;
    if (cudaMalloc(&pool, 2 * 16 * 64 * 2) != cudaSuccess || cudaMalloc(&said, 16) != cudaSuccess) return 1;
    const wsp_cache_memory memory{pool, static_cast<char*>(pool) + 16 * 64 * 2, nullptr, nullptr, 1024, 1024, 64};
    std::vector<wsp_cache*> caches(wsp::kStatusWords + 2);
    for (auto& c : caches) expect(wsp_cache_create(&shape, 0, &memory, &c) == WSP_OK, "wsp_cache_create");
    if (failures) return 1;
    wsp_cache *first = caches.front(), *same = caches[wsp::kStatusWords], *other = caches[1];
    expect(first->status == same->status && first->status != other->status, "the words");

    waits<<<1, 32>>>(first->status, first->mark, said);
    int got[4] = {};
    cudaMemcpy(got, said, sizeof got, cudaMemcpyDeviceToHost);
    expect(got[0] == 1 && got[1] == 0 && got[2] == 0 && got[3] == 1, "the waits");
    expect(wsp_cache_check(other) == WSP_OK, "a cache of another word");
    expect(wsp_cache_check(same) == WSP_OK, "a cache of the same word");
    expect(wsp_cache_check(first) == WSP_CUDA_ERROR, "the cache whose wait gave up");
    expect(std::string(wsp_last_error()).find("(9)") != std::string::npos, "which wait it was");
    expect(wsp_cache_check(first) == WSP_OK, "asked again");
    for (auto c : caches) wsp_cache_destroy(c);
    if (!failures) std::printf("ok\n");
    return failures != 0;
}

}  // namespace

int main() { return run(); }
