// The paged cache through include/wsp_cache.hpp alone: a window's rows appended
// in two calls to a cache of its own memory, read back, and attended, against
// the same sums in double precision here; a refusal as its exception.
//
//   cache_binding_test      prints "ok", or the first failure and exits 1
#include "wsp_cache.hpp"

#include <cuda_runtime_api.h>

#include <cmath>
#include <cstdio>
#include <stdexcept>
#include <vector>

namespace {

constexpr int kHeads = 2, kWidth = 64, kRows = 21, kPageRows = 16;

template <typename T>
T* on_device(const std::vector<T>& host) {
    void* p = nullptr;
    if (cudaMalloc(&p, host.size() * sizeof(T)) != cudaSuccess ||
        cudaMemcpy(p, host.data(), host.size() * sizeof(T), cudaMemcpyHostToDevice) != cudaSuccess)
        throw std::runtime_error("device memory");
    return static_cast<T*>(p);
}

// bf16 bits of small multiples of 1/8, exact
uint16_t bf16(float v) {
    union { float f; uint32_t u; } x{v};
    return (uint16_t)(x.u >> 16);
}
float value(int row, int head, int d, int which) { return (float)((row * 7 + head * 5 + d * 3 + which * 11) % 17 - 8) / 8.f; }

std::vector<uint16_t> rows_of(int which) {
    std::vector<uint16_t> v((size_t)kRows * kHeads * kWidth);
    for (int r = 0; r < kRows; ++r)
        for (int h = 0; h < kHeads; ++h)
            for (int d = 0; d < kWidth; ++d) v[((size_t)r * kHeads + h) * kWidth + d] = bf16(value(r, h, d, which));
    return v;
}

int run() {
    const wsp::CacheShape shape{kHeads, kWidth, kPageRows, 4, WSP_CACHE_BFLOAT16};
    wsp::CudaCache cache(shape, 0);
    const std::vector<uint16_t> q = rows_of(0), k = rows_of(1), v = rows_of(2);
    uint16_t *dq = on_device(q), *dk = on_device(k), *dv = on_device(v);
    uint16_t *ok = on_device(std::vector<uint16_t>(q.size())), *ov = on_device(std::vector<uint16_t>(q.size()));
    uint16_t* out = on_device(std::vector<uint16_t>(q.size()));
    float* lse = on_device(std::vector<float>(kRows * kHeads));
    int32_t* table = on_device(std::vector<int32_t>{3, 1});
    // 18 rows, then 3 more
    int32_t *first = on_device(std::vector<int32_t>{18, 0, 18}), *all = on_device(std::vector<int32_t>{kRows, 18, kRows}),
            *whole = on_device(std::vector<int32_t>{kRows, 0, kRows});
    wsp::CacheBatch batch{table, first, first + 1, 2, 2, 1, 18};
    const auto keys = cache.rows(dk, kHeads, WSP_BFLOAT16), values = cache.rows(dv, kHeads, WSP_BFLOAT16);
    cache.append(batch, 18, keys, values);
    batch.lengths = all;
    batch.starts = all + 1;
    batch.max_rows = 3;
    cache.append(batch, kRows, keys, values);
    batch.lengths = whole;
    batch.starts = whole + 1;
    batch.max_rows = kRows;
    cache.read(batch, kRows, cache.rows(ok, kHeads, WSP_BFLOAT16), cache.rows(ov, kHeads, WSP_BFLOAT16));
    const size_t bytes = cache.attendWorkspace(batch, kRows, kHeads);
    void* workspace = on_device(std::vector<uint8_t>(bytes + 16));
    cache.attend(batch, kRows, kHeads, cache.rows(dq, kHeads, WSP_BFLOAT16), cache.rows(out, kHeads, WSP_BFLOAT16), lse,
                 0.125f, true, workspace, bytes);
    cache.checkDevice();
    std::vector<uint16_t> rk(q.size()), rv(q.size()), ro(q.size());
    cudaMemcpy(rk.data(), ok, rk.size() * 2, cudaMemcpyDeviceToHost);
    cudaMemcpy(rv.data(), ov, rv.size() * 2, cudaMemcpyDeviceToHost);
    cudaMemcpy(ro.data(), out, ro.size() * 2, cudaMemcpyDeviceToHost);
    if (rk != k || rv != v) return std::printf("read back\n"), 1;
    for (int r = 0; r < kRows; ++r)
        for (int h = 0; h < kHeads; ++h) {
            std::vector<double> p(r + 1);
            double sum = 0;
            for (int j = 0; j <= r; ++j) {
                double s = 0;
                for (int d = 0; d < kWidth; ++d) s += (double)value(r, h, d, 0) * value(j, h, d, 1);
                sum += p[j] = std::exp(s * 0.125);
            }
            for (int d = 0; d < kWidth; ++d) {
                double o = 0, size = 0;
                for (int j = 0; j <= r; ++j) {
                    o += p[j] / sum * value(j, h, d, 2);
                    size += p[j] / sum * std::fabs(value(j, h, d, 2));
                }
                union { uint32_t u; float f; } got{(uint32_t)ro[((size_t)r * kHeads + h) * kWidth + d] << 16};
                // half a step of bf16 for the result and for each probability
                if (std::fabs(got.f - o) > (std::fabs(o) + size) / 256 + size * 1e-4)
                    return std::printf("row %d head %d: %g, not %g\n", r, h, got.f, o), 1;
            }
        }
    try {
        cache.attend(batch, kRows, 3, cache.rows(dq, 3, WSP_BFLOAT16), cache.rows(out, 3, WSP_BFLOAT16), nullptr, 1.f, true,
                     workspace, bytes);
        return std::printf("3 query heads over 2 were taken\n"), 1;
    } catch (const wsp::ModelError&) {
    }
    std::printf("ok\n");
    return 0;
}

}  // namespace

int main() {
    try {
        return run();
    } catch (const std::exception& e) {
        std::printf("%s\n", e.what());
        return 1;
    }
}
