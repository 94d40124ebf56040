// The paged cache's entry points (include/wsp_cache.h), their refusals checked
// on the host: a cache made here by hand, over addresses that no call may
// reach, and calls that must come back with a status before anything is
// launched.  Calls that have nothing to do must come back with WSP_OK.
//
//   cache_test      prints "ok", or the first failure and exits 1
#include "../../whispereacp_b200/csrc/cache.cu"

#include <cmath>
#include <cstdio>
#include <cstring>

namespace {

int failures = 0;

void expect(int status, int wanted, const char* text, const char* call) {
    const std::string said = wsp_last_error();
    if (status == wanted && said.find(text) != std::string::npos) return;
    std::printf("%s: status %d (wanted %d), \"%s\" (wanted \"%s\")\n", call, status, wanted, said.c_str(), text);
    ++failures;
}
#define EXPECT(call, wanted, text) expect((call), (wanted), (text), #call)

void* at(size_t address) { return reinterpret_cast<void*>(address); }

}  // namespace

int main() {
    // ---- creation
    wsp_cache* none = nullptr;
    wsp_cache_shape shape{4, 64, 16, 100, WSP_CACHE_FLOAT16};
    EXPECT(wsp_cache_create(nullptr, 0, nullptr, &none), WSP_INVALID_ARGUMENT, "NULL");
    EXPECT(wsp_cache_create(&shape, 0, nullptr, nullptr), WSP_INVALID_ARGUMENT, "NULL");
    for (int width : {0, 32, 63, 80, 96, 256}) {
        wsp_cache_shape s = shape;
        s.head_width = width;
        EXPECT(wsp_cache_create(&s, 0, nullptr, &none), WSP_MODEL_ERROR, "64 or 128 wide");
    }
    for (int rows : {0, 1, 8, 17, 48, 512, -16}) {
        wsp_cache_shape s = shape;
        s.page_rows = rows;
        EXPECT(wsp_cache_create(&s, 0, nullptr, &none), WSP_MODEL_ERROR, "a page has");
    }
    for (int storage : {0, 5, -1}) {
        wsp_cache_shape s = shape;
        s.storage = storage;
        EXPECT(wsp_cache_create(&s, 0, nullptr, &none), WSP_MODEL_ERROR, "storage");
    }
    for (int bad : {0, -3}) {
        wsp_cache_shape s = shape, t = shape;
        s.heads = bad;
        t.pages = bad;
        EXPECT(wsp_cache_create(&s, 0, nullptr, &none), WSP_MODEL_ERROR, "needs heads and pages");
        EXPECT(wsp_cache_create(&t, 0, nullptr, &none), WSP_MODEL_ERROR, "needs heads and pages");
    }
    const wsp_cache_memory memory{at(4096), at(8192), nullptr, nullptr, 4096, 1024, 64};
    wsp_cache_memory m = memory;
    m.values = nullptr;
    EXPECT(wsp_cache_create(&shape, 0, &m, &none), WSP_INVALID_ARGUMENT, "NULL");
    m = memory;
    m.keys = at(4096 + 8);
    EXPECT(wsp_cache_create(&shape, 0, &m, &none), WSP_INVALID_ARGUMENT, "16-byte aligned");
    m = memory;
    m.row_stride = 60;
    EXPECT(wsp_cache_create(&shape, 0, &m, &none), WSP_INVALID_ARGUMENT, "strides");
    m = memory;
    m.head_stride = 1028;
    EXPECT(wsp_cache_create(&shape, 0, &m, &none), WSP_INVALID_ARGUMENT, "strides");
    wsp_cache_shape eight = shape;
    eight.storage = WSP_CACHE_INT8;
    EXPECT(wsp_cache_create(&eight, 0, &memory, &none), WSP_INVALID_ARGUMENT, "NULL");
    if (none) ++failures;

    // ---- calls, over a cache made by hand
    wsp_cache cache{};
    cache.shape = shape;
    cache.memory = memory;
    cache.sms = 148;
    wsp_cache_batch batch{};
    batch.table = static_cast<const int32_t*>(at(1 << 20));
    batch.lengths = batch.starts = batch.table;
    batch.table_stride = batch.table_columns = 80;  // 1280 rows a sequence: the attention needs its workspace
    batch.sequences = 3;
    batch.max_rows = 2;
    const wsp_cache_rows rows{at(1 << 21), 256, 64, WSP_FLOAT16};
    wsp_cache_rows r = rows;
    size_t bytes = 0;

    EXPECT(wsp_cache_append(nullptr, &batch, 6, &rows, &rows, nullptr), WSP_INVALID_ARGUMENT, "cache must not be NULL");
    EXPECT(wsp_cache_append(&cache, nullptr, 6, &rows, &rows, nullptr), WSP_INVALID_ARGUMENT, "batch must not be NULL");
    EXPECT(wsp_cache_read(&cache, &batch, -1, &rows, &rows, nullptr), WSP_INVALID_ARGUMENT, "rows must not be negative");
    EXPECT(wsp_cache_read(&cache, &batch, 6, nullptr, &rows, nullptr), WSP_INVALID_ARGUMENT, "keys must not be NULL");
    EXPECT(wsp_cache_read(&cache, &batch, 6, &rows, nullptr, nullptr), WSP_INVALID_ARGUMENT, "values must not be NULL");
    for (auto change : {+[](wsp_cache_batch& b) { b.sequences = -1; }, +[](wsp_cache_batch& b) { b.max_rows = -1; },
                        +[](wsp_cache_batch& b) { b.table_columns = -1; }, +[](wsp_cache_batch& b) { b.lengths = nullptr; },
                        +[](wsp_cache_batch& b) { b.table = nullptr; }, +[](wsp_cache_batch& b) { b.table_stride = 79; },
                        +[](wsp_cache_batch& b) { b.starts = static_cast<const int32_t*>(at((1 << 20) + 2)); }}) {
        wsp_cache_batch b = batch;
        change(b);
        EXPECT(wsp_cache_append(&cache, &b, 6, &rows, &rows, nullptr), WSP_INVALID_ARGUMENT, "");
        EXPECT(wsp_cache_attend(&cache, &b, 6, 4, &rows, &rows, nullptr, 1.f, 1, at(4096), 1 << 30, nullptr),
               WSP_INVALID_ARGUMENT, "");
        EXPECT(wsp_cache_attend_workspace(&cache, &b, 6, 4, &bytes), WSP_INVALID_ARGUMENT, "");
    }
    for (auto change : {+[](wsp_cache_rows& x) { x.data = nullptr; }, +[](wsp_cache_rows& x) { x.data = at((1 << 21) + 2); },
                        +[](wsp_cache_rows& x) { x.row_stride = 260; }, +[](wsp_cache_rows& x) { x.head_stride = 68; },
                        +[](wsp_cache_rows& x) { x.row_stride = 0; }, +[](wsp_cache_rows& x) { x.head_stride = 56; },
                        +[](wsp_cache_rows& x) { x.dtype = 7; }}) {
        r = rows;
        change(r);
        EXPECT(wsp_cache_append(&cache, &batch, 6, &rows, &r, nullptr), WSP_INVALID_ARGUMENT, "values");
        EXPECT(wsp_cache_read(&cache, &batch, 6, &r, &rows, nullptr), WSP_INVALID_ARGUMENT, "keys");
        EXPECT(wsp_cache_attend(&cache, &batch, 6, 4, &r, &rows, nullptr, 1.f, 1, at(4096), 1 << 30, nullptr),
               WSP_INVALID_ARGUMENT, "queries");
        EXPECT(wsp_cache_attend(&cache, &batch, 6, 4, &rows, &r, nullptr, 1.f, 1, at(4096), 1 << 30, nullptr),
               WSP_INVALID_ARGUMENT, "out");
    }
    r = rows;
    r.dtype = WSP_FLOAT32;
    EXPECT(wsp_cache_append(&cache, &batch, 6, &rows, &r, nullptr), WSP_INVALID_ARGUMENT, "one dtype");
    EXPECT(wsp_cache_attend(&cache, &batch, 6, 4, &r, &r, nullptr, 1.f, 1, at(4096), 1 << 30, nullptr), WSP_MODEL_ERROR,
           "16-bit");
    r.dtype = WSP_BFLOAT16;
    EXPECT(wsp_cache_attend(&cache, &batch, 6, 4, &r, &r, nullptr, 1.f, 1, at(4096), 1 << 30, nullptr), WSP_MODEL_ERROR,
           "have its type");
    EXPECT(wsp_cache_attend(&cache, &batch, 6, 4, &rows, &r, nullptr, 1.f, 1, at(4096), 1 << 30, nullptr),
           WSP_MODEL_ERROR, "one 16-bit type");
    for (int heads : {0, -4, 3, 6})
        EXPECT(wsp_cache_attend(&cache, &batch, 6, heads, &rows, &rows, nullptr, 1.f, 1, at(4096), 1 << 30, nullptr),
               WSP_MODEL_ERROR, "multiple of the cache's heads");
    for (float scale : {NAN, INFINITY, -INFINITY})
        EXPECT(wsp_cache_attend(&cache, &batch, 6, 4, &rows, &rows, nullptr, scale, 1, at(4096), 1 << 30, nullptr),
               WSP_INVALID_ARGUMENT, "scale");
    EXPECT(wsp_cache_attend(&cache, &batch, 6, 4, &rows, &rows, static_cast<float*>(at(4098)), 1.f, 1, at(4096), 1 << 30,
                            nullptr),
           WSP_INVALID_ARGUMENT, "lse");
    EXPECT(wsp_cache_attend_workspace(&cache, &batch, 6, 4, nullptr), WSP_INVALID_ARGUMENT, "NULL");
    EXPECT(wsp_cache_attend_workspace(&cache, &batch, 6, 4, &bytes), WSP_OK, "");
    if (!bytes) ++failures, std::printf("no workspace\n");
    {
        EXPECT(wsp_cache_attend(&cache, &batch, 6, 4, &rows, &rows, nullptr, 1.f, 1, nullptr, 0, nullptr),
               WSP_INVALID_ARGUMENT, "workspace");
        EXPECT(wsp_cache_attend(&cache, &batch, 6, 4, &rows, &rows, nullptr, 1.f, 1, at(4096), bytes - 1, nullptr),
               WSP_INVALID_ARGUMENT, "workspace");
        EXPECT(wsp_cache_attend(&cache, &batch, 6, 4, &rows, &rows, nullptr, 1.f, 1, at(4104), bytes, nullptr),
               WSP_INVALID_ARGUMENT, "workspace");
    }
    EXPECT(wsp_cache_attend(&cache, &batch, 6, 4, &rows, &rows, nullptr, 1.f, 1, at(4096), bytes, nullptr),
           WSP_INVALID_ARGUMENT, "one memory");
    {
        // The rows of a sequence: 2^31 - 256 are the most.
        wsp_cache_batch b = batch;
        b.table_stride = b.table_columns = (0x7fffff00 >> 4) + 1;
        EXPECT(wsp_cache_attend(&cache, &b, 6, 4, &rows, &rows, nullptr, 1.f, 1, at(4096), bytes, nullptr),
               WSP_INVALID_ARGUMENT, "at most 2147483392 rows");
        EXPECT(wsp_cache_append(&cache, &b, 6, &rows, &rows, nullptr), WSP_INVALID_ARGUMENT, "at most 2147483392 rows");
        EXPECT(wsp_cache_read(&cache, &b, 6, &rows, &rows, nullptr), WSP_INVALID_ARGUMENT, "at most 2147483392 rows");
        b.table_stride = --b.table_columns;
        EXPECT(wsp_cache_attend_workspace(&cache, &b, 6, 4, &bytes), WSP_OK, "");
    }
    EXPECT(wsp_cache_get_memory(&cache, nullptr), WSP_INVALID_ARGUMENT, "NULL");
    wsp_cache_memory got{};
    EXPECT(wsp_cache_get_memory(&cache, &got), WSP_OK, "");
    if (std::memcmp(&got, &memory, sizeof got)) ++failures, std::printf("wsp_cache_get_memory\n");
    EXPECT(wsp_cache_check(nullptr), WSP_INVALID_ARGUMENT, "NULL");
    wsp_cache_destroy(nullptr);

    // ---- nothing to do
    batch.sequences = 0;
    batch.table = batch.lengths = batch.starts = nullptr;
    EXPECT(wsp_cache_append(&cache, &batch, 6, &rows, &rows, nullptr), WSP_OK, "");
    EXPECT(wsp_cache_attend(&cache, &batch, 6, 4, &rows, &rows, nullptr, 1.f, 1, nullptr, 0, nullptr), WSP_OK, "");
    EXPECT(wsp_cache_read(&cache, &batch, 0, &rows, &rows, nullptr), WSP_OK, "");

    if (failures == 0) std::printf("ok\n");
    return failures != 0;
}
