// The paged key/value cache: the C ABI of include/wsp_cache.h, and the
// kernels that write rows into the pages and read them back (sm_100a).
#include "../../include/wsp_cache.h"

#include "cache.cuh"
#include "cache_attend.cuh"
#include "host.h"

#include <algorithm>
#include <atomic>
#include <memory>
#include <tuple>
#include <utility>

namespace wsp {
namespace {

// ---------------------------------------------------------- append and read
//
// Bound by the bytes of the rows and the pages.  A block takes up to 16 rows,
// finds each one's place once, and goes over (head, row, piece), pieces
// fastest: a warp's lanes then cover 4 or 8 neighbouring rows of one head,
// which lie next to one another in the page.  A thread holds a piece of 16 (8-bit
// pages) or 8 values of the key and of the value: 16 bytes of the page each,
// and 2 x 16 or 2 x 32 of the rows in flight.  The D / 16 lanes of an 8-bit row
// agree on its scale.
//
// Measured: 48 x 1500 rows of 20 heads, 64 wide, fp16 to e4m3 and back, 205 us
// for 1.11 GB, 5.4 TB/s of a copy's 6.54 (what is left is the conversions and
// the scales' agreement); ragged rows of 32 windows read back from int8, 24.4 us
// for 100 MB; one step's rows of 64 windows 2.5 us, a launch and two loads that
// depend on one another.

struct RowsView {
    unsigned char* data;
    long long row_bytes, head_bytes;
};

struct CopyArgs {
    CacheView cache;
    CacheBatchView batch;
    RowsView keys, values;
    int rows, block_rows;  // rows of the arrays, and of a block: 2^n
};

// dtype codes of wsp_decoder.h as types
template <int T> struct RowType;
template <> struct RowType<WSP_FLOAT32> { static constexpr int bytes = 4; };
template <> struct RowType<WSP_FLOAT16> { static constexpr int bytes = 2; using type = __half; };
template <> struct RowType<WSP_BFLOAT16> { static constexpr int bytes = 2; using type = __nv_bfloat16; };

// A piece of kE values as it lies in memory, 4 bytes a word.
template <int kWords>
struct Piece {
    uint32_t w[kWords];
};
template <int kWords>
__device__ __forceinline__ Piece<kWords> fetch_piece(const unsigned char* p) {
    Piece<kWords> v;
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
        const uint4 x = load_stream(p + i * 4);
        v.w[i] = x.x, v.w[i + 1] = x.y, v.w[i + 2] = x.z, v.w[i + 3] = x.w;
    }
    return v;
}
template <int kWords>
__device__ __forceinline__ void put_piece(unsigned char* p, const Piece<kWords>& v) {
#pragma unroll
    for (int i = 0; i < kWords; i += 4)
        *reinterpret_cast<uint4*>(p + i * 4) = make_uint4(v.w[i], v.w[i + 1], v.w[i + 2], v.w[i + 3]);
}

// Values 2 i and 2 i + 1 of a piece of rows, and the way back.
template <int T, int kWords>
__device__ __forceinline__ float2 row_pair(const Piece<kWords>& v, int i) {
    if constexpr (T == WSP_FLOAT32) return make_float2(__uint_as_float(v.w[2 * i]), __uint_as_float(v.w[2 * i + 1]));
    else return Half16<typename RowType<T>::type>::pair_to_float2(v.w[i]);
}
template <int T, int kWords>
__device__ __forceinline__ void set_row_pair(Piece<kWords>& v, int i, float x, float y) {
    if constexpr (T == WSP_FLOAT32) v.w[2 * i] = __float_as_uint(x), v.w[2 * i + 1] = __float_as_uint(y);
    else v.w[i] = Half16<typename RowType<T>::type>::pack2(x, y);
}

// The largest magnitude of a piece, through the values' bits: without the
// sign they order as the values do, and keep a NaN on top.
template <int T, int kWords>
__device__ __forceinline__ float largest(const Piece<kWords>& v) {
    if constexpr (T == WSP_FLOAT32) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < kWords; ++i) top = max(top, v.w[i] & 0x7fffffffu);
        return __uint_as_float(top);
    } else {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < kWords; ++i)
            asm("max.u16x2 %0, %1, %2;" : "=r"(top) : "r"(top), "r"(v.w[i] & 0x7fff7fffu));
        const uint32_t one = max(top & 0xffffu, top >> 16);
        if constexpr (T == WSP_BFLOAT16) return __uint_as_float(one << 16);
        else return __half2float(__ushort_as_half((unsigned short)one));
    }
}

// The scale byte of a row whose largest magnitude is `top`: E + 127 with E
// the smallest integer for which top <= L 2^E.  top = m 2^e with m in [1, 2)
// (the exponent bits), and L = 448 is 1.75 2^8, 127 is 1.984375 2^6: E is e
// minus L's exponent, and one more where m is above L's mantissa.  Magnitudes
// so small that E would be below -126 keep E = -126.
template <int S>
__device__ __forceinline__ uint32_t scale_byte(float top) {
    const uint32_t bits = __float_as_uint(top);
    if (bits >= 0x7f800000u) return 255u;
    constexpr int kExponent = S == kCacheE4m3 ? 8 : 6;
    constexpr uint32_t kMantissa = S == kCacheE4m3 ? 0x600000u : 0x7e0000u;
    const int e = (int)(bits >> 23) - kExponent + ((bits & 0x7fffffu) > kMantissa ? 1 : 0);
    return (uint32_t)max(e, 1);
}

// A piece of rows as a piece of a page; the row's lanes agree on its scale
// byte.  A row that holds an infinity or NaN has byte 255, and its values no
// meaning.
template <int S, int T, int D, int kIn, int kOut>
__device__ __forceinline__ uint32_t narrow_piece(const Piece<kIn>& in, Piece<kOut>& out) {
    if constexpr (!cache_eight(S)) {
        constexpr int kStored = S == kCacheF16 ? WSP_FLOAT16 : WSP_BFLOAT16;
#pragma unroll
        for (int i = 0; i < kOut; ++i) {
            if constexpr (T == kStored) {
                out.w[i] = in.w[i];
            } else {
                const float2 x = row_pair<T>(in, i);
                set_row_pair<kStored>(out, i, x.x, x.y);
            }
        }
        return 0;
    } else {
        float top = largest<T>(in);
        // NaN above all: an order of the bits again
        uint32_t bits = __float_as_uint(top);
#pragma unroll
        for (int o = D / 32; o > 0; o >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, o));
        const uint32_t byte = scale_byte<S>(__uint_as_float(bits));
        // 2^(127 - byte); byte is 1..249, or 255 and then any finite factor
        const float inverse = __uint_as_float((254u - min(byte, 253u)) << 23);
#pragma unroll
        for (int h = 0; h < kOut; ++h) {
            const float2 x = row_pair<T>(in, 2 * h), y = row_pair<T>(in, 2 * h + 1);
            if constexpr (S == kCacheE4m3) {
                const uint32_t lo =
                    __nv_cvt_float2_to_fp8x2(make_float2(x.x * inverse, x.y * inverse), __NV_SATFINITE, __NV_E4M3);
                const uint32_t hi =
                    __nv_cvt_float2_to_fp8x2(make_float2(y.x * inverse, y.y * inverse), __NV_SATFINITE, __NV_E4M3);
                out.w[h] = lo | (hi << 16);
            } else {
                // 1.5 2^23 + x rounds x to an integer, ties to even, in the low
                // bits; the product is exact
                const float magic = 12582912.f;
                const uint32_t a = __float_as_uint(fmaf(x.x, inverse, magic)), b = __float_as_uint(fmaf(x.y, inverse, magic));
                const uint32_t c = __float_as_uint(fmaf(y.x, inverse, magic)), d = __float_as_uint(fmaf(y.y, inverse, magic));
                out.w[h] = __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
            }
        }
        return byte;
    }
}

// The way back: the values a piece of a page stands for, rounded once.
template <int S, int T, int kIn, int kOut>
__device__ __forceinline__ void widen_piece(const Piece<kIn>& in, uint32_t byte, Piece<kOut>& out) {
    if constexpr (!cache_eight(S)) {
        constexpr int kStored = S == kCacheF16 ? WSP_FLOAT16 : WSP_BFLOAT16;
#pragma unroll
        for (int i = 0; i < kIn; ++i) {
            if constexpr (T == kStored) {
                out.w[i] = in.w[i];
            } else {
                const float2 x = row_pair<kStored>(in, i);
                set_row_pair<T>(out, i, x.x, x.y);
            }
        }
    } else {
        const float s = cache_scale(byte);
#pragma unroll
        for (int e = 0; e < 2 * kIn; ++e) {
            const float2 f = cache_pair<S>((in.w[e / 2] >> (16 * (e & 1))) & 0xffffu);
            set_row_pair<T>(out, e, f.x * s, f.y * s);
        }
    }
}

constexpr int kCopyThreads = 256;
constexpr int kCopyRows = 16;  // of a block, at most

template <int S, int T, int D, bool kWrite>
__global__ void __launch_bounds__(kCopyThreads) cache_copy_kernel(const __grid_constant__ CopyArgs a) {
    constexpr int kE = cache_eight(S) ? 16 : 8;  // values of a piece
    constexpr int kLanes = D / kE;               // pieces of a row
    __shared__ long long pool_at[kCopyRows], scale_at[kCopyRows];  // a row's place in head 0; -1: no page, -2: no row
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int first = (int)blockIdx.x * a.block_rows;
    wait_for_kernel_before();
    for (int i = warp; i < a.block_rows; i += kCopyThreads / 32) {
        const int r = first + i;
        // The row's sequence: as many as end at or before it lie in front.
        int s = 0;
        for (int base = 0; base < a.batch.sequences; base += 32) {
            const bool before = base + lane < a.batch.sequences && __ldg(a.batch.starts + base + lane + 1) <= r;
            s += __popc(__ballot_sync(0xffffffffu, before));
        }
        if (lane == 0) {
            long long at = -2, si = 0;
            if (r < a.rows && s < a.batch.sequences) {
                const CacheSequence q = cache_sequence(a.cache, a.batch, s);
                if (r >= q.first) {
                    const int position = q.before + (r - q.first);
                    const int page = cache_page(a.cache, a.batch, s, position);
                    const int slot = position & ((1 << a.cache.page_shift) - 1);
                    at = page < 0 ? -1 : cache_offset(a.cache, page, 0, slot);
                    si = page < 0 ? 0 : cache_scale_index(a.cache, page, 0, slot);
                }
            }
            pool_at[i] = at;
            scale_at[i] = si;
        }
    }
    __syncthreads();
    constexpr int kPage = kE * cache_bytes(S) / 4, kRow = kE * RowType<T>::bytes / 4;  // words of a piece
    constexpr int kAtOnce = 2;  // pieces of the key and of the value on their way
    const int items = a.cache.heads * a.block_rows * kLanes;
    const int row_shift = 31 - __clz(a.block_rows);
    // Whole warps stay for the rows' shuffles.
    for (int base = warp * 32; base < items; base += kAtOnce * kCopyThreads) {
        Piece<kWrite ? kRow : kPage> key_in[kAtOnce], value_in[kAtOnce];
        unsigned char *key_out[kAtOnce], *value_out[kAtOnce];
        uint8_t *key_scale[kAtOnce], *value_scale[kAtOnce];
        uint32_t key_byte[kAtOnce], value_byte[kAtOnce];
        int state[kAtOnce];  // 1: a row and its page, 0: a row of no page, -1: none
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int item = base + i * kCopyThreads + lane;
            const int piece = item % kLanes, in_block = (item / kLanes) & (a.block_rows - 1);
            const int head = (item / kLanes) >> row_shift;
            const long long at = pool_at[in_block];
            state[i] = item < items && at >= -1 ? (at >= 0) : -1;
            const long long to = at + head * a.cache.head_bytes + piece * (kE * cache_bytes(S));
            const long long r = first + in_block;
            unsigned char* key = a.keys.data + r * a.keys.row_bytes + head * a.keys.head_bytes + piece * (kRow * 4);
            unsigned char* value = a.values.data + r * a.values.row_bytes + head * a.values.head_bytes + piece * (kRow * 4);
            if constexpr (cache_eight(S)) {
                const long long si = scale_at[in_block] + ((long long)head << a.cache.page_shift);
                key_scale[i] = a.cache.key_scales + si;
                value_scale[i] = a.cache.value_scales + si;
                if (piece != 0 && kWrite) key_scale[i] = nullptr;
            }
            key_out[i] = kWrite ? a.cache.keys + to : key;
            value_out[i] = kWrite ? a.cache.values + to : value;
            key_in[i] = value_in[i] = {};
            key_byte[i] = value_byte[i] = 0;
            if (state[i] == 1) {
                key_in[i] = fetch_piece<kWrite ? kRow : kPage>(kWrite ? key : a.cache.keys + to);
                value_in[i] = fetch_piece<kWrite ? kRow : kPage>(kWrite ? value : a.cache.values + to);
                if constexpr (cache_eight(S) && !kWrite) {
                    key_byte[i] = __ldg(key_scale[i]);
                    value_byte[i] = __ldg(value_scale[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            if constexpr (kWrite) {
                Piece<kPage> k, v;
                const uint32_t kb = narrow_piece<S, T, D>(key_in[i], k), vb = narrow_piece<S, T, D>(value_in[i], v);
                if (state[i] == 1) {
                    put_piece(key_out[i], k);
                    put_piece(value_out[i], v);
                    if constexpr (cache_eight(S))
                        if (key_scale[i]) {
                            *key_scale[i] = (uint8_t)kb;
                            *value_scale[i] = (uint8_t)vb;
                        }
                }
            } else if (state[i] >= 0) {
                Piece<kRow> k, v;
                widen_piece<S, T>(key_in[i], key_byte[i], k);
                widen_piece<S, T>(value_in[i], value_byte[i], v);
                put_piece(key_out[i], k);
                put_piece(value_out[i], v);
            }
        }
    }
}

template <int S, int T, bool kWrite>
void launch_copy(const CopyArgs& a, int width, cudaStream_t stream) {
    const unsigned grid = (unsigned)(((long long)a.rows + a.block_rows - 1) / a.block_rows);
    CUDA_CHECK(launch_early(width == 64 ? cache_copy_kernel<S, T, 64, kWrite> : cache_copy_kernel<S, T, 128, kWrite>,
                            dim3(grid), kCopyThreads, 0, stream, a));
}

template <int S, bool kWrite>
void launch_copy(const CopyArgs& a, int dtype, int width, cudaStream_t stream) {
    if (dtype == WSP_FLOAT32) launch_copy<S, WSP_FLOAT32, kWrite>(a, width, stream);
    else if (dtype == WSP_FLOAT16) launch_copy<S, WSP_FLOAT16, kWrite>(a, width, stream);
    else launch_copy<S, WSP_BFLOAT16, kWrite>(a, width, stream);
}

template <bool kWrite>
void launch_copy(const CopyArgs& a, int storage, int dtype, int width, cudaStream_t stream) {
    if (storage == kCacheF16) launch_copy<kCacheF16, kWrite>(a, dtype, width, stream);
    else if (storage == kCacheBf16) launch_copy<kCacheBf16, kWrite>(a, dtype, width, stream);
    else if (storage == kCacheE4m3) launch_copy<kCacheE4m3, kWrite>(a, dtype, width, stream);
    else launch_copy<kCacheInt8, kWrite>(a, dtype, width, stream);
}

// ------------------------------------------------------------------- host

class CurrentDevice {
public:
    explicit CurrentDevice(int device) {
        CUDA_CHECK(cudaGetDevice(&before_));
        if (before_ != device) CUDA_CHECK(cudaSetDevice(device));
        else before_ = -1;
    }
    ~CurrentDevice() {
        if (before_ >= 0) cudaSetDevice(before_);
    }
    CurrentDevice(const CurrentDevice&) = delete;
    CurrentDevice& operator=(const CurrentDevice&) = delete;

private:
    int before_ = -1;
};

int row_size(int dtype) { return dtype == WSP_FLOAT32 ? 4 : 2; }

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace wsp

struct wsp_cache {
    wsp_cache_shape shape;
    wsp_cache_memory memory;
    wsp::CacheView view;
    wsp::CacheMaps maps;
    int device = 0;
    int sms = 0;
    wsp::DeviceBuffer owned[4];
    int* status = nullptr;  // which wait of a kernel gave up: the kind of the last, and the mark of its cache
    int mark = 0;
};

namespace wsp {
namespace {

using std::to_string;

const wsp_cache& checked(const wsp_cache* cache) {
    if (!cache) throw InvalidArgument("cache must not be NULL");
    return *cache;
}

// Positions and what a kernel adds to them (a block of 128 keys, the copies'
// boxes) stay in 31 bits.
constexpr long long kMostHeld = 0x7fffff00ll;

void check_batch(const wsp_cache& c, const wsp_cache_batch* b, int rows) {
    if (!b) throw InvalidArgument("batch must not be NULL");
    if (rows < 0) throw InvalidArgument("rows must not be negative, got " + to_string(rows));
    if (b->sequences < 0 || b->table_columns < 0 || b->max_rows < 0)
        throw InvalidArgument("a batch's sequences, table_columns and max_rows must not be negative");
    if ((long long)b->table_columns * c.shape.page_rows > kMostHeld)
        throw InvalidArgument("a table's columns hold at most " + to_string(kMostHeld) + " rows of a sequence, not " +
                              to_string((long long)b->table_columns * c.shape.page_rows));
    if (b->sequences == 0) return;
    if (!b->lengths || !b->starts || (!b->table && b->table_columns > 0))
        throw InvalidArgument("a batch's table, lengths and starts must not be NULL");
    if (b->sequences > 1 && b->table_stride < b->table_columns)
        throw InvalidArgument("table_stride (" + to_string(b->table_stride) + ") must hold table_columns (" +
                              to_string(b->table_columns) + ")");
    for (const void* p : {(const void*)b->table, (const void*)b->lengths, (const void*)b->starts})
        if (reinterpret_cast<uintptr_t>(p) & 3) throw InvalidArgument("a batch's arrays must be 4-byte aligned");
}

// A row array's view; heads 1 wide need no head stride.
RowsView check_rows(const wsp_cache_rows* r, const char* name, int rows, int heads, int width) {
    if (!r) throw InvalidArgument(std::string(name) + " must not be NULL");
    if (r->dtype != WSP_FLOAT32 && r->dtype != WSP_FLOAT16 && r->dtype != WSP_BFLOAT16)
        throw InvalidArgument(std::string(name) + ": not a wsp_dtype: " + to_string(r->dtype));
    if (rows > 0 && !r->data) throw InvalidArgument(std::string(name) + "' data must not be NULL");
    const int size = row_size(r->dtype);
    if (!aligned(r->data) || (rows > 1 && r->row_stride * size % 16) || (heads > 1 && r->head_stride * size % 16))
        throw InvalidArgument(std::string(name) + " must be 16-byte aligned, its strides multiples of 16 bytes");
    if ((rows > 1 && r->row_stride < width) || (heads > 1 && r->head_stride < width))
        throw InvalidArgument(std::string(name) + ": strides must be at least head_width (" + to_string(width) + ")");
    return {static_cast<unsigned char*>(r->data), r->row_stride * size, r->head_stride * size};
}

CacheBatchView batch_view(const wsp_cache_batch& b) {
    return {b.table, b.lengths, b.starts, b.table_stride, b.table_columns, b.sequences};
}

// The caches' status words: static device memory, one after another, so that
// making a cache allocates and waits for nothing.  Caches 1024 apart share one,
// which then holds the last wait that gave up: their marks tell whose it was
// (2^22 of them, so that none is used again while a cache of it lives).
constexpr int kStatusWords = 1024;
__device__ int status_words[kStatusWords];

std::pair<int*, int> next_status() {
    static std::atomic<unsigned> made{0};
    void* words = nullptr;
    CUDA_CHECK(cudaGetSymbolAddress(&words, status_words));
    const unsigned n = made++;
    return {static_cast<int*>(words) + n % kStatusWords, (int)((n % (1u << 22) + 1) << 8)};
}

using EncodeTiled = decltype(&cuTensorMapEncodeTiled);

EncodeTiled encode_tiled() {
    static const EncodeTiled found = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult result{};
        CUDA_CHECK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &result));
        if (result != cudaDriverEntryPointSuccess || !f) throw CudaFailure("the driver has no cuTensorMapEncodeTiled", false);
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return found;
}

// A pool as the copy engine sees it: [pages][heads][page_rows][width], a box
// a page's rows (64 at most) of up to 128 bytes, swizzled over its row.
CUtensorMap pool_map(const wsp_cache_shape& s, const wsp_cache_memory& m, void* pool) {
    const int size = cache_bytes(s.storage);
    const cuuint64_t extents[4] = {(cuuint64_t)s.head_width, (cuuint64_t)s.page_rows, (cuuint64_t)s.heads,
                                   (cuuint64_t)s.pages};
    const cuuint64_t strides[3] = {(cuuint64_t)(m.row_stride * size), (cuuint64_t)(m.head_stride * size),
                                   (cuuint64_t)(m.page_stride * size)};
    const cuuint32_t columns = std::min(s.head_width, 128 / size);
    const cuuint32_t box[4] = {columns, (cuuint32_t)std::min(s.page_rows, 64), 1, 1}, steps[4] = {1, 1, 1, 1};
    const CUtensorMapDataType type = s.storage == WSP_CACHE_FLOAT16    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                     : s.storage == WSP_CACHE_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                       : CU_TENSOR_MAP_DATA_TYPE_UINT8;
    CUtensorMap map;
    const CUresult result = encode_tiled()(&map, type, 4, pool, extents, strides, box, steps,
                                           CU_TENSOR_MAP_INTERLEAVE_NONE,
                                           columns * size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (result != CUDA_SUCCESS)
        throw ModelError("the pools' strides are not ones the copy engine takes (status " + to_string((int)result) + ")");
    return map;
}

CacheAttendShape attend_shape(const wsp_cache& c, int dtype, const wsp_cache_batch& batch) {
    return {c.shape.storage,    dtype == WSP_BFLOAT16,
            c.shape.head_width, batch.max_rows,
            (long long)batch.table_columns * c.shape.page_rows, c.sms};
}

size_t checked_workspace(const wsp_cache& c, const wsp_cache_batch* batch, int rows, int query_heads) {
    check_batch(c, batch, rows);
    if (query_heads <= 0 || query_heads % c.shape.heads)
        throw ModelError("query_heads (" + to_string(query_heads) + ") must be a multiple of the cache's heads (" +
                         to_string(c.shape.heads) + ")");
    return cache_attend_workspace(attend_shape(c, WSP_FLOAT16, *batch), query_heads / c.shape.heads);
}

template <bool kWrite>
void copy_rows(wsp_cache* cache, const wsp_cache_batch* batch, int rows, const wsp_cache_rows* keys,
               const wsp_cache_rows* values, void* stream) {
    const wsp_cache& c = checked(cache);
    check_batch(c, batch, rows);
    CopyArgs a{};
    a.keys = check_rows(keys, "keys", rows, c.shape.heads, c.shape.head_width);
    a.values = check_rows(values, "values", rows, c.shape.heads, c.shape.head_width);
    if (keys->dtype != values->dtype) throw InvalidArgument("keys and values must have one dtype");
    if (rows == 0 || batch->sequences == 0) return;
    a.cache = c.view;
    a.batch = batch_view(*batch);
    a.rows = rows;
    // As many rows a block as leave every SM two blocks: 72000 int8 rows x 16
    // heads are written in 66 us by 16 rows a block and in 194 by one, 64 in 5.9
    // and in 2.9.
    a.block_rows = 1;
    while (a.block_rows < kCopyRows && rows / (2 * a.block_rows) >= 2 * c.sms) a.block_rows *= 2;
    CurrentDevice device(c.device);
    launch_copy<kWrite>(a, c.shape.storage, keys->dtype, c.shape.head_width, static_cast<cudaStream_t>(stream));
}

}  // namespace
}  // namespace wsp

using wsp::guarded;

extern "C" {

int wsp_cache_create(const wsp_cache_shape* shape, int device, const wsp_cache_memory* memory, wsp_cache** out) {
    return guarded([&] {
        using wsp::ModelError;
        using std::to_string;
        if (!shape || !out) throw wsp::InvalidArgument("shape and out must not be NULL");
        const wsp_cache_shape& s = *shape;
        if (s.storage < WSP_CACHE_FLOAT16 || s.storage > WSP_CACHE_INT8)
            throw ModelError("a cache's storage is one of WSP_CACHE_FLOAT16, _BFLOAT16, _E4M3 and _INT8, not " +
                             to_string(s.storage));
        if (s.head_width != 64 && s.head_width != 128)
            throw ModelError("a cache's heads are 64 or 128 wide, not " + to_string(s.head_width));
        if (s.page_rows < 16 || s.page_rows > 256 || (s.page_rows & (s.page_rows - 1)))
            throw ModelError("a page has 16, 32, 64, 128 or 256 rows, not " + to_string(s.page_rows));
        if (s.heads <= 0 || s.pages <= 0) throw ModelError("a cache needs heads and pages");
        if (s.heads > 65535) throw ModelError("a cache has at most 65535 heads, not " + to_string(s.heads));
        const bool eight = wsp::cache_eight(s.storage);
        const int size = wsp::cache_bytes(s.storage);
        if (memory) {
            const wsp_cache_memory& m = *memory;
            if (!m.keys || !m.values || (eight && (!m.key_scales || !m.value_scales)))
                throw wsp::InvalidArgument("a cache's memory must not be NULL");
            for (int64_t stride : {m.page_stride, m.head_stride, m.row_stride})
                if (stride < s.head_width || stride * size % 16)
                    throw wsp::InvalidArgument("a pool's strides are at least head_width and multiples of 16 bytes, not " +
                                               to_string(stride) + " elements");
            if (!wsp::aligned(m.keys) || !wsp::aligned(m.values) ||
                (eight && (!wsp::aligned(m.key_scales) || !wsp::aligned(m.value_scales))))
                throw wsp::InvalidArgument("the pools and the scale bytes must be 16-byte aligned");
        }
        int count = 0;
        wsp::cuda_check(cudaGetDeviceCount(&count), "cudaGetDeviceCount");
        if (device < 0 || device >= count) throw wsp::InvalidArgument("no CUDA device " + to_string(device));
        wsp::CurrentDevice current(device);
        std::unique_ptr<wsp_cache> c(new wsp_cache{});
        c->shape = s;
        c->device = device;
        wsp::cuda_check(cudaDeviceGetAttribute(&c->sms, cudaDevAttrMultiProcessorCount, device),
                        "cudaDeviceGetAttribute");
        if (memory) {
            c->memory = *memory;
            if (!eight) c->memory.key_scales = c->memory.value_scales = nullptr;
        } else {
            const size_t rows = (size_t)s.pages * s.heads * s.page_rows;
            for (int i = 0; i < 2; ++i) {
                c->owned[i].allocate(rows * s.head_width * size);
                if (eight) c->owned[2 + i].allocate(rows);
            }
            c->memory = {c->owned[0].get(), c->owned[1].get(), c->owned[2].get<uint8_t>(), c->owned[3].get<uint8_t>(),
                         (int64_t)s.heads * s.page_rows * s.head_width, (int64_t)s.page_rows * s.head_width,
                         s.head_width};
        }
        const wsp_cache_memory& m = c->memory;
        int shift = 0;
        while ((1 << shift) < s.page_rows) ++shift;
        c->view = {static_cast<unsigned char*>(m.keys), static_cast<unsigned char*>(m.values), m.key_scales,
                   m.value_scales, m.page_stride * size, m.head_stride * size, m.row_stride * size, s.heads, s.pages,
                   shift};
        c->maps.keys = wsp::pool_map(s, m, m.keys);
        c->maps.values = wsp::pool_map(s, m, m.values);
        wsp::prepare_cache_attend(s.storage, s.head_width);
        std::tie(c->status, c->mark) = wsp::next_status();
        *out = c.release();
    });
}

void wsp_cache_destroy(wsp_cache* cache) {
    if (!cache) return;
    guarded([&] {
        wsp::CurrentDevice current(cache->device);
        delete cache;
    });
}

int wsp_cache_get_memory(const wsp_cache* cache, wsp_cache_memory* memory) {
    return guarded([&] {
        if (!memory) throw wsp::InvalidArgument("memory must not be NULL");
        *memory = wsp::checked(cache).memory;
    });
}

int wsp_cache_append(wsp_cache* cache, const wsp_cache_batch* batch, int rows, const wsp_cache_rows* keys,
                     const wsp_cache_rows* values, void* stream) {
    return guarded([&] { wsp::copy_rows<true>(cache, batch, rows, keys, values, stream); });
}

int wsp_cache_read(wsp_cache* cache, const wsp_cache_batch* batch, int rows, const wsp_cache_rows* keys,
                   const wsp_cache_rows* values, void* stream) {
    return guarded([&] { wsp::copy_rows<false>(cache, batch, rows, keys, values, stream); });
}

int wsp_cache_attend_workspace(const wsp_cache* cache, const wsp_cache_batch* batch, int rows, int query_heads,
                               size_t* bytes) {
    return guarded([&] {
        const wsp_cache& c = wsp::checked(cache);
        if (!bytes) throw wsp::InvalidArgument("bytes must not be NULL");
        *bytes = wsp::checked_workspace(c, batch, rows, query_heads);
    });
}

int wsp_cache_attend(wsp_cache* cache, const wsp_cache_batch* batch, int rows, int query_heads,
                     const wsp_cache_rows* queries, const wsp_cache_rows* out, float* lse, float scale, int causal,
                     void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        using std::to_string;
        const wsp_cache& c = wsp::checked(cache);
        const size_t needed = wsp::checked_workspace(c, batch, rows, query_heads);
        const wsp::RowsView q = wsp::check_rows(queries, "queries", rows, query_heads, c.shape.head_width);
        const wsp::RowsView o = wsp::check_rows(out, "out", rows, query_heads, c.shape.head_width);
        if (queries->dtype != out->dtype || queries->dtype == WSP_FLOAT32)
            throw wsp::ModelError("queries and out are of one 16-bit type");
        if (!wsp::cache_eight(c.shape.storage) && queries->dtype != c.shape.storage)
            throw wsp::ModelError("queries of a 16-bit cache have its type");
        if (!(scale == scale) || scale - scale != 0.f) throw wsp::InvalidArgument("scale must be finite");
        if (reinterpret_cast<uintptr_t>(lse) & 3) throw wsp::InvalidArgument("lse must be 4-byte aligned");
        if (rows == 0 || batch->sequences == 0) return;
        if ((long long)rows * query_heads > 0x7fff0000ll)
            throw wsp::InvalidArgument("too many rows for one call: " + to_string(rows));
        if (needed && (!workspace || !wsp::aligned(workspace) || workspace_bytes < needed))
            throw wsp::InvalidArgument("the workspace must be 16-byte aligned and hold " + to_string(needed) + " bytes, not " +
                                       to_string(workspace ? workspace_bytes : 0));
        if (q.data == o.data) throw wsp::InvalidArgument("queries and out must not be one memory");
        wsp::CacheAttendArgs a{};
        a.cache = c.view;
        a.batch = wsp::batch_view(*batch);
        a.queries = q.data;
        a.q_row = q.row_bytes;
        a.q_head = q.head_bytes;
        a.out = o.data;
        a.o_row = o.row_bytes;
        a.o_head = o.head_bytes;
        a.lse = lse;
        a.rows = rows;
        a.query_heads = query_heads;
        a.group = query_heads / c.shape.heads;
        a.scale = scale;
        a.causal = causal != 0;
        a.status = c.status;
        a.mark = c.mark;
        a.workspace = static_cast<unsigned char*>(workspace);
        wsp::CurrentDevice device(c.device);
        wsp::launch_cache_attend(a, c.maps, wsp::attend_shape(c, queries->dtype, *batch),
                                 static_cast<cudaStream_t>(stream));
    });
}

int wsp_cache_check(wsp_cache* cache) {
    return guarded([&] {
        const wsp_cache& c = wsp::checked(cache);
        wsp::CurrentDevice device(c.device);
        wsp::cuda_check(cudaDeviceSynchronize(), "wsp_cache_check");
        int status = 0;
        wsp::cuda_check(cudaMemcpy(&status, c.status, sizeof status, cudaMemcpyDeviceToHost), "wsp_cache_check");
        if ((status & ~255) != c.mark) return;
        wsp::cuda_check(cudaMemset(c.status, 0, sizeof status), "wsp_cache_check");
        throw wsp::CudaFailure("a wait of the cache's attention gave up (" + std::to_string(status & 255) + ")", false);
    });
}

}  // extern "C"
