/*
 * wsp_cache.h -- the C ABI of a paged key/value cache on a B200: new rows
 * appended (and quantised, where the cache holds 8 bits), rows read back, and
 * the attention of new rows over the pages.  Same conventions as
 * wsp_decoder.h for status codes and wsp_last_error.
 *
 * The decoder of wsp_decoder.h keeps contiguous caches for windows that step
 * together.  A host that serves windows standing at their own tokens -- one
 * brings a prompt of previous text, the next a single token, all attend over
 * what they hold -- keeps their rows in pages and runs the two cache ops of
 * the reference's Net interface here, for every window of a batch in one
 * launch: appendLinear's cache write (Lib/WhisperEACP/Net/Net.h:110-171) is
 * wsp_cache_append, the attention over a Cache is wsp_cache_attend.
 *
 * All data pointers below are device pointers on the cache's device.  The
 * calls queue their work on `stream` (a cudaStream_t; NULL: the legacy
 * stream) and return without waiting; they allocate nothing, keep nothing
 * between calls and may be captured into a CUDA graph (what the arrays hold
 * is read when the work runs).  Calls on several streams or host threads may
 * use one cache at once, each wsp_cache_attend with a workspace of its own;
 * reading rows while another stream writes them is the caller's to order.
 * The current device is left as it was.
 */
#ifndef WSP_CACHE_H
#define WSP_CACHE_H

#include "wsp_decoder.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * What a held element is.  The 8-bit forms keep, for each row of each head,
 * one scale byte b beside the `head_width` values: a value stands for itself
 * times 2^(b - 127), b = 0 for zero rows of untouched memory, b = 255 for a
 * row that held an infinity or NaN (it reads back as NaN).  b is the
 * smallest that keeps the row's largest magnitude within 448 (E4M3) or 127
 * (INT8); the division by a power of two is exact, so a value is rounded
 * once, to nearest even.
 */
enum {
    WSP_CACHE_FLOAT16 = 1,  /* = WSP_FLOAT16  */
    WSP_CACHE_BFLOAT16 = 2, /* = WSP_BFLOAT16 */
    WSP_CACHE_E4M3 = 3,     /* 8-bit float, 4 exponent bits, 3 mantissa bits */
    WSP_CACHE_INT8 = 4
};

typedef struct wsp_cache_shape {
    int32_t heads;      /* key/value heads                                  */
    int32_t head_width; /* 64 or 128                                        */
    int32_t page_rows;  /* rows of a page: 16, 32, 64, 128 or 256           */
    int32_t pages;
    int32_t storage;    /* WSP_CACHE_*                                      */
} wsp_cache_shape;

/*
 * The two pools, [pages, heads, page_rows, head_width] in any order of the
 * first three (strides in elements, at least head_width and multiples of 16
 * bytes; the base 16-byte aligned; distinct rows must not overlap), and the
 * scale bytes [pages, heads, page_rows], contiguous and 16-byte aligned (8-bit
 * storage only).
 */
typedef struct wsp_cache_memory {
    void* keys;
    void* values;
    uint8_t* key_scales;
    uint8_t* value_scales;
    int64_t page_stride;
    int64_t head_stride;
    int64_t row_stride;
} wsp_cache_memory;

typedef struct wsp_cache wsp_cache;

/*
 * A cache over the caller's memory, or, with memory NULL, over zeroed memory
 * of its own ([pages][heads][page_rows][head_width]) that
 * wsp_cache_destroy frees.
 */
int wsp_cache_create(const wsp_cache_shape* shape, int device, const wsp_cache_memory* memory, wsp_cache** out);
void wsp_cache_destroy(wsp_cache* cache);
int wsp_cache_get_memory(const wsp_cache* cache, wsp_cache_memory* memory);

/*
 * The sequences of a call.  Sequence s holds lengths[s] rows, the new ones
 * counted; row p of them stands in page table[s * table_stride + p /
 * page_rows], row p % page_rows.  Its new rows are rows starts[s] ..
 * starts[s + 1] - 1 of the call's row arrays and its LAST rows: row i of n
 * stands at position lengths[s] - n + i.  n may be 0, and so may a length.
 * starts must not decrease, starts[0] may be any row, and rows before
 * starts[0] or from starts[sequences] on belong to no sequence and are left
 * alone.  A page id outside the pool, and a position outside the table, is
 * no page: appending there does nothing, and its rows read as zeros.  In the
 * attention rows of such pages take part as zeros, positions outside the
 * table do not take part, and a sequence whose rows lie outside the call's
 * arrays has none.  table_columns * page_rows is at most 2^31 - 256.  max_rows
 * is a bound of n, the same or larger; it chooses
 * kernels only.
 */
typedef struct wsp_cache_batch {
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* starts;
    int64_t table_stride;
    int32_t table_columns;
    int32_t sequences;
    int32_t max_rows;
} wsp_cache_batch;

/* Row arrays [rows, heads, head_width]: strides in elements, multiples of 16
   bytes, the base 16-byte aligned. */
typedef struct wsp_cache_rows {
    void* data;
    int64_t row_stride;
    int64_t head_stride;
    int32_t dtype; /* a wsp_dtype */
} wsp_cache_rows;

/*
 * Writes the new rows of keys and values (any wsp_dtype) into the pages,
 * rounded once to the storage.  Two sequences of a call that name one place
 * race on it.
 */
int wsp_cache_append(wsp_cache* cache, const wsp_cache_batch* batch, int rows, const wsp_cache_rows* keys,
                     const wsp_cache_rows* values, void* stream);

/*
 * Reads the sequences' last rows back, as appended ones lie: the values they
 * stand for, rounded once to the row arrays' type (any wsp_dtype).
 */
int wsp_cache_read(wsp_cache* cache, const wsp_cache_batch* batch, int rows, const wsp_cache_rows* keys,
                   const wsp_cache_rows* values, void* stream);

/*
 * Attention of the new rows over the sequences' held rows, these included
 * (append first): out = softmax(scale q . k) v over the keys at positions up
 * to the row's own (causal) or over every held row.  queries and out are
 * [rows, query_heads, head_width] of one 16-bit type, which a 16-bit cache
 * shares; query_heads is a multiple of the cache's heads, and query head h
 * reads head h / (query_heads / heads); out overlaps neither queries nor the
 * pools.  lse (NULL: none), [rows,
 * query_heads] contiguous, gets the natural logarithm of the sum of
 * exponentials.  A row that sees no key gets zeros and -infinity.  Keys and
 * values a row does not see cannot change its result, whatever they hold.
 * Scores, softmax and sums are kept in fp32.  A probability (over 8 bits, times
 * its value's scale) meets its value rounded to 16 bits or to two of them: by
 * 2^-8 (bf16) or 2^-11 (fp16, and over 8 bits) of itself at most, fp16 by 2^-32
 * of the row's largest where that is more.  A row whose result is not finite, or
 * whose numbers the 16 bits do not reach, is computed again alone in fp32, at
 * up to some hundred times the cost.
 *
 * workspace: wsp_cache_attend_workspace bytes, 16-byte aligned, of any
 * content; two calls that may overlap on the device need two.
 */
int wsp_cache_attend(wsp_cache* cache, const wsp_cache_batch* batch, int rows, int query_heads,
                     const wsp_cache_rows* queries, const wsp_cache_rows* out, float* lse, float scale, int causal,
                     void* workspace, size_t workspace_bytes, void* stream);
int wsp_cache_attend_workspace(const wsp_cache* cache, const wsp_cache_batch* batch, int rows, int query_heads,
                               size_t* bytes);

/*
 * Waits for the device's queued work and reports a wait inside a kernel that
 * gave up after 2 s (WSP_CUDA_ERROR; none should).  The attention's calls do
 * not say so themselves: rows that such a wait held up are computed again
 * without waits, slowly.
 */
int wsp_cache_check(wsp_cache* cache);

#ifdef __cplusplus
}
#endif

#endif
