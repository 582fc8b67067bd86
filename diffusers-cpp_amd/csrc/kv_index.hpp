// kv_index.hpp -- which rows, places and pages belong together in a call on a paged
// cache, in plain C++ that the kernels (kv_cache.hip, kv_attention.hip) and a host
// program can build.  Nothing here trusts the device arrays: whatever they hold, rows
// stay within [0, rows), places within the table and pages within the pool.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define DT_KV_FN __host__ __device__ __forceinline__
#else
#define DT_KV_FN inline
#endif

namespace dit {
namespace kv {

struct Seqs {
    const int32_t* table;
    int64_t table_stride;
    const int32_t* seq_start;
    const int32_t* past;
    int32_t table_pages, seqs, rows;
    int32_t pages, page_log2;  // of the pool
};

DT_KV_FN int clamped(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// Where sequence b's rows start (b = seqs: where the last one's end).
DT_KV_FN int start_of(const Seqs& s, int b) { return clamped(s.seq_start[b], 0, s.rows); }

struct Seq {
    int row, n;     // first row, rows
    int past, len;  // tokens before, and with the rows (places past the table's end are none)
    DT_KV_FN Seq(const Seqs& s, int b) : Seq(s, s.seq_start[b], s.seq_start[b + 1], s.past[b]) {}
    DT_KV_FN Seq(const Seqs& s, int start, int end, int before) {
        row = clamped(start, 0, s.rows);
        end = clamped(end, 0, s.rows);
        n = end > row ? end - row : 0;
        past = clamped(before, 0, 1 << 30);
        const int64_t cap = (int64_t)s.table_pages << s.page_log2;
        len = past + n < cap ? past + n : (int)cap;
    }
};

// The page that holds place t of sequence b, or -1.
DT_KV_FN int page_of(const Seqs& s, int b, int t) {
    const int j = t >> s.page_log2;
    if (j >= s.table_pages) return -1;
    const int p = s.table[b * s.table_stride + j];
    return (uint32_t)p < (uint32_t)s.pages ? p : -1;
}

// The pages that are written are numbered without knowing how many each sequence touches: b's
// numbers begin here, n rows touch at most n / page + 2 pages, and there are items() in all.
DT_KV_FN int64_t first_item(const Seqs& s, int start, int b) { return (int64_t)(start >> s.page_log2) + 2 * b; }
DT_KV_FN int64_t items(const Seqs& s) { return first_item(s, s.rows, s.seqs); }

// Item `item` of sequence b: which rows of its page (page_of(begin)) are new.  False: none.
struct PageItem {
    int begin, first, last;  // begin: the place of the page's row 0; new rows [first, last)
};
DT_KV_FN bool page_item(const Seqs& s, const Seq& q, int b, int64_t item, PageItem* out) {
    const int64_t j = item - first_item(s, q.row, b) + (q.past >> s.page_log2), begin = j * (1 << s.page_log2);
    if (j < 0 || q.n == 0 || q.len <= q.past || begin >= q.len) return false;
    const int size = 1 << s.page_log2;
    out->begin = (int)begin;
    out->first = q.past > begin ? (int)(q.past - begin) : 0;
    out->last = q.len - begin < size ? (int)(q.len - begin) : size;
    return out->first < out->last;
}

}  // namespace kv
}  // namespace dit
