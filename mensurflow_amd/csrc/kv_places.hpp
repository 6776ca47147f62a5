// Where the rows of a step stand (mfr_kv_batch): which sequence a row belongs to, which tokens it has,
// which page holds a token. Everything read from device memory passes these functions, and none of
// what they give leads outside the arrays. No HIP header, so that the CPU tests run them on any values.
#pragma once

#include <cstdint>

#if defined(__HIPCC__)
#define MFR_KV_BOTH __host__ __device__ inline
#else
#define MFR_KV_BOTH inline
#endif

namespace mfr::kv {

struct Batch {
    int32_t rows, sequences;
    int32_t each;               // rows of every sequence, where starts is null
    const int32_t* starts;
    const int32_t* lengths;
    const int32_t* table;
    int64_t table_rs;
    int32_t width;              // entries of a table's row
    int32_t page_log2;          // tokens of a page
    int32_t pages;              // of the cache
    const int32_t* prefix_pages;
    int32_t prefix;             // tokens
};

struct Span {
    int32_t first, count;
};

MFR_KV_BOTH int32_t within(int32_t v, int32_t low, int32_t high) {
    return v < low ? low : v > high ? high : v;
}

MFR_KV_BOTH int32_t capacity_of(const Batch& b) { return b.width << b.page_log2; }

// The rows of sequence s, inside 0 .. rows.
MFR_KV_BOTH Span span_of(const Batch& b, int32_t s) {
    if (b.starts == nullptr) {
        return {s * b.each, b.each};
    }
    const int32_t first = within(b.starts[s], 0, b.rows);
    return {first, within(b.starts[s + 1], first, b.rows) - first};
}

// The tokens of a sequence that its table has room for.
MFR_KV_BOTH int32_t tokens_of(const Batch& b, int32_t length) {
    return within(length, 0, capacity_of(b));
}

// The place of a sequence's first row of `count`: below 0, or past the table, it has none.
MFR_KV_BOTH int64_t first_place(int32_t length, int32_t count) {
    return static_cast<int64_t>(length) - count;
}

// Where a row stands: its sequence (-1: none), that one's rows, and its length as it is in memory.
struct Standing {
    int32_t seq;
    Span span;
    int32_t length;
};

// `leading(low, step, count)`: of the starts low, low + step, low + 2 step, ... in front of low + count, 64 at
// most, how many are at or before the row until the first that is not (a wavefront's ballot).
template <typename Leading>
MFR_KV_BOTH Standing standing_of(const Batch& b, int32_t row, Leading leading) {
    int32_t low = 0;
    if (b.starts == nullptr) {
        low = row / b.each;
    } else {
        // The last sequence that starts at or before the row (empty ones of the same start come first).
        int32_t count = b.sequences;
        while (count > 1) {
            const int32_t step = (count - 1) / 64 + 1;
            const int32_t before = leading(low, step, count);
            const int32_t skip = before > 1 ? (before - 1) * step : 0;
            low += skip;
            count = step < count - skip ? step : count - skip;
        }
    }
    const int32_t length = b.lengths[low]; // under way with the starts
    const Span span = span_of(b, low);
    const bool here = row >= span.first && row - span.first < span.count;
    return {here ? low : -1, span, length};
}

// A page number that the cache has, or -1.
MFR_KV_BOTH int32_t page_checked(const Batch& b, int32_t page) {
    return page >= 0 && page < b.pages ? page : -1;
}

// The page of token `place` of sequence s, -1 if it has none.
MFR_KV_BOTH int32_t page_of(const Batch& b, int32_t s, int64_t place) {
    if (place < 0 || place >= capacity_of(b)) {
        return -1;
    }
    return page_checked(b, b.table[s * b.table_rs + (place >> b.page_log2)]);
}

} // namespace mfr::kv
