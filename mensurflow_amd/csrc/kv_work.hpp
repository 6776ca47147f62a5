// How the work of one attention launch over a paged cache is cut over its workgroups. No HIP header, so
// that the CPU tests walk it whole.
//
// The work of a sequence is a list of items, one for each head of the cache and tile of `tile_rows` rows
// (query, query head of that head), and an item a list of units, `unit` tokens of the keys; an item
// without tokens has one empty unit, so that its rows are written. All units in a row, sequence by
// sequence, head by head, tile by tile, are cut into equal chunks, one a workgroup, by the lengths that
// the kernel finds: a chunk may end inside an item, or hold many. An item inside one chunk is finished
// there. Of others every chunk writes a part: to the first of its two places if the item began before
// the chunk, to the second if it began in it (and ends behind it). The chunk where it began names the
// workgroup that joins the parts, in order.
#pragma once

#include "kv_places.hpp"

namespace mfr::kv {

struct Work {
    Batch batch;
    int32_t heads, group;
    int32_t tile_rows;
    int32_t unit;   // tokens
    int32_t shared; // the prefix of all rows instead of the sequences' own tokens
};

// A sequence (or, for the prefix, all rows as one).
struct Shape {
    Span span;
    int32_t tokens;
    int64_t first_place;
    int32_t tiles;  // of rows
    int32_t units;  // of an item
    int64_t count;  // units in all
};

MFR_KV_BOTH int32_t sequences_of(const Work& w) { return w.shared != 0 ? 1 : w.batch.sequences; }

MFR_KV_BOTH Shape shape_of(const Work& w, int32_t s) {
    Shape p;
    if (w.shared != 0) {
        p.span = {0, w.batch.rows};
        p.tokens = w.batch.prefix;
        p.first_place = 0;
    } else {
        const int32_t length = w.batch.lengths[s]; // under way with the starts
        p.span = span_of(w.batch, s);
        p.tokens = tokens_of(w.batch, length);
        p.first_place = first_place(length, p.span.count);
    }
    p.tiles = (p.span.count * w.group + w.tile_rows - 1) / w.tile_rows;
    p.units = p.tokens > 0 ? (p.tokens - 1) / w.unit + 1 : 1;
    p.count = static_cast<int64_t>(p.tiles) * p.units * w.heads;
    return p;
}

MFR_KV_BOTH int64_t quotient(int64_t a, int64_t b) { // a not below 0, b above; most often of 32 bits
    return ((a | b) >> 32) == 0 ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}

// The chunk that each of `groups` workgroups takes.
MFR_KV_BOTH int64_t chunk_of(int64_t total, int32_t groups) {
    return total > 0 ? quotient(total - 1, groups) + 1 : 1;
}

// An item from the place of one of its units in the list.
struct Item {
    int32_t head, tile;
    int32_t first;   // the unit, from the item's start
    int64_t begin;   // the item's place in the list
};

MFR_KV_BOTH Item item_of(const Shape& p, int64_t base, int64_t at) {
    const int64_t off = at - base;
    const int64_t item = quotient(off, p.units);
    Item i;
    i.first = static_cast<int32_t>(off - item * p.units);
    i.head = static_cast<int32_t>(quotient(item, p.tiles));
    i.tile = static_cast<int32_t>(item - static_cast<int64_t>(i.head) * p.tiles);
    i.begin = at - i.first;
    return i;
}

// The place of a chunk's part of an item that began at `begin`.
MFR_KV_BOTH int64_t part_of(int64_t chunk_index, int64_t chunk, int64_t begin) {
    return 2 * chunk_index + (begin >= chunk_index * chunk ? 1 : 0);
}

// The tokens of the sequence that row `i` of its own sees.
MFR_KV_BOTH int32_t seen_by(const Shape& p, int32_t i, bool causal) {
    if (!causal) {
        return p.tokens;
    }
    const int64_t place = p.first_place + i;
    return place < 0 ? 0 : place + 1 < p.tokens ? static_cast<int32_t>(place + 1) : p.tokens;
}

} // namespace mfr::kv
