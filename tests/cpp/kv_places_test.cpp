// Where rows and tokens of a paged batch stand (csrc/kv_places.hpp), on the CPU: against a plain
// search on good batches, and inside the arrays on any values.
#include "kv_places.hpp"

#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <limits>
#include <random>
#include <vector>

using namespace mfr::kv;

namespace {

void require(bool ok, const char* what) {
    if (!ok) {
        std::printf("kv_places_test: FAILED: %s\n", what);
        std::exit(1);
    }
}

struct Held {
    std::vector<int32_t> starts, lengths, table, prefix;
    Batch b{};
};

// A batch whose arrays lie in vectors of exactly their sizes.
void point(Held& h, int rows, int sequences, int width, int log2, int pages, int prefix) {
    h.b = {rows,  sequences, sequences > 0 ? rows / sequences : 0, h.starts.empty() ? nullptr : h.starts.data(),
           h.lengths.data(), h.table.data(), width, width, log2, pages, h.prefix.data(), prefix};
}

// standing_of as a wavefront takes it, 64 starts a step.
Standing standing(const Batch& b, int32_t row) {
    return standing_of(b, row, [&](int32_t low, int32_t step, int32_t count) {
        int32_t n = 0;
        while (n < 64 && n * step < count && b.starts[low + n * step] <= row) {
            ++n;
        }
        return n;
    });
}

int32_t sequence_of(const Batch& b, int32_t row) { return standing(b, row).seq; }

void good_batches() {
    std::mt19937 gen(1);
    for (int round = 0; round < 300; ++round) {
        Held h;
        const int sequences = 1 + gen() % (round % 20 == 0 ? 9000 : round % 4 == 0 ? 200 : 9);
        const int width = 1 + gen() % 5, log2 = 4 + gen() % 3;
        std::vector<int> owner;
        h.starts = {static_cast<int32_t>(gen() % 3)};
        owner.assign(h.starts[0], -1);
        for (int s = 0; s < sequences; ++s) {
            const int n = gen() % 4;
            h.starts.push_back(h.starts.back() + n);
            owner.insert(owner.end(), n, s);
            h.lengths.push_back(gen() % ((width << log2) + 1));
        }
        owner.insert(owner.end(), gen() % 3, -1);
        for (int i = 0; i < sequences * width; ++i) {
            h.table.push_back(gen() % 40);
        }
        const int rows = static_cast<int>(owner.size());
        point(h, rows, sequences, width, log2, 40, 0);
        for (int r = 0; r < rows; ++r) {
            const Standing at = standing(h.b, r);
            require(at.seq == owner[r], "the sequence of a row");
            require(at.seq < 0 || (at.span.first == h.starts[at.seq] && at.length == h.lengths[at.seq]),
                    "its rows and its length");
        }
        for (int s = 0; s < sequences; ++s) {
            const Span span = span_of(h.b, s);
            require(span.first == h.starts[s] && span.count == h.starts[s + 1] - h.starts[s],
                    "the rows of a sequence");
            require(tokens_of(h.b, h.lengths[s]) == h.lengths[s], "the tokens of a sequence");
            require(first_place(h.lengths[s], span.count) == h.lengths[s] - span.count, "first place");
            for (int t = 0; t < width << log2; ++t) {
                require(page_of(h.b, s, t) == h.table[s * width + t / (1 << log2)], "page");
            }
        }
    }
}

void even_batches() {
    Held h;
    h.lengths = {5, 6, 7};
    h.table = {0, 1, 2};
    point(h, 12, 3, 1, 4, 3, 0);
    for (int r = 0; r < 12; ++r) {
        require(sequence_of(h.b, r) == r / 4, "the sequence of a row, four each");
    }
    require(span_of(h.b, 2).first == 8 && span_of(h.b, 2).count == 4, "four rows each");
}

// Nothing read from the arrays leads outside rows, the table or the pages.
void any_values() {
    std::mt19937 gen(2);
    const int32_t least = std::numeric_limits<int32_t>::min();
    const int32_t most = std::numeric_limits<int32_t>::max();
    const int32_t odd[] = {least, least + 1, -1, 0, 1, 2, 15, 16, 17, 1000, most - 1, most};
    for (int round = 0; round < 20000; ++round) {
        Held h;
        const int sequences = 1 + gen() % 6, width = gen() % 4, log2 = 4 + gen() % 3;
        const int rows = sequences * (gen() % 5), pages = gen() % 4;
        const auto any = [&] {
            return gen() % 2 != 0 ? odd[gen() % 12] : static_cast<int32_t>(gen());
        };
        if (gen() % 4 != 0) {
            for (int s = 0; s <= sequences; ++s) {
                h.starts.push_back(gen() % 2 != 0 ? any() : static_cast<int32_t>(gen() % (rows + 1)));
            }
        }
        for (int s = 0; s < sequences; ++s) {
            h.lengths.push_back(any());
        }
        for (int i = 0; i < sequences * width; ++i) {
            h.table.push_back(any());
        }
        const int prefix = gen() % 40;
        for (int i = 0; i < prefix; i += 1 << log2) {
            h.prefix.push_back(any());
        }
        point(h, rows, sequences, width, log2, pages, prefix);
        for (int s = 0; s < sequences; ++s) {
            const Span span = span_of(h.b, s);
            require(span.first >= 0 && span.count >= 0 && span.first + span.count <= rows,
                    "rows inside the arrays");
            require(tokens_of(h.b, h.lengths[s]) >= 0 && tokens_of(h.b, h.lengths[s]) <= width << log2,
                    "tokens inside the table");
            const int64_t first = first_place(h.lengths[s], span.count);
            for (int64_t place : {first, first + span.count - 1, int64_t{0}, int64_t{-1},
                                  static_cast<int64_t>(width) << log2, int64_t{any()},
                                  static_cast<int64_t>(tokens_of(h.b, h.lengths[s])) - 1}) {
                // The vectors hold exactly the table: a read past it would not pass a checked build.
                const int32_t page = page_of(h.b, s, place);
                require(page >= -1 && page < pages, "a page that the cache has");
                require(page < 0 || (place >= 0 && place < width << log2), "no page past the table");
            }
        }
        for (int r = 0; r < rows; ++r) {
            const int32_t s = sequence_of(h.b, r);
            require(s >= -1 && s < sequences, "a sequence that there is");
            require(s < 0 || (r >= span_of(h.b, s).first &&
                              r - span_of(h.b, s).first < span_of(h.b, s).count),
                    "a row of its sequence");
        }
        for (int t = 0; t < prefix; ++t) {
            const int32_t page = page_checked(h.b, h.prefix[t >> log2]);
            require(page >= -1 && page < pages, "a prefix page that the cache has");
        }
    }
}

} // namespace

int main() {
    good_batches();
    even_batches();
    any_values();
    std::printf("kv_places_test passed\n");
    return 0;
}
