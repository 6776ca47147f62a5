// How attention over a paged cache is cut over workgroups (csrc/kv_work.hpp), on the CPU: every unit is
// taken once, items are finished once, and their parts are read where they were written.
#include "kv_work.hpp"

#include <cstdio>
#include <cstdlib>
#include <limits>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>

using namespace mfr::kv;

namespace {

void require(bool ok, const char* what) {
    if (!ok) {
        std::printf("kv_work_test: FAILED: %s\n", what);
        std::exit(1);
    }
}

using Key = std::tuple<int, int, int>; // sequence, head, tile

struct Found {
    int64_t total = 0, chunk = 0, base = 0;
    int seq = -1;
};

// What a workgroup finds for a unit of the list (the search of the kernels, one sequence at a time).
Found find(const Work& w, int groups, int64_t target_of(int64_t, int64_t, int64_t), int64_t index) {
    Found f;
    for (int s = 0; s < sequences_of(w); ++s) {
        f.total += shape_of(w, s).count;
    }
    f.chunk = chunk_of(f.total, groups);
    const int64_t target = target_of(f.total, f.chunk, index);
    if (target < 0) {
        return f;
    }
    for (int s = 0; s < sequences_of(w); ++s) {
        const int64_t count = shape_of(w, s).count;
        if (target < f.base + count) {
            f.seq = s;
            return f;
        }
        f.base += count;
    }
    require(false, "a unit that no sequence has");
    return f;
}

void walk(const Work& w, int groups) {
    std::map<Key, std::set<int>> taken;
    std::map<int64_t, Key> parts;
    std::map<Key, std::vector<int64_t>> written;
    std::set<Key> finished;
    for (int64_t g = 0; g < groups; ++g) {
        const Found f = find(w, groups, [](int64_t total, int64_t chunk, int64_t i) {
            return i * chunk < total ? i * chunk : int64_t{-1};
        }, g);
        if (f.seq < 0) {
            continue;
        }
        const int64_t end = std::min(g * f.chunk + f.chunk, f.total);
        int seq = f.seq;
        int64_t base = f.base;
        Shape shape = shape_of(w, seq);
        for (int64_t at = g * f.chunk; at < end;) {
            while (at >= base + shape.count) {
                base += shape.count;
                require(++seq < sequences_of(w), "a chunk past the last sequence");
                shape = shape_of(w, seq);
            }
            const Item item = item_of(shape, base, at);
            const int64_t item_end = item.begin + shape.units;
            const int units = static_cast<int>(std::min(item_end, end) - at);
            require(units > 0 && item.head < w.heads && item.tile < shape.tiles, "an item's place");
            const Key key{seq, item.head, item.tile};
            for (int u = 0; u < units; ++u) {
                require(taken[key].insert(item.first + u).second, "a unit taken twice");
            }
            if (item.first == 0 && units == shape.units) {
                require(finished.insert(key).second, "an item finished twice");
            } else {
                const int64_t part = part_of(g, f.chunk, item.begin);
                require(part >= 0 && part < 2 * groups, "a part's place");
                require(parts.emplace(part, key).second, "two parts in one place");
                written[key].push_back(part);
            }
            at += units;
        }
    }
    for (int64_t g = 0; g < groups; ++g) {
        const Found f = find(w, groups, [](int64_t total, int64_t chunk, int64_t i) {
            return (i + 1) * chunk < total ? (i + 1) * chunk - 1 : int64_t{-1};
        }, g);
        if (f.seq < 0) {
            continue;
        }
        const Shape shape = shape_of(w, f.seq);
        const int64_t edge = (g + 1) * f.chunk;
        const Item item = item_of(shape, f.base, edge - 1);
        const int64_t end = item.begin + shape.units;
        if (item.begin < g * f.chunk || end <= edge) {
            continue;
        }
        const Key key{f.seq, item.head, item.tile};
        std::vector<int64_t> read;
        for (int64_t i = g; i <= (end - 1) / f.chunk; ++i) {
            read.push_back(part_of(i, f.chunk, item.begin));
        }
        require(read == written[key], "the parts of an item");
        require(finished.insert(key).second, "an item joined twice");
    }
    for (int s = 0; s < sequences_of(w); ++s) {
        const Shape shape = shape_of(w, s);
        for (int h = 0; h < w.heads; ++h) {
            for (int t = 0; t < shape.tiles; ++t) {
                const Key key{s, h, t};
                require(static_cast<int>(taken[key].size()) == shape.units, "a unit left out");
                require(finished.count(key) == 1, "an item left out");
            }
        }
    }
}

void cuts() {
    std::mt19937 gen(3);
    for (int round = 0; round < 3000; ++round) {
        const int sequences = 1 + gen() % 8, width = 1 + gen() % 12;
        std::vector<int32_t> starts{static_cast<int32_t>(gen() % 2)}, lengths;
        for (int s = 0; s < sequences; ++s) {
            starts.push_back(starts.back() + (gen() % 3 == 0 ? 0 : gen() % 40));
            lengths.push_back(gen() % 4 == 0 ? 0 : gen() % (16 * width + 20));
        }
        Work w{};
        w.batch = {starts.back() + 1, sequences, 0,     starts.data(), lengths.data(), nullptr, 0,
                   width,             4,         100,   nullptr,       static_cast<int32_t>(gen() % 200)};
        w.heads = 1 + gen() % 3;
        w.group = 1 + gen() % 5;
        const int32_t rows_of_forms[] = {16, 32, 128};
        w.tile_rows = rows_of_forms[gen() % 3];
        w.unit = gen() % 2 != 0 ? 64 : 16;
        w.shared = gen() % 4 == 0;
        walk(w, 1 + gen() % 40);
    }
}

void rows_see() {
    Work w{};
    const int32_t starts[] = {0, 5}, lengths[] = {7};
    w.batch = {5, 1, 0, starts, lengths, nullptr, 0, 1, 4, 1, nullptr, 0};
    w.heads = w.group = 1;
    w.tile_rows = 16;
    w.unit = 16;
    Shape p = shape_of(w, 0);
    for (int i = 0; i < 5; ++i) {
        require(seen_by(p, i, true) == 3 + i && seen_by(p, i, false) == 7, "tokens that a row sees");
    }
    const int32_t odd[] = {3, -4, 100, std::numeric_limits<int32_t>::min(),
                           std::numeric_limits<int32_t>::max()};
    for (int32_t length : odd) {
        w.batch.lengths = &length;
        p = shape_of(w, 0);
        int32_t before = 0;
        for (int i = 0; i < 5; ++i) {
            const int32_t seen = seen_by(p, i, true);
            require(seen >= before && seen <= p.tokens && p.tokens <= 16, "tokens inside the table");
            before = seen;
        }
    }
}

} // namespace

int main() {
    cuts();
    rows_see();
    std::printf("kv_work_test passed\n");
    return 0;
}
