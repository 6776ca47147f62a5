// mfr_f8gemm: checks, and the choice between the tiles (f8gemm_kernel.hpp), the depth in ranges
// (f8gemm_finish.hpp) and the form for few rows (f8gemm_few.hpp).
#include "f8gemm_few.hpp"
#include "f8gemm_finish.hpp"
#include "f8gemm_ring.hpp"

#include <algorithm>
#include <limits>
#include <utility>

namespace {

using mfr::f8::blocks_of;
using mfr::f8gemm::Params;

constexpr int64_t kMostOutputs = int64_t{1} << 44;

// The descriptor's checks (of shapes, layouts and pointers: no device is needed).
Params checked(const mfr_f8gemm_desc* desc) {
    using mfr::require;
    require(desc != nullptr, "f8gemm: null descriptor");
    const mfr_f8gemm_desc& d = *desc;
    require(d.m >= 0 && d.n >= 0 && d.k >= 0, "f8gemm: negative dimension");
    require(d.act >= MFR_ACT_NONE && d.act <= MFR_ACT_SILU, "f8gemm: unknown activation");
    const bool gated = d.up.values != nullptr;
    require(!gated || (d.c0 == nullptr && d.bias == nullptr),
            "f8gemm: the gated form takes no c0 and no bias");
    require(d.beta == 0.0f || d.c0 != nullptr, "f8gemm: beta requires c0");
    Params p{};
    p.m = d.m, p.n = d.n, p.k = d.k;
    p.a = mfr::f8::checked(d.a, d.m, d.k, 1, false, "f8gemm", "a");
    p.b = mfr::f8::checked(d.b, d.n, d.k, 128, false, "f8gemm", "b");
    if (gated) {
        p.up = mfr::f8::checked(d.up, d.n, d.k, 128, false, "f8gemm", "up");
    }
    if (d.out_f8.values != nullptr) {
        p.q = mfr::f8::checked(d.out_f8, d.m, d.n, 1, true, "f8gemm", "out_f8");
    }
    if (d.m == 0 || d.n == 0) {
        return p;
    }
    const bool add = d.c0 != nullptr && d.beta != 0.0f;
    require(d.c != nullptr || d.out_f8.values != nullptr,
            "f8gemm: neither c nor out_f8 is given");
    require(d.m <= kMostOutputs / d.n, "f8gemm: problem too large");
    require(d.c == nullptr || d.c_rs >= d.n, "f8gemm: c has rows that overlap");
    require(!add || d.c0_rs >= d.n, "f8gemm: c0 has rows that overlap");
    require(!add || d.c0 != d.c || d.c0_rs == d.c_rs,
            "f8gemm: c0 in place of c needs its row stride");
    p.c = d.c, p.c_rs = d.c_rs;
    p.c0 = add ? d.c0 : nullptr, p.c0_rs = d.c0_rs;
    p.bias = d.bias;
    p.beta = d.beta, p.act = d.act;
    return p;
}

// ---- which form ---------------------------------------------------------------------------------
//
// The times of a call in microseconds, by what was measured on an MI355X (256 CUs) over m = 1 ..
// 8192, n = 1024 .. 16384 and k = 1024 .. 8192: a fixed part, and one per block of the depth that a
// workgroup or wavefront walks, by how many workgroups a CU has. The least of them is taken.

enum class Form : int32_t {
    kFew16 = MFR_F8_FEW_16,
    kFew32 = MFR_F8_FEW_32,
    kFew32Wide = MFR_F8_FEW_32_WIDE,
    kFew64 = MFR_F8_FEW_64,
    kRing32 = MFR_F8_RING_32,
    kRing32Wide = MFR_F8_RING_32_WIDE,
    kRing64 = MFR_F8_RING_64,
    kRing64Pair = MFR_F8_RING_64_PAIR,
    kRing128 = MFR_F8_RING_128,
    kTile64 = MFR_F8_TILE_64,
    kTile128 = MFR_F8_TILE_128
};

// A workgroup's rows and columns, the wavefronts that share the depth, and a wavefront's time per
// block with one workgroup per CU. Measured, k = 4096 (32 blocks): 16 x 4096 5.8 us and 16 x 16384
// 18.7; 32 x 4096 8.7; 32 x 16384 18.4 wide (28.5 narrow); 128 x 4096 15.5 in the last form. Gated:
// 1 x 10240 17.6, 32 x 4096 11.5, 64 x 4096 16.6.
struct Few {
    Form form;
    int64_t rows, cols, waves;
    double block;
};
constexpr double kFewFixed = 2.6;
constexpr Few kFew[] = {{Form::kFew16, 16, 16, 8, 1.0},
                        {Form::kFew32, 32, 16, 8, 1.45},
                        {Form::kFew32Wide, 32, 32, 4, 1.0},
                        {Form::kFew64, 64, 32, 8, 3.15}};
constexpr Few kFewGated[] = {{Form::kFew16, 16, 16, 8, 1.5},
                             {Form::kFew32, 32, 16, 8, 2.3},
                             {Form::kFew64, 64, 16, 4, 1.7}};

// A ring's rows and columns, the slices of a turn, how many share a CU, what a workgroup takes
// besides its turns, and the time of a turn when every CU has them all, or one alone. Measured, a
// round of every CU at k = 1024, 4096, 8192: 32 x 32 4.3, 7.9, 13.4 us; 32 x 64 5.4, 9.8, 16.3; 64 x 64
// 7.6, 14.6, 24.5, two on a CU 9.5, 23, 43; gated, k = 4096: 32 x 32 12, 64 x 32 15.5, two 23.5. The
// one of 128 columns makes 8 bits by itself: 8-bit output of 32 x 16384 x 4096 17.4 us (18.9 with a
// second launch), of the gated 32 x 14336 x 4096 28.6 (30.2), of few rows without a workspace, 1 x 4096
// x 4096, 16.7 (64-row tiles 22.1), gated 1 x 10240 x 4096 26.5 (33.5).
struct Ring {
    Form form;
    int64_t rows, cols, slices, at_once;
    double start, full, alone;
};
constexpr double kRingFixed = 2.0;
constexpr int64_t kMostRingThreads = 768;
constexpr Ring kRings[] = {{Form::kRing32, 32, 32, 8, 1, 3.0, 1.28, 1.28},
                           {Form::kRing32Wide, 32, 64, 4, 1, 3.7, 0.78, 0.78},
                           {Form::kRing64, 64, 64, 3, 1, 4.5, 0.88, 0.88},
                           {Form::kRing64Pair, 64, 64, 2, 2, 3.0, 1.26, 1.0},
                           {Form::kRing128, 32, 128, 2, 1, 3.7, 0.75, 0.75}};
constexpr Ring kRingsGated[] = {{Form::kRing32, 32, 32, 4, 1, 3.7, 1.04, 1.04},
                                {Form::kRing64, 64, 32, 4, 1, 3.5, 1.5, 1.5},
                                {Form::kRing64Pair, 64, 32, 2, 2, 3.0, 1.28, 0.95},
                                {Form::kRing128, 32, 128, 2, 1, 3.7, 1.42, 1.42}};

// The rate at which a ring's weights come from memory at most (32 x 16384 x 4096).
constexpr double kBytesPerUs = 4.6e6;

// A tile's workgroups per CU at once, what a round of them takes besides its blocks (the first
// loads and the outputs, 32 MB a round of the larger tile), and the time of a block when every CU
// has them all, or one alone on few CUs. Measured, n = 8192, every CU full: 64 x 128 tiles, one round,
// k = 1024 16.3 us, 2304 27.8; 128 x 128 25.1, 45.4 and 76 at 4096, two rounds of 1024 48.6; gated
// 64 x 128 37 us a round of k = 4096, 128 x 128 59.
struct Tile {
    Form form;
    int64_t rows, at_once;
    double start, full, alone;
};
constexpr double kTileFixed = 2.5;
constexpr Tile kTiles[] = {{Form::kTile64, 64, 2, 4.0, 1.2, 0.55},
                           {Form::kTile128, 128, 2, 6.3, 1.95, 0.8}};
constexpr Tile kTilesGated[] = {{Form::kTile64, 64, 1, 3.8, 1.1, 0.92},
                                {Form::kTile128, 128, 1, 6.0, 1.75, 1.29}};
constexpr int64_t kTileCols = 128;

// The second launch of a depth in ranges and the memory it reads; the second launch of few rows
// with an 8-bit output.
constexpr double kFinishFixed = 3.0;
constexpr double kFinishBytesPerUs = 4e6;
constexpr double kConvertFixed = 2.6;
constexpr int64_t kMostPartialBytes = int64_t{256} << 20;

// Up to here a call that is given c and an 8-bit output never takes the workspace, so that a captured
// one runs as an eager one does, in the same order of summation. What that costs: the depth in ranges
// would be faster for one such call in nine, by 8 % in the mean and up to 1.4 times (gated 35 x 1510 x
// 8992, priced at 18.3 us in ranges and 25.9 without).
constexpr int64_t kAlikeRows = 64;

struct Plan {
    Form form = Form::kTile64;
    int64_t splits = 1;
    double time = std::numeric_limits<double>::infinity();
    int64_t workspace = 0; // bytes
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether the form leaves an 8-bit output to a second launch: several workgroups hold a block.
bool converts(Form f) {
    return f != Form::kRing128 && f != Form::kTile64 && f != Form::kTile128;
}

Plan choose(const Params& p, int64_t cus, bool workspace) {
    const bool gated = p.up.values != nullptr;
    const int64_t blocks = blocks_of(p.k);
    Plan best;
    const auto offer = [&](Form form, int64_t splits, double time, int64_t bytes) {
        if (time < best.time && (bytes == 0 || (workspace && bytes <= kMostPartialBytes))) {
            best = {form, splits, time, bytes};
        }
    };
    const auto few = [&](const Few& f) {
        // The CUs' share of the workgroups: the memory sees the mean, a CU's wavefronts the most;
        // between them where small workgroups mingle.
        const int64_t groups = ceil_div(p.m, f.rows) * ceil_div(p.n, f.cols);
        const double most = static_cast<double>(ceil_div(groups, cus));
        const double mean = std::max(1.0, static_cast<double>(groups) / static_cast<double>(cus));
        double time = kFewFixed + static_cast<double>(ceil_div(blocks, f.waves)) * f.block *
                                      (f.rows < 64 ? (most + mean) / 2.0 : most);
        int64_t bytes = 0;
        if (p.q.values != nullptr) {
            time += kConvertFixed;
            bytes = p.c != nullptr ? 0 : 4 * p.m * p.n;
        }
        if (ceil_div(p.m, f.rows) < 65536 && mfr::one_launch(groups, 64 * f.waves)) {
            offer(f.form, 1, time, bytes);
        }
    };
    const double weights = (gated ? 2.0 : 1.0) * static_cast<double>(p.n) * static_cast<double>(p.k);
    const auto ring = [&](const Ring& r) {
        const int64_t groups = ceil_div(p.m, r.rows) * ceil_div(p.n, r.cols);
        const int64_t slots = cus * r.at_once;
        const int64_t rest = groups % slots;
        const double turns = static_cast<double>(ceil_div(blocks, r.slices));
        double time = static_cast<double>(groups / slots) * (r.start + turns * r.full);
        if (rest > 0) {
            time += r.start + turns * (rest > cus ? r.full : r.alone);
        }
        time = kRingFixed + std::max(time, weights / kBytesPerUs);
        int64_t bytes = 0;
        if (p.q.values != nullptr && converts(r.form)) {
            time += kConvertFixed;
            bytes = p.c != nullptr ? 0 : 4 * p.m * p.n;
        }
        if (mfr::one_launch(groups, kMostRingThreads)) {
            offer(r.form, 1, time, bytes);
        }
    };
    const bool alike = p.m <= kAlikeRows && p.c != nullptr && p.q.values != nullptr;
    const int64_t most_splits = alike ? 1 : std::clamp(blocks, int64_t{1}, int64_t{8});
    const auto tiles = [&](const Tile& t) {
        for (int64_t splits = 1; splits <= most_splits; splits *= 2) {
            const int64_t groups = ceil_div(p.m, t.rows) * ceil_div(p.n, kTileCols) * splits;
            const int64_t slots = cus * t.at_once;
            const int64_t rest = groups % slots;
            const double walked = static_cast<double>(ceil_div(blocks, splits));
            // The second workgroup of a CU, and the CUs' rivalry when all are busy, bring `alone`
            // to `full`.
            const double share = static_cast<double>(rest) / static_cast<double>(slots);
            double time = kTileFixed + static_cast<double>(groups / slots) * (t.start + walked * t.full);
            if (rest > 0) {
                time += t.start * (0.5 + 0.5 * share) +
                        walked * (t.alone + (t.full - t.alone) * share * share);
            }
            int64_t bytes = 0;
            if (splits > 1) {
                bytes = splits * (gated ? 2 : 1) * 4 * p.m * p.n;
                time += kFinishFixed + 2.0 * static_cast<double>(bytes) / kFinishBytesPerUs;
            }
            offer(t.form, splits, time, bytes);
        }
    };
    if (gated) {
        for (const Few& f : kFewGated) {
            few(f);
        }
        for (const Ring& r : kRingsGated) {
            ring(r);
        }
        for (const Tile& t : kTilesGated) {
            tiles(t);
        }
    } else {
        for (const Few& f : kFew) {
            few(f);
        }
        for (const Ring& r : kRings) {
            ring(r);
        }
        for (const Tile& t : kTiles) {
            tiles(t);
        }
    }
    return best;
}

void launch(const mfr_stream& s, const Plan& plan, const Params& p) {
    using namespace mfr::f8gemm;
    const bool gated = p.up.values != nullptr;
    switch (plan.form) {
    case Form::kFew16:
        (gated ? launch_few<1, 1, 8, 2, true> : launch_few<1, 1, 8, 2, false>)(s, p);
        break;
    case Form::kFew32:
        (gated ? launch_few<2, 1, 8, 1, true> : launch_few<2, 1, 8, 2, false>)(s, p);
        break;
    case Form::kFew32Wide:
        launch_few<2, 2, 4, 2, false>(s, p);
        break;
    case Form::kFew64:
        (gated ? launch_few<4, 1, 4, 1, true> : launch_few<4, 2, 8, 1, false>)(s, p);
        break;
    case Form::kRing32:
        (gated ? launch_ring<1, 1, 4, 3, true> : launch_ring<1, 1, 8, 2, false>)(s, p);
        break;
    case Form::kRing32Wide:
        launch_ring<1, 2, 4, 3, false>(s, p);
        break;
    case Form::kRing64:
        (gated ? launch_ring<2, 1, 4, 2, true> : launch_ring<2, 2, 3, 3, false>)(s, p);
        break;
    case Form::kRing64Pair:
        (gated ? launch_ring<2, 1, 2, 2, true> : launch_ring<2, 2, 2, 2, false>)(s, p);
        break;
    case Form::kRing128:
        (gated ? launch_ring<1, 4, 2, 2, true> : launch_ring<1, 4, 2, 3, false>)(s, p);
        break;
    case Form::kTile64:
        (gated ? launch_tiles<64, 128, 2, 4, 3, true> : launch_tiles<64, 128, 1, 4, 2, false>)(
            s, p, plan.splits);
        break;
    case Form::kTile128:
        (gated ? launch_tiles<128, 128, 2, 4, 2, true> : launch_tiles<128, 128, 2, 2, 2, false>)(
            s, p, plan.splits);
        break;
    }
}

// The ranges of the depth that are not empty.
int64_t ranges_of(const Params& p, const Plan& plan) {
    const int64_t blocks = blocks_of(p.k);
    return plan.splits > 1 ? ceil_div(blocks, ceil_div(blocks, plan.splits)) : 1;
}

void run_region(mfr_stream& s, Params p, Plan plan) {
    std::unique_lock<std::mutex> hold(s.workspace_mutex, std::defer_lock);
    void* memory = nullptr;
    if (plan.workspace > 0) {
        // Held until all kernels are queued: another thread's reserve() may not free the memory.
        // Under stream capture none is used: a graph would keep its address, which a later call may
        // free to grow it, and its replays may run beside calls that use it. (The default stream
        // cannot be asked while another captures: none then, too.)
        hold.lock();
        hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing(s.stream, &capture) != hipSuccess) {
            (void)hipGetLastError();
        } else if (capture == hipStreamCaptureStatusNone) {
            try {
                memory = s.reserve(static_cast<size_t>(plan.workspace));
            } catch (const mfr::Error&) {
                (void)hipGetLastError();
            }
        }
        if (memory == nullptr) {
            plan = choose(p, s.compute_units, false);
        }
    }
    if (converts(plan.form)) {
        Params sums = p;
        if (p.c == nullptr) {
            sums.c = static_cast<float*>(memory);
            sums.c_rs = p.n;
        }
        launch(s, plan, sums);
        if (p.q.values != nullptr) {
            mfr::f8::quantize_rows(s, sums.c, sums.c_rs, p.m, p.n, p.q);
        }
        return;
    }
    p.split_blocks = ceil_div(blocks_of(p.k), plan.splits);
    if (plan.splits > 1) {
        p.partial = static_cast<float*>(memory);
        plan.splits = ranges_of(p, plan);
    }
    launch(s, plan, p);
    if (p.partial != nullptr) {
        mfr::f8gemm::launch_finish(s, p, plan.splits);
    }
}

// Rows [first, m) or columns [first, n) of the problem, and what comes before them; first a multiple
// of 128.
Params rows_from(Params p, int64_t first) {
    p.m -= first;
    p.a.values += first * p.a.rs;
    p.a.scales += first * p.a.srs;
    p.c += p.c != nullptr ? first * p.c_rs : 0;
    p.c0 += p.c0 != nullptr ? first * p.c0_rs : 0;
    p.q.values += p.q.values != nullptr ? first * p.q.rs : 0;
    p.q.scales += p.q.values != nullptr ? first * p.q.srs : 0;
    return p;
}

Params cols_from(Params p, int64_t first) {
    const int64_t block = first / mfr::f8::kBlock;
    p.n -= first;
    for (mfr::f8::Matrix* w : {&p.b, &p.up}) {
        if (w->values != nullptr) {
            w->values += first * w->rs;
            w->scales += block * w->srs;
        }
    }
    p.c += p.c != nullptr ? first : 0;
    p.c0 += p.c0 != nullptr ? first : 0;
    p.bias += p.bias != nullptr ? first : 0;
    p.q.values += p.q.values != nullptr ? first : 0;
    p.q.scales += p.q.values != nullptr ? block * p.q.scs : 0;
    return p;
}

// Launches of their own, each part of the outputs.
struct Region {
    Params p;
    Plan plan;
};
struct Regions {
    Region list[3];
    int count = 0;
};

// The problem whole, or, where the model prices that lower, without the rows and columns past the
// last multiple of 128, which run by themselves: 3 columns more than 32 x 32 tiles of two on each CU
// cost a third turn of every CU (4093 x 4099 x 1023 58.9 -> 54.0 us). Short calls are not worth the
// question.
constexpr double kShortCall = 20.0;

Regions regions_of(const Params& p, int64_t cus) {
    const auto priced = [&](const Params& x) { return choose(x, cus, true); };
    Regions out;
    const auto add = [&](const Params& x, const Plan& plan) { out.list[out.count++] = {x, plan}; };
    const Plan whole = priced(p);
    const int64_t m = p.m / 128 * 128;
    const int64_t n = p.n / 128 * 128;
    const auto head = [](Params x, int64_t rows, int64_t cols) {
        x.m = rows;
        x.n = cols;
        return x;
    };
    double best = whole.time;
    int64_t rows = p.m;
    int64_t cols = p.n;
    for (const auto& [r, c] : {std::pair{p.m, n}, std::pair{m, p.n}, std::pair{m, n}}) {
        if (whole.time < kShortCall || r == 0 || c == 0 || (r == p.m && c == p.n)) {
            continue;
        }
        double time = priced(head(p, r, c)).time;
        if (c < p.n) {
            time += priced(cols_from(head(p, r, p.n), c)).time;
        }
        if (r < p.m) {
            time += priced(rows_from(p, r)).time;
        }
        if (time < best) {
            best = time;
            rows = r;
            cols = c;
        }
    }
    if (rows == p.m && cols == p.n) {
        add(p, whole);
        return out;
    }
    const auto region = [&](const Params& x) { add(x, priced(x)); };
    region(head(p, rows, cols));
    if (cols < p.n) {
        region(cols_from(head(p, rows, p.n), cols));
    }
    if (rows < p.m) {
        region(rows_from(p, rows));
    }
    return out;
}

} // namespace

extern "C" {

int mfr_f8gemm(mfr_stream_t stream, const mfr_f8gemm_desc* desc) {
    return mfr::guarded([&] {
        const Params p = checked(desc);
        auto& s = mfr::stream_of(stream);
        if (p.m == 0 || p.n == 0) {
            return;
        }
        const Regions regions = regions_of(p, s.compute_units);
        for (int i = 0; i < regions.count; ++i) {
            run_region(s, regions.list[i].p, regions.list[i].plan);
        }
    });
}

int mfr_f8gemm_plan(int device, const mfr_f8gemm_desc* desc, int32_t* form, int32_t* splits,
                    int32_t* regions, size_t* workspace) {
    return mfr::guarded([&] {
        mfr::require(form != nullptr && splits != nullptr && regions != nullptr &&
                         workspace != nullptr,
                     "f8gemm_plan: null argument");
        const Params p = checked(desc);
        int cus = 0;
        const int status = mfr_get_device_info(device, nullptr, 0, nullptr, &cus, nullptr);
        if (status != MFR_OK) {
            throw mfr::Error(status, mfr_last_error());
        }
        *form = MFR_F8_NOTHING;
        *splits = *regions = 0;
        *workspace = 0;
        if (p.m == 0 || p.n == 0) {
            return;
        }
        const Regions made = regions_of(p, cus);
        *form = static_cast<int32_t>(made.list[0].plan.form);
        *splits = static_cast<int32_t>(ranges_of(made.list[0].p, made.list[0].plan));
        *regions = made.count;
        for (int i = 0; i < made.count; ++i) {
            *workspace = std::max(*workspace, static_cast<size_t>(made.list[i].plan.workspace));
        }
    });
}

} // extern "C"
