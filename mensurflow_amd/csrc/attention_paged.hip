// mfr_attention_paged: checks, the choice of the form, workspace and launches.
#include "attention_paged.hpp"

#include <algorithm>
#include <cmath>

namespace {

using mfr::paged::Params;

// One launch over the prefix or over the sequences' own tokens.
struct Launch {
    Params p;
    size_t parts; // rows of parts
};

struct Plan {
    Launch shared, own;
    bool has_prefix;
    size_t bytes;
};

size_t aligned(size_t bytes) { return (bytes + 255) / 256 * 256; }

size_t parts_bytes(size_t rows, int depth) {
    return aligned(rows * depth * sizeof(float)) + aligned(rows * 2 * sizeof(float));
}

mfr::paged::Parts parts_at(uint8_t* at, size_t rows, int depth) {
    return {reinterpret_cast<float*>(at),
            reinterpret_cast<float*>(at + aligned(rows * depth * sizeof(float)))};
}

Launch launch_of(Params p, int32_t type, int shared, int cus) {
    mfr::kv::Work& w = p.work;
    w.shared = shared;
    const int64_t sequences = mfr::kv::sequences_of(w);
    const int64_t rows = static_cast<int64_t>(w.batch.rows) * w.group;
    // By the rows of a sequence, on average. 32 sequences of up to 4096 tokens, 8 heads of 128, us in tiles
    // of 16, 32 and 128 rows, bf16 (8 bits): 16 rows 83, 88, 202 (60, 74, 202); 24 rows 120, 94, 202 (94, 80,
    // 202); 64 rows 248, 167, 221 (183, 148, 228); 96 rows -, 225, 241 (-, 189, 244); 128 rows -, 317, 263
    // (-, 275, 264). The large tiles save reading the keys again. It is not the better one everywhere: few
    // sequences, whose keys stay in a cache, and short ones do as well or better in tiles of 32 (4 of 512 rows
    // on 600 tokens 36 and 49 us, on 4800 131 and 146; 1024 rows on a prefix of 4096 96 and 105, in 8 bits of
    // 16384 313 and 296), and where rows differ much most items get the other ones' height (7 single queries
    // and a piece of 512 rows on 4096 tokens each 162 us, 35 and 120 by themselves).
    const bool many = type != MFR_KV_F32 && rows > 96 * sequences;
    w.tile_rows = many ? mfr::paged::kManyRows : rows <= 16 * sequences ? 16 : 32;
    w.unit = many || type == MFR_KV_F32 ? 64 : 128; // a workgroup's step
    const int64_t tokens =
        shared != 0 ? w.batch.prefix : static_cast<int64_t>(mfr::kv::capacity_of(w.batch));
    const int64_t units = std::max<int64_t>(1, (tokens + w.unit - 1) / w.unit);
    const int64_t items = (rows / w.tile_rows + sequences) * w.heads;
    const int64_t wanted =
        static_cast<int64_t>(cus) * mfr::paged::per_unit(type, p.depth, w.tile_rows);
    p.groups = static_cast<int32_t>(items >= wanted ? wanted : std::min(wanted, items * units));
    return {p, 2 * static_cast<size_t>(p.groups) * static_cast<size_t>(w.tile_rows)};
}

// The descriptor's checks (of shapes, layouts and pointers: no device is needed), and the plan of a call
// on a device of `cus` compute units. The workspace: the parts of one launch after the other, then what
// the prefix gave.
Plan planned(const mfr_attention_paged_desc* desc, int cus) {
    using mfr::require;
    require(desc != nullptr, "attention_paged: null descriptor");
    const mfr_attention_paged_desc& d = *desc;
    Params p{};
    p.cache = mfr::kv::checked(d.cache, false, "attention_paged");
    p.work.batch = mfr::kv::checked(d.batch, d.cache, "attention_paged");
    require(d.q_heads >= 1 && d.q_heads % d.cache.heads == 0,
            "attention_paged: q's heads are no multiple of the cache's");
    mfr::kv::supported(d.q_heads <= mfr::kv::kMostHeads, "attention_paged: too many heads");
    require(std::isfinite(d.scale), "attention_paged: scale is not finite");
    Plan plan{};
    if (p.work.batch.rows == 0) {
        return plan;
    }
    mfr::kv::check_heads(d.q, d.q_ts, d.q_hs, d.batch.rows, d.q_heads, d.cache.d, false,
                         "attention_paged: q");
    mfr::kv::check_heads(d.out, d.out_ts, d.out_hs, d.batch.rows, d.q_heads, d.cache.d, true,
                         "attention_paged: out");
    // Rows of an item, and of parts, are counted in 32 bits.
    mfr::kv::supported(d.batch.rows * d.q_heads < (int64_t{1} << 30),
                       "attention_paged: too many rows");
    if (d.cache.pages == 0) { // no token is anywhere, and no address may be read
        p.work.batch.width = 0;
        p.work.batch.prefix = 0;
    }
    p.work.heads = p.cache.heads;
    p.work.group = static_cast<int32_t>(d.q_heads / d.cache.heads);
    p.q = {d.q, d.q_ts, d.q_hs};
    p.out = d.out;
    p.out_ts = d.out_ts;
    p.out_hs = d.out_hs;
    p.q_heads = static_cast<int32_t>(d.q_heads);
    p.causal = d.causal;
    const float scale =
        d.scale != 0.0f ? d.scale : static_cast<float>(1.0 / std::sqrt(static_cast<double>(d.cache.d)));
    p.scale = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
    p.depth = d.cache.d <= 64 ? 64 : 128;
    plan.has_prefix = p.work.batch.prefix > 0;
    plan.own = launch_of(p, d.cache.type, 0, cus);
    plan.bytes = parts_bytes(plan.own.parts, p.depth);
    if (plan.has_prefix) {
        Params shared = p;
        shared.causal = 0;
        plan.shared = launch_of(shared, d.cache.type, 1, cus);
        const size_t rows = static_cast<size_t>(d.batch.rows) * static_cast<size_t>(d.q_heads);
        plan.bytes = std::max(plan.bytes, parts_bytes(plan.shared.parts, p.depth)) +
                     parts_bytes(rows, p.depth);
    }
    return plan;
}

void run(Plan& plan, const mfr_attention_paged_desc& d, uint8_t* workspace, hipStream_t stream) {
    const int depth = plan.own.p.depth;
    if (plan.has_prefix) {
        const size_t rows = static_cast<size_t>(d.batch.rows) * static_cast<size_t>(d.q_heads);
        const mfr::paged::Parts prefix =
            parts_at(workspace + plan.bytes - parts_bytes(rows, depth), rows, depth);
        plan.own.p.prefix = plan.shared.p.prefix = prefix;
    }
    for (Launch* l : {&plan.shared, &plan.own}) {
        if (l == &plan.shared && !plan.has_prefix) {
            continue;
        }
        l->p.parts = parts_at(workspace, l->parts, depth);
        if (l->p.work.tile_rows == mfr::paged::kManyRows) {
            mfr::paged::launch_tiles(l->p, d.cache.type, stream);
        } else {
            mfr::paged::launch_few(l->p, d.cache.type, stream);
        }
        mfr::paged::launch_join(l->p, stream);
    }
}

} // namespace

extern "C" {

int mfr_attention_paged(mfr_stream_t stream, const mfr_attention_paged_desc* desc) {
    return mfr::guarded([&] {
        (void)planned(desc, 256); // before the stream is looked at
        auto& s = mfr::stream_of(stream);
        Plan plan = planned(desc, s.compute_units);
        if (desc->batch.rows == 0 || desc->batch.sequences == 0) {
            return;
        }
        if (desc->workspace != nullptr) {
            mfr::require(mfr::aligned16(desc->workspace) && desc->workspace_bytes >= plan.bytes,
                         "attention_paged: the workspace is too small (" +
                             std::to_string(plan.bytes) + " bytes) or not 16-byte aligned");
            run(plan, *desc, static_cast<uint8_t*>(desc->workspace), s.stream);
            return;
        }
        // A graph would keep the address of the stream's workspace, which a later call may free to grow
        // it, and its replays may run beside calls that use it. (A stream that cannot be asked is
        // taken as one that captures.)
        hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing(s.stream, &capture) != hipSuccess) {
            (void)hipGetLastError();
            capture = hipStreamCaptureStatusActive;
        }
        mfr::require(capture == hipStreamCaptureStatusNone,
                     "attention_paged: a captured call needs a workspace of its own (" +
                         std::to_string(plan.bytes) + " bytes)");
        // Held until the last launch is queued: another thread's reserve() may not free it before.
        const std::lock_guard<std::mutex> hold(s.workspace_mutex);
        run(plan, *desc, static_cast<uint8_t*>(s.reserve(plan.bytes)), s.stream);
    });
}

int mfr_attention_paged_workspace(int device, const mfr_attention_paged_desc* desc, size_t* bytes) {
    return mfr::guarded([&] {
        (void)planned(desc, 256);
        mfr::require(bytes != nullptr, "attention_paged: null result");
        int cus = 0;
        if (const int status =
                mfr_get_device_info(device, nullptr, 0, nullptr, &cus, nullptr)) {
            throw mfr::Error(status, mfr_last_error());
        }
        *bytes = planned(desc, cus).bytes;
    });
}

} // extern "C"
