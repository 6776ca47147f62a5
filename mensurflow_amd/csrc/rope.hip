// mfr_rope and mfr_kv_append: queries and keys turned by their positions (rotary.hpp), keys and values
// into the pages of a cache (kv.hpp).
#include "kv.hpp"
#include "rotary.hpp"

#include "f8.hpp"

#include <algorithm>

namespace {

using mfr::kv::Batch;
using mfr::kv::Cache;
using mfr::kv::Heads;
using mfr::rotary::kMostPairs;
using mfr::rotary::Rotary;
namespace rdev = mfr::rotary::dev;

constexpr int kThreads = 256;

// Workgroups of a launch whose tokens are cut into `groups` pieces each; they walk what is more.
constexpr int64_t kMostBlocks = int64_t{1} << 20;

// Pieces of a token's heads, `per_step` heads a step: enough to fill the chip where tokens are few,
// whole steps.
int64_t groups_of(const mfr_stream& s, int64_t tokens, int64_t heads, int64_t per_step) {
    const int64_t steps = (heads + per_step - 1) / per_step;
    const int64_t wanted = (4 * static_cast<int64_t>(s.compute_units) + tokens - 1) / tokens;
    return std::max<int64_t>(1, std::min(wanted, steps));
}

struct RopeParams {
    int64_t rows;
    int32_t heads, d;
    Heads x;
    float* out;
    int64_t out_ts, out_hs;
    const int32_t* positions;
    int64_t first;
    int32_t backward;
    int32_t columns;   // of a head that are written: all, or in place those that turn
    int32_t lane_log2; // lanes of a head, 4 columns each
    int32_t groups;    // pieces of a token's heads
    int32_t group_heads;
    Rotary rotary;
};

// A workgroup takes a token's heads, or some of them where tokens are few.
template <bool QUADS> __global__ __launch_bounds__(kThreads) void rope_kernel(RopeParams p) {
    __shared__ float2 table[kMostPairs];
    const int lanes = 1 << p.lane_log2;
    const int c0 = 4 * (threadIdx.x & (lanes - 1));
    const int per_step = kThreads >> p.lane_log2;
    const int64_t blocks = p.rows * p.groups;
    for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
        const int64_t row = b / p.groups;
        const int h0 = static_cast<int>(b - row * p.groups) * p.group_heads;
        const int h1 = min(h0 + p.group_heads, p.heads);
        const int64_t position = p.positions != nullptr ? p.positions[row] : p.first + row;
        rdev::fill_angles(p.rotary, position, p.backward != 0, table, kThreads);
        __syncthreads();
        for (int h = h0 + (threadIdx.x >> p.lane_log2); h < h1; h += per_step) {
            const float* x = p.x.p + row * p.x.ts + h * p.x.hs;
            float* out = p.out + row * p.out_ts + h * p.out_hs;
            // In place the columns are at most 256, a single step: no load follows a store.
            for (int c = c0; c < p.columns; c += 4 * lanes) {
                const float4 v = rdev::turned_quad<QUADS>(x, c, p.d, p.rotary, table);
                rdev::loads_before_stores();
                mfr::f8::dev::store_quad(out + c, v, p.columns - c);
            }
        }
        __syncthreads();
    }
}

void run_rope(mfr_stream& s, const RopeParams& p, int64_t blocks) {
    const unsigned grid = static_cast<unsigned>(std::min(blocks, kMostBlocks));
    if (p.rotary.quads != 0) {
        rope_kernel<true><<<grid, kThreads, 0, s.stream>>>(p);
    } else {
        rope_kernel<false><<<grid, kThreads, 0, s.stream>>>(p);
    }
    mfr::check_launch("rope_kernel");
}

// ---- appending to a cache ---------------------------------------------------------------------

struct AppendParams {
    Cache cache;
    Batch batch;
    Heads k, v, q;
    float* q_out;
    int64_t q_out_ts, q_out_hs;
    int32_t q_heads;
    const int32_t* positions;
    int32_t groups;
    int32_t group_items;
    Rotary rotary;
};

constexpr int kRowLanes = 32; // a head of at most 128 columns

__device__ inline uint32_t two_bf16(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, v);
}

// Four columns from c on of a row of the cache; all 32 lanes of a row call it, `live` those that hold
// columns of a row that is written.
template <int TYPE>
__device__ inline void store_row(uint8_t* row, float* scale, int c, float4 v, bool live) {
    if constexpr (TYPE == MFR_KV_F32) {
        if (live) {
            *reinterpret_cast<float4*>(row + 4 * c) = v;
        }
    } else if constexpr (TYPE == MFR_KV_BF16) {
        if (live) {
            *reinterpret_cast<uint2*>(row + 2 * c) = make_uint2(two_bf16(v.x, v.y), two_bf16(v.z, v.w));
        }
    } else {
        namespace dev = mfr::f8::dev;
        const uint32_t top = dev::half_max(live ? dev::magnitude(v) : 0u);
        if (live) {
            *reinterpret_cast<uint32_t*>(row + c) = dev::pack(v, dev::quotient_of(top));
            if (c == 0) {
                *scale = dev::scale_of(top);
            }
        }
    }
}

// A workgroup takes a row of the batch: its keys' heads, its values' and its queries', 8 at a time, or
// some of them where rows are few.
template <int TYPE, bool QUADS>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(AppendParams p) {
    __shared__ float2 table[kMostPairs];
    const int c = 4 * (threadIdx.x % kRowLanes);
    const int heads = p.cache.heads, d = p.cache.d;
    const int64_t blocks = static_cast<int64_t>(p.batch.rows) * p.groups;
    for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
        const int32_t row = static_cast<int32_t>(b / p.groups);
        const int32_t seq = mfr::kv::sequence_of(p.batch, row);
        if (seq < 0) {
            continue; // the whole workgroup
        }
        const mfr::kv::Span span = mfr::kv::span_of(p.batch, seq);
        const int64_t place = mfr::kv::first_place(p.batch, seq, span.count) + (row - span.first);
        const int32_t page = mfr::kv::page_of(p.batch, seq, place);
        const int64_t slot = place & ((1 << p.cache.page_log2) - 1);
        if (p.rotary.rot > 0) {
            const int64_t position = p.positions != nullptr ? p.positions[row]
                                                            : p.batch.prefix + place;
            rdev::fill_angles(p.rotary, position, false, table, kThreads);
        }
        __syncthreads();
        const int first = static_cast<int>(b - static_cast<int64_t>(row) * p.groups) * p.group_items;
        const int items = 2 * heads + p.q_heads;
        const int end = min(first + p.group_items, items);
        for (int i = first; i < end; i += kThreads / kRowLanes) {
            const int item = i + static_cast<int>(threadIdx.x / kRowLanes);
            // Keys, then values, then queries.
            const int what = item >= end ? 3 : item < heads ? 0 : item < 2 * heads ? 1 : 2;
            const int h = what == 0 ? item : what == 1 ? item - heads : item - 2 * heads;
            const bool live = what < 3 && c < d && (what == 2 || page >= 0);
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (live) {
                const Heads& from = what == 0 ? p.k : what == 1 ? p.v : p.q;
                const float* x = from.p + row * from.ts + h * from.hs;
                v = what == 1 ? mfr::dev::load_loose(x + c)
                              : rdev::turned_quad<QUADS>(x, c, d, p.rotary, table);
            }
            rdev::loads_before_stores();
            if (what == 2 && live) {
                mfr::dev::store_loose(p.q_out + row * p.q_out_ts + h * p.q_out_hs + c, v);
            }
            uint8_t* base = what == 0 ? p.cache.k : p.cache.v;
            float* scales = what == 0 ? p.cache.k_scales : p.cache.v_scales;
            store_row<TYPE>(base + page * p.cache.page_stride + slot * p.cache.token_stride +
                                h * p.cache.head_stride,
                            scales + (((static_cast<int64_t>(page) * heads + h)
                                       << p.cache.page_log2) +
                                      slot),
                            c, v, live && what < 2);
        }
        __syncthreads();
    }
}

template <int TYPE> void launch_append(const AppendParams& p, unsigned grid, hipStream_t stream) {
    if (p.rotary.quads != 0) {
        kv_append_kernel<TYPE, true><<<grid, kThreads, 0, stream>>>(p);
    } else {
        kv_append_kernel<TYPE, false><<<grid, kThreads, 0, stream>>>(p);
    }
    mfr::check_launch("kv_append_kernel");
}

} // namespace

extern "C" {

int mfr_rotary_init(mfr_rotary* rotary, int32_t rot, int32_t layout, double base, double amplitude,
                    double factor, double original, double slow, double fast) {
    return mfr::guarded([&] {
        using mfr::require;
        require(rotary != nullptr, "rotary: null rotation");
        require(rot >= 0 && rot % 2 == 0 && rot <= MFR_ROTARY_MOST,
                "rotary: an even number of columns is needed, at most 256");
        require(layout == MFR_ROTARY_HALVES || layout == MFR_ROTARY_PAIRS,
                "rotary: unknown layout");
        require(std::isfinite(base) && base >= 1.0, "rotary: base has to be 1 or more");
        require(std::isfinite(amplitude) && std::isfinite(static_cast<float>(amplitude)),
                "rotary: amplitude is not finite");
        require(std::isfinite(factor) && factor >= 1.0, "rotary: factor has to be 1 or more");
        require(std::isfinite(original) && original >= 0.0, "rotary: negative original length");
        require(original == 0.0 || (std::isfinite(slow) && std::isfinite(fast) && slow < fast),
                "rotary: slow has to be less than fast");
        mfr_rotary out{};
        out.rot = rot;
        out.layout = layout;
        out.amplitude = static_cast<float>(amplitude);
        for (int i = 0; i < rot / 2; ++i) {
            const double step = std::pow(base, -2.0 * i / rot);
            double kept = 0.0;
            if (original > 0.0) {
                const double turns = original * step / 6.283185307179586476925;
                kept = std::min(1.0, std::max(0.0, (turns - slow) / (fast - slow)));
            }
            out.steps[i] = step * (kept + (1.0 - kept) / factor);
        }
        *rotary = out;
    });
}

int mfr_rope(mfr_stream_t stream, const mfr_rope_desc* desc) {
    return mfr::guarded([&] {
        using mfr::require;
        require(desc != nullptr, "rope: null descriptor");
        const mfr_rope_desc& d = *desc;
        require(d.rows >= 0 && d.heads >= 0 && d.d >= 0, "rope: negative dimension");
        mfr::kv::supported(d.rows < (int64_t{1} << 40) && d.heads <= mfr::kv::kMostHeads &&
                               d.d <= (1 << 20),
                           "rope: too large");
        const Rotary rotary = mfr::rotary::checked(d.rotary, d.d, "rope");
        const bool empty = d.rows == 0 || d.heads == 0 || d.d == 0;
        if (!empty) {
            mfr::kv::check_heads(d.x, d.x_ts, d.x_hs, d.rows, d.heads, d.d, false, "rope: x");
            mfr::kv::check_heads(d.out, d.out_ts, d.out_hs, d.rows, d.heads, d.d, true,
                                 "rope: out");
            require(d.x != d.out || ((d.rows == 1 || d.x_ts == d.out_ts) &&
                                     (d.heads == 1 || d.x_hs == d.out_hs)),
                    "rope: an output in place of its input needs its strides");
            constexpr int64_t kFar = int64_t{1} << 31;
            require(d.positions != nullptr || (d.first >= -kFar && d.first + d.rows <= kFar),
                    "rope: positions past 2^31");
        }
        auto& s = mfr::stream_of(stream);
        const int64_t columns = d.x == d.out ? rotary.rot : d.d;
        if (empty || columns == 0) {
            return;
        }
        RopeParams p{};
        p.rows = d.rows;
        p.heads = static_cast<int32_t>(d.heads);
        p.d = static_cast<int32_t>(d.d);
        p.x = {d.x, d.x_ts, d.x_hs};
        p.out = d.out;
        p.out_ts = d.out_ts;
        p.out_hs = d.out_hs;
        p.positions = d.positions;
        p.first = d.first;
        p.backward = d.backward;
        p.columns = static_cast<int32_t>(columns);
        p.rotary = rotary;
        while (p.lane_log2 < 6 && (4 << p.lane_log2) < columns) {
            ++p.lane_log2;
        }
        const int64_t per_step = kThreads >> p.lane_log2;
        const int64_t groups = groups_of(s, d.rows, d.heads, per_step);
        const int64_t steps = (d.heads + per_step - 1) / per_step;
        p.groups = static_cast<int32_t>(groups);
        p.group_heads = static_cast<int32_t>((steps + groups - 1) / groups * per_step);
        run_rope(s, p, d.rows * groups);
    });
}

int mfr_kv_append(mfr_stream_t stream, const mfr_kv_append_desc* desc) {
    return mfr::guarded([&] {
        using mfr::require;
        require(desc != nullptr, "kv_append: null descriptor");
        const mfr_kv_append_desc& d = *desc;
        AppendParams p{};
        p.cache = mfr::kv::checked(d.cache, true, "kv_append");
        p.batch = mfr::kv::checked(d.batch, d.cache, "kv_append");
        p.rotary = mfr::rotary::checked(d.rotary, d.cache.d, "kv_append");
        require(d.q_heads >= 0 && (d.q == nullptr || d.q_heads > 0),
                "kv_append: q needs its number of heads");
        mfr::kv::supported(d.q_heads <= mfr::kv::kMostHeads, "kv_append: too many heads");
        const bool empty = d.batch.rows == 0 || d.batch.sequences == 0;
        if (!empty) {
            const int64_t rows = d.batch.rows, depth = d.cache.d;
            mfr::kv::check_heads(d.k, d.k_ts, d.k_hs, rows, d.cache.heads, depth, false,
                                 "kv_append: k");
            mfr::kv::check_heads(d.v, d.v_ts, d.v_hs, rows, d.cache.heads, depth, false,
                                 "kv_append: v");
            if (d.q != nullptr) {
                mfr::kv::check_heads(d.q, d.q_ts, d.q_hs, rows, d.q_heads, depth, false,
                                     "kv_append: q");
                mfr::kv::check_heads(d.q_out, d.q_out_ts, d.q_out_hs, rows, d.q_heads, depth, true,
                                     "kv_append: q_out");
                require(d.q != d.q_out || ((rows == 1 || d.q_ts == d.q_out_ts) &&
                                           (d.q_heads == 1 || d.q_hs == d.q_out_hs)),
                        "kv_append: an output in place of its input needs its strides");
            }
        }
        auto& s = mfr::stream_of(stream);
        if (empty) {
            return;
        }
        p.k = {d.k, d.k_ts, d.k_hs};
        p.v = {d.v, d.v_ts, d.v_hs};
        p.q = {d.q, d.q_ts, d.q_hs};
        p.q_out = d.q_out;
        p.q_out_ts = d.q_out_ts;
        p.q_out_hs = d.q_out_hs;
        p.q_heads = d.q != nullptr ? static_cast<int32_t>(d.q_heads) : 0;
        p.positions = d.positions;
        constexpr int64_t kPerStep = kThreads / kRowLanes;
        const int64_t items = 2 * d.cache.heads + p.q_heads;
        const int64_t steps = (items + kPerStep - 1) / kPerStep;
        const int64_t groups = groups_of(s, d.batch.rows, items, kPerStep);
        p.groups = static_cast<int32_t>(groups);
        p.group_items = static_cast<int32_t>((steps + groups - 1) / groups * kPerStep);
        const unsigned grid =
            static_cast<unsigned>(std::min(d.batch.rows * groups, kMostBlocks));
        switch (d.cache.type) {
        case MFR_KV_F32: launch_append<MFR_KV_F32>(p, grid, s.stream); break;
        case MFR_KV_BF16: launch_append<MFR_KV_BF16>(p, grid, s.stream); break;
        default: launch_append<MFR_KV_F8>(p, grid, s.stream); break;
        }
    });
}

} // extern "C"
