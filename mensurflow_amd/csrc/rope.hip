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

constexpr int kWaves = kThreads / 64;

// How a launch is cut: a token's heads into groups, a wavefront each, neighbours in one workgroup, and
// `tokens` at once, which walk what is more.
struct Cut {
    int32_t groups, group_heads;
    uint32_t tokens;
};

// `per_step` heads a step of a wavefront, whole steps, `most` of them at most. Where tokens are few, as
// many groups as give 16 wavefronts a compute unit.
Cut cut_of(const mfr_stream& s, int64_t tokens, int64_t heads, int64_t per_step, int64_t most) {
    const int64_t steps = (heads + per_step - 1) / per_step;
    const int64_t wanted = (16 * static_cast<int64_t>(s.compute_units) + tokens - 1) / tokens;
    const int64_t groups = std::max(std::min(wanted, steps), (steps + most - 1) / most);
    const int64_t group_heads = (steps + groups - 1) / groups * per_step;
    const int64_t count = (heads + group_heads - 1) / group_heads; // 2^20 at most
    const int64_t at_once = std::max<int64_t>(1, std::min(int64_t{1} << 20, (int64_t{1} << 24) / count));
    return {static_cast<int32_t>(count), static_cast<int32_t>(group_heads),
            static_cast<uint32_t>(std::min(tokens, at_once))};
}

unsigned blocks_of(const Cut& cut) {
    const int64_t waves = static_cast<int64_t>(cut.tokens) * cut.groups;
    return static_cast<unsigned>((waves + kWaves - 1) / kWaves);
}

// A wavefront's first token and group. (No token: behind all.)
struct Share {
    uint32_t token;
    int32_t first;
};
__device__ inline Share share_of(const Cut& cut) {
    const uint32_t wave = blockIdx.x * kWaves + threadIdx.x / 64;
    const uint32_t u = __builtin_amdgcn_readfirstlane(static_cast<int>(wave));
    const uint32_t token = u / static_cast<uint32_t>(cut.groups);
    return {token, static_cast<int32_t>(u - token * cut.groups) * cut.group_heads};
}

struct RopeParams {
    int64_t rows;
    int32_t heads;
    Heads x;
    float* out;
    int64_t out_ts, out_hs;
    const int32_t* positions;
    int64_t first;
    int32_t backward;
    int32_t columns; // of a head that are written: all, or in place those that turn
    int32_t pieces;  // of them
    Cut cut;
    Rotary rotary;
};

// A wavefront takes a token's heads, or some of them where tokens are few: their pieces in a row, 64 at a
// time, all of them under way while the angles are made. Bound by memory: 16384 tokens of 40 heads of 128
// take 117 us (5.75 TB/s) in groups of two steps (8 heads), which keep the wavefronts of a moment near to
// one another in memory, 125 in groups of four and 133 with a wavefront a token. 64 tokens take 5.7.
constexpr int kAhead = 2;
template <bool QUADS> __global__ __launch_bounds__(kThreads) void rope_kernel(RopeParams p) {
    __shared__ float2 tables[kWaves][kMostPairs];
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64));
    const Share share = share_of(p.cut);
    const int h0 = share.first;
    const int h1 = min(h0 + p.cut.group_heads, p.heads);
    const int over = 64 / p.pieces, rest = 64 - over * p.pieces; // how far 64 pieces reach
    const int lane_h = lane / p.pieces, lane_i = lane - lane_h * p.pieces;
    if (share.token >= p.cut.tokens) {
        return;
    }
    for (int64_t row = share.token; row < p.rows; row += p.cut.tokens) {
        const float* x = p.x.p + row * p.x.ts;
        float* out = p.out + row * p.out_ts;
        bool angles = false;
        int h = h0 + lane_h, i = lane_i;
        while (__any(h < h1)) {
            rdev::Piece piece[kAhead];
            rdev::Numbers v[kAhead];
            int head[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                head[k] = h;
                piece[k] = rdev::piece_of(p.rotary, i, p.columns);
                if (h < h1) {
                    v[k] = rdev::load_piece<QUADS>(x + h * p.x.hs, piece[k]);
                }
                i += rest;
                h += over + (i >= p.pieces ? 1 : 0);
                i -= i >= p.pieces ? p.pieces : 0;
            }
            if (!angles) {
                angles = true;
                const int64_t position = p.positions != nullptr ? p.positions[row] : p.first + row;
                rdev::fill_angles(p.rotary, position, p.backward != 0, tables[wave]);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (head[k] < h1) {
                    const rdev::Numbers w =
                        rdev::turned_piece<QUADS>(v[k], piece[k], p.rotary, tables[wave]);
                    float* to = out + head[k] * p.out_hs;
                    mfr::f8::dev::store_quad(to + piece[k].a, w.a, QUADS ? 4 : piece[k].na);
                    if (piece[k].nb > 0) {
                        mfr::f8::dev::store_quad(to + piece[k].b, w.b, QUADS ? 4 : piece[k].nb);
                    }
                }
            }
        }
    }
}

void run_rope(mfr_stream& s, const RopeParams& p) {
    if (p.rotary.quads != 0) {
        rope_kernel<true><<<blocks_of(p.cut), kThreads, 0, s.stream>>>(p);
    } else {
        rope_kernel<false><<<blocks_of(p.cut), kThreads, 0, s.stream>>>(p);
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
    Cut cut;
    Rotary rotary;
};

__device__ inline uint32_t two_bf16(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, v);
}

// The largest of v over the LANES lanes that hold a row, in each of them.
template <int LANES> __device__ inline uint32_t row_top(uint32_t v) {
    const auto with = [&](float other) { v = mfr::f8::most(v, __float_as_uint(other)); };
    if constexpr (LANES == 32) {
        float a, b;
        mfr::dev::swap_pair<false>(__uint_as_float(v), a, b);
        v = mfr::f8::most(__float_as_uint(a), __float_as_uint(b));
    }
    with(mfr::dev::xor_lane<8>(__uint_as_float(v)));
    with(mfr::dev::xor_lane<4>(__uint_as_float(v)));
    with(mfr::dev::xor_lane<2>(__uint_as_float(v)));
    with(mfr::dev::xor_lane<1>(__uint_as_float(v)));
    return v;
}

// The first n of four columns from c on of a row of the cache; whole quads are at a multiple of 4.
template <int TYPE, bool QUADS>
__device__ inline void store_columns(uint8_t* row, int32_t c, float4 v, int32_t n,
                                     const mfr::f8::dev::Quotient& by) {
    if (n <= 0) {
        return;
    }
    if constexpr (TYPE == MFR_KV_F32) {
        mfr::f8::dev::store_quad(reinterpret_cast<float*>(row) + c, v, QUADS ? 4 : n);
    } else if constexpr (TYPE == MFR_KV_BF16) {
        const uint2 w = make_uint2(two_bf16(v.x, v.y), two_bf16(v.z, v.w));
        uint16_t* to = reinterpret_cast<uint16_t*>(row) + c;
        if constexpr (QUADS) {
            *reinterpret_cast<uint2*>(to) = w;
        } else {
            for (int i = 0; i < n; ++i) {
                to[i] = static_cast<uint16_t>((i < 2 ? w.x : w.y) >> (16 * (i % 2)));
            }
        }
    } else {
        const uint32_t w = mfr::f8::dev::pack(v, by);
        if constexpr (QUADS) {
            *reinterpret_cast<uint32_t*>(row + c) = w;
        } else {
            for (int i = 0; i < n; ++i) {
                row[c + i] = static_cast<uint8_t>(w >> (8 * i));
            }
        }
    }
}

// A wavefront takes a row of the batch: its keys' heads, its values' and its queries', or some of them
// where rows are few; LANES lanes a head, a piece each (16 hold the pieces of 128 columns, but where a half
// is no whole number of quads 17 may be needed). The first ones are under way while the row's place is
// looked up and the angles are made. Bound by memory for prompts (8 of 2048 tokens, 8 heads of 128 into
// bf16: 45 us, 4.5 TB/s; 52 with the row's items in two wavefronts, which both look it up), by that chain
// of loads for a step (64 rows into 8 bits with 32 heads of queries: 6.6 us).
template <int TYPE, bool QUADS>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(AppendParams p) {
    constexpr int kLanes = QUADS ? 16 : 32;
    __shared__ float2 tables[kWaves][kMostPairs];
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64));
    const int heads = p.cache.heads, d = p.cache.d;
    const int items = 2 * heads + p.q_heads;
    const Share share = share_of(p.cut);
    const int end = min(share.first + p.cut.group_heads, items);
    const rdev::Piece turned = rdev::piece_of(p.rotary, lane % kLanes, d);
    const int32_t c = 8 * (lane % kLanes);
    const rdev::Piece plain{c, c + 4, min(4, d - c), min(4, d - c - 4), -1};
    if (share.token >= p.cut.tokens) {
        return;
    }
    for (int64_t at = share.token; at < p.batch.rows; at += p.cut.tokens) {
        const int32_t row = static_cast<int32_t>(at);
        bool found = false;
        int32_t page = -1;
        int64_t slot = 0;
        for (int i0 = share.first; i0 < end; i0 += kAhead * (64 / kLanes)) {
            // Keys, then values, then queries.
            int what[kAhead], head[kAhead];
            rdev::Numbers v[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int item = i0 + k * (64 / kLanes) + lane / kLanes;
                what[k] = item >= end ? 3 : item < heads ? 0 : item < 2 * heads ? 1 : 2;
                head[k] = what[k] == 0 ? item : what[k] == 1 ? item - heads : item - 2 * heads;
                v[k] = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
                if (what[k] < 3) {
                    const float* x =
                        what[k] == 0   ? p.k.p + row * p.k.ts + head[k] * p.k.hs
                        : what[k] == 1 ? p.v.p + row * p.v.ts + head[k] * p.v.hs
                                       : p.q.p + row * p.q.ts + head[k] * p.q.hs;
                    v[k] = rdev::load_piece<QUADS>(x, what[k] == 1 ? plain : turned);
                }
            }
            if (!found) {
                found = true;
                const mfr::kv::Standing at_row = mfr::kv::dev::standing_of_wave(p.batch, row);
                if (at_row.seq < 0) {
                    break;
                }
                const int64_t place = mfr::kv::first_place(at_row.length, at_row.span.count) +
                                      (row - at_row.span.first);
                page = mfr::kv::page_of(p.batch, at_row.seq, place);
                slot = place & ((1 << p.cache.page_log2) - 1);
                if (p.rotary.rot > 0) {
                    const int64_t position = p.positions != nullptr ? p.positions[row]
                                                                    : p.batch.prefix + place;
                    rdev::fill_angles(p.rotary, position, false, tables[wave]);
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const rdev::Piece piece = what[k] == 1 ? plain : turned;
                const rdev::Numbers w =
                    rdev::turned_piece<QUADS>(v[k], piece, p.rotary, tables[wave]);
                mfr::f8::dev::Quotient by{};
                uint32_t top = 0;
                if constexpr (TYPE == MFR_KV_F8) { // all lanes
                    top = row_top<kLanes>(mfr::f8::most(mfr::f8::dev::magnitude(w.a),
                                                        mfr::f8::dev::magnitude(w.b)));
                    by = mfr::f8::dev::quotient_of(top);
                }
                if (what[k] == 2 && piece.na > 0) {
                    float* to = p.q_out + row * p.q_out_ts + head[k] * p.q_out_hs;
                    mfr::f8::dev::store_quad(to + piece.a, w.a, QUADS ? 4 : piece.na);
                    if (piece.nb > 0) {
                        mfr::f8::dev::store_quad(to + piece.b, w.b, QUADS ? 4 : piece.nb);
                    }
                } else if (what[k] < 2 && page >= 0) {
                    uint8_t* to = (what[k] == 0 ? p.cache.k : p.cache.v) + page * p.cache.page_stride +
                                  slot * p.cache.token_stride + head[k] * p.cache.head_stride;
                    store_columns<TYPE, QUADS>(to, piece.a, w.a, piece.na, by);
                    store_columns<TYPE, QUADS>(to, piece.b, w.b, piece.nb, by);
                    if (TYPE == MFR_KV_F8 && lane % kLanes == 0) {
                        float* scales = what[k] == 0 ? p.cache.k_scales : p.cache.v_scales;
                        scales[(((static_cast<int64_t>(page) * heads + head[k]) << p.cache.page_log2) +
                                slot)] = mfr::f8::dev::scale_of(top);
                    }
                }
            }
        }
    }
}

template <int TYPE> void launch_append(const AppendParams& p, hipStream_t stream) {
    const unsigned grid = blocks_of(p.cut);
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
        p.x = {d.x, d.x_ts, d.x_hs};
        p.out = d.out;
        p.out_ts = d.out_ts;
        p.out_hs = d.out_hs;
        p.positions = d.positions;
        p.first = d.first;
        p.backward = d.backward;
        p.columns = static_cast<int32_t>(columns);
        p.rotary = rotary;
        p.pieces = mfr::rotary::pieces_of(rotary, p.columns);
        p.cut = cut_of(s, d.rows, d.heads, std::max(1, 64 / p.pieces), kAhead);
        run_rope(s, p);
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
        const int64_t per_step = p.rotary.quads != 0 ? 4 : 2;
        const int64_t items = 2 * d.cache.heads + p.q_heads;
        p.cut = cut_of(s, d.batch.rows, items, per_step, items);
        switch (d.cache.type) {
        case MFR_KV_F32: launch_append<MFR_KV_F32>(p, s.stream); break;
        case MFR_KV_BF16: launch_append<MFR_KV_BF16>(p, s.stream); break;
        default: launch_append<MFR_KV_F8>(p, s.stream); break;
        }
    });
}

} // extern "C"
