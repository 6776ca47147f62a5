// Rotation by position (mfr_rotary), for the kernels that turn queries and keys.
//
// A wavefront works on one token at a time: the cosines and sines of its rot / 2 angles are made once,
// into LDS, for all heads that it has of the token. Columns that turn together are in one lane: a piece of
// a head is two times 4 columns, those of four pairs where any of them turns, so that every number is
// loaded once and a head may be turned in place.
#pragma once

#include "common.hpp"
#include "rotary_angle.hpp"

namespace mfr::rotary {

constexpr int kMostPairs = MFR_ROTARY_MOST / 2;

// As a kernel's argument.
struct Rotary {
    int32_t rot;
    int32_t pairs; // neighbours turn together
    float amplitude;
    int32_t quads; // a piece is whole quads of columns, at multiples of 4
    double quarters[kMostPairs]; // of a turn, a position
};

// Checks a rotation of heads of d and takes it over.
inline Rotary checked(const mfr_rotary& r, int64_t d, const char* what) {
    const std::string at = std::string(what) + ": the rotation ";
    require(r.rot >= 0 && r.rot % 2 == 0 && r.rot <= MFR_ROTARY_MOST,
            at + "needs an even number of columns, at most 256");
    require(r.rot <= d, at + "turns more columns than a head has");
    require(r.layout == MFR_ROTARY_HALVES || r.layout == MFR_ROTARY_PAIRS,
            at + "has an unknown layout");
    require(std::isfinite(r.amplitude), at + "has an amplitude that is not finite");
    Rotary out{};
    out.rot = r.rot;
    out.pairs = r.layout == MFR_ROTARY_PAIRS;
    out.amplitude = r.amplitude;
    out.quads = d % 4 == 0 && (out.pairs != 0 || r.rot % 8 == 0);
    for (int i = 0; i < r.rot / 2; ++i) {
        require(std::abs(r.steps[i]) <= 1e6, at + "has steps past 10^6 or not finite");
        out.quarters[i] = quarters_of(r.steps[i]);
    }
    return out;
}

// Pieces (dev::piece_of) of a head's first `columns`.
inline int32_t pieces_of(const Rotary& r, int32_t columns) {
    return r.pairs != 0 ? (columns + 7) / 8 : (r.rot / 2 + 3) / 4 + (columns - r.rot + 7) / 8;
}

} // namespace mfr::rotary

namespace mfr::rotary::dev {

// The angles of a token into the wavefront's `table` [rot / 2], times the amplitude, rounded once.
__device__ inline void fill_angles(const Rotary& r, int64_t position, bool backward, float2* table) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    for (int i = threadIdx.x % 64; i < r.rot / 2; i += 64) {
        const Angle t = angle_of(static_cast<double>(position), r.quarters[i]);
        const double amplitude = r.amplitude;
        table[i] = make_float2(static_cast<float>(amplitude * t.cosine),
                               static_cast<float>(amplitude * (backward ? -t.sine : t.sine)));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
}

// na columns of a head from a on, and nb from b on (each up to 4, nb perhaps 0). Where pieces are whole quads
// (Rotary::quads) a quad is taken whole if it has any of them: what does not turn is written as it was.
struct Piece {
    int32_t a, b, na, nb;
    int32_t angles; // from here on are its pairs'; -1: nothing turns
};

// Piece i of a head's first `columns`, which hold at least all that turn. Past the last one na <= 0.
__device__ inline Piece piece_of(const Rotary& r, int32_t i, int32_t columns) {
    const int32_t half = r.rot / 2;
    const int32_t turning = (half + 3) / 4;
    if (r.pairs == 0 && i < turning) {
        const int32_t n = min(4, half - 4 * i);
        return {4 * i, half + 4 * i, n, n, 4 * i};
    }
    const int32_t a = r.pairs != 0 ? 8 * i : r.rot + 8 * (i - turning);
    return {a, a + 4, min(4, columns - a), max(0, min(4, columns - a - 4)), a < r.rot ? 4 * i : -1};
}

// The numbers of a piece of a head at x. QUADS: Rotary::quads, and whole quads of columns.
struct Numbers {
    float4 a, b;
};
template <bool QUADS>
__device__ inline float4 load_columns(const float* x, int32_t n) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if constexpr (QUADS) {
        if (n > 0) {
            v = mfr::dev::load_loose(x);
        }
    } else {
        v.x = n > 0 ? x[0] : 0.0f;
        v.y = n > 1 ? x[1] : 0.0f;
        v.z = n > 2 ? x[2] : 0.0f;
        v.w = n > 3 ? x[3] : 0.0f;
    }
    return v;
}
template <bool QUADS>
__device__ inline Numbers load_piece(const float* x, const Piece& p) {
    return {load_columns<QUADS>(x + p.a, p.na), load_columns<QUADS>(x + p.b, p.nb)};
}

// A pair turned, or as it is: each product and their sum rounded to fp32 as the formula stands, so that a key
// next to a border between two numbers of a cache falls as it does for any other program in fp32.
struct Pair {
    float own, other;
};
__device__ inline Pair turned(float own, float other, float2 t, bool turns) {
    return {turns ? own * t.x - other * t.y : own, turns ? other * t.x + own * t.y : other};
}

// Columns past the piece's stay zeros.
template <bool QUADS>
__device__ inline Numbers turned_piece(const Numbers& v, const Piece& p, const Rotary& r,
                                       const float2* table) {
    if (p.angles < 0) {
        return v;
    }
    const float2* t = table + p.angles;
    if (r.pairs != 0) {
        const bool a = p.a < r.rot, b = p.b < r.rot;
        const Pair p0 = turned(v.a.x, v.a.y, t[0], a);
        const Pair p1 = turned(v.a.z, v.a.w, t[1], p.a + 2 < r.rot);
        const Pair p2 = turned(v.b.x, v.b.y, t[2], b);
        const Pair p3 = turned(v.b.z, v.b.w, t[3], p.b + 2 < r.rot);
        return {make_float4(p0.own, p0.other, p1.own, p1.other),
                make_float4(p2.own, p2.other, p3.own, p3.other)};
    }
    const Pair p0 = turned(v.a.x, v.b.x, t[0], true);
    const Pair p1 = turned(v.a.y, v.b.y, t[1], QUADS || p.na > 1);
    const Pair p2 = turned(v.a.z, v.b.z, t[2], QUADS || p.na > 2);
    const Pair p3 = turned(v.a.w, v.b.w, t[3], QUADS || p.na > 3);
    return {make_float4(p0.own, p1.own, p2.own, p3.own),
            make_float4(p0.other, p1.other, p2.other, p3.other)};
}

} // namespace mfr::rotary::dev
