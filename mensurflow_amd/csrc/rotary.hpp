// Rotation by position (mfr_rotary), for the kernels that turn queries and keys.
//
// A workgroup works on one token at a time: the cosines and sines of its rot / 2 angles are made once,
// into LDS, for all heads of the token. A lane holds 4 columns of a head from 4 lane on and loads its
// pairs' other halves as well, so that every layout has one form; the second loads find the first ones'
// lines in the L1 cache.
#pragma once

#include "common.hpp"

#include <cmath>

namespace mfr::rotary {

constexpr int kMostPairs = MFR_ROTARY_MOST / 2;

// As a kernel's argument.
struct Rotary {
    int32_t rot;
    int32_t pairs; // neighbours turn together
    float amplitude;
    int32_t quads; // no four columns straddle a half's, the rotated part's or the head's end
    double turns[kMostPairs]; // a position, in whole turns
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
    out.quads = d % 4 == 0 && r.rot % (out.pairs != 0 ? 4 : 8) == 0;
    for (int i = 0; i < r.rot / 2; ++i) {
        require(std::abs(r.steps[i]) <= 1e6, at + "has steps past 10^6 or not finite");
        out.turns[i] = r.steps[i] / 6.283185307179586476925;
    }
    return out;
}

} // namespace mfr::rotary

namespace mfr::rotary::dev {

// (cosine, sine) of position * turns whole turns: the distance to the nearest quarter of a turn is
// taken in double and is at most pi / 4, where the Taylor series to x^10 and x^9 are 1e-9 off; the
// quarter then chooses sign and place.
__device__ inline float2 angle_of(double position, double turns) {
    const double quarters = 4.0 * (position * turns);
    const double whole = rint(quarters);
    const float x = static_cast<float>(quarters - whole) * 1.57079632679489662f;
    const int quarter = static_cast<int>(whole - 4.0 * floor(0.25 * whole));
    const float z = x * x;
    float s = fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
    s = fmaf(z, s, 8.33333333e-3f);
    s = fmaf(z, s, -1.66666667e-1f);
    s = fmaf(x * z, s, x);
    float c = fmaf(z, -2.75573192e-7f, 2.48015873e-5f);
    c = fmaf(z, c, -1.38888889e-3f);
    c = fmaf(z, c, 4.16666667e-2f);
    c = fmaf(z * z, c, fmaf(z, -0.5f, 1.0f));
    const float a = (quarter & 1) != 0 ? s : c;
    const float b = (quarter & 1) != 0 ? c : s;
    return make_float2(quarter == 1 || quarter == 2 ? -a : a, quarter >= 2 ? -b : b);
}

// The angles of a token into `table` [rot / 2], by all threads of the workgroup. A barrier has to
// follow.
__device__ inline void fill_angles(const Rotary& r, int64_t position, bool backward, float2* table,
                                   int threads) {
    for (int i = threadIdx.x; i < r.rot / 2; i += threads) {
        const float2 t = angle_of(static_cast<double>(position), r.turns[i]);
        table[i] = make_float2(r.amplitude * t.x, r.amplitude * (backward ? -t.y : t.y));
    }
}

// One column: own * cos +- other * sin.
__device__ inline float turned(float own, float other, float2 t, bool first) {
    return first ? fmaf(own, t.x, -(other * t.y)) : fmaf(own, t.x, other * t.y);
}

// Up to 4 columns from c on (c < d, a multiple of 4) of the head of d columns at x, turned. QUADS:
// Rotary::quads.
template <bool QUADS>
__device__ inline float4 turned_quad(const float* x, int c, int d, const Rotary& r,
                                     const float2* table) {
    const int half = r.rot / 2;
    if constexpr (QUADS) {
        float4 v = mfr::dev::load_loose(x + c);
        if (c < r.rot) {
            if (r.pairs != 0) {
                const float2 t0 = table[c / 2], t1 = table[c / 2 + 1];
                return make_float4(turned(v.x, v.y, t0, true), turned(v.y, v.x, t0, false),
                                   turned(v.z, v.w, t1, true), turned(v.w, v.z, t1, false));
            }
            const bool first = c < half;
            const float4 o = mfr::dev::load_loose(x + (first ? c + half : c - half));
            const float2* t = table + (first ? c : c - half);
            v = make_float4(turned(v.x, o.x, t[0], first), turned(v.y, o.y, t[1], first),
                            turned(v.z, o.z, t[2], first), turned(v.w, o.w, t[3], first));
        }
        return v;
    } else {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int at = c + e;
            v[e] = at < d ? x[at] : 0.0f;
            if (at < r.rot) {
                const bool first = r.pairs != 0 ? at % 2 == 0 : at < half;
                const int step = r.pairs != 0 ? 1 : half;
                const int pair = r.pairs != 0 ? at / 2 : first ? at : at - half;
                v[e] = turned(v[e], x[first ? at + step : at - step], table[pair], first);
            }
        }
        return make_float4(v[0], v[1], v[2], v[3]);
    }
}

// Between a wavefront's loads of a head and its stores over it: no store is moved up into one side of
// a branch whose other side still loads.
__device__ inline void loads_before_stores() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
}

} // namespace mfr::rotary::dev
