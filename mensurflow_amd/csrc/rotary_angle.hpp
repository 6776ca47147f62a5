// The cosine and sine of a position's angle. No HIP header, so that the CPU tests run it on any values.
#pragma once

#include <cmath>
#include <cstdint>

#if defined(__HIPCC__)
#define MFR_ROTARY_BOTH __host__ __device__ inline
#else
#define MFR_ROTARY_BOTH inline
#endif

namespace mfr::rotary {

struct Angle {
    double cosine, sine;
};

// A step of `radians` a position, in quarter turns: within 1.5e-16 of itself.
inline double quarters_of(double radians) { return radians / 1.57079632679489661923; }

// A number that is made where it is used: those of the series, kept through the kernels' loops in every
// lane's registers, let fewer wavefronts fit (37 ragged pieces into fp32 15.7 us, 13.0 so).
MFR_ROTARY_BOTH double constant(double v) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("" : "+s"(v));
#endif
    return v;
}

// Of position * quarters quarter turns (less than 2^51). Behind 1.5 * 2^52 the sum's last bits are the nearest
// whole one's. What is left of it is one rounding of the exact product, so that a far position's angle is
// as good as its step; it is at most pi / 4, where the Taylor series to x^13 and x^14 are 1e-15 off. Their
// terms from x^7 and x^8 on are summed in fp32, 5e-12 off at most. The quarter then chooses sign and place.
MFR_ROTARY_BOTH Angle angle_of(double position, double quarters) {
    constexpr double kWhole = 6755399441055744.0;
    const double behind = fma(position, quarters, kWhole);
    const int quarter = static_cast<int>(__builtin_bit_cast(int64_t, behind) & 3);
    const double x = fma(position, quarters, kWhole - behind) * 1.57079632679489661923;
    const double z = x * x;
    const float zf = static_cast<float>(z);
    float sf = fmaf(zf, 1.0f / 6227020800.0f, -1.0f / 39916800.0f);
    sf = fmaf(zf, sf, 1.0f / 362880.0f);
    sf = fmaf(zf, sf, -1.0f / 5040.0f);
    double s = fma(z, static_cast<double>(sf), constant(1.0 / 120.0));
    s = fma(z, s, constant(-1.0 / 6.0));
    s = fma(x * z, s, x);
    float cf = fmaf(zf, -1.0f / 87178291200.0f, 1.0f / 479001600.0f);
    cf = fmaf(zf, cf, -1.0f / 3628800.0f);
    cf = fmaf(zf, cf, 1.0f / 40320.0f);
    double c = fma(z, static_cast<double>(cf), constant(-1.0 / 720.0));
    c = fma(z, c, constant(1.0 / 24.0));
    c = fma(z, c, -0.5);
    c = fma(z, c, 1.0);
    const double a = (quarter & 1) != 0 ? s : c;
    const double b = (quarter & 1) != 0 ? c : s;
    return {quarter == 1 || quarter == 2 ? -a : a, quarter >= 2 ? -b : b};
}

} // namespace mfr::rotary
