// The cosine and sine of far and near positions (csrc/rotary_angle.hpp) against long double's, on the CPU.
#include "rotary_angle.hpp"

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>

using namespace mfr::rotary;

namespace {

double worst = 0.0; // of the bound

void check(int64_t position, double radians) {
    const Angle got = angle_of(static_cast<double>(position), quarters_of(radians));
    const long double w = static_cast<long double>(position) * radians;
    // The terms in fp32: half a step of x^7 / 5040 and of -1 / 5040, (pi / 4)^7 / 5040 2^-24 each, and less
    // of what follows. The step in quarter turns: two roundings of pi / 2, one of the quotient.
    const double off = 5e-12 + 1.8e-16 * std::fabs(static_cast<double>(w));
    const long double dc = std::fabs(got.cosine - std::cos(w)), ds = std::fabs(got.sine - std::sin(w));
    worst = std::fmax(worst, static_cast<double>(std::fmax(dc, ds)) / off);
    if (!(dc <= off && ds <= off)) {
        std::printf("rotary_angle_test: FAILED: position %lld, step %.17g: off by %.3Lg and %.3Lg of %.3g\n",
                    static_cast<long long>(position), radians, dc, ds, off);
        std::exit(1);
    }
}

} // namespace

int main() {
    constexpr int64_t kFar = int64_t{1} << 31;
    std::mt19937_64 rng(1);
    std::uniform_real_distribution<double> unit(0.0, 1.0);
    for (int i = 0; i < 1000000; ++i) {
        check(static_cast<int64_t>(std::exp(unit(rng) * std::log(2.0 * kFar))) - 1,
              std::exp(-unit(rng) * std::log(1e6)));
        check(static_cast<int64_t>(rng() % 200000) - 100000, std::pow(10000.0, -unit(rng)));
    }
    for (const int64_t position : {-kFar, -kFar + 1, int64_t{-1}, int64_t{0}, int64_t{1}, kFar - 1, kFar,
                                   kFar + (int64_t{1} << 30) - 1}) {
        for (const double radians : {0.0, -1.0, 1.0, 1e6, -1e6, 1.57079632679489661923, 0.785398163397448309616,
                                     3.14159265358979323846, 1e-300}) {
            check(position, radians);
        }
    }
    // The edges of a quarter's half, where series and quarter change.
    for (int i = -4000; i <= 4000; ++i) {
        for (int j = -2; j <= 2; ++j) {
            check(1, i * 0.785398163397448309616 + j * 1e-13);
        }
    }
    std::printf("rotary_angle_test passed (%.2f of the bound)\n", worst);
    return 0;
}
