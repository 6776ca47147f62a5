// 8-bit matrices (mfr_f8_matrix): what the kernels that write and read them share.
//
// A block of values x is held as e4m3 numbers v and one fp32 scale s, x ~ v s. With the largest
// magnitude of the block put on e4m3's largest number, 448, a value is off by at most half a step:
// 2^-4 of itself, or 2^-10 s below the least normal number 2^-6. The scale is at least 2^-126, so
// that its reciprocal is a normal number; blocks below 448 2^-126 lose bits there.
#pragma once

#include "common.hpp"

#include <string>

namespace mfr::f8 {

constexpr int kBlock = MFR_F8_BLOCK;
constexpr float kTop = 448.0f;
constexpr float kLeastScale = 0x1p-126f;

// A tile's rows (up to 128), and 64 rows' scales, are addressed with 31 and 32 bits.
constexpr int64_t kMostRowBytes = int64_t{1} << 24;
constexpr int64_t kMostScaleStride = int64_t{1} << 23;

// More rows, or column blocks of scales further apart, are no memory's: their products stay inside
// 64 bits.
constexpr int64_t kMostRows = int64_t{1} << 40;
constexpr int64_t kMostScaleStep = int64_t{1} << 40;

// Of two values of one type. (HIP's own min and max take 64-bit values for ints in host code.)
template <typename T> __host__ __device__ constexpr T least(T a, T b) { return b < a ? b : a; }
template <typename T> __host__ __device__ constexpr T most(T a, T b) { return a < b ? b : a; }

constexpr int64_t blocks_of(int64_t n) { return (n + kBlock - 1) / kBlock; }

// One matrix as a kernel's argument.
struct Matrix {
    uint8_t* values;
    int64_t rs;
    float* scales;
    int64_t srs, scs;
};

// Checks `d` as a [rows, cols] matrix with `block_rows`, and takes it over. An empty matrix may
// have null pointers and any strides: it is taken over with none, since a kernel forms addresses and
// a buffer's size from them also where the depth is 0 and nothing is read.
inline Matrix checked(const mfr_f8_matrix& d, int64_t rows, int64_t cols, int block_rows,
                      bool output, const char* what, const char* name) {
    const std::string at = std::string(what) + ": " + name;
    require(d.block_rows == 1 || d.block_rows == 128, at + " needs block_rows 1 or 128");
    if (d.block_rows != block_rows) {
        throw Error(MFR_E_UNSUPPORTED,
                    at + " is taken with block_rows " + std::to_string(block_rows) + " only");
    }
    if (rows == 0 || cols == 0) {
        return {d.values, 0, d.scales, 0, 0};
    }
    const Matrix m{d.values, d.rs, d.scales, d.scales_rs, d.scales_cs};
    require(d.values != nullptr && d.scales != nullptr, at + " has a null pointer");
    require(rows <= kMostRows, at + " has too many rows");
    require(d.rs >= cols, at + " has rows that overlap");
    if (d.rs > kMostRowBytes || d.scales_rs > kMostScaleStride || d.scales_cs > kMostScaleStep) {
        throw Error(MFR_E_UNSUPPORTED, at + " has rows or scales that lie too far apart");
    }
    require(d.scales_rs >= 0 && d.scales_cs >= 0, at + " has negative scale strides");
    if (!aligned16(d.values) || d.rs % 16 != 0) {
        throw Error(MFR_E_UNSUPPORTED, at + " needs 16-byte aligned rows");
    }
    if (output) {
        // No two scales in one place.
        const int64_t r = (rows + block_rows - 1) / block_rows;
        const int64_t c = blocks_of(cols);
        const auto apart = [](int64_t inner, int64_t count, int64_t outer, int64_t others) {
            return (count == 1 || inner >= 1) && (others == 1 || outer > inner * (count - 1));
        };
        require(apart(d.scales_rs, r, d.scales_cs, c) || apart(d.scales_cs, c, d.scales_rs, r),
                at + " has scales that overlap");
    }
    return m;
}

// x in 8 bits, a scale per row and 128 columns (mfr_f8_quantize's launch).
void quantize_rows(const mfr_stream& s, const float* x, int64_t x_rs, int64_t rows, int64_t cols,
                   const Matrix& q);

} // namespace mfr::f8

namespace mfr::f8::dev {

// A magnitude as its bits, which order like the magnitude with infinity and then NaN on top: an
// unsigned maximum over a block finds its NaN where fmaxf would pass it by.
__device__ inline uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ inline uint32_t magnitude(float4 v) {
    return most(most(magnitude(v.x), magnitude(v.y)), most(magnitude(v.z), magnitude(v.w)));
}

// The block's scale from its largest magnitude's bits; NaN stays.
__device__ inline float scale_of(uint32_t top) {
    const float s = __uint_as_float(top) / kTop;
    return s < kLeastScale ? kLeastScale : s;
}

// Four values in e4m3, the first in the low byte (v_cvt_pk_fp8_f32: nearest, ties to even).
__device__ inline uint32_t pack(float4 v) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(v.x, v.y, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(v.z, v.w, w, true);
    return static_cast<uint32_t>(w);
}

// `near`, a float next to or at a number that lies `beyond` (its sign alone counts) past it, as the
// one of the number's neighbours whose last bit is set; `near` itself if it is the number. A later
// rounding to fewer bits then goes the number's way.
__device__ inline float to_odd(float near, float beyond) {
    const int bits = __float_as_int(near);
    const int step = (bits ^ __float_as_int(beyond)) >> 31 | 1; // away from zero, or towards it
    return __int_as_float((beyond > 0.0f || beyond < 0.0f) && (bits & 1) == 0 ? bits + step : bits);
}

// What takes the values x of a block to x / s, s = max(top / 448, 2^-126) unrounded: the e4m3 value of
// x is the nearest to that quotient, as if there were no rounding between.
struct Quotient {
    float up;      // a power of two that brings top to [4, 8)
    float top;     // top up
    float inverse; // 448 / (top up), within 2 units of the last place
};

__device__ inline Quotient quotient_of(uint32_t top) {
    if (__uint_as_float(top) < kTop * kLeastScale) {
        return {0x1p126f, kTop, 1.0f};
    }
    if (top >= 0x7f800000u) { // with an infinity, the others are 0; with a NaN, all are NaN
        return {top == 0x7f800000u ? 0.0f : __uint_as_float(top), 0.0f, 1.0f};
    }
    const float up = __uint_as_float((256u - (top >> 23)) << 23);
    const float at = __uint_as_float(top) * up;
    return {up, at, kTop * __builtin_amdgcn_rcpf(at)};
}

// x / s, its last bit as to_odd() has it. p top and 448 x are compared exactly: the first as two
// floats, their difference then fits one.
__device__ inline float quotient(float x, const Quotient& by) {
    const float v = x * by.up;
    const auto beyond = [&](float p) {
        const float product = p * by.top;
        return fmaf(v, kTop, -product) - fmaf(p, by.top, -product);
    };
    float p = v * by.inverse;
    // Within 3 units of the last place; then within one.
    p = fmaf(beyond(p) * by.inverse, 1.0f / kTop, p);
    return copysignf(to_odd(p, beyond(p)), x); // -0 + 0 above is 0
}

// Four values of a block in e4m3. A product with 448 / top, rounded, is within 4 units of the last
// place of the quotient: where a little less and a little more of it round alike, the quotient does
// too. Otherwise, 2 values in 10^5, it is taken exactly.
__device__ inline uint32_t pack(float4 v, const Quotient& by) {
    const float less = by.up * by.inverse * (1.0f - 0x1p-20f);
    const float more = by.up * by.inverse * (1.0f + 0x1p-20f);
    const uint32_t low = pack(make_float4(v.x * less, v.y * less, v.z * less, v.w * less));
    const uint32_t high = pack(make_float4(v.x * more, v.y * more, v.z * more, v.w * more));
    if (low == high) {
        return low;
    }
    return pack(make_float4(quotient(v.x, by), quotient(v.y, by), quotient(v.z, by),
                            quotient(v.w, by)));
}

// Stores the first `count` (up to 4) bytes of w at p, which is 4-byte aligned.
__device__ inline void store_bytes(uint8_t* p, uint32_t w, int64_t count) {
    if (count >= 4) {
        *reinterpret_cast<uint32_t*>(p) = w;
        return;
    }
    for (int64_t e = 0; e < count; ++e) {
        p[e] = static_cast<uint8_t>(w >> (8 * e));
    }
}

// The largest of v over the 32 lanes of a half wavefront, in each of them.
__device__ inline uint32_t half_max(uint32_t v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
        v = most(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), m, 64)));
    }
    return v;
}

// Four columns from `col` on of row r, in 8 bits. 32 lanes hold a block: columns past the row are
// zeros and count for nothing.
__device__ inline void write_f8(const Matrix& q, int64_t r, int64_t col, int64_t cols, float4 v) {
    const uint32_t top = half_max(magnitude(v));
    if (col < cols) {
        store_bytes(q.values + r * q.rs + col, pack(v, quotient_of(top)), cols - col);
        if (col % kBlock == 0) {
            q.scales[r * q.srs + col / kBlock * q.scs] = scale_of(top);
        }
    }
}

// Up to four floats of a row from p on, zeros behind `count`. 4-byte alignment.
__device__ inline float4 load_quad(const float* p, int64_t count) {
    if (count >= 4) {
        return mfr::dev::load_loose(p);
    }
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (count > 0) {
        v.x = p[0];
    }
    if (count > 1) {
        v.y = p[1];
    }
    if (count > 2) {
        v.z = p[2];
    }
    return v;
}

__device__ inline void store_quad(float* p, float4 v, int64_t count) {
    if (count >= 4) {
        mfr::dev::store_loose(p, v);
        return;
    }
    if (count > 0) {
        p[0] = v.x;
    }
    if (count > 1) {
        p[1] = v.y;
    }
    if (count > 2) {
        p[2] = v.z;
    }
}

} // namespace mfr::f8::dev
