// mfr_f8_quantize and mfr_rms_norm: passes over the rows of an fp32 matrix that end in e4m3 values
// with a scale per block (f8.hpp), in fp32, or in both.
#include "f8.hpp"

#include <algorithm>
#include <cmath>

namespace {

using mfr::dev::kWave;
using mfr::f8::kBlock;
using mfr::f8::Matrix;
namespace dev = mfr::f8::dev;

constexpr int kThreads = 256;
constexpr int kStep = 4 * kThreads; // columns per workgroup step

// A workgroup takes 1024 columns of a row at a time, a thread 4, 32 lanes a block: one read, one
// write, no LDS. 2000 x 1960: 6.0 us, 3.3 TB/s, of which launch and tail are half.
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(const float* x, int64_t x_rs,
                                                                 int64_t groups, int64_t cols,
                                                                 uint32_t col_groups, Matrix q) {
    for (int64_t i = blockIdx.x; i < groups; i += gridDim.x) {
        const int64_t r = i / col_groups;
        const int64_t col = (i - r * col_groups) * kStep + 4 * threadIdx.x;
        dev::write_f8(q, r, col, cols, dev::load_quad(x + r * x_rs + col, cols - col));
    }
}

// A workgroup per 128 x 128 block, all of it in registers between the one read and the one write:
// bound by memory. 16384 x 4096: 62 us, 5.4 TB/s.
__global__ __launch_bounds__(kThreads) void quantize_blocks_kernel(const float* x, int64_t x_rs,
                                                                   int64_t rows, int64_t cols,
                                                                   Matrix q, int64_t col_blocks) {
    __shared__ uint32_t tops[kThreads / 32];
    const int64_t rb = blockIdx.x / col_blocks;
    const int64_t cb = blockIdx.x % col_blocks;
    const int64_t col = cb * kBlock + 4 * (threadIdx.x % 32);
    const int64_t row = rb * kBlock + threadIdx.x / 32;
    float4 v[16];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int64_t r = row + 8 * i;
        v[i] = dev::load_quad(x + r * x_rs + col, r < rows ? cols - col : 0);
        top = mfr::f8::most(top, dev::magnitude(v[i]));
    }
    tops[threadIdx.x / 32] = dev::half_max(top); // the 32 lanes store one value
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) {
        top = mfr::f8::most(top, tops[i]);
    }
    const dev::Quotient by = dev::quotient_of(top);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int64_t r = row + 8 * i;
        if (r < rows && col < cols) {
            dev::store_bytes(q.values + r * q.rs + col, dev::pack(v[i], by), cols - col);
        }
    }
    if (threadIdx.x == 0) {
        q.scales[rb * q.srs + cb * q.scs] = dev::scale_of(top);
    }
}

struct NormParams {
    int64_t rows, cols;
    const float* x;
    int64_t x_rs;
    const float* residual;
    int64_t residual_rs;
    const float* weight;
    float* sum;
    int64_t sum_rs;
    float* out;
    int64_t out_rs;
    Matrix q; // values null: none
    float eps;

    // `count` rows from `first` on.
    NormParams from(int64_t first, int64_t count) const {
        NormParams n = *this;
        n.rows = count;
        n.x += first * x_rs;
        n.residual += residual != nullptr ? first * residual_rs : 0;
        n.sum += sum != nullptr ? first * sum_rs : 0;
        n.out += out != nullptr ? first * out_rs : 0;
        n.q.values += q.values != nullptr ? first * q.rs : 0;
        n.q.scales += q.values != nullptr ? first * q.srs : 0;
        return n;
    }
};

__device__ inline float4 add(float4 a, float4 b) {
    return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}

__device__ inline double squares(float4 v) {
    const double x = v.x, y = v.y, z = v.z, w = v.w;
    return fma(x, x, fma(y, y, fma(z, z, w * w)));
}

// Four columns from `col` on of row r in 8 bits, as dev::write_f8, from numbers before their rounding
// to fp32: no value is on the wrong side of a border between two codes.
__device__ inline void write_f8(const Matrix& q, int64_t r, int64_t col, int64_t cols,
                                const double (&y)[4]) {
    // Magnitudes as bits, a NaN on top (dev::magnitude).
    uint64_t top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        top = mfr::f8::most(top, static_cast<uint64_t>(__double_as_longlong(fabs(y[e]))));
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) {
        top = mfr::f8::most(top, static_cast<uint64_t>(__shfl_xor(
                                     static_cast<unsigned long long>(top), m, 64)));
    }
    if (col >= cols) {
        return;
    }
    const double largest = __longlong_as_double(static_cast<long long>(top));
    const double least = mfr::f8::kLeastScale;
    const double top_code = mfr::f8::kTop;
    const bool clamped = largest < top_code * least;
    const double by = clamped ? 1.0 / least : top_code / largest;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const double x = y[e] * by;
        const float near = static_cast<float>(x);
        v[e] = dev::to_odd(near, static_cast<float>(x - static_cast<double>(near)));
    }
    dev::store_bytes(q.values + r * q.rs + col, dev::pack(make_float4(v[0], v[1], v[2], v[3])),
                     cols - col);
    if (col % kBlock == 0) {
        q.scales[r * q.srs + col / kBlock * q.scs] =
            static_cast<float>(clamped ? least : largest / top_code);
    }
}

// The sum of v over a workgroup of WAVES wavefronts, in each thread: over the lanes by halves, then
// over the wavefronts in order.
template <int WAVES> __device__ inline double group_sum(double v, double* sums) {
    v = mfr::dev::wave_sum(v);
    if constexpr (WAVES > 1) {
        if (threadIdx.x % kWave == 0) {
            sums[threadIdx.x / kWave] = v;
        }
        __syncthreads();
        v = 0.0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            v += sums[i];
        }
    }
    return v;
}

__device__ inline double norm_scale(const NormParams& p, double squares) {
    return 1.0 / sqrt(squares / static_cast<double>(p.cols) + static_cast<double>(p.eps));
}

// What follows the sum of squares: four columns of the result, in the forms that are asked for.
__device__ inline void write_normed(const NormParams& p, int64_t r, int64_t col, float4 t,
                                    double scale, float4 w) {
    const int64_t count = p.cols - col;
    const float from[4] = {t.x, t.y, t.z, t.w};
    const float by[4] = {w.x, w.y, w.z, w.w};
    double y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        y[e] = e < count ? from[e] * scale * by[e] : 0.0; // behind the row 0 * scale may be NaN
    }
    if (p.out != nullptr) {
        dev::store_quad(p.out + r * p.out_rs + col,
                        make_float4(static_cast<float>(y[0]), static_cast<float>(y[1]),
                                    static_cast<float>(y[2]), static_cast<float>(y[3])),
                        count);
    }
    if (p.q.values != nullptr) {
        write_f8(p.q, r, col, p.cols, y);
    }
}

__device__ inline float4 weight_at(const NormParams& p, int64_t col) {
    return p.weight != nullptr ? dev::load_quad(p.weight + col, p.cols - col)
                               : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
}

// A row in the registers of THREADS threads, QUADS x 4 columns each: every element is read once,
// all of a thread's loads before the first use. A workgroup takes one row, or 4 where a wavefront
// holds a row. Bound by memory; the arithmetic, most of it in double, takes 57 % of the vector units'
// time at that rate with 8 bits out. With residual, sum and 8 bits: 16384 x 8192 335 us, 5.2 TB/s (two
// passes over the row 364), 1 x 4096 4.4 us (6.4); fp32 alone, 4093 x 1023 8.6 us (10.8).
template <int THREADS, int QUADS>
__global__ __launch_bounds__(THREADS == kWave ? 4 * kWave : THREADS) void rms_norm_kernel(
    NormParams p) {
    constexpr int kRows = THREADS == kWave ? 4 : 1;
    __shared__ double sums[THREADS / kWave];
    const int64_t r = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / THREADS;
    if (r >= p.rows) {
        return; // a whole wavefront, where that has a row of its own
    }
    const int64_t col0 = 4 * (threadIdx.x % THREADS);
    const float* x = p.x + r * p.x_rs;
    float4 t[QUADS];
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
        const int64_t col = col0 + i * 4 * THREADS;
        t[i] = dev::load_quad(x + col, p.cols - col);
    }
    if (p.residual != nullptr) {
        const float* residual = p.residual + r * p.residual_rs;
        float4 u[QUADS];
#pragma unroll
        for (int i = 0; i < QUADS; ++i) {
            const int64_t col = col0 + i * 4 * THREADS;
            u[i] = dev::load_quad(residual + col, p.cols - col);
        }
#pragma unroll
        for (int i = 0; i < QUADS; ++i) {
            t[i] = add(t[i], u[i]);
        }
    }
    if (p.sum != nullptr) {
#pragma unroll
        for (int i = 0; i < QUADS; ++i) {
            const int64_t col = col0 + i * 4 * THREADS;
            dev::store_quad(p.sum + r * p.sum_rs + col, t[i], p.cols - col);
        }
    }
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
        total += squares(t[i]);
    }
    const double scale = norm_scale(p, group_sum<THREADS / kWave>(total, sums));
#pragma unroll
    for (int i = 0; i < QUADS; ++i) {
        const int64_t col = col0 + i * 4 * THREADS;
        write_normed(p, r, col, t[i], scale, weight_at(p, col));
    }
}

// Rows of any length, a workgroup each, in two passes over them.
constexpr int kLongThreads = 1024;

__global__ __launch_bounds__(kLongThreads) void rms_norm_long_kernel(NormParams p) {
    __shared__ double sums[kLongThreads / kWave];
    const int64_t r = blockIdx.x;
    const float* x = p.x + r * p.x_rs;
    const float* residual = p.residual != nullptr ? p.residual + r * p.residual_rs : nullptr;
    float* sum = p.sum != nullptr ? p.sum + r * p.sum_rs : nullptr;
    double total = 0.0;
    for (int64_t col = 4 * threadIdx.x; col < p.cols; col += 4 * kLongThreads) {
        float4 t = dev::load_quad(x + col, p.cols - col);
        if (residual != nullptr) {
            t = add(t, dev::load_quad(residual + col, p.cols - col));
        }
        if (sum != nullptr) {
            dev::store_quad(sum + col, t, p.cols - col);
        }
        total += squares(t);
    }
    const double scale = norm_scale(p, group_sum<kLongThreads / kWave>(total, sums));
    for (int64_t c0 = 0; c0 < p.cols; c0 += 4 * kLongThreads) {
        const int64_t col = c0 + 4 * threadIdx.x;
        float4 t;
        if (sum != nullptr) {
            t = dev::load_quad(sum + col, p.cols - col);
        } else {
            t = dev::load_quad(x + col, p.cols - col);
            if (residual != nullptr) {
                t = add(t, dev::load_quad(residual + col, p.cols - col));
            }
        }
        write_normed(p, r, col, t, scale, weight_at(p, col));
    }
}

template <int THREADS, int QUADS> void launch_norm(const mfr_stream& s, const NormParams& p) {
    constexpr int kRows = THREADS == kWave ? 4 : 1;
    rms_norm_kernel<THREADS, QUADS>
        <<<static_cast<unsigned>((p.rows + kRows - 1) / kRows), kRows * THREADS, 0, s.stream>>>(p);
}

// The rows of one launch. A wavefront holds up to 1024 columns; longer rows go over 256 threads
// where there are rows for every compute unit, over 1024 where there are few and a row's own time
// counts.
void norm_rows(const mfr_stream& s, const NormParams& p) {
    const int64_t quads = (p.cols + 3) / 4;
    if (quads <= kWave * 4) {
        if (quads <= kWave) {
            launch_norm<kWave, 1>(s, p);
        } else if (quads <= kWave * 2) {
            launch_norm<kWave, 2>(s, p);
        } else {
            launch_norm<kWave, 4>(s, p);
        }
    } else if (quads <= 256 * 8 && p.rows > 2 * s.compute_units) {
        if (quads <= 256 * 2) {
            launch_norm<256, 2>(s, p);
        } else if (quads <= 256 * 4) {
            launch_norm<256, 4>(s, p);
        } else {
            launch_norm<256, 8>(s, p);
        }
    } else if (quads <= 1024) {
        launch_norm<1024, 1>(s, p);
    } else if (quads <= 1024 * 2) {
        launch_norm<1024, 2>(s, p);
    } else if (quads <= 1024 * 4) {
        launch_norm<1024, 4>(s, p);
    } else {
        rms_norm_long_kernel<<<static_cast<unsigned>(p.rows), kLongThreads, 0, s.stream>>>(p);
    }
    mfr::check_launch("rms_norm_kernel");
}

// The descriptor's checks (of shapes, layouts and pointers: no device is needed).
NormParams checked(const mfr_rms_norm_desc* desc) {
    using mfr::require;
    require(desc != nullptr, "rms_norm: null descriptor");
    const mfr_rms_norm_desc& d = *desc;
    require(d.rows >= 0 && d.cols >= 0, "rms_norm: negative dimension");
    require(d.eps >= 0.0f && std::isfinite(d.eps), "rms_norm: eps is negative or not finite");
    NormParams p{d.rows,   d.cols, d.x,      d.x_rs, d.residual, d.residual_rs,
                 d.weight, d.sum,  d.sum_rs, d.out,  d.out_rs,   Matrix{},
                 d.eps};
    if (d.out_f8.values != nullptr) {
        p.q = mfr::f8::checked(d.out_f8, d.rows, d.cols, 1, true, "rms_norm", "out_f8");
    }
    if (d.rows == 0 || d.cols == 0) {
        return p;
    }
    require(d.out != nullptr || d.out_f8.values != nullptr,
            "rms_norm: neither out nor out_f8 is given");
    require(d.x != nullptr, "rms_norm: null input");
    const auto apart = [&](const float* t, int64_t rs) { return t == nullptr || rs >= d.cols; };
    require(apart(d.x, d.x_rs) && apart(d.residual, d.residual_rs) && apart(d.sum, d.sum_rs) &&
                apart(d.out, d.out_rs),
            "rms_norm: a matrix has rows that overlap");
    require(d.sum == nullptr || d.sum != d.out, "rms_norm: sum and out are one array");
    const auto in_place = [&](const float* t, int64_t rs) {
        return t == nullptr ||
               ((t != d.x || rs == d.x_rs) && (t != d.residual || rs == d.residual_rs));
    };
    require(in_place(d.sum, d.sum_rs) && in_place(d.out, d.out_rs),
            "rms_norm: an output in place of an input needs its row stride");
    return p;
}

} // namespace

namespace mfr::f8 {

void quantize_rows(const mfr_stream& s, const float* x, int64_t x_rs, int64_t rows, int64_t cols,
                   const Matrix& q) {
    const int64_t col_groups = (cols + kStep - 1) / kStep;
    require(col_groups < (int64_t{1} << 32) && rows < (int64_t{1} << 62) / col_groups,
            "f8_quantize: matrix too large");
    const int64_t groups = rows * col_groups;
    quantize_rows_kernel<<<grid_blocks(groups, 1, int64_t{1} << 20), kThreads, 0, s.stream>>>(
        x, x_rs, groups, cols, static_cast<uint32_t>(col_groups), q);
    check_launch("quantize_rows_kernel");
}

} // namespace mfr::f8

extern "C" {

int mfr_f8_quantize(mfr_stream_t stream, int64_t rows, int64_t cols, const float* x, int64_t x_rs,
                    const mfr_f8_matrix* out) {
    return mfr::guarded([&] {
        mfr::require(out != nullptr, "f8_quantize: null output");
        mfr::require(rows >= 0 && cols >= 0, "f8_quantize: negative dimension");
        mfr::require(out->block_rows == 1 || out->block_rows == 128,
                     "f8_quantize: out needs block_rows 1 or 128");
        const Matrix q =
            mfr::f8::checked(*out, rows, cols, out->block_rows, true, "f8_quantize", "out");
        const bool empty = rows == 0 || cols == 0;
        mfr::require(empty || x != nullptr, "f8_quantize: null input");
        mfr::require(empty || x_rs >= cols, "f8_quantize: x has rows that overlap");
        auto& s = mfr::stream_of(stream);
        if (empty) {
            return;
        }
        if (out->block_rows == 1) {
            mfr::f8::quantize_rows(s, x, x_rs, rows, cols, q);
            return;
        }
        const int64_t col_blocks = mfr::f8::blocks_of(cols);
        const int64_t blocks = mfr::f8::blocks_of(rows) * col_blocks;
        mfr::require(mfr::one_launch(blocks, kThreads), "f8_quantize: matrix too large");
        quantize_blocks_kernel<<<static_cast<unsigned>(blocks), kThreads, 0, s.stream>>>(
            x, x_rs, rows, cols, q, col_blocks);
        mfr::check_launch("quantize_blocks_kernel");
    });
}

int mfr_rms_norm(mfr_stream_t stream, const mfr_rms_norm_desc* desc) {
    return mfr::guarded([&] {
        const NormParams p = checked(desc);
        auto& s = mfr::stream_of(stream);
        if (p.rows == 0 || p.cols == 0) {
            return;
        }
        // 2^21 rows a launch: fewer than 2^32 threads.
        constexpr int64_t kMostRows = int64_t{1} << 21;
        for (int64_t r = 0; r < p.rows; r += kMostRows) {
            norm_rows(s, p.from(r, std::min(p.rows - r, kMostRows)));
        }
    });
}

} // extern "C"
