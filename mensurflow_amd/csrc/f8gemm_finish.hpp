// What follows mfr_f8gemm's kernels where they leave sums instead of outputs: ranges of the depth
// that are still to be added, or columns of a block of 128 that several workgroups hold.
#pragma once

#include "f8gemm_kernel.hpp"

namespace mfr::f8gemm {

// Adds the ranges in order and applies the epilogue. A workgroup takes 1024 columns of a row, a
// thread 4, 32 lanes a block of the 8-bit output.
template <bool GATED>
__global__ __launch_bounds__(256) void finish_kernel(Params p, int splits, uint32_t col_groups) {
    namespace dev = f8::dev;
    const int64_t row = blockIdx.x / col_groups;
    const int64_t col = static_cast<int64_t>(blockIdx.x % col_groups) * 1024 + 4 * threadIdx.x;
    const int64_t count = p.n - col;
    constexpr int kWeights = GATED ? 2 : 1;
    const float* at = p.partial + row * p.n + col;
    const int64_t step = p.m * p.n;
    float4 sum[kWeights];
#pragma unroll
    for (int w = 0; w < kWeights; ++w) {
        sum[w] = dev::load_quad(at + w * step, count);
    }
    for (int x = 1; x < splits; ++x) {
#pragma unroll
        for (int w = 0; w < kWeights; ++w) {
            const float4 y = dev::load_quad(at + (x * kWeights + w) * step, count);
            sum[w].x += y.x, sum[w].y += y.y, sum[w].z += y.z, sum[w].w += y.w;
        }
    }
    float v[4] = {sum[0].x, sum[0].y, sum[0].z, sum[0].w};
    if (!GATED && p.c0 != nullptr) {
        const float4 c0 = dev::load_quad(p.c0 + row * p.c0_rs + col, count);
        v[0] += p.beta * c0.x, v[1] += p.beta * c0.y;
        v[2] += p.beta * c0.z, v[3] += p.beta * c0.w;
    }
    if (!GATED && p.bias != nullptr) {
        const float4 bias = dev::load_quad(p.bias + col, count);
        v[0] += bias.x, v[1] += bias.y, v[2] += bias.z, v[3] += bias.w;
    }
    const float other[4] = {sum[kWeights - 1].x, sum[kWeights - 1].y, sum[kWeights - 1].z,
                            sum[kWeights - 1].w};
    for (int e = 0; e < 4; ++e) {
        v[e] = p.act == MFR_ACT_SILU ? silu(v[e]) : mfr::dev::activate(v[e], p.act);
        if constexpr (GATED) {
            v[e] = v[e] * other[e];
        }
        v[e] = e < count ? v[e] : 0.0f; // counts for nothing in the block's scale
    }
    const float4 y = make_float4(v[0], v[1], v[2], v[3]);
    if (p.c != nullptr) {
        dev::store_quad(p.c + row * p.c_rs + col, y, count);
    }
    if (p.q.values != nullptr) {
        dev::write_f8(p.q, row, col, p.n, y);
    }
}

inline void launch_finish(const mfr_stream& s, const Params& p, int64_t splits) {
    const int64_t col_groups = (p.n + 1023) / 1024;
    require(one_launch(p.m * col_groups, 256), "f8gemm: problem too large for one launch");
    const unsigned grid = static_cast<unsigned>(p.m * col_groups);
    const uint32_t groups = static_cast<uint32_t>(col_groups);
    if (p.up.values != nullptr) {
        finish_kernel<true><<<grid, 256, 0, s.stream>>>(p, static_cast<int>(splits), groups);
    } else {
        finish_kernel<false><<<grid, 256, 0, s.stream>>>(p, static_cast<int>(splits), groups);
    }
    check_launch("f8gemm finish_kernel");
}

} // namespace mfr::f8gemm
