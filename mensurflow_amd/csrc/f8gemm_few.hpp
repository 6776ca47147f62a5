// The form of mfr_f8gemm for few rows of A, where the weights' bytes bound the time: they go from
// memory straight to registers, once, in the layout of the matrix cores' operand, every wavefront a
// run of depths of its own.
//
// A lane of a wavefront takes, per block of 128 depths, two 16-byte pieces of one weight row (16
// rows, 64 neighbouring bytes of each per load) and the same pieces of its rows of A, widens both to
// bf16 and multiplies: 4 v_mfma_f32_16x16x32_bf16 per 16 x 16 block, added to the outer sum with the
// two scales. DEEP blocks are in flight. The wavefronts' sums are added through LDS in the order of
// the depths' runs, so nothing here needs memory of its own and a captured call is like any other.
// 1 x 4096 x 4096: 6.0 us, launch and 4 blocks a wavefront at memory's latency (tiles 26.7); gated
// 1 x 10240 x 4096: 17.3 us, 4.9 TB/s.
#pragma once

#include "f8gemm_kernel.hpp"

namespace mfr::f8gemm {

// A workgroup: 16 MT rows of A against 16 NT rows of each weight, WK wavefronts along the depth.
template <int MT, int NT, int WK, int DEEP, bool GATED>
__global__ __launch_bounds__(64 * WK) void few_rows_kernel(Params p) {
    constexpr int kWeights = GATED ? 2 : 1;
    constexpr int kTiles = kWeights * NT * MT;
    __shared__ float4 sums[WK][kTiles][64];

    const int lane = static_cast<int>(threadIdx.x % 64);
    const int wk = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64));
    const int r16 = lane % 16;
    const int g = lane / 16;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * NT);
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);

    // Rows past the matrices repeat their last one: their sums are not stored.
    const uint8_t* rows_a[MT];
    const float* scales_a[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t row = f8::least(m0 + 16 * i + r16, p.m - 1);
        rows_a[i] = p.a.values + row * p.a.rs;
        scales_a[i] = p.a.scales + row * p.a.srs;
    }
    const uint8_t* rows_b[kWeights][NT];
    const float* scales_b[kWeights];
#pragma unroll
    for (int w = 0; w < kWeights; ++w) {
        const Matrix& from = w == 1 ? p.up : p.b;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            rows_b[w][j] = from.values + f8::least(n0 + 16 * j + r16, p.n - 1) * from.rs;
        }
        // 16 NT divides 128: one block of columns.
        scales_b[w] = from.scales + f8::least(n0, p.n - 1) / kBlock * from.srs;
    }

    const int64_t depth_blocks = blocks_of(p.k);
    const int64_t last_piece = (p.k + 15) / 16 - 1;
    struct Block {
        uint4 a[MT][2];
        uint4 b[kWeights][NT][2];
        float sa[MT];
        float sb[kWeights];
    };
    Block ring[DEEP];
    const auto load = [&](Block& to, int64_t kb) __attribute__((always_inline)) {
        const int64_t at[2] = {f8::least(kb * 8 + g, last_piece) * 16,
                               f8::least(kb * 8 + 4 + g, last_piece) * 16};
#pragma unroll
        for (int w = 0; w < kWeights; ++w) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    to.b[w][j][h] = *reinterpret_cast<const uint4*>(rows_b[w][j] + at[h]);
                }
            }
            to.sb[w] = scales_b[w][kb * (w == 1 ? p.up.scs : p.b.scs)];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                to.a[i][h] = *reinterpret_cast<const uint4*>(rows_a[i] + at[h]);
            }
            to.sa[i] = scales_a[i][kb * p.a.scs];
        }
    };
    // Zeros for the depths behind k.
    const auto clear = [&](uint4 (&v)[2], int64_t left) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t words[4] = {v[h].x, v[h].y, v[h].z, v[h].w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int64_t bytes = left - 16 * (g + 4 * h) - 4 * x;
                words[x] &= bytes >= 4 ? ~0u : bytes <= 0 ? 0u : (1u << (8 * bytes)) - 1;
            }
            v[h] = make_uint4(words[0], words[1], words[2], words[3]);
        }
    };

    floatx4 acc[kWeights][NT][MT] = {};
    const auto multiply = [&](Block& s, int64_t kb) __attribute__((always_inline)) {
        if (kb + 1 == depth_blocks && p.k % kBlock != 0) {
            const int64_t left = p.k - kb * kBlock;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                clear(s.a[i], left);
            }
#pragma unroll
            for (int w = 0; w < kWeights; ++w) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    clear(s.b[w][j], left);
                }
            }
        }
        bf16x8 fa[MT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                fa[i][2 * h] = widen(s.a[i][h].x, s.a[i][h].y);
                fa[i][2 * h + 1] = widen(s.a[i][h].z, s.a[i][h].w);
            }
        }
#pragma unroll
        for (int w = 0; w < kWeights; ++w) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                bf16x8 fb[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    fb[2 * h] = widen(s.b[w][j][h].x, s.b[w][j][h].y);
                    fb[2 * h + 1] = widen(s.b[w][j][h].z, s.b[w][j][h].w);
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    floatx4 part = {};
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[t], fa[i][t], part, 0, 0,
                                                                       0);
                    }
                    const float scale = s.sa[i] * s.sb[w];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc[w][j][i][e] = fmaf(part[e], scale, acc[w][j][i][e]);
                    }
                }
            }
        }
    };
    // Wavefront wk takes a run of neighbouring blocks.
    const int64_t run = (depth_blocks + WK - 1) / WK;
    const int64_t begin = wk * run;
    const int64_t end = f8::least(begin + run, depth_blocks);
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
        if (begin + d < end) {
            load(ring[d], begin + d);
        }
    }
    for (int64_t kb = begin; kb < end; kb += DEEP) {
#pragma unroll
        for (int d = 0; d < DEEP; ++d) {
            if (kb + d < end) {
                multiply(ring[d], kb + d);
                if (kb + d + DEEP < end) {
                    load(ring[d], kb + d + DEEP);
                }
            }
        }
    }

#pragma unroll
    for (int w = 0; w < kWeights; ++w) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const floatx4 v = acc[w][j][i];
                sums[wk][(j * MT + i) * kWeights + w][lane] = make_float4(v[0], v[1], v[2], v[3]);
            }
        }
    }
    __syncthreads();
    // Block u = (j, i) falls to wavefront u % WK. A lane holds 4 neighbouring columns of one row.
    namespace dev = f8::dev;
    const auto total = [&](int u, int w) {
        float4 v = sums[0][u * kWeights + w][lane];
        for (int x = 1; x < WK; ++x) {
            const float4 y = sums[x][u * kWeights + w][lane];
            v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
        }
        return v;
    };
    for (int u = wk; u < NT * MT; u += WK) {
        const int64_t row = m0 + 16 * (u % MT) + r16;
        const int64_t col = n0 + 16 * (u / MT) + 4 * g;
        const int64_t count = row < p.m ? p.n - col : 0;
        float4 sum = total(u, 0);
        float v[4] = {sum.x, sum.y, sum.z, sum.w};
        float other[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        if constexpr (GATED) {
            sum = total(u, 1);
            other[0] = sum.x, other[1] = sum.y, other[2] = sum.z, other[3] = sum.w;
        } else {
            if (p.c0 != nullptr) {
                const float4 c0 = dev::load_quad(p.c0 + row * p.c0_rs + col, count);
                v[0] += p.beta * c0.x, v[1] += p.beta * c0.y;
                v[2] += p.beta * c0.z, v[3] += p.beta * c0.w;
            }
            if (p.bias != nullptr) {
                const float4 bias = dev::load_quad(p.bias + col, p.n - col);
                v[0] += bias.x, v[1] += bias.y, v[2] += bias.z, v[3] += bias.w;
            }
        }
        for (int e = 0; e < 4; ++e) {
            v[e] = p.act == MFR_ACT_SILU ? silu(v[e]) : mfr::dev::activate(v[e], p.act);
            if constexpr (GATED) {
                v[e] = v[e] * other[e];
            }
        }
        dev::store_quad(p.c + row * p.c_rs + col, make_float4(v[0], v[1], v[2], v[3]), count);
    }
}

template <int MT, int NT, int WK, int DEEP, bool GATED>
void launch_few(const mfr_stream& s, const Params& p) {
    const int64_t columns = 16 * NT;
    const int64_t x = (p.n + columns - 1) / columns;
    const int64_t y = (p.m + 16 * MT - 1) / (16 * MT);
    require(x < (int64_t{1} << 31) && y < 65536 && one_launch(x * y, 64 * WK),
            "f8gemm: problem too large for one launch");
    few_rows_kernel<MT, NT, WK, DEEP, GATED>
        <<<dim3(static_cast<unsigned>(x), static_cast<unsigned>(y)), 64 * WK, 0, s.stream>>>(p);
    check_launch("f8gemm few_rows_kernel");
}

} // namespace mfr::f8gemm
