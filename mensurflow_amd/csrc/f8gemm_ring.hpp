// The form of mfr_f8gemm for products of some tens to some hundreds of rows, or of few rows against
// weights of tens of megabytes: there is a tile a CU or less, and what bounds the time is how fast
// bytes reach that CU. So the tiles are small enough to give every CU one, and the depth's slices
// pass through a ring in LDS that keeps 64 to 100 KB of copies under way without a register.
//
// Measured at 128 x 4096 x 4096: 12.4 us, without the multiplication 11.0, without the copies 10.0;
// a CU's LDS fills at 56 GB/s then, 0.4 of the nominal 64 bytes a clock: a ring of two turns has no copy
// under way while it waits, and the scalar registers of the offsets are spilled in most of these loops.
// few_rows_kernel, whose wavefronts load for themselves: 16.5 us.
// 32 x 16384 x 4096: 14.4 us, 4.8 TB/s of memory (19.9). 128 x 5120 x 4096: 15.4 (28.8). 256 x 4096 x
// 4096: 16.0 (23.9). Gated, 256 x 2048 x 4096: 17.1 (23.8). Two workgroups on a CU with half the
// ring each win where one would leave a second round: 128 x 14336 x 4096 25.2 against 30.1.
#pragma once

#include "f8gemm_kernel.hpp"

namespace mfr::f8gemm {

// The wavefronts of a SIMD: of the one workgroup whose ring fits the 160 KB of LDS, or of two.
constexpr int ring_waves(int wm, int wn, int wk, int turns, bool gated) {
    const int rows = 32 * wm + 32 * wn * (gated ? 2 : 1);
    const int bytes = turns * wk * (rows * 128 + (gated ? 3 : 2) * 256);
    const int waves = wm * wn * wk * (2 * bytes <= 160 * 1024 ? 2 : 1);
    return (waves + 3) / 4;
}

// A workgroup: 32 WM rows of A against 32 WN rows of each weight, WK slices of the depth a turn, a
// wavefront for each 32 x 32 block of each slice. TURNS turns' slices lie in LDS, all but one under
// way. The wavefronts' sums are added through LDS in the order of their slices.
template <int WM, int WN, int WK, int TURNS, bool GATED>
__global__ __launch_bounds__(64 * WM * WN * WK, ring_waves(WM, WN, WK, TURNS, GATED)) void ring_kernel(
    Params p) {
    constexpr int kWeights = GATED ? 2 : 1;
    constexpr int kWaves = WM * WN * WK;
    constexpr int kRowsA = 32 * WM;
    constexpr int kRowsB = 32 * WN;
    // Rounds of copies of a turn, 8 rows a wavefront: of A's rows, and of each weight's.
    constexpr int kRoundsA = WK * kRowsA / 8 / kWaves;
    constexpr int kRoundsB = WK * kRowsB / 8 / kWaves;
    constexpr int kRounds = kRoundsA + kWeights * kRoundsB;
    static_assert(kRoundsA * 8 * kWaves == WK * kRowsA && kRoundsB * 8 * kWaves == WK * kRowsB &&
                      kWaves % 2 == 0,
                  "whole rounds of copies; a wavefront's groups of 8 rows are all odd or all even");
    static_assert(kRowsA <= 64 && kBlock % kRowsB == 0, "one copy of A's scales, one block of B's");
    struct Turn {
        uint4 a[WK][kRowsA * 8];
        uint4 b[kWeights][WK][kRowsB * 8];
        float scales[WK][1 + kWeights][64];
    };
    __shared__ __align__(16) Turn ring[TURNS];

    const int lane = static_cast<int>(threadIdx.x % 64);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64));
    const int wk = wave % WK;
    const int wm = wave / WK % WM;
    const int wn = wave / WK / WM;
    const int r32 = lane % 32;
    const int half = lane / 32;

    // Workgroup -> tile: consecutive ones on one XCD, rows fastest: an XCD's L2 reads its columns'
    // weights once.
    const uint32_t total = p.tiles_m * p.tiles_n;
    const uint32_t per_xcd = total / 8;
    const uint32_t logical =
        blockIdx.x < per_xcd * 8 ? blockIdx.x % 8 * per_xcd + blockIdx.x / 8 : blockIdx.x;
    const int64_t m0 = static_cast<int64_t>(logical % p.tiles_m) * kRowsA;
    const int64_t n0 = static_cast<int64_t>(logical / p.tiles_m) * kRowsB;

    const int blocks = static_cast<int>(blocks_of(p.k)); // rows are at most 2^24 bytes
    const int turns = (blocks + WK - 1) / WK;
    // As in tile_kernel: a resource from the tile's first row to the matrix's end; rows past it are
    // zeros, and so is what an offset of kNothing reads. (Slices past the last in the last turn are
    // whatever lies there, and are not multiplied.)
    constexpr uint32_t kNothing = 0x80000000u;
    const int64_t row_bytes = (p.k + 15) / 16 * 16;
    const auto operand = [&](const Matrix& m, int64_t row, int64_t rows) {
        const int64_t bytes = (rows - row - 1) * m.rs + row_bytes;
        return resource(m.values + row * m.rs,
                        static_cast<uint32_t>(f8::least(bytes, static_cast<int64_t>(kNothing))));
    };
    const intx4 from_a = operand(p.a, m0, p.m);
    const intx4 from_b = operand(p.b, n0, p.n);
    const intx4 from_up = GATED ? operand(p.up, n0, p.n) : intx4{};
    const uint32_t a_rs = static_cast<uint32_t>(p.a.rs);
    const uint32_t b_rs = static_cast<uint32_t>(p.b.rs);
    const uint32_t up_rs = static_cast<uint32_t>(p.up.rs);
    // Piece c of row r lies at place c ^ (r / 2 % 8).
    const uint32_t lane_row = static_cast<uint32_t>(lane) / 8;
    const uint32_t lane_piece =
        static_cast<uint32_t>((lane ^ (wave % 2 * 4 + lane / 16)) % 8) * 16;
    const uint32_t lane_a = lane_row * a_rs + lane_piece;
    const uint32_t lane_b = lane_row * b_rs + lane_piece;
    const uint32_t lane_up = lane_row * up_rs + lane_piece;
    // Of `rows` rows a slice, the offset of the 8 that round x gives this wavefront.
    const auto group_offset = [&](int x, int rows, uint32_t rs) __attribute__((always_inline)) {
        const int group = x * kWaves + wave;
        return static_cast<uint32_t>(group % (rows / 8) * 8) * rs +
               static_cast<uint32_t>(group / (rows / 8)) * kBlock;
    };
    // Wavefront w < WK copies the scales of slice w: A's rows, then a weight's one.
    const auto scale_source = [&](const Matrix& m, int64_t first) {
        const uint64_t at = reinterpret_cast<uint64_t>(m.scales + first * m.srs + wave * m.scs);
        const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(at));
        const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<int>(at >> 32));
        return static_cast<uint64_t>(hi) << 32 | lo;
    };
    uint64_t scales_a = scale_source(p.a, m0);
    uint64_t scales_b = scale_source(p.b, n0 / kBlock);
    uint64_t scales_up = GATED ? scale_source(p.up, n0 / kBlock) : 0;
    const uint32_t scale_offset =
        static_cast<uint32_t>(f8::least(static_cast<int64_t>(lane % kRowsA), p.m - 1 - m0)) *
        static_cast<uint32_t>(p.a.srs) * 4;
    constexpr int kScaleCopies = 1 + kWeights;
    const auto copy = [&](Turn& to, int turn) __attribute__((always_inline)) {
        if (wave < WK) {
            const uint32_t bytes = turn * WK + wave < blocks ? 0xffffffffu : 0u;
            copy_to_lds<4>(resource(reinterpret_cast<const void*>(scales_a), bytes), scale_offset, 0,
                           to.scales[wave][0]);
            copy_to_lds<4>(resource(reinterpret_cast<const void*>(scales_b), bytes), 0, 0,
                           to.scales[wave][1]);
            scales_a += static_cast<uint64_t>(p.a.scs) * (4 * WK);
            scales_b += static_cast<uint64_t>(p.b.scs) * (4 * WK);
            if constexpr (GATED) {
                copy_to_lds<4>(resource(reinterpret_cast<const void*>(scales_up), bytes), 0, 0,
                               to.scales[wave][2]);
                scales_up += static_cast<uint64_t>(p.up.scs) * (4 * WK);
            }
        }
        const uint32_t depth = turn < turns ? static_cast<uint32_t>(turn) * (WK * kBlock) : kNothing;
#pragma unroll
        for (int x = 0; x < kRoundsA; ++x) {
            copy_to_lds<16>(from_a, lane_a, depth + group_offset(x, kRowsA, a_rs),
                            &to.a[0][0] + (x * kWaves + wave) * 64);
        }
#pragma unroll
        for (int x = 0; x < kRoundsB; ++x) {
            copy_to_lds<16>(from_b, lane_b, depth + group_offset(x, kRowsB, b_rs),
                            &to.b[0][0][0] + (x * kWaves + wave) * 64);
        }
        if constexpr (GATED) {
#pragma unroll
            for (int x = 0; x < kRoundsB; ++x) {
                copy_to_lds<16>(from_up, lane_up, depth + group_offset(x, kRowsB, up_rs),
                                &to.b[1][0][0] + (x * kWaves + wave) * 64);
            }
        }
    };

    const int row_a = wm * 32 + r32;
    const int row_b = wn * 32 + r32;
    floatx16 acc[kWeights] = {};
    uint4 raw[1 + kWeights][4];
    float sa = 0.0f;
    float sb[kWeights] = {};
    const auto read = [&](const Turn& here) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int at = (4 * half + q) ^ (r32 / 2 % 8);
            raw[0][q] = here.a[wk][row_a * 8 + at];
#pragma unroll
            for (int w = 0; w < kWeights; ++w) {
                raw[1 + w][q] = here.b[w][wk][row_b * 8 + at];
            }
        }
        sa = here.scales[wk][0][row_a];
#pragma unroll
        for (int w = 0; w < kWeights; ++w) {
            sb[w] = here.scales[wk][1 + w][0];
        }
    };
    const auto multiply = [&](int kb) __attribute__((always_inline)) {
        if (kb + 1 == blocks && p.k % kBlock != 0) {
            // Zeros for the depths behind k.
            const int depths = static_cast<int>(p.k % kBlock) - 64 * half;
#pragma unroll
            for (int o = 0; o < 1 + kWeights; ++o) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t words[4] = {raw[o][q].x, raw[o][q].y, raw[o][q].z, raw[o][q].w};
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int bytes = depths - 16 * q - 4 * x;
                        words[x] &= bytes >= 4 ? ~0u : bytes <= 0 ? 0u : (1u << (8 * bytes)) - 1;
                    }
                    raw[o][q] = make_uint4(words[0], words[1], words[2], words[3]);
                }
            }
        }
        floatx16 part[kWeights] = {};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const bf16x8 a0 = widen(raw[0][q].x, raw[0][q].y);
            const bf16x8 a1 = widen(raw[0][q].z, raw[0][q].w);
#pragma unroll
            for (int w = 0; w < kWeights; ++w) {
                part[w] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                    widen(raw[1 + w][q].x, raw[1 + w][q].y), a0, part[w], 0, 0, 0);
                part[w] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                    widen(raw[1 + w][q].z, raw[1 + w][q].w), a1, part[w], 0, 0, 0);
            }
        }
#pragma unroll
        for (int w = 0; w < kWeights; ++w) {
            const float scale = sa * sb[w];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                acc[w][e] = fmaf(part[w][e], scale, acc[w][e]);
            }
        }
    };

#pragma unroll
    for (int t = 0; t < TURNS - 1; ++t) {
        copy(ring[t], t);
    }
    for (int turn = 0; turn < turns; turn += TURNS) {
#pragma unroll
        for (int t = 0; t < TURNS; ++t) {
            if (turn + t < turns) {
                if (wave < WK) {
                    wait_copies<(TURNS - 2) * (kRounds + kScaleCopies)>();
                } else {
                    wait_copies<(TURNS - 2) * kRounds>();
                }
                bare_barrier();
                read(ring[t]);
                copy(ring[(t + TURNS - 1) % TURNS], turn + t + TURNS - 1);
                if ((turn + t) * WK + wk < blocks) {
                    multiply((turn + t) * WK + wk);
                }
            }
        }
    }
    wait_copies<0>();
    __syncthreads();

    // The sums: quad x of a lane (columns 8 x + 4 half on) of row r32. Its place among a row's 8
    // quads is (2 x + half) ^ (r32 / 2 % 8).
    float4(*const sums)[32 * 8] = reinterpret_cast<float4(*)[32 * 8]>(&ring);
    static_assert(sizeof(ring) >= sizeof(float4) * 32 * 8 * kWaves * kWeights, "all sums");
#pragma unroll
    for (int w = 0; w < kWeights; ++w) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            sums[wave * kWeights + w][r32 * 8 + ((2 * x + half) ^ (r32 / 2 % 8))] =
                make_float4(acc[w][4 * x], acc[w][4 * x + 1], acc[w][4 * x + 2], acc[w][4 * x + 3]);
        }
    }
    __syncthreads();
    namespace dev = f8::dev;
    const auto total_of = [&](int block, int at, int w) {
        float4 v = sums[block * WK * kWeights + w][at];
#pragma unroll
        for (int x = 1; x < WK; ++x) {
            const float4 y = sums[(block * WK + x) * kWeights + w][at];
            v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
        }
        return v;
    };
    // Quads in the order of rows. With 128 columns half a wavefront holds a row's block, and makes
    // its 8 bits; otherwise they are another launch's.
    constexpr int kQuads = 8 * WN;
    for (int i = static_cast<int>(threadIdx.x); i < kRowsA * kQuads; i += 64 * kWaves) {
        const int r = i / kQuads;
        const int quad = i % kQuads;
        const int block = quad / 8 * WM + r / 32;
        const int at = r % 32 * 8 + ((quad % 8) ^ (r / 2 % 8));
        const int64_t row = m0 + r;
        const int64_t col = n0 + quad * 4;
        const int64_t count = row < p.m ? p.n - col : 0;
        float4 sum = total_of(block, at, 0);
        float v[4] = {sum.x, sum.y, sum.z, sum.w};
        float other[4] = {1.0f, 1.0f, 1.0f, 1.0f};
        if constexpr (GATED) {
            sum = total_of(block, at, 1);
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
#pragma nounroll
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
        if constexpr (kRowsB == kBlock) {
            if (p.q.values != nullptr && row < p.m) {
                dev::write_f8(p.q, row, col, p.n, y);
            }
        }
    }
}

template <int WM, int WN, int WK, int TURNS, bool GATED>
void launch_ring(const mfr_stream& s, Params p) {
    const int64_t tiles_m = (p.m + 32 * WM - 1) / (32 * WM);
    const int64_t tiles_n = (p.n + 32 * WN - 1) / (32 * WN);
    require(tiles_m < (int64_t{1} << 31) && tiles_n < (int64_t{1} << 31) &&
                one_launch(tiles_m * tiles_n, 64 * WM * WN * WK),
            "f8gemm: problem too large for one launch");
    p.tiles_m = static_cast<uint32_t>(tiles_m);
    p.tiles_n = static_cast<uint32_t>(tiles_n);
    ring_kernel<WM, WN, WK, TURNS, GATED>
        <<<static_cast<unsigned>(tiles_m * tiles_n), 64 * WM * WN * WK, 0, s.stream>>>(p);
    check_launch("f8gemm ring_kernel");
}

} // namespace mfr::f8gemm
