// The tile kernel of mfr_f8gemm: e4m3 operands with block scales, multiplied on the bf16 matrix cores.
//
// Every e4m3 number is a bf16 number, so the operands go to the matrix cores exactly, as bf16
// (v_cvt_scalef32_pk_bf16_fp8, two at once, one in the time of an fma). The 8-bit matrix cores run at
// twice the rate, but add the 8 products of neighbouring depths with what is 2^13 times smaller than
// the largest of them cut off (found by feeding them powers of two): sums over 128 normal values came
// out 1.4e-5 off in the 2-norm, whole products 2.3e-5 to 4.2e-5, against 1e-8 and 5e-7 here. That is
// no fp32 sum, so they are not used.
#pragma once

#include "f8.hpp"

namespace mfr::f8gemm {

using f8::blocks_of;
using f8::kBlock;
using f8::Matrix;

struct Params {
    int64_t m, n, k;
    Matrix a, b, up;
    float* c; // null: none
    int64_t c_rs;
    const float* c0; // null: none (beta is not 0 otherwise)
    int64_t c0_rs;
    const float* bias;
    Matrix q; // values null: none
    float beta;
    int act;
    uint32_t tiles_m, tiles_n;
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

// Eight e4m3 values as bf16, exactly.
__device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi) {
    const bf16x2 v[4] = {
        __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false),
        __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true),
        __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false),
        __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true),
    };
    bf16x8 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        out[2 * i] = v[i][0];
        out[2 * i + 1] = v[i][1];
    }
    return out;
}

__device__ inline float activate(float v, int act) {
    if (act == MFR_ACT_SILU) {
        return v / (1.0f + expf(-v));
    }
    return mfr::dev::activate(v, act);
}

// The copies into LDS have landed, and the LDS reads before have been done (a later copy may write there).
__device__ __forceinline__ void wait_copies() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(7 << 4); // vmcnt 0, lgkmcnt 0
}

// A workgroup barrier that waits for no memory operation by itself.
__device__ __forceinline__ void bare_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// 16 bytes from global memory to LDS, lane l's to `to` + 16 l (`to` is the wavefront's).
__device__ __forceinline__ void copy16(const uint8_t* from, void* to) {
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)(from),
        (__attribute__((address_space(3))) void*)(to), 16, 0, 0);
}

__device__ __forceinline__ void copy4(const float* from, void* to) {
    __builtin_amdgcn_global_load_lds(
        (const __attribute__((address_space(1))) void*)(from),
        (__attribute__((address_space(3))) void*)(to), 4, 0, 0);
}

// A tile of BM x BN outputs (BN of each projection when GATED) by WM x WN wavefronts. Depth slices
// of one block (128 bytes of a row) are copied to LDS in 16-byte pieces, piece c of row r at place
// c ^ (r % 8), so that the 16 rows of a fragment lie in different banks; while one slice is
// multiplied the next is on its way.
//
// A wavefront keeps its columns' fragments of a slice in registers, as bf16, and takes its rows 16
// at a time: 4 v_mfma_f32_16x16x32_bf16 give the block's inner sums of 16 x 16 outputs, which the
// vector units add, times the two scales, to the outer sums. The weight is the instruction's first
// operand: a lane then holds 4 neighbouring columns of one row of C. The 32 depths that a lane
// gives to an instruction's 4 rounds are 32 neighbouring ones for both operands: which depth stands
// where does not matter to a sum as long as it is the same for both.
template <int BM, int BN, int WM, int WN, bool GATED>
__global__ __launch_bounds__(64 * WM * WN) void tile_kernel(Params p) {
    constexpr int kThreads = 64 * WM * WN;
    constexpr int kWeights = GATED ? 2 : 1;
    constexpr int FM = BM / WM / 16;
    constexpr int FN = BN / WN / 16; // of each projection
    constexpr int kRowsB = BN * kWeights;
    constexpr int kRowStep = kThreads / 8; // rows per round of copies
    constexpr int kCopiesA = BM / kRowStep;
    constexpr int kCopiesB = kRowsB / kRowStep;
    static_assert(BM % kRowStep == 0 && BN % kRowStep == 0 && BM % 64 == 0, "whole rounds of copies");
    static_assert(kBlock % (BN / WN) == 0 && BN % kBlock == 0, "blocks of columns within a tile");
    struct Slice {
        uint4 a[BM * 8];
        uint4 b[kRowsB * 8];
        float scales[BM];
    };
    // Two objects, so that the compiler sees that the copy into one does not write the other.
    __shared__ __align__(16) Slice slice0;
    __shared__ __align__(16) Slice slice1;

    const int lane = static_cast<int>(threadIdx.x % 64);
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64));
    const int wm = wave % WM;
    const int wn = wave / WM;
    const int r16 = lane % 16;
    const int g = lane / 16;

    // Workgroup -> tile: consecutive logical indices on one XCD (the hardware sends workgroup i to
    // XCD i % 8), in groups of 8 tile-rows, rows fastest, whose operands that XCD's L2 keeps.
    const uint32_t total = p.tiles_m * p.tiles_n;
    const uint32_t per_xcd = total / 8;
    const uint32_t logical =
        blockIdx.x < per_xcd * 8 ? blockIdx.x % 8 * per_xcd + blockIdx.x / 8 : blockIdx.x;
    const uint32_t group_rows = p.tiles_m < 8 ? p.tiles_m : 8;
    const uint32_t group = logical / (group_rows * p.tiles_n);
    const uint32_t rows_here = min(group_rows, p.tiles_m - group * group_rows);
    const uint32_t in_group = logical - group * group_rows * p.tiles_n;
    const int64_t m0 = static_cast<int64_t>(group * group_rows + in_group % rows_here) * BM;
    const int64_t n0 = static_cast<int64_t>(in_group / rows_here) * BN;

    const int64_t depth_blocks = blocks_of(p.k);
    const int64_t last_piece = (p.k + 15) / 16 - 1;

    // This thread's rows of a slice; rows past the matrix repeat its last one (their sums are not
    // stored). A row's pieces past its last one repeat that, and clear() removes them.
    const int row_in_round = static_cast<int>(threadIdx.x) / 8;
    const int64_t piece = (threadIdx.x % 8) ^ (row_in_round % 8);
    const uint8_t* from_a[kCopiesA];
    const uint8_t* from_b[kCopiesB];
#pragma unroll
    for (int i = 0; i < kCopiesA; ++i) {
        from_a[i] = p.a.values + min(m0 + row_in_round + i * kRowStep, p.m - 1) * p.a.rs;
    }
#pragma unroll
    for (int i = 0; i < kCopiesB; ++i) {
        const Matrix& w = GATED && i * kRowStep >= BN ? p.up : p.b;
        from_b[i] =
            w.values + min(n0 + row_in_round + (i * kRowStep) % BN, p.n - 1) * w.rs;
    }
    const float* from_scales =
        p.a.scales + min(m0 + (wave * 64 + lane) % BM, p.m - 1) * p.a.srs;

    const auto copy = [&](Slice& to, int64_t kb) {
        const int64_t offset = min(kb * 8 + piece, last_piece) * 16;
#pragma unroll
        for (int i = 0; i < kCopiesA; ++i) {
            copy16(from_a[i] + offset, to.a + i * kThreads + wave * 64);
        }
#pragma unroll
        for (int i = 0; i < kCopiesB; ++i) {
            copy16(from_b[i] + offset, to.b + i * kThreads + wave * 64);
        }
        if (wave * 64 < BM) {
            copy4(from_scales + kb * p.a.scs, to.scales + wave * 64);
        }
    };
    // Zeros for the depths of the last slice that lie behind k.
    const auto clear = [&](Slice& s) {
        const int depths = static_cast<int>(p.k - (depth_blocks - 1) * kBlock);
        for (int i = static_cast<int>(threadIdx.x); i < (BM + kRowsB) * 8; i += kThreads) {
            const int inside = depths - 16 * ((i % 8) ^ (i / 8 % 8));
            uint4* const at = i < BM * 8 ? s.a + i : s.b + (i - BM * 8);
            if (inside <= 0) {
                *at = make_uint4(0, 0, 0, 0);
            } else if (inside < 16) {
                uint32_t* const words = reinterpret_cast<uint32_t*>(at);
                for (int w = 0; w < 4; ++w) {
                    const int bytes = inside - 4 * w;
                    words[w] &= bytes >= 4 ? ~0u : bytes <= 0 ? 0u : (1u << (8 * bytes)) - 1;
                }
            }
        }
    };

    floatx4 acc[kWeights][FM][FN] = {};
    // One for the wavefront: its columns lie within a block.
    const int64_t col_block = min(n0 + wn * (BN / WN), p.n - 1) / kBlock;
    const float* scale_b[2] = {p.b.scales + col_block * p.b.srs, p.up.scales + col_block * p.up.srs};

    const auto multiply = [&](const Slice& s, int64_t kb) {
        float sb[kWeights];
        sb[0] = scale_b[0][kb * p.b.scs];
        if constexpr (GATED) {
            sb[1] = scale_b[1][kb * p.up.scs];
        }
        const auto piece_at = [&](const uint4* tile, int row, int half) {
            return tile[row * 8 + ((2 * g + half) ^ (row % 8))];
        };
        bf16x8 fb[kWeights][FN][4];
#pragma unroll
        for (int w = 0; w < kWeights; ++w) {
#pragma unroll
            for (int j = 0; j < FN; ++j) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint4 v =
                        piece_at(s.b, w * BN + wn * (BN / WN) + 16 * j + r16, half);
                    fb[w][j][2 * half] = widen(v.x, v.y);
                    fb[w][j][2 * half + 1] = widen(v.z, v.w);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int row = wm * (BM / WM) + 16 * i + r16;
            floatx4 part[kWeights][FN] = {};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint4 v = piece_at(s.a, row, half);
                const bf16x8 fa[2] = {widen(v.x, v.y), widen(v.z, v.w)};
#pragma unroll
                for (int t = 0; t < 2; ++t) {
#pragma unroll
                    for (int w = 0; w < kWeights; ++w) {
#pragma unroll
                        for (int j = 0; j < FN; ++j) {
                            part[w][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                fb[w][j][2 * half + t], fa[t], part[w][j], 0, 0, 0);
                        }
                    }
                }
            }
            const float sa = s.scales[row];
#pragma unroll
            for (int w = 0; w < kWeights; ++w) {
                const float scale = sa * sb[w];
#pragma unroll
                for (int j = 0; j < FN; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc[w][i][j][e] = fmaf(part[w][j][e], scale, acc[w][i][j][e]);
                    }
                }
            }
        }
    };
    const auto step = [&](Slice& here, Slice& next, int64_t kb) {
        wait_copies();
        bare_barrier(); // everyone's copies have landed, and `next` has been read
        if (kb + 1 < depth_blocks) {
            copy(next, kb + 1);
        } else if (p.k % kBlock != 0) {
            clear(here);
            __syncthreads();
        }
        multiply(here, kb);
    };

    if (depth_blocks > 0) {
        copy(slice0, 0);
    }
    for (int64_t kb = 0; kb < depth_blocks; kb += 2) {
        step(slice0, slice1, kb);
        if (kb + 1 < depth_blocks) {
            step(slice1, slice0, kb + 1);
        }
    }

    // The epilogue. Element e of block (i, j) is row 16 i + r16, column 16 j + 4 g + e.
    namespace dev = f8::dev;
    uint32_t top[FM];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int64_t row = m0 + wm * (BM / WM) + 16 * i + r16;
        top[i] = 0;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int64_t col = n0 + wn * (BN / WN) + 16 * j + 4 * g;
            floatx4 v = acc[0][i][j];
            const int64_t count = row < p.m ? p.n - col : 0;
            if (!GATED && p.c0 != nullptr) {
                const float4 c0 = dev::load_quad(p.c0 + row * p.c0_rs + col, count);
                v[0] += p.beta * c0.x, v[1] += p.beta * c0.y;
                v[2] += p.beta * c0.z, v[3] += p.beta * c0.w;
            }
            if (!GATED && p.bias != nullptr) {
                const float4 bias = dev::load_quad(p.bias + col, p.n - col);
                v[0] += bias.x, v[1] += bias.y, v[2] += bias.z, v[3] += bias.w;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = activate(v[e], p.act);
                if constexpr (GATED) {
                    v[e] = v[e] * acc[1][i][j][e];
                }
                v[e] = e < count ? v[e] : 0.0f;
            }
            acc[0][i][j] = v;
            const float4 y = make_float4(v[0], v[1], v[2], v[3]);
            top[i] = max(top[i], dev::magnitude(y));
            if (p.c != nullptr) {
                dev::store_quad(p.c + row * p.c_rs + col, y, count);
            }
        }
    }
    if (p.q.values == nullptr) {
        return;
    }
    // The largest magnitude of a row's 128 columns: over the lanes of a row, then over the
    // wavefronts that share the block.
    uint32_t(&tops)[WN][BM] = *reinterpret_cast<uint32_t(*)[WN][BM]>(&slice0);
    __syncthreads(); // the slices have been read
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        top[i] = max(top[i], static_cast<uint32_t>(__shfl_xor(static_cast<int>(top[i]), 16, 64)));
        top[i] = max(top[i], static_cast<uint32_t>(__shfl_xor(static_cast<int>(top[i]), 32, 64)));
        if (g == 0) {
            tops[wn][wm * (BM / WM) + 16 * i + r16] = top[i];
        }
    }
    __syncthreads();
    constexpr int kSharing = kBlock / (BN / WN);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const int in_tile = wm * (BM / WM) + 16 * i + r16;
        const int64_t row = m0 + in_tile;
#pragma unroll
        for (int w = 0; w < kSharing; ++w) {
            top[i] = max(top[i], tops[wn / kSharing * kSharing + w][in_tile]);
        }
        const float scale = dev::scale_of(top[i]);
        const int64_t first = n0 + wn / kSharing * kSharing * (BN / WN);
        if (row < p.m && first < p.n && wn % kSharing == 0 && g == 0) {
            p.q.scales[row * p.q.srs + first / kBlock * p.q.scs] = scale;
        }
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const int64_t col = n0 + wn * (BN / WN) + 16 * j + 4 * g;
            const floatx4 v = acc[0][i][j];
            if (row < p.m && col < p.n) {
                dev::store_bytes(p.q.values + row * p.q.rs + col,
                                 dev::pack(make_float4(v[0], v[1], v[2], v[3]), 1.0f / scale),
                                 p.n - col);
            }
        }
    }
}

template <int BM, int BN, int WM, int WN> void launch(const mfr_stream& s, Params p) {
    const int64_t tiles_m = (p.m + BM - 1) / BM;
    const int64_t tiles_n = (p.n + BN - 1) / BN;
    require(tiles_m < (int64_t{1} << 31) && tiles_n < (int64_t{1} << 31) &&
                one_launch(tiles_m * tiles_n, 64 * WM * WN),
            "f8gemm: problem too large for one launch");
    p.tiles_m = static_cast<uint32_t>(tiles_m);
    p.tiles_n = static_cast<uint32_t>(tiles_n);
    const unsigned grid = static_cast<unsigned>(tiles_m * tiles_n);
    tile_kernel<BM, BN, WM, WN, false><<<grid, 64 * WM * WN, 0, s.stream>>>(p);
    check_launch("f8gemm tile_kernel");
}

// Gated: BN of each projection.
template <int BM, int BN, int WM, int WN> void launch_gated(const mfr_stream& s, Params p) {
    const int64_t tiles_m = (p.m + BM - 1) / BM;
    const int64_t tiles_n = (p.n + BN - 1) / BN;
    require(tiles_m < (int64_t{1} << 31) && tiles_n < (int64_t{1} << 31) &&
                one_launch(tiles_m * tiles_n, 64 * WM * WN),
            "f8gemm: problem too large for one launch");
    p.tiles_m = static_cast<uint32_t>(tiles_m);
    p.tiles_n = static_cast<uint32_t>(tiles_n);
    const unsigned grid = static_cast<unsigned>(tiles_m * tiles_n);
    tile_kernel<BM, BN, WM, WN, true><<<grid, 64 * WM * WN, 0, s.stream>>>(p);
    check_launch("f8gemm tile_kernel");
}

} // namespace mfr::f8gemm
