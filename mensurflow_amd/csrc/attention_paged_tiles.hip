// mfr_attention_paged for items of many rows (a prefix that a batch shares, pieces of prompts), caches in
// bf16 and e4m3: bound by the matrix cores.
//
// A workgroup's four wavefronts hold 32 rows each and walk the item's tokens together, 64 at a time: the
// keys, then the values of the next 64 come into registers under the products of these, are turned into
// the operands' layouts there, and go to the other of two buffers in LDS.
//   - S^T = K Q^T by 32 x 32 x 16 products: a wavefront keeps the parts of its queries in registers; keys
//     lie by 16-byte pieces. Row 8 g + 4 h + r of a product (h: the half of the lanes that gets its scores,
//     r < 4) is token 16 (g / 2) + 8 h + 4 (g % 2) + r, so that a lane's scores of 16 tokens are of 8
//     neighbours.
//   - O^T += V^T P^T: those are the B operand, and the A operand is 8 neighbouring tokens of one column,
//     which is how the values lie.
// bf16 caches: three bf16 parts of queries and weights. e4m3 numbers are exact in fp16 too, whose parts
// hold 11 bits, so two do: queries are brought to 2^15 by a power of two for each row, weights (with
// the values' scales) by the softmax's reference, which is 2^15 below the largest of them.
#include "attention_paged.hpp"

namespace {

using namespace mfr::paged;
using namespace mfr::paged::dev;
namespace dev = mfr::paged::dev;

constexpr int kKeys = 64; // tokens of a unit

template <int TYPE, int D> struct Tile {
    static constexpr int kPieces = kKeys * D * kBytes<TYPE> / 16 / kThreads; // of keys, a thread
    static constexpr int kRowPieces = D * kBytes<TYPE> / 16;                 // of a token's keys
    static constexpr int kColumns = 4;                                       // of values, a thread
    static constexpr int kValueBytes = kColumns * kBytes<TYPE>;
};

// A tile in LDS.
template <int D> struct Shared {
    uint4 keys[D / 8][kKeys + 4];       // 16-byte pieces of tokens; the pad turns the banks
    uint4 values[kKeys / 8][4][D / 4];  // [8 tokens][column % 4][column / 4]
    float scales[3][kKeys];             // keys', values', log2 of the values'
    int odd[kWaves];                    // at edges: whether 16 tokens have values that are no numbers
};
constexpr int kAllThere = 15; // a bit for each 16 tokens whose page is one of the cache's

// The numbers of the matrix cores: bf16 as it is, e4m3 as fp16.
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
template <int TYPE> constexpr int kParts = TYPE == MFR_KV_BF16 ? 3 : 2;

template <int TYPE>
__device__ __forceinline__ floatx16 product(const uint4& a, const uint4& b, const floatx16& c) {
    if constexpr (TYPE == MFR_KV_BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, a),
                                                      __builtin_bit_cast(halfx8, b), c, 0, 0, 0);
    }
}

// Two e4m3 numbers of a half of w as fp16.
template <bool HIGH> __device__ __forceinline__ uint32_t widen_half(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HIGH));
}

// Eight floats (up to 2^16 in fp16) cut into their parts.
template <int TYPE> struct Parts8 {
    uint4 part[kParts<TYPE>];
};
template <int TYPE>
__device__ __forceinline__ Parts8<TYPE> cut(float a, float b, float c, float d, float e, float f,
                                            float g, float h) {
    Parts8<TYPE> to;
    if constexpr (TYPE == MFR_KV_BF16) {
        cut_pair(a, b, to.part[0].x, to.part[1].x, to.part[2].x);
        cut_pair(c, d, to.part[0].y, to.part[1].y, to.part[2].y);
        cut_pair(e, f, to.part[0].z, to.part[1].z, to.part[2].z);
        cut_pair(g, h, to.part[0].w, to.part[1].w, to.part[2].w);
    } else {
        const auto round = [](float u, float v) { // towards zero: no overflow
            return __builtin_bit_cast(halfx2, __builtin_amdgcn_cvt_pkrtz(u, v));
        };
        const auto pair = [&](float x, float y, uint32_t& p0, uint32_t& p1) {
            const halfx2 h0 = round(x, y);
            p0 = __builtin_bit_cast(uint32_t, h0);
            p1 = __builtin_bit_cast(uint32_t, round(fmaf(static_cast<float>(h0[0]), -1.0f, x),
                                                    fmaf(static_cast<float>(h0[1]), -1.0f, y)));
        };
        pair(a, b, to.part[0].x, to.part[1].x);
        pair(c, d, to.part[0].y, to.part[1].y);
        pair(e, f, to.part[0].z, to.part[1].z);
        pair(g, h, to.part[0].w, to.part[1].w);
    }
    return to;
}

// A thread's share of a tile on its way from memory to LDS.
template <int TYPE, int D> struct StagedKeys {
    uint4 k[Tile<TYPE, D>::kPieces];
};
template <int TYPE, int D> struct StagedValues {
    uint32_t v[8][Tile<TYPE, D>::kValueBytes / 4];
    float scale;
    int32_t first;
    bool there; // the page of this wavefront's values
};

template <int TYPE, int D> struct Loader {
    using T = Tile<TYPE, D>;
    const Params& p;
    const Shape& shape;
    const Pages& pages;
    const int wave, lane;

    // The page numbers of a tile's tokens, 16 by 16.
    struct Numbers {
        int32_t page[4];
    };
    __device__ __forceinline__ Numbers numbers(int32_t first) const {
        Numbers n;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            n.page[i] = pages.page(p, first + 16 * i);
        }
        return n;
    }

    __device__ __forceinline__ int there(const Numbers& n) const {
        int bits = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bits |= mfr::kv::page_checked(p.work.batch, n.page[i]) >= 0 ? 1 << i : 0;
        }
        return bits;
    }
    // (Not an array's element: its index is not known before the run.)
    __device__ __forceinline__ static int32_t page_of(const Numbers& n, int i) {
        return i == 0 ? n.page[0] : i == 1 ? n.page[1] : i == 2 ? n.page[2] : n.page[3];
    }

    // Addresses are a uniform part and 32 bits of the lane's. Lanes past a row's end load its last piece
    // again: the queries are zeros there, and those columns of the output are not written.
    __device__ __forceinline__ void load_keys(StagedKeys<TYPE, D>& to, int32_t first,
                                              const Numbers& n) const {
        constexpr int kTokens = kThreads / T::kRowPieces; // of the workgroup's loads
        constexpr int kWaveTokens = 64 / T::kRowPieces;
        const uint32_t lane_at = lane / T::kRowPieces * p.cache.token_stride +
                                 min(16 * (lane % T::kRowPieces), p.cache.d * kBytes<TYPE> - 16);
#pragma unroll
        for (int i = 0; i < T::kPieces; ++i) {
            const int32_t token = i * kTokens + wave * kWaveTokens;
            const TileAt at = pages.at(p, first + (token & ~15), page_of(n, token / 16));
            const uint8_t* base = uniform(
                p.cache.k + at.at + static_cast<int64_t>(token & 15) * p.cache.token_stride);
            to.k[i] = *reinterpret_cast<const uint4*>(base + lane_at);
        }
    }

    // Values: this wavefront's 16 tokens, a thread 8 of them and four columns (at a depth of 64 half of the
    // threads load what the others do).
    __device__ __forceinline__ void load_values(StagedValues<TYPE, D>& to, int32_t first,
                                                const Numbers& n) const {
        const TileAt at = pages.at(p, first + 16 * wave, page_of(n, wave));
        to.first = first;
        to.there = at.there;
        const int half = lane / 32;
        const uint32_t lane_at = 8 * half * p.cache.token_stride +
                                 min(T::kValueBytes * (lane % (D / 4)),
                                     p.cache.d * kBytes<TYPE> - T::kValueBytes);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const uint8_t* from =
                uniform(p.cache.v + at.at + static_cast<int64_t>(r) * p.cache.token_stride) + lane_at;
            if constexpr (T::kValueBytes == 8) {
                const uint2 w = *reinterpret_cast<const uint2*>(from);
                to.v[r][0] = w.x;
                to.v[r][1] = w.y;
            } else {
                to.v[r][0] = *reinterpret_cast<const uint32_t*>(from);
            }
        }
        if constexpr (TYPE == MFR_KV_F8) {
            to.scale = 0.0f;
            if (half == 0) {
                const float* scales = lane < 16 ? p.cache.k_scales : p.cache.v_scales;
                to.scale = scales[at.scale_at + lane % 16];
            }
        }
    }

    // What was loaded, turned into the operands' layouts, to a buffer that nothing reads.
    __device__ __forceinline__ void store_keys(const StagedKeys<TYPE, D>& from, Shared<D>& to) const {
        constexpr int kWaveTokens = 64 / T::kRowPieces;
        constexpr int kTokens = kThreads / T::kRowPieces;
#pragma unroll
        for (int i = 0; i < T::kPieces; ++i) {
            const int token = i * kTokens + wave * kWaveTokens + lane / T::kRowPieces;
            const int piece = lane % T::kRowPieces;
            if constexpr (TYPE == MFR_KV_BF16) {
                to.keys[piece][token] = from.k[i];
            } else {
                const uint4 w = from.k[i];
                to.keys[2 * piece][token] =
                    make_uint4(widen_half<false>(w.x), widen_half<true>(w.x), widen_half<false>(w.y),
                               widen_half<true>(w.y));
                to.keys[2 * piece + 1][token] =
                    make_uint4(widen_half<false>(w.z), widen_half<true>(w.z), widen_half<false>(w.w),
                               widen_half<true>(w.w));
            }
        }
    }

    // Values of tokens that there are not are zeros; `edge`: some row does not see some token.
    __device__ __forceinline__ void store_values(StagedValues<TYPE, D>& from, Shared<D>& to,
                                                 bool edge) const {
        const int half = lane / 32;
        if (from.first + kKeys > shape.tokens || !from.there) {
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                const int32_t token = from.first + 16 * wave + 8 * half + r;
                const bool keep = from.there && token < shape.tokens;
#pragma unroll
                for (int i = 0; i < T::kValueBytes / 4; ++i) {
                    from.v[r][i] = keep ? from.v[r][i] : 0u;
                }
            }
        }
        if (edge) {
            bool odd = false;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
#pragma unroll
                for (int i = 0; i < T::kValueBytes / 4; ++i) {
                    const uint32_t w = from.v[r][i];
                    if constexpr (TYPE == MFR_KV_BF16) {
                        odd |= (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            odd |= ((w >> (8 * e)) & 0x7fu) == 0x7fu;
                        }
                    }
                }
            }
            const int any = __any(odd) ? 1 : 0;
            if (lane == 0) {
                to.odd[wave] = any;
            }
        }
        if (TYPE == MFR_KV_F8 && half == 0) {
            to.scales[lane / 16][16 * wave + lane % 16] = from.scale;
            if (lane >= 16) {
                // No further down, so that a weight over its value's scale stays inside fp32: values under
                // a scale of 2^-96 lose bits.
                to.scales[2][16 * wave + lane % 16] =
                    fmaxf(__builtin_amdgcn_logf(from.scale), -96.0f);
            }
        }
        // Column j of the 8 tokens.
#pragma unroll
        for (int j = 0; j < T::kColumns; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                constexpr int kPerWord = TYPE == MFR_KV_BF16 ? 2 : 4;
                const uint32_t a = from.v[2 * i][j / kPerWord], b = from.v[2 * i + 1][j / kPerWord];
                if constexpr (TYPE == MFR_KV_BF16) {
                    w[i] = __builtin_amdgcn_perm(b, a, j % 2 == 0 ? 0x05040100u : 0x07060302u);
                } else {
                    const uint32_t both =
                        __builtin_amdgcn_perm(b, a, j % 4 < 2 ? 0x05010400u : 0x07030602u);
                    w[i] = j % 2 == 0 ? widen_half<false>(both) : widen_half<true>(both);
                }
            }
            to.values[2 * wave + half][j][lane % (D / 4)] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
};

// The queries of a wavefront's rows as B operands, in parts.
template <int TYPE, int D> using Queries = uint4[kParts<TYPE>][D / 16];

// Loads them, times the scale in bf16; in 8 bits brought to 2^14 .. 2^15. Returns what scores have to be
// multiplied by.
template <int TYPE, int D>
__device__ __forceinline__ float load_queries(Queries<TYPE, D>& to, const Params& p,
                                              const Shape& shape, int32_t head, int32_t rr, int half) {
    const int32_t rows = shape.span.count * p.work.group;
    const int32_t i = rr / p.work.group;
    const float* q = p.q.p + (shape.span.first + static_cast<int64_t>(i)) * p.q.ts +
                     (head * p.work.group + (rr - i * p.work.group)) * p.q.hs;
    const auto quad = [&](int c) {
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (rr < rows && c < p.cache.d) {
            v = mfr::dev::load_loose(q + c);
        }
        return v;
    };
    float by = p.scale, rest = 1.0f;
    if constexpr (TYPE != MFR_KV_BF16) {
        float top = 0.0f;
#pragma unroll 2
        for (int s = 0; s < D / 16; ++s) {
            const float4 a = quad(16 * s + 8 * half), b = quad(16 * s + 8 * half + 4);
            top = fmaxf(top, fmaxf(fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(a.z), fabsf(a.w))),
                                   fmaxf(fmaxf(fabsf(b.x), fabsf(b.y)), fmaxf(fabsf(b.z), fabsf(b.w)))));
        }
        top = max_halves(top);
        // A power of two, so that the largest gets the exponent 14; of 0, infinities and subnormal
        // numbers as near as there is one.
        const int exponent = static_cast<int>(__float_as_uint(top) >> 23) - 127;
        const int shift = max(-112, min(14 - exponent, 126));
        by = __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
        rest = p.scale / by;
    }
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        const float4 a = scaled(quad(16 * s + 8 * half), by);
        const float4 b = scaled(quad(16 * s + 8 * half + 4), by);
        const Parts8<TYPE> w = cut<TYPE>(a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w);
#pragma unroll
        for (int part = 0; part < kParts<TYPE>; ++part) {
            to[part][s] = w.part[part];
        }
    }
    return rest;
}

template <int D> using Sums = floatx16[D / 32];

// 32 tokens of a tile. Element 4 g + r of the scores: token 16 (g / 2) + 8 half + 4 (g % 2) + r of them.
// `edge` (uniform): some row does not see some token, or a page is not there. One code for both: a second
// one, run once at an item's end, takes longer to come into the instruction cache than to run.
template <int TYPE, int D>
__device__ __forceinline__ void step(Sums<D>& acc, Running& run, const Queries<TYPE, D>& queries,
                                     float rest, const Shared<D>& tile, int sub, int32_t first,
                                     int lane, bool edge, int there) {
    const int half = lane / 32, m = lane % 32;
    // The keys of product row m; this half's tokens.
    const int token = 32 * sub + 16 * (m / 16) + 8 * (m / 4 % 2) + 4 * (m / 8 % 2) + m % 4;
    const int mine = 32 * sub + 8 * half;
    floatx16 s;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        s[e] = 0.0f;
    }
    // A piece of the keys is read under the products of the ones before; the barriers keep the compiler
    // from reading all of them at once, for which there are no registers.
    const uint4* pieces = &tile.keys[half][token];
    constexpr int kPitch = 2 * (kKeys + 4);
    uint4 k[2] = {pieces[0], pieces[kPitch]};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
        const uint4 now = k[i % 2];
        if (i + 2 < D / 16) {
            k[i % 2] = pieces[(i + 2) * kPitch];
        }
        // The smallest parts first.
#pragma unroll
        for (int part = kParts<TYPE> - 1; part >= 0; --part) {
            s = product<TYPE>(now, queries[part][i], s);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    const auto token_of = [&](int e) { return 16 * (e / 8) + 4 * (e / 4 % 2) + e % 4; };
    const auto visible = [&](int e) {
        const int at = mine + token_of(e);
        return first + at < run.seen && (there >> (at / 16) & 1) != 0;
    };
    const auto scales_of = [&](int which, int g) {
        return *reinterpret_cast<const float4*>(&tile.scales[which][mine + token_of(4 * g)]);
    };
    // Base-2 scores, and the largest; in 8 bits of what a weight is times its value's scale.
    if constexpr (TYPE == MFR_KV_F8) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 by = scaled(scales_of(0, g), rest);
            s[4 * g] *= by.x;
            s[4 * g + 1] *= by.y;
            s[4 * g + 2] *= by.z;
            s[4 * g + 3] *= by.w;
        }
    }
    if (edge) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = visible(e) ? s[e] : -INFINITY;
        }
    }
    float most = -INFINITY;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        float4 up = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if constexpr (TYPE == MFR_KV_F8) {
            up = scales_of(2, g);
        }
        most = fmaxf(fmaxf(most, s[4 * g] + up.x), s[4 * g + 1] + up.y);
        most = fmaxf(fmaxf(most, s[4 * g + 2] + up.z), s[4 * g + 3] + up.w);
    }
    // In 8 bits the reference is 2^15 below the largest.
    most = max_halves(most) - (TYPE == MFR_KV_F8 ? 15.0f : 0.0f);
    most = fmaxf(run.top, most);
    // Nothing seen yet: any finite reference gives weights of 0.
    const float reference = most == -INFINITY ? 0.0f : most;
    if (__any(most != run.top)) {
        const float shrink = __builtin_amdgcn_exp2f(run.top - reference);
        run.top = most;
        run.sum *= shrink;
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                acc[b][e] *= shrink;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        s[e] = __builtin_amdgcn_exp2f(s[e] - reference);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) { // a short chain of sums
        run.sum += (s[4 * g] + s[4 * g + 1]) + (s[4 * g + 2] + s[4 * g + 3]);
    }
    if constexpr (TYPE == MFR_KV_F8) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 by = scales_of(1, g);
            s[4 * g] *= by.x;
            s[4 * g + 1] *= by.y;
            s[4 * g + 2] *= by.z;
            s[4 * g + 3] *= by.w;
        }
        if (edge) { // a scale that is not seen may be anything
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = visible(e) ? s[e] : 0.0f;
            }
        }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const Parts8<TYPE> weights =
            cut<TYPE>(s[8 * q], s[8 * q + 1], s[8 * q + 2], s[8 * q + 3], s[8 * q + 4], s[8 * q + 5],
                      s[8 * q + 6], s[8 * q + 7]);
        const uint4* values = &tile.values[4 * sub + 2 * q + half][0][0] + m;
        uint4 v[2] = {values[0], values[32]};
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
            const uint4 now = v[b % 2];
            if (b + 2 < D / 32) {
                v[b % 2] = values[32 * (b + 2)];
            }
#pragma unroll
            for (int part = kParts<TYPE> - 1; part >= 0; --part) {
                acc[b] = product<TYPE>(now, weights.part[part], acc[b]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// A tile with values that are no numbers, some of which some rows do not see: these must not meet the
// weights of 0 of such rows. Rows that see one become NaN in its column, and then there are zeros in their
// place. All wavefronts.
template <int TYPE, int D>
__device__ __forceinline__ void settle_odd(Sums<D>& acc, const Running& run, Shared<D>& tile,
                                           int32_t first, int lane, int there) {
    const int half = lane / 32;
#pragma unroll 1
    for (int group = 0; group < kKeys / 16; ++group) {
        const int at = first + 16 * group + 8 * half;
        const auto sees = [&](int i) { return at + i < run.seen && (there >> group & 1) != 0; };
        const uint4 seen = make_uint4(ones<TYPE>(sees(0), sees(1)), ones<TYPE>(sees(2), sees(3)),
                                      ones<TYPE>(sees(4), sees(5)), ones<TYPE>(sees(6), sees(7)));
        const uint4* values = &tile.values[2 * group + half][0][0] + lane % 32;
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
            floatx16 count;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                count[e] = 0.0f;
            }
            count = product<TYPE>(odd_ones<TYPE>(values[32 * b]), seen, count);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                acc[b][e] = count[e] > 0.0f ? NAN : acc[b][e];
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    __syncthreads();
    uint4* const values = &tile.values[0][0][0];
#pragma unroll 1
    for (int i = threadIdx.x; i < kKeys * D / 8; i += kThreads) {
        values[i] = without_odd<TYPE>(values[i]);
    }
    __syncthreads();
}

template <int TYPE, int D>
__global__ __launch_bounds__(kThreads, 2) void attention_paged_tiles_kernel(Params p) {
    extern __shared__ uint4 lds[];
    Shared<D>* const tiles = reinterpret_cast<Shared<D>*>(lds);
    const int64_t index = blockIdx.x;
    const dev::Place place = dev::find(p.work, p.groups, [&](int64_t total, int64_t chunk) {
        return index * chunk < total ? index * chunk : int64_t{-1};
    });
    if (place.seq < 0) {
        return;
    }
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64));
    const int half = lane / 32;
    const int64_t begin = index * place.chunk;
    const int64_t end = begin + place.chunk < place.total ? begin + place.chunk : place.total;
    int32_t seq = place.seq;
    int64_t base = place.base;
    Shape shape = mfr::kv::shape_of(p.work, seq);
    for (int64_t at = begin; at < end;) {
        while (at >= base + shape.count) { // the next sequence that has units
            base += shape.count;
            shape = mfr::kv::shape_of(p.work, ++seq);
        }
        const Item item = mfr::kv::item_of(shape, base, at);
        const int64_t item_end = item.begin + shape.units;
        const int32_t units = static_cast<int32_t>((item_end < end ? item_end : end) - at);

        const int32_t rows = shape.span.count * p.work.group;
        const int32_t row0 = item.tile * kManyRows;
        const int32_t wave0 = row0 + 32 * wave;
        const int32_t rr = wave0 + lane % 32;
        const auto seen_at = [&](int32_t row) {
            return mfr::kv::seen_by(shape, min(row, rows - 1) / p.work.group, p.causal != 0);
        };
        Running run;
        run.seen = seen_at(rr);
        // Tokens that every row of the workgroup sees, and that some row sees.
        const int32_t group_all = seen_at(row0);
        const int32_t group_some = seen_at(row0 + kManyRows - 1);

        Queries<TYPE, D> queries;
        const float rest = load_queries<TYPE, D>(queries, p, shape, item.head, rr, half);
        Sums<D> acc;
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                acc[b][e] = 0.0f;
            }
        }
        int32_t first = item.first * kKeys;
        const int32_t last = min(group_some, (item.first + units) * kKeys);
        if (first < last) {
            const Pages pages(p, shape, seq, item.head);
            const Loader<TYPE, D> loader{p, shape, pages, wave, lane};
            typename Loader<TYPE, D>::Numbers numbers = loader.numbers(first);
            StagedKeys<TYPE, D> keys;
            StagedValues<TYPE, D> values;
            loader.load_keys(keys, first, numbers);
            loader.load_values(values, first, numbers);
            int there = loader.there(numbers);
            numbers = loader.numbers(first + kKeys);
            loader.store_keys(keys, tiles[0]);
            loader.store_values(values, tiles[0], first + kKeys > group_all);
            __syncthreads();
            // The next tile's keys are on their way under the first half of this one, its values under the
            // second, so that the registers hold one of the two; behind the last tile there is something to
            // load all the same.
            for (int buffer = 0; first < last; buffer ^= 1) {
                const int32_t next = first + kKeys;
                const bool edge = next > group_all || there != kAllThere;
                if (edge) {
                    const int4 f = *reinterpret_cast<const int4*>(tiles[buffer].odd);
                    if (__builtin_amdgcn_readfirstlane(f.x | f.y | f.z | f.w) != 0) {
                        settle_odd<TYPE, D>(acc, run, tiles[buffer], first, lane, there);
                    }
                }
                loader.load_keys(keys, next, numbers);
                step<TYPE, D>(acc, run, queries, rest, tiles[buffer], 0, first, lane, edge, there);
                loader.store_keys(keys, tiles[buffer ^ 1]);
                loader.load_values(values, next, numbers);
                step<TYPE, D>(acc, run, queries, rest, tiles[buffer], 1, first, lane, edge, there);
                loader.store_values(values, tiles[buffer ^ 1], next + kKeys > group_all);
                there = loader.there(numbers);
                numbers = loader.numbers(next + kKeys);
                first = next;
                __syncthreads();
            }
        }
        // Results to rows in LDS, in place of the tiles, and from there to memory in whole rows.
        const float sum = sum_halves(run.sum);
        float* const out = reinterpret_cast<float*>(lds);
        constexpr int kPitch = D + 4; // values, the maximum and the sum
        float* const mine = out + (32 * wave + lane % 32) * kPitch;
#pragma unroll
        for (int e = 0; e < D / 8; ++e) {
            // Element e of block b: place 32 b + 8 (e / 4) + 4 half + e % 4 of [column % 4][column / 4].
            const int c = 4 * (8 * (e / 4) + 4 * half + e % 4);
            *reinterpret_cast<float4*>(mine + c) =
                D == 128 ? make_float4(acc[0][e], acc[1][e], acc[2 % (D / 32)][e], acc[3 % (D / 32)][e])
                         : make_float4(acc[0][e % 8], acc[0][e % 8 + 8], acc[1][e % 8],
                                       acc[1][e % 8 + 8]);
        }
        if (half == 0) {
            *reinterpret_cast<float2*>(mine + D) = make_float2(run.top, sum);
        }
        __syncthreads();
        const bool whole = item.first == 0 && units == shape.units;
        const int64_t part0 = mfr::kv::part_of(index, place.chunk, item.begin) * kManyRows;
        const int32_t here = min(kManyRows, rows - row0);
        constexpr int kLanes = D / 4;
#pragma unroll 1
        for (int32_t r = threadIdx.x / kLanes; r < here; r += kThreads / kLanes) {
            const int c = 4 * (threadIdx.x % kLanes);
            const float4 v = *reinterpret_cast<const float4*>(out + r * kPitch + c);
            const float2 stats = *reinterpret_cast<const float2*>(out + r * kPitch + D);
            if (whole) {
                const int32_t i = (row0 + r) / p.work.group;
                dev::finish(p, shape.span.first + static_cast<int64_t>(i),
                            item.head * p.work.group + (row0 + r - i * p.work.group), c, v, stats.x,
                            stats.y);
            } else {
                *reinterpret_cast<float4*>(p.parts.values + (part0 + r) * D + c) = v;
                if (c == 0) {
                    *reinterpret_cast<float2*>(p.parts.stats + 2 * (part0 + r)) = stats;
                }
            }
        }
        __syncthreads(); // the rows have been read
        at += units;
    }
}

template <int TYPE, int D> void launch(const Params& p, hipStream_t stream) {
    constexpr unsigned kBytesOfLds = 2 * sizeof(Shared<D>);
    static_assert(kBytesOfLds >= kManyRows * (D + 4) * sizeof(float), "room for the results");
    static_assert(2 * kBytesOfLds <= 160 * 1024, "two workgroups a compute unit");
    mfr::check(hipFuncSetAttribute(
                   reinterpret_cast<const void*>(attention_paged_tiles_kernel<TYPE, D>),
                   hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kBytesOfLds)),
               "hipFuncSetAttribute");
    attention_paged_tiles_kernel<TYPE, D>
        <<<static_cast<unsigned>(p.groups), kThreads, kBytesOfLds, stream>>>(p);
    mfr::check_launch("attention_paged_tiles_kernel");
}

template <int TYPE> void launch_depth(const Params& p, hipStream_t stream) {
    if (p.depth == 64) {
        launch<TYPE, 64>(p, stream);
    } else {
        launch<TYPE, 128>(p, stream);
    }
}

} // namespace

namespace mfr::paged {

void launch_tiles(const Params& p, int32_t type, hipStream_t stream) {
    if (type == MFR_KV_BF16) {
        launch_depth<MFR_KV_BF16>(p, stream);
    } else {
        launch_depth<MFR_KV_F8>(p, stream);
    }
}

} // namespace mfr::paged
