// mfr_attention_paged for items of many rows (a prefix that a batch shares, pieces of prompts), caches in
// bf16 and e4m3: bound by the matrix cores.
//
// A workgroup's four wavefronts, one a SIMD, hold 32 rows each and walk the item's tokens together, 64 at
// a time, through three buffers in LDS: one that is multiplied, one that is written, and one that a
// wavefront behind may still read. There is no second wavefront to fill a SIMD's pauses, so that every
// stretch of products has vector work of another 32 tokens between them, chunk by chunk (a barrier to the
// compiler's scheduling ends each): scores of the next 32 beside the weights of these, weights times
// values beside the maximum of the next scores and the turning of the next tile into the operands'
// layouts, whose numbers come into registers a whole tile ahead. (Two wavefronts a SIMD of half the
// registers, without this, ran the matrix cores at a fifth of their rate: each waited for its own
// results, and what spilled came back behind the loads that were under way.)
//   - S^T = K Q^T by 32 x 32 x 16 products: a wavefront keeps the parts of its queries in registers; keys
//     lie by 16-byte pieces. Row 8 g + 4 h + r of a product (h: the half of the lanes that gets its scores,
//     r < 4) is token 16 (g / 2) + 8 h + 4 (g % 2) + r, so that a lane's scores of 16 tokens are of 8
//     neighbours.
//   - O^T += V^T P^T: those are the B operand, and the A operand is 8 neighbouring tokens of one column,
//     which is how the values lie.
// bf16 caches: three bf16 parts of queries and weights. e4m3 numbers are exact in fp16 too, whose parts
// hold 11 bits and a sign, so two hold 23: queries are brought to 2^15 by a power of two for each row, weights
// (with the values' scales) by the softmax's reference, 2^7 to 2^15 below the largest of them.
//
// 4 x 512 queries of 8 x 4 heads of 128 on up to 8192 tokens in bf16: 500 us (517-529 with the join), 980
// TFLOP/s of products (the matrix cores' power: 2.2 GHz); they are 41 % busy, the vector units 42 %; in 8 bits
// 475 with the join. 1024 rows a head on 16383 tokens in 8 bits: 179 us, 770 TFLOP/s, bound by the vector
// instructions of a wavefront (670 a tile of 64 tokens beside 64 products: widening, scales and cuts), which
// fill 43 % of the time and cannot be issued beside others of the same SIMD.
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

// Tokens of a tile and one more: pieces of a row, which a thread's neighbours write, are in different banks.
constexpr int kPitch = kKeys + 1;

// A tile in LDS.
template <int D> struct Shared {
    uint4 keys[D / 8][kPitch];          // 16-byte pieces of tokens
    uint4 values[kKeys / 8][4][D / 4];  // [8 tokens][column % 4][column / 4]
    float scales[4][kKeys];             // keys', values', log2 of the values', nothing
    uint32_t odd[kWaves];               // at edges: tokens of 16 with values that are no numbers
};
// Sums of 128 products of a query of up to 2^15 with numbers of up to 448 stay below 2^31: keys' scales are
// taken times 2^-31, so that no finite one leads a score out of fp32's range before the query's power (and
// this one) is taken back. (Below 2^-95 they lose bits: 2^-102 of the scale times a query's largest.)
constexpr int kKeyPower = 31;
constexpr float kKeyUnit = 0x1p-31f;
constexpr int kAllThere = 15; // a bit for each 16 tokens whose page is one of the cache's

// The numbers of the matrix cores: bf16 as it is, e4m3 as fp16.
typedef float floatx2 __attribute__((ext_vector_type(2)));
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

// Two floats (up to 2^15) cut into two fp16 parts each, both rounded to nearest (v_cvt_pk_f16_f32): what the
// first leaves is up to 2^12 of fp32's last places, of either sign, and the second holds it to within one,
// ties to even. (Cut towards zero, they were up to three last places off, and always below.)
__device__ __forceinline__ halfx2 halves(float x, float y) {
    return __builtin_convertvector((floatx2{x, y}), halfx2);
}
__device__ __forceinline__ void cut_halves(float x, float y, uint32_t& p0, uint32_t& p1) {
    const halfx2 h = halves(x, y);
    p0 = __builtin_bit_cast(uint32_t, h);
    p1 = __builtin_bit_cast(uint32_t, halves(fmaf(static_cast<float>(h[0]), -1.0f, x),
                                             fmaf(static_cast<float>(h[1]), -1.0f, y)));
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
    static constexpr int kTokens = kThreads / T::kRowPieces; // of the workgroup's loads of keys
    static constexpr int kWaveTokens = 64 / T::kRowPieces;

    const Params& p;
    const Shape& shape;
    const Pages& pages;
    const int wave, lane;
    // From a tile's first token to the lane's piece of its keys (of 16 tokens' pieces) and values (of its
    // 16 tokens), and to the scales: 16 lanes of the keys', 16 of the values', and the same again.
    GlobalBytes keys, values, scales;
    float unit; // of the scales that this lane loads

    __device__ __forceinline__ Loader(const Params& params, const Shape& of, const Pages& at, int w,
                                      int l)
        : p(params), shape(of), pages(at), wave(w), lane(l) {
        const int row_bytes = p.cache.d * kBytes<TYPE>;
        keys = lane_address(p.cache.k + at.head * p.cache.head_stride,
                            (wave * kWaveTokens % 16 + lane / T::kRowPieces) * p.cache.token_stride +
                                min(16 * (lane % T::kRowPieces), row_bytes - 16));
        values = lane_address(p.cache.v + at.head * p.cache.head_stride,
                              8 * (lane / 32) * p.cache.token_stride +
                                  min(T::kValueBytes * (lane % (D / 4)), row_bytes - T::kValueBytes));
        unit = (lane & 16) != 0 ? 1.0f : kKeyUnit;
        scales = lane_address((lane & 16) != 0 ? p.cache.v_scales : p.cache.k_scales, 4 * (lane % 16));
    }

    // The page numbers of a tile: of this wavefront's pieces of the keys and of its values, and whether
    // they are all there, 16 tokens a bit.
    struct Numbers {
        int32_t key[T::kPieces];
        int32_t value;
        int there;
    };
    // The tokens, of 16, that piece i of this wavefront's keys is among.
    __device__ __forceinline__ int key_tile(int i) const {
        return kTokens == 16 ? i : kTokens == 32 ? 2 * i + wave / 2 : 4 * i + wave;
    }
    __device__ __forceinline__ Numbers numbers(int32_t first) const {
        Numbers n;
#pragma unroll
        for (int i = 0; i < T::kPieces; ++i) {
            n.key[i] = pages.page(p, first + 16 * key_tile(i));
        }
        n.value = pages.page(p, first + 16 * wave);
        n.there = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t page = static_cast<uint32_t>(pages.page(p, first + 16 * i));
            n.there |= page < static_cast<uint32_t>(p.work.batch.pages) ? 1 << i : 0;
        }
        return n;
    }

    // Lanes past a row's end load its last piece again: the queries are zeros there, and those columns of
    // the output are not written. Piece i of the keys.
    __device__ __forceinline__ void load_key(StagedKeys<TYPE, D>& to, int i, int32_t first,
                                             const Numbers& n) const {
        to.k[i] = load_at<uint4>(keys, pages.at(p, first + 16 * key_tile(i), n.key[i]).at);
    }

    // Values: this wavefront's 16 tokens, a thread 8 of them and four columns (at a depth of 64 half of the
    // threads load what the others do). Token r of them.
    __device__ __forceinline__ TileAt values_at(StagedValues<TYPE, D>& to, int32_t first,
                                                const Numbers& n) const {
        const TileAt at = pages.at(p, first + 16 * wave, n.value);
        to.first = first;
        to.there = at.there;
        if constexpr (TYPE == MFR_KV_F8) {
            to.scale = load_at<float>(scales, at.scale_at);
        }
        return at;
    }
    __device__ __forceinline__ void load_value(StagedValues<TYPE, D>& to, int r, const TileAt& at) const {
        const int64_t from = at.at + static_cast<int64_t>(r) * p.cache.token_stride;
        if constexpr (T::kValueBytes == 8) {
            const uint2 w = load_at<uint2>(values, from);
            to.v[r][0] = w.x;
            to.v[r][1] = w.y;
        } else {
            to.v[r][0] = load_at<uint32_t>(values, from);
        }
    }

    __device__ __forceinline__ void load(StagedKeys<TYPE, D>& k, StagedValues<TYPE, D>& v,
                                         int32_t first, const Numbers& n) const {
#pragma unroll
        for (int i = 0; i < T::kPieces; ++i) {
            load_key(k, i, first, n);
        }
        const TileAt at = values_at(v, first, n);
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            load_value(v, r, at);
        }
    }

    // What was loaded, turned into the operands' layouts, to a buffer that nothing reads: a piece of the
    // keys, ...
    __device__ __forceinline__ void store_key(const StagedKeys<TYPE, D>& from, int i,
                                              Shared<D>& to) const {
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

    // ... the scales (lanes write what others write too, and one row that nothing reads, rather than take a
    // branch), ...
    __device__ __forceinline__ void store_scales(const StagedValues<TYPE, D>& from,
                                                 Shared<D>& to) const {
        if constexpr (TYPE == MFR_KV_F8) {
            const int which = lane >> 4 & 1;
            to.scales[which][16 * wave + lane % 16] = from.scale * unit;
            // No further down, so that a weight over its value's scale stays inside fp32 (far_row).
            to.scales[3 - which][16 * wave + lane % 16] =
                fmaxf(__builtin_amdgcn_logf(fabsf(from.scale)), -96.0f);
        }
    }

    // ... what the values need before where some row does not see some token of the tile, or a page is
    // not there (zeros for tokens that there are not, and for numbers that are none), ...
    __device__ __forceinline__ void settle(StagedValues<TYPE, D>& from, Shared<D>& to) const {
        const int half = lane / 32;
        // Values under a scale that is no number are none. (Their tokens: 16 lanes of the scales.)
        uint64_t bad = 0;
        if constexpr (TYPE == MFR_KV_F8) {
            const bool mine = (lane & 16) != 0 && !(fabsf(from.scale) < INFINITY);
            bad = __ballot(mine && lane < 32) >> 16;
            from.scale = mine ? 1.0f : from.scale;
        }
        uint32_t tokens = 0;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const bool keep = from.there && from.first + 16 * wave + 8 * half + r < shape.tokens;
            const bool under = (bad >> (8 * half + r) & 1) != 0;
            bool odd = keep && under;
#pragma unroll
            for (int i = 0; i < T::kValueBytes / 4; ++i) {
                const uint32_t w = keep && !under ? from.v[r][i] : 0u;
                odd |= is_odd<TYPE>(w);
                from.v[r][i] = without_odd<TYPE>(w);
            }
            const uint64_t lanes = __ballot(odd);
            tokens |= static_cast<uint32_t>(lanes) != 0 ? 1u << r : 0u;
            tokens |= static_cast<uint32_t>(lanes >> 32) != 0 ? 0x100u << r : 0u;
        }
        if (lane == 0) {
            to.odd[wave] = tokens;
        }
    }

    // ... and column j of this thread's 8 tokens.
    __device__ __forceinline__ void store_value(const StagedValues<TYPE, D>& from, int j,
                                                Shared<D>& to) const {
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
        to.values[2 * wave + lane / 32][j][lane % (D / 4)] = make_uint4(w[0], w[1], w[2], w[3]);
    }

    // All of it.
    __device__ __forceinline__ void store(const StagedKeys<TYPE, D>& k, StagedValues<TYPE, D>& v,
                                          Shared<D>& to, bool edge) const {
#pragma unroll
        for (int i = 0; i < T::kPieces; ++i) {
            store_key(k, i, to);
        }
        if (edge) {
            settle(v, to);
        }
        store_scales(v, to);
#pragma unroll
        for (int j = 0; j < T::kColumns; ++j) {
            store_value(v, j, to);
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
        const int shift = min(14 - exponent, 126);
        by = __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
        // Above 0, so that scores of tokens that are not seen stay -infinity. Queries past 2^112 meet the
        // largest there is.
        rest = fminf(fmaxf(ldexpf(fabsf(p.scale), kKeyPower - shift), 0x1p-126f), 0x1.fffffep127f);
        by = copysignf(by, p.scale);
    }
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        const float4 a = scaled(quad(16 * s + 8 * half), by);
        const float4 b = scaled(quad(16 * s + 8 * half + 4), by);
        if constexpr (TYPE == MFR_KV_BF16) {
            cut_pair(a.x, a.y, to[0][s].x, to[1][s].x, to[2][s].x);
            cut_pair(a.z, a.w, to[0][s].y, to[1][s].y, to[2][s].y);
            cut_pair(b.x, b.y, to[0][s].z, to[1][s].z, to[2][s].z);
            cut_pair(b.z, b.w, to[0][s].w, to[1][s].w, to[2][s].w);
        } else {
            cut_halves(a.x, a.y, to[0][s].x, to[1][s].x);
            cut_halves(a.z, a.w, to[0][s].y, to[1][s].y);
            cut_halves(b.x, b.y, to[0][s].z, to[1][s].z);
            cut_halves(b.z, b.w, to[0][s].w, to[1][s].w);
        }
    }
    return rest;
}

template <int D> using Sums = floatx16[D / 32];

// Scores of 32 tokens: element e is token token_of(e) + 8 half of them.
__device__ __forceinline__ constexpr int token_of(int e) {
    return 16 * (e / 8) + 4 * (e / 4 % 2) + e % 4;
}

// Where a wavefront reads 32 tokens of a tile.
template <int TYPE, int D> struct Reader {
    const Shared<D>& tile;
    const int sub, lane;

    __device__ __forceinline__ uint4 key(int i) const {
        const int m = lane % 32;
        const int token = 32 * sub + 16 * (m / 16) + 8 * (m / 4 % 2) + 4 * (m / 8 % 2) + m % 4;
        return (&tile.keys[lane / 32][token])[i * 2 * kPitch];
    }
    // Of tokens 16 q + 8 half on, block b of the columns.
    __device__ __forceinline__ uint4 value(int q, int b) const {
        return (&tile.values[4 * sub + lane / 32][0][0] + lane % 32)[q * 2 * D + 32 * b];
    }
    __device__ __forceinline__ float scale(int which, int e) const {
        return (&tile.scales[which][32 * sub + 8 * (lane / 32)])[token_of(e)];
    }
};

// Weights of 32 tokens as B operands: pairs of them, in parts.
template <int TYPE> struct Weights {
    uint32_t pair[kParts<TYPE>][8];

    __device__ __forceinline__ void cut(float x, float y, int i) {
        if constexpr (TYPE == MFR_KV_BF16) {
            cut_pair(x, y, pair[0][i], pair[1][i], pair[2][i]);
        } else {
            cut_halves(x, y, pair[0][i], pair[1][i]);
        }
    }
    __device__ __forceinline__ uint4 operand(int part, int q) const {
        return make_uint4(pair[part][4 * q], pair[part][4 * q + 1], pair[part][4 * q + 2],
                          pair[part][4 * q + 3]);
    }
};

// Fragments of keys or values on their way from LDS, four products ahead.
struct Fragments {
    uint4 at[4];
};

// The scales of a lane's 16 tokens, in 8 bits.
template <int TYPE> struct Scales {
    float of[TYPE == MFR_KV_F8 ? 16 : 1];

    template <int D> __device__ __forceinline__ void load(const Reader<TYPE, D>& from, int which) {
        if constexpr (TYPE == MFR_KV_F8) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                of[e] = from.scale(which, e);
            }
        }
    }
};

// The next scores, whose first keys are in `keys`, and beside them the weights of these: a chunk of 16
// depths' products has 256 / D weights between them. The first values come into `values`.
template <int TYPE, int D>
__device__ __forceinline__ void scores_and_weights(floatx16& next, Fragments& keys,
                                                   const Reader<TYPE, D>& ahead,
                                                   const Queries<TYPE, D>& queries,
                                                   Weights<TYPE>& weights, const floatx16& s,
                                                   Fragments& values, const Reader<TYPE, D>& from,
                                                   Running& run, float reference, float rest) {
    constexpr int kChunks = D / 16, kEach = 16 / kChunks;
    Scales<TYPE> by;
    by.load(from, 1);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        next[e] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const uint4 now = keys.at[i % 4];
        if (i + 4 < kChunks) {
            keys.at[i % 4] = ahead.key(i + 4);
        } else {
            const int j = i + 4 - kChunks;
            values.at[j] = from.value(j / (D / 32), j % (D / 32));
        }
        // The smallest parts first.
#pragma unroll
        for (int part = kParts<TYPE> - 1; part >= 0; --part) {
            next = product<TYPE>(now, queries[part][i], next);
        }
#pragma unroll
        for (int e = kEach * i; e < kEach * (i + 1); e += 2) {
            float w[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                w[j] = __builtin_amdgcn_exp2f(TYPE == MFR_KV_F8 ? fmaf(s[e + j], rest, -reference)
                                                                : s[e + j] - reference);
            }
            run.sum += w[0] + w[1];
            if constexpr (TYPE == MFR_KV_F8) {
                w[0] *= by.of[e];
                w[1] *= by.of[e + 1];
            }
            weights.cut(w[0], w[1], e / 2);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Weights times values, whose first are in `values`, and beside them the next scores' maximum and, chunk by
// chunk, `other(chunk)`. In 8 bits scores are multiplied by their keys' scales (times `rest` they are base-2
// scores then), and the maximum is of what a weight is times its value's scale.
template <int TYPE, int D, typename Other>
__device__ __forceinline__ void add_values(Sums<D>& acc, const Weights<TYPE>& weights,
                                           Fragments& values, const Reader<TYPE, D>& from,
                                           floatx16& next, float& most, const Reader<TYPE, D>& ahead,
                                           float rest, Other other) {
    constexpr int kBlocks = D / 32, kChunks = 2 * kBlocks, kEach = 16 / kChunks;
    Scales<TYPE> by, up;
    by.load(ahead, 0);
    up.load(ahead, 2);
    most = -INFINITY;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
        const uint4 now = values.at[i % 4];
        if (i + 4 < kChunks) {
            values.at[i % 4] = from.value((i + 4) / kBlocks, (i + 4) % kBlocks);
        }
#pragma unroll
        for (int part = kParts<TYPE> - 1; part >= 0; --part) {
            acc[i % kBlocks] = product<TYPE>(now, weights.operand(part, i / kBlocks), acc[i % kBlocks]);
        }
#pragma unroll
        for (int e = kEach * i; e < kEach * (i + 1); ++e) {
            if constexpr (TYPE == MFR_KV_F8) {
                next[e] *= by.of[e];
                most = fmaxf(most, fmaf(next[e], rest, up.of[e]));
            } else {
                most = fmaxf(most, next[e]);
            }
        }
        other(i);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// What the scores that are ready need before they become weights: tokens that a row does not see (`edge`,
// uniform: there are some), the running maximum, and the output so far rescaled where it moved. Returns
// the reference of the weights.
template <int TYPE, int D>
__device__ __forceinline__ float settle_scores(floatx16& s, float most, Sums<D>& acc, Running& run,
                                               const Reader<TYPE, D>& from, float rest, int32_t first,
                                               bool edge, int there) {
    if (__builtin_expect(edge, 0)) {
        const int half = from.lane / 32;
        const int32_t left = run.seen - first - 32 * from.sub - 8 * half; // tokens of this half's
        Scales<TYPE> up;
        up.load(from, 2);
        const uint32_t* tokens = &from.tile.odd[2 * from.sub];
        const uint32_t odd = (tokens[0] >> (8 * half) & 0xffu) | (tokens[1] >> (8 * half) & 0xffu) << 8;
        const uint32_t pages = there >> (2 * from.sub);
        const uint32_t here = ((pages & 1) != 0 ? 0xffu : 0u) | ((pages & 2) != 0 ? 0xff00u : 0u);
        uint32_t sees = 0; // element e: bit e, as in `odd`
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            sees |= token_of(e) < left ? 1u << e : 0u;
        }
        sees &= here;
        most = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float t = TYPE == MFR_KV_F8 ? fmaf(s[e], rest, up.of[TYPE == MFR_KV_F8 ? e : 0]) : s[e];
            most = (sees >> e & 1) != 0 ? fmaxf(most, t) : most;
            s[e] = (sees >> e & 1) != 0 ? s[e] : -INFINITY;
        }
        // A value that is no number was taken out, and makes the row NaN.
        run.sum = (sees & odd) != 0 ? NAN : run.sum;
    }
    // Weights are taken against a reference that follows the maximum in steps: it moves, and the output so
    // far with it, where the maximum has grown by more than 2^8, so that few steps do. In bf16 it is 2^8
    // above the maximum then, and no weight is above 1; in 8 bits 2^7 below: fp16 holds weights up to 2^15.
    constexpr float kBelow = TYPE == MFR_KV_F8 ? 7.0f : -8.0f;
    most = max_halves(most) - kBelow;
    if (__builtin_expect(__any(most > run.top + 8.0f), 0)) {
        const float top = fmaxf(run.top, most);
        // In 8 bits half of the step at a time: weights over small scales may be as large as steps to those of
        // large scales are deep.
        const float steps = TYPE == MFR_KV_F8 ? 0.5f : 1.0f;
        float shrink = run.top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(steps * (run.top - top));
        asm volatile("" : "+v"(shrink)); // no products with it ahead of the branch
        run.top = top;
        run.sum *= TYPE == MFR_KV_F8 ? shrink : 1.0f;
        run.sum *= shrink;
        shrink *= TYPE == MFR_KV_F8 ? shrink : 1.0f;
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                acc[b][e] *= shrink;
            }
        }
    }
    // Nothing seen yet: any finite reference gives weights of 0.
    const float reference = run.top == -INFINITY ? 0.0f : run.top;
    return reference;
}

// In 8 bits a weight's exponent is taken from a score before its last rounding, and the reference has one: past
// 2^20 they no longer agree to the last places of a weight, past 2^24 not at all. And scales below 2^-96 are
// weighed as that, so that fp32 can sum the weights over them: they lose bits. The rows of far scores, and those
// whose weights' sum says that such scales lead (not where all values are zeros), are done again, a wavefront
// a row, in fp32 throughout: tokens `first` .. `last` - 1, a lane a token for scores, a lane two columns for
// values: 300 us for 64 tokens of 128 rows, but no model is meant to have such numbers.
constexpr float kFar = 0x1p20f;

// Where a token is (in bytes from a head's first row, in scales from the first).
struct FarToken {
    int64_t at, scale_at;
    bool there;

    __device__ __forceinline__ FarToken(const Params& p, const Pages& pages, int32_t token) {
        const int32_t page = mfr::kv::page_checked(p.work.batch, pages.table[token >> p.cache.page_log2]);
        const int64_t number = max(page, 0);
        const int32_t slot = token & ((1 << p.cache.page_log2) - 1);
        at = number * p.cache.page_stride + static_cast<int64_t>(slot) * p.cache.token_stride;
        scale_at = ((number * p.cache.heads + pages.head) << p.cache.page_log2) + slot;
        there = page >= 0;
    }
};

// Whether the tokens first .. last - 1 have any value that is not 0.
__device__ __forceinline__ bool any_value(const Params& p, const Pages& pages, int32_t first, int32_t last,
                                          int lane) {
    const uint8_t* const values = p.cache.v + pages.head * p.cache.head_stride;
    bool found = false;
#pragma unroll 1
    for (; first < last && !__any(found); first += 64) {
        const FarToken of(p, pages, min(first + lane, last - 1));
        uint32_t bits = 0;
#pragma unroll 1
        for (int c = 0; c < p.cache.d; c += 16) {
            const uint4 w = *reinterpret_cast<const uint4*>(values + of.at + c);
            bits |= (w.x | w.y | w.z | w.w) & 0x7f7f7f7fu;
        }
        found = of.there && bits != 0 && p.cache.v_scales[of.scale_at] != 0.0f;
    }
    return __any(found);
}

template <int D>
__device__ __forceinline__ void far_row(const Params& p, const Pages& pages, const float* q, int32_t first,
                                        int32_t last, int lane, float* out) {
    const uint8_t* const keys = p.cache.k + pages.head * p.cache.head_stride;
    const uint8_t* const values = p.cache.v + pages.head * p.cache.head_stride;
    float top = -INFINITY, sum = 0.0f, acc[2] = {0.0f, 0.0f};
#pragma unroll 1
    for (; first < last; first += 64) {
        const int32_t token = min(first + lane, last - 1);
        const FarToken of(p, pages, token);
        float s = 0.0f;
#pragma unroll 1
        for (int c = 0; c < p.cache.d; c += 4) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(keys + of.at + c);
            s = fmaf(__builtin_amdgcn_cvt_f32_fp8(w, 0), q[c], s);
            s = fmaf(__builtin_amdgcn_cvt_f32_fp8(w, 1), q[c + 1], s);
            s = fmaf(__builtin_amdgcn_cvt_f32_fp8(w, 2), q[c + 2], s);
            s = fmaf(__builtin_amdgcn_cvt_f32_fp8(w, 3), q[c + 3], s);
        }
        s *= p.cache.k_scales[of.scale_at] * p.scale;
        s = of.there && first + lane < last ? s : -INFINITY;
        float most = s;
#pragma unroll
        for (int step = 32; step > 0; step /= 2) {
            most = fmaxf(most, __shfl_xor(most, step, 64));
        }
        most = fmaxf(most, top);
        const float shrink = part_weight(top, most);
        top = most;
        const float weight = s == -INFINITY ? 0.0f : exp2_native(s - top);
        sum = fmaf(sum, shrink, weight);
        acc[0] *= shrink;
        acc[1] *= shrink;
        const float by = p.cache.v_scales[of.scale_at];
#pragma unroll 1
        for (int j = 0; j < 64; ++j) {
            const uint8_t* const row = values + __shfl(static_cast<long long>(of.at), j, 64);
            const float w = __shfl(weight, j, 64), unit = __shfl(by, j, 64);
            if (w == 0.0f) { // tokens that there are not, too
                continue;
            }
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const int c = lane + 64 * i;
                const float v = c < p.cache.d ? __builtin_amdgcn_cvt_f32_fp8(row[c], 0) : 0.0f;
                acc[i] = fmaf(w, v * unit, acc[i]);
            }
        }
    }
#pragma unroll
    for (int step = 32; step > 0; step /= 2) {
        sum += __shfl_xor(sum, step, 64);
    }
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        out[lane + 64 * i] = acc[i];
    }
    if (lane == 0) {
        *reinterpret_cast<float2*>(out + D) = make_float2(top, sum);
    }
}

// Sums of weights over very small or large scales are brought near 1, with the reference: what joins parts
// weighs them by their references alone, and two of 2^48 and 2^-48 leave fp32 room for 2^-30 between their
// shares. (Both by what the rounded reference moves.)
constexpr int kWide = 48;

template <int D> __device__ __forceinline__ void wide_row(float2 stats, int lane, float* out) {
    const float top = stats.x + static_cast<float>(__builtin_amdgcn_frexp_expf(stats.y));
    const float by = __builtin_amdgcn_exp2f(0.5f * (stats.x - top));
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        out[lane + 64 * i] = out[lane + 64 * i] * by * by;
    }
    if (lane == 0) {
        *reinterpret_cast<float2*>(out + D) = make_float2(top, stats.y * by * by);
    }
}

template <int TYPE, int D>
__global__ __launch_bounds__(kThreads, 1) void attention_paged_tiles_kernel(Params p) {
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
            if (!dev::advance(p.work, seq, shape)) {
                return; // (lengths that changed meanwhile)
            }
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
            const Pages pages(p, last, seq, item.head);
            const Loader<TYPE, D> loader(p, shape, pages, wave, lane);
            typename Loader<TYPE, D>::Numbers numbers = loader.numbers(first);
            StagedKeys<TYPE, D> keys;
            StagedValues<TYPE, D> values;
            loader.load(keys, values, first, numbers);
            int there = numbers.there; // of the tile, and of the one that is under way
            numbers = loader.numbers(first + kKeys);
            loader.store(keys, values, tiles[0], first + kKeys > group_all || there != kAllThere);
            loader.load(keys, values, first + kKeys, numbers);
            int there_next = numbers.there;
            numbers = loader.numbers(first + 2 * kKeys);
            __syncthreads();
            // The first 32 tokens' scores, as they stand after add_values.
            floatx16 s0, s1;
            float most = -INFINITY;
            {
                const Reader<TYPE, D> from{tiles[0], 0, lane};
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s0[e] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const uint4 k = from.key(i);
#pragma unroll
                    for (int part = kParts<TYPE> - 1; part >= 0; --part) {
                        s0 = product<TYPE>(k, queries[part][i], s0);
                    }
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    if constexpr (TYPE == MFR_KV_F8) {
                        s0[e] *= from.scale(0, e);
                        most = fmaxf(most, fmaf(s0[e], rest, from.scale(2, e)));
                    } else {
                        most = fmaxf(most, s0[e]);
                    }
                }
            }
            Fragments keys_ahead, values_ahead;
            const auto first_keys = [&](const Reader<TYPE, D>& from) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    keys_ahead.at[i] = from.key(i);
                }
            };
            first_keys(Reader<TYPE, D>{tiles[0], 1, lane});
            Weights<TYPE> weights;
#pragma unroll 1
            for (int buffer = 0; first < last; first += kKeys) {
                Shared<D>& tile = tiles[buffer];
                buffer = buffer == 2 ? 0 : buffer + 1;
                Shared<D>& other = tiles[buffer];
                const bool edge = first + kKeys > group_all || there != kAllThere;
                const Reader<TYPE, D> low{tile, 0, lane}, high{tile, 1, lane}, ahead{other, 0, lane};
                if (__builtin_expect(first + 2 * kKeys > group_all || there_next != kAllThere, 0)) {
                    loader.settle(values, other);
                }
                float reference =
                    settle_scores<TYPE, D>(s0, most, acc, run, low, rest, first, edge, there);
                scores_and_weights<TYPE, D>(s1, keys_ahead, high, queries, weights, s0, values_ahead, low,
                                            run, reference, rest);
                // The next tile's pieces and columns, in the chunks that there are.
                constexpr int kPieces = Tile<TYPE, D>::kPieces;
                constexpr int kStores = kPieces + Tile<TYPE, D>::kColumns, kChunks = D / 16;
                add_values<TYPE, D>(
                    acc, weights, values_ahead, low, s1, most, high, rest, [&](int chunk) {
#pragma unroll
                        for (int i = chunk * kStores / kChunks; i < (chunk + 1) * kStores / kChunks;
                             ++i) {
                            if (i == 0) {
                                loader.store_scales(values, other);
                            }
                            if (i < kPieces) {
                                loader.store_key(keys, i, other);
                            } else {
                                loader.store_value(values, i - kPieces, other);
                            }
                        }
                    });
                lds_barrier();
                first_keys(ahead);
                reference =
                    settle_scores<TYPE, D>(s1, most, acc, run, high, rest, first, edge, there);
                scores_and_weights<TYPE, D>(s0, keys_ahead, ahead, queries, weights, s1, values_ahead,
                                            high, run, reference, rest);
                // Loads of the tile behind the next, and the first keys of the next half.
                const TileAt at = loader.values_at(values, first + 2 * kKeys, numbers);
                constexpr int kLoads = kPieces + 8;
                const Reader<TYPE, D> behind{other, 1, lane};
                add_values<TYPE, D>(
                    acc, weights, values_ahead, high, s0, most, ahead, rest, [&](int chunk) {
#pragma unroll
                        for (int i = chunk * kLoads / kChunks; i < (chunk + 1) * kLoads / kChunks; ++i) {
                            if (i < kPieces) {
                                loader.load_key(keys, i, first + 2 * kKeys, numbers);
                            } else {
                                loader.load_value(values, i - kPieces, at);
                            }
                        }
                        if (chunk >= kChunks - 4) {
                            const int i = chunk + 4 - kChunks;
                            keys_ahead.at[i] = behind.key(i);
                        }
                    });
                there = there_next;
                there_next = numbers.there;
                numbers = loader.numbers(first + 3 * kKeys);
            }
            __syncthreads(); // the tiles have been read
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
        if constexpr (TYPE == MFR_KV_F8) {
            const auto stats_of = [&](int32_t r) {
                return *reinterpret_cast<const float2*>(out + min(r, here - 1) * kPitch + D);
            };
            const auto is_far = [&](float2 stats) {
                return fabsf(stats.x) > kFar && stats.x != -INFINITY;
            };
            const auto is_wide = [&](float2 stats) {
                return abs(__builtin_amdgcn_frexp_expf(stats.y)) > kWide;
            };
            const auto is_small = [&](float2 stats) { return stats.y >= 0x1p102f; }; // infinities, too
            const float2 mine_of = stats_of(32 * wave + lane % 32);
            if (__builtin_expect(__any(is_far(mine_of) || is_wide(mine_of) || is_small(mine_of)), 0)) {
                const int32_t from = item.first * kKeys;
                const bool small = __any(is_small(mine_of)) &&
                                   any_value(p, Pages(p, last, seq, item.head), from, last, lane);
#pragma unroll 1
                for (int32_t r = 32 * wave; r < min(32 * (wave + 1), here); ++r) { // its own rows alone
                    const float2 stats = stats_of(r);
                    if (is_far(stats) || (small && is_small(stats)) || stats.y == INFINITY) {
                        const int32_t i = (row0 + r) / p.work.group;
                        const float* q = p.q.p + (shape.span.first + static_cast<int64_t>(i)) * p.q.ts +
                                         (item.head * p.work.group + (row0 + r - i * p.work.group)) *
                                             p.q.hs;
                        const int32_t to = min(seen_at(row0 + r), last);
                        far_row<D>(p, Pages(p, to, seq, item.head), q, from, to, lane, out + r * kPitch);
                    } else if (is_wide(stats)) {
                        wide_row<D>(stats, lane, out + r * kPitch);
                    }
                }
            }
            __syncthreads();
        }
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
    constexpr unsigned kBytesOfLds = 3 * sizeof(Shared<D>);
    static_assert(kBytesOfLds <= 160 * 1024 && kBytesOfLds >= kManyRows * (D + 4) * sizeof(float), "room for the results");
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
