// mfr_attention_paged for items of few rows (one query, or a few drafted ones, of the query heads that
// share a head of the cache): bound by reading the cache once.
//
// A wavefront takes KEYS tokens at a time straight from memory into the operands of the matrix cores,
// with no LDS between, and the four of a workgroup take turns along the item's tokens, each with its own
// running softmax; they join through LDS at the item's end.
//   - S^T = K Q^T by 16 x 16 products: the A operand of K is a lane's 16 bytes of its token's row (the
//     depth in the order that the loads give, the queries cut alike), so a lane gets 4 tokens' scores
//     of one row of the item.
//   - O^T += V^T P^T: those scores are the B operand already, for tokens in the order in which lanes hold
//     them. A lane loads D / 16 neighbouring columns of each of its 4 tokens; column j of all lanes'
//     pieces is an A operand, made by byte permutations inside the lane, and the output's columns come
//     out in that order.
// bf16 and e4m3 numbers are exact in bf16. Queries, and weights (times the scales of the values), are
// cut into three bf16 parts, so that products and sums are fp32's; fp32 caches use the fp32 products.
//
// One query of each of 64 sequences on up to 8191 tokens in 8 bits (8 heads of 128, 4 query heads each): 119 to
// 122 us, 4.7 TB/s; the same loads without any arithmetic take 110 to 116, more wavefronts a compute unit no less:
// pages lie at random, and an eighth goes to the scales, in arrays of their own. 256 sequences of up to 1023
// tokens: 98 us, 2.9 TB/s, four items a workgroup, at whose ends nothing is under way. One query against 4096
// tokens in bf16: 7.5 us, one step a wavefront.
#include "attention_paged.hpp"

#include <type_traits>

namespace {

using namespace mfr::paged;
using namespace mfr::paged::dev;
namespace dev = mfr::paged::dev;

// TILES: tokens of a step, in tiles of 16. PIECES: 16-byte pieces of a token's row that a lane loads.
// VBYTES: bytes of a token's values that a lane loads.
template <int TYPE, int D> struct Form {
    static constexpr int kTiles = TYPE == MFR_KV_F32 ? 1 : 2;
    static constexpr int kKeys = 16 * kTiles;
    static constexpr int kPieces = D * kBytes<TYPE> / 64;
    static constexpr int kValueBytes = D * kBytes<TYPE> / 16;
    static constexpr int kColumns = D / 16;                       // of the values that a lane loads
    static constexpr int kValueWords = (kValueBytes + 3) / 4;
    static constexpr int kSteps = D / 32;                         // of depth, bf16 products
};

// The loads of a step: keys, values and scales of 16 tokens each tile.
template <int TYPE, int D> struct Keys {
    uint4 k[Form<TYPE, D>::kTiles][Form<TYPE, D>::kPieces];
    float4 scale[Form<TYPE, D>::kTiles];
};
template <int TYPE, int D> struct Values {
    uint32_t v[Form<TYPE, D>::kTiles][4][Form<TYPE, D>::kValueWords];
    float4 scale[Form<TYPE, D>::kTiles];
};

// A lane's constant place in the loads.
struct Lanes {
    int row;               // of the item's tile, and token of a key tile: lane % 16
    int quad;              // lane / 16
    uint32_t key_at;       // bytes from a tile's first token to the lane's first piece of its key
    uint32_t value_at;     // to the lane's columns of its first value
    uint32_t key_most;     // the last piece's distance from the first, of a row of fewer than D
    uint32_t value_most;   // likewise, in fp32
};

// Of RT tiles of 16 rows: scores or weights (lane: its row, tokens 4 quad + r of each tile), and weighted
// values (lane: its row, column j of rows 4 quad + r of the pieces).
template <int TYPE, int D, int RT> using Scores = floatx4[RT][Form<TYPE, D>::kTiles];
template <int TYPE, int D, int RT> using Sums = floatx4[RT][Form<TYPE, D>::kColumns];
template <int TYPE, int D> using Tiles = TileAt[Form<TYPE, D>::kTiles];
template <int TYPE, int D> using There = bool[Form<TYPE, D>::kTiles];

template <int RT> using Rows = Running[RT];

// FULL: rows of D.
template <int TYPE, int D, bool FULL> struct Segment {
    using F = Form<TYPE, D>;
    const Params& p;
    const Lanes& lanes;
    // From a tile's first token to the lane's first piece of its key, to the lane's columns of its first
    // value, and to its four scales.
    GlobalBytes keys, values, key_scales, value_scales;

    __device__ __forceinline__ Segment(const Params& params, const Lanes& l, int32_t head)
        : p(params), lanes(l) {
        const int64_t at = head * p.cache.head_stride;
        keys = lane_address(p.cache.k + at, lanes.key_at);
        values = lane_address(p.cache.v + at, lanes.value_at);
        key_scales = lane_address(p.cache.k_scales, 16 * lanes.quad);
        value_scales = lane_address(p.cache.v_scales, 16 * lanes.quad);
    }

    // Lanes past a row's end load its last piece again: the queries are zeros there, and those columns of
    // the output are not written.
    __device__ __forceinline__ void load_keys(Keys<TYPE, D>& to, const Tiles<TYPE, D>& at) const {
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) {
#pragma unroll
            for (int i = 0; i < F::kPieces; ++i) {
                to.k[t][i] = load_at<uint4>(keys + at[t].at,
                                            FULL ? 64 * i : min(64u * i, lanes.key_most));
            }
            if constexpr (TYPE == MFR_KV_F8) {
                to.scale[t] = load_at<float4>(key_scales, at[t].scale_at);
            }
        }
    }

    __device__ __forceinline__ void load_values(Values<TYPE, D>& to,
                                                const Tiles<TYPE, D>& at) const {
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const GlobalBytes base =
                    values + (at[t].at + static_cast<int64_t>(r) * p.cache.token_stride);
                auto& v = to.v[t][r];
                if constexpr (TYPE == MFR_KV_F32) {
#pragma unroll
                    for (int i = 0; i < F::kValueWords / 4; ++i) {
                        const uint4 w =
                            load_at<uint4>(base, FULL ? 256 * i : min(256u * i, lanes.value_most));
                        v[4 * i] = w.x;
                        v[4 * i + 1] = w.y;
                        v[4 * i + 2] = w.z;
                        v[4 * i + 3] = w.w;
                    }
                } else if constexpr (F::kValueWords == 4) {
                    const uint4 w = load_at<uint4>(base, 0);
                    v[0] = w.x;
                    v[1] = w.y;
                    v[2] = w.z;
                    v[3] = w.w;
                } else if constexpr (F::kValueWords == 2) {
                    const uint2 w = load_at<uint2>(base, 0);
                    v[0] = w.x;
                    v[1] = w.y;
                } else {
                    v[0] = load_at<uint32_t>(base, 0);
                }
            }
            if constexpr (TYPE == MFR_KV_F8) {
                to.scale[t] = load_at<float4>(value_scales, at[t].scale_at);
            }
        }
    }
};

// The queries of an item's rows as B operands: three bf16 parts, or fp32. Where the registers that they
// take let one more workgroup run on a compute unit, the parts lie in LDS, once for the workgroup's
// wavefronts, which read them at every step (24 rows a sequence on up to 4096 tokens in 8 bits: 121 us and
// 153 in registers; 4 rows of 64 on up to 8191: 70 and 74). With one tile of rows of 128 that is not so, and
// they stay in registers: no barrier holds an item's first loads back then (256 sequences of up to 1023
// tokens in 8 bits 103 us and 108 in LDS).
template <int TYPE, int D, int RT>
constexpr bool kQueriesInLds = TYPE != MFR_KV_F32 && (D == 64 || RT == 2);

template <int TYPE, int D, int RT> struct Queries {
    static constexpr int kLanes = kQueriesInLds<TYPE, D, RT> ? 64 : 1;
    uint4 part[RT][3][Form<TYPE, D>::kSteps][kLanes];
};
template <int D, int RT> struct Queries<MFR_KV_F32, D, RT> {
    float4 q[RT][D / 16];
};

// By every wavefront for itself, but into LDS, where each takes some steps of the depth, and a barrier has to
// follow.
template <int TYPE, int D, int RT, bool FULL>
__device__ __forceinline__ void load_queries(Queries<TYPE, D, RT>& to, const Params& p,
                                             const Shape& shape, int32_t head, int32_t tile,
                                             const Lanes& lanes, int wave) {
    constexpr bool kLds = kQueriesInLds<TYPE, D, RT>;
    const int32_t rows = shape.span.count * p.work.group;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int32_t rr = tile * (16 * RT) + 16 * rt + lanes.row;
        const int32_t i = rr / p.work.group;
        const float* q = p.q.p + (shape.span.first + static_cast<int64_t>(i)) * p.q.ts +
                         (head * p.work.group + (rr - i * p.work.group)) * p.q.hs;
        const auto quad = [&](int c) {
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (rr < rows && (FULL || c < p.cache.d)) {
                v = mfr::dev::load_loose(q + c);
            }
            return v;
        };
        if constexpr (TYPE == MFR_KV_F32) {
#pragma unroll
            for (int s = 0; s < D / 16; ++s) {
                to.q[rt][s] = quad(16 * s + 4 * lanes.quad);
            }
        } else {
            static_assert(!kLds || Form<TYPE, D>::kSteps <= kWaves);
#pragma unroll
            for (int j = 0; j < (kLds ? 1 : Form<TYPE, D>::kSteps); ++j) {
                const int s = kLds ? wave : j;
                if (kLds && s >= Form<TYPE, D>::kSteps) {
                    break;
                }
                // The depths of piece s of a key: 8 neighbours, or in 8 bits half of 16.
                const int c = TYPE == MFR_KV_BF16 ? 32 * s + 8 * lanes.quad
                                                  : 64 * (s / 2) + 16 * lanes.quad + 8 * (s % 2);
                const float4 a = quad(c), b = quad(c + 4);
                uint4 part[3];
                cut_pair(a.x, a.y, part[0].x, part[1].x, part[2].x);
                cut_pair(a.z, a.w, part[0].y, part[1].y, part[2].y);
                cut_pair(b.x, b.y, part[0].z, part[1].z, part[2].z);
                cut_pair(b.z, b.w, part[0].w, part[1].w, part[2].w);
#pragma unroll
                for (int i = 0; i < 3; ++i) {
                    to.part[rt][i][s][kLds ? 16 * lanes.quad + lanes.row : 0] = part[i];
                }
            }
        }
    }
}

// Scores of a step's tokens, unscaled.
template <int TYPE, int D, int RT>
__device__ __forceinline__ void scores_of(Scores<TYPE, D, RT>& s,
                                          const Keys<TYPE, D>& keys,
                                          const Queries<TYPE, D, RT>& queries, const Lanes& lanes) {
    using F = Form<TYPE, D>;
    const int lane = kQueriesInLds<TYPE, D, RT> ? 16 * lanes.quad + lanes.row : 0;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) {
            s[rt][t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    if constexpr (TYPE == MFR_KV_F32) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const float k[4] = {__uint_as_float(keys.k[0][i].x), __uint_as_float(keys.k[0][i].y),
                                __uint_as_float(keys.k[0][i].z), __uint_as_float(keys.k[0][i].w)};
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float4 q = queries.q[rt][i];
                s[rt][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[0], q.x, s[rt][0], 0, 0, 0);
                s[rt][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[1], q.y, s[rt][0], 0, 0, 0);
                s[rt][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[2], q.z, s[rt][0], 0, 0, 0);
                s[rt][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[3], q.w, s[rt][0], 0, 0, 0);
            }
        }
    } else {
#pragma unroll
        for (int step = 0; step < F::kSteps; ++step) {
            bf16x8 k[F::kTiles];
#pragma unroll
            for (int t = 0; t < F::kTiles; ++t) {
                if constexpr (TYPE == MFR_KV_BF16) {
                    k[t] = __builtin_bit_cast(bf16x8, keys.k[t][step]);
                } else {
                    const uint4 w = keys.k[t][step / 2];
                    const uint32_t lo = step % 2 == 0 ? w.x : w.z, hi = step % 2 == 0 ? w.y : w.w;
                    k[t] = __builtin_bit_cast(bf16x8,
                                              make_uint4(widen<false>(lo), widen<true>(lo),
                                                         widen<false>(hi), widen<true>(hi)));
                }
            }
            // The smallest parts first.
#pragma unroll
            for (int part = 2; part >= 0; --part) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const bf16x8 q =
                        __builtin_bit_cast(bf16x8, queries.part[rt][part][step][lane]);
#pragma unroll
                    for (int t = 0; t < F::kTiles; ++t) {
                        s[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[t], q, s[rt][t], 0, 0, 0);
                    }
                }
            }
        }
    }
}

__device__ __forceinline__ float element(const float4& v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}
__device__ __forceinline__ float& element(float4& v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// Scores to weights (not yet times the values' scales); the output so far is rescaled where a
// maximum moved. `edge` (uniform): some row does not see some token; `first` is the step's first token.
template <int TYPE, int D, int RT>
__device__ __forceinline__ void softmax_step(Scores<TYPE, D, RT>& s,
                                             Sums<TYPE, D, RT>& acc,
                                             Rows<RT>& run, const Keys<TYPE, D>& keys,
                                             float scale, int32_t first, const Lanes& lanes,
                                             bool edge, const There<TYPE, D>& there) {
    using F = Form<TYPE, D>;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[rt][t][r] *= TYPE == MFR_KV_F8 ? element(keys.scale[t], r) * scale : scale;
            }
        }
        if (edge) {
#pragma unroll
            for (int t = 0; t < F::kTiles; ++t) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int32_t token = first + 16 * t + 4 * lanes.quad + r;
                    s[rt][t][r] = there[t] && token < run[rt].seen ? s[rt][t][r] : -INFINITY;
                }
            }
        }
        float most = -INFINITY;
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                most = fmaxf(most, s[rt][t][r]);
            }
        }
        // Weights are taken against a reference that follows the maximum in steps, 2^7 above it where it
        // moves, and the output so far with it: few steps do, and no weight is above 1. (Far scores, whose
        // last place is 16, are then taken as their own reference.)
        most = row_max(most);
        if (__any(most > run[rt].top)) {
            const float top = most > run[rt].top ? most + 7.0f : run[rt].top;
            float shrink = run[rt].top == -INFINITY ? 0.0f : exp2_native(run[rt].top - top);
            asm volatile("" : "+v"(shrink)); // no products with it ahead of the branch
            run[rt].top = top;
            run[rt].sum *= shrink;
#pragma unroll
            for (int j = 0; j < F::kColumns; ++j) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    acc[rt][j][r] *= shrink;
                }
            }
        }
        // Nothing seen yet: any finite reference gives weights of 0.
        const float reference = run[rt].top == -INFINITY ? 0.0f : run[rt].top;
#pragma unroll
        for (int t = 0; t < F::kTiles; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float w = exp2_native(s[rt][t][r] - reference);
                run[rt].sum += w;
                s[rt][t][r] = w;
            }
        }
    }
}

// Column j of the values as an A operand of bf16 products.
template <int TYPE, int D>
__device__ __forceinline__ bf16x8 column_of(const Values<TYPE, D>& values, int j) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { // tokens 2 (i % 2), 2 (i % 2) + 1 of tile i / 2
        constexpr int kPerWord = TYPE == MFR_KV_BF16 ? 2 : 4;
        const uint32_t a = values.v[i / 2][2 * (i % 2)][j / kPerWord];
        const uint32_t b = values.v[i / 2][2 * (i % 2) + 1][j / kPerWord];
        if constexpr (TYPE == MFR_KV_BF16) {
            w[i] = __builtin_amdgcn_perm(b, a, j % 2 == 0 ? 0x05040100u : 0x07060302u);
        } else {
            const uint32_t both =
                __builtin_amdgcn_perm(b, a, j % 4 < 2 ? 0x05010400u : 0x07030602u);
            w[i] = j % 2 == 0 ? widen<false>(both) : widen<true>(both);
        }
    }
    return __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
}

// acc += V^T P^T.
template <int TYPE, int D, int RT>
__device__ __forceinline__ void add_values(Sums<TYPE, D, RT>& acc, const Scores<TYPE, D, RT>& w,
                                           const Values<TYPE, D>& values) {
    using F = Form<TYPE, D>;
    if constexpr (TYPE == MFR_KV_F32) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
            for (int j = 0; j < F::kColumns; ++j) {
                const float v = __uint_as_float(values.v[0][r][j]);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    acc[rt][j] =
                        __builtin_amdgcn_mfma_f32_16x16x4f32(v, w[rt][0][r], acc[rt][j], 0, 0, 0);
                }
            }
        }
    } else {
        Cut cut[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            cut[rt] = cut_weights(w[rt][0], w[rt][1]);
        }
#pragma unroll
        for (int j = 0; j < F::kColumns; ++j) {
            const bf16x8 v = column_of<TYPE, D>(values, j);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                acc[rt][j] = add_column(acc[rt][j], v, cut[rt]);
            }
        }
    }
}

// Before a step that some row does not see whole: zeros for values of tokens that there are not, and for
// ones that are no numbers, which must not meet the weights of 0 of rows that do not see them. Rows that
// do see one become NaN through their sum.
template <int TYPE, int D, int RT>
__device__ __forceinline__ void settle_values(Values<TYPE, D>& values, Rows<RT>& run, int32_t tokens,
                                              int32_t first, const Lanes& lanes,
                                              const There<TYPE, D>& there) {
    using F = Form<TYPE, D>;
#pragma unroll
    for (int t = 0; t < F::kTiles; ++t) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int32_t token = first + 16 * t + 4 * lanes.quad + r;
            const bool keep = there[t] && token < tokens;
            bool odd = false;
#pragma unroll
            for (int i = 0; i < F::kValueWords; ++i) {
                const uint32_t w = keep ? values.v[t][r][i] : 0u;
                odd |= is_odd<TYPE>(w);
                values.v[t][r][i] = without_odd<TYPE>(w);
            }
            if constexpr (TYPE == MFR_KV_F8) { // (values under a scale that is none are none)
                float& scale = element(values.scale[t], r);
                odd |= keep && !(fabsf(scale) < INFINITY);
                scale = fabsf(scale) < INFINITY ? scale : 0.0f;
            }
            // The token's columns are in the 16 lanes of the quad, and so are the rows.
            const uint64_t lanes_odd = __ballot(odd) >> (16 * lanes.quad) & 0xffffu;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                run[rt].sum = lanes_odd != 0 && token < run[rt].seen ? NAN : run[rt].sum;
            }
        }
    }
}

// Weights times the scales of the values, in 8 bits.
template <int TYPE, int D, int RT>
__device__ __forceinline__ void scale_weights(Scores<TYPE, D, RT>& w, Values<TYPE, D>& values) {
    if constexpr (TYPE == MFR_KV_F8) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int t = 0; t < Form<TYPE, D>::kTiles; ++t) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    w[rt][t][r] *= element(values.scale[t], r);
                }
            }
        }
    }
}

// The first of four neighbouring columns that a lane holds in acc[4 q ..][r].
template <int TYPE, int D> __device__ __forceinline__ int column_at(int quad, int r, int q) {
    return TYPE == MFR_KV_F32 ? 16 * quad + 4 * r + 64 * q
                              : Form<TYPE, D>::kColumns * (4 * quad + r) + 4 * q;
}

template <int TYPE, int D, int RT, bool FULL>
__global__ __launch_bounds__(kThreads, (per_unit(TYPE, D, 16 * RT))) void attention_paged_few_kernel(Params p) {
    using F = Form<TYPE, D>;
    constexpr int kPitch = D + 4;
    __shared__ float joined[kWaves][16][kPitch];
    __shared__ float stats[kWaves][16][2];
    __shared__ std::conditional_t<kQueriesInLds<TYPE, D, RT>, Queries<TYPE, D, RT>, int> held;
    const int64_t index = blockIdx.x;
    const dev::Place place = dev::find(p.work, p.groups, [&](int64_t total, int64_t chunk) {
        return index * chunk < total ? index * chunk : int64_t{-1};
    });
    if (place.seq < 0) {
        return;
    }
    const int lane = threadIdx.x % 64;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x / 64));
    Lanes lanes;
    lanes.row = lane % 16;
    lanes.quad = lane / 16;
    const int row_bytes = p.cache.d * kBytes<TYPE>;
    const int key_piece = min(16 * lanes.quad, row_bytes - 16);
    constexpr int kPiece = TYPE == MFR_KV_F32 ? 16 : F::kValueBytes;
    const int value_piece = min(kPiece * lanes.row, row_bytes - kPiece);
    lanes.key_at = lanes.row * p.cache.token_stride + key_piece;
    lanes.value_at = 4 * lanes.quad * p.cache.token_stride + value_piece;
    lanes.key_most = row_bytes - 16 - key_piece;
    lanes.value_most = row_bytes - kPiece - value_piece;
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

        Rows<RT> run;
        const int32_t rows = shape.span.count * p.work.group;
        const int32_t row0 = item.tile * (16 * RT);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int32_t rr = min(row0 + 16 * rt + lanes.row, rows - 1);
            run[rt].seen = mfr::kv::seen_by(shape, rr / p.work.group, p.causal != 0);
        }
        // Tokens that every row sees, and that some row sees.
        const int32_t all_see = mfr::kv::seen_by(shape, row0 / p.work.group, p.causal != 0);
        const int32_t some_see = mfr::kv::seen_by(
            shape, (min(row0 + 16 * RT, rows) - 1) / p.work.group, p.causal != 0);
        const Segment<TYPE, D, FULL> segment(p, lanes, item.head);
        // This wavefront's tokens: a step of every unit.
        constexpr int kUnit = kWaves * F::kKeys;
        int32_t first = item.first * kUnit + wave * F::kKeys;
        const int32_t last = min(some_see, (item.first + units) * kUnit);
        const Pages pages(p, last, seq, item.head);
        // Page numbers are read a step before they are used.
        int32_t numbers[F::kTiles];
        const auto numbers_of = [&](int32_t token) {
#pragma unroll
            for (int t = 0; t < F::kTiles; ++t) {
                numbers[t] = pages.page(p, token + 16 * t);
            }
        };
        if (first < last) {
            numbers_of(first);
        }
        // (What is in LDS of the item before was read before the barriers at its end.)
        constexpr bool kLds = kQueriesInLds<TYPE, D, RT>;
        std::conditional_t<kLds, int, Queries<TYPE, D, RT>> own;
        auto& queries = [&]() -> auto& {
            if constexpr (kLds) {
                return held;
            } else {
                return own;
            }
        }();
        load_queries<TYPE, D, RT, FULL>(queries, p, shape, item.head, item.tile, lanes, wave);
        if constexpr (kLds) {
            __syncthreads();
        }
        Sums<TYPE, D, RT> acc;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int j = 0; j < F::kColumns; ++j) {
                acc[rt][j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
        if (first < last) {
            Tiles<TYPE, D> tiles;
            Keys<TYPE, D> keys;
            Values<TYPE, D> values;
            const auto tiles_of = [&](int32_t token) {
#pragma unroll
                for (int t = 0; t < F::kTiles; ++t) {
                    tiles[t] = pages.at(p, token + 16 * t, numbers[t]);
                }
            };
            tiles_of(first);
            numbers_of(first + kUnit);
            segment.load_keys(keys, tiles);
            segment.load_values(values, tiles);
            // The next step's keys are under way from the scores on, its values from the end; behind the
            // last step there is something to load all the same. One code for steps that some row does not
            // see whole and the others: a second one, run once at an item's end, takes longer to come into
            // the instruction cache than to run.
#pragma unroll 1
            for (; first < last; first += kUnit) {
                There<TYPE, D> there;
                bool edge = first + F::kKeys > all_see;
#pragma unroll
                for (int t = 0; t < F::kTiles; ++t) {
                    there[t] = tiles[t].there;
                    edge = edge || !there[t];
                }
                tiles_of(first + kUnit);
                if constexpr (!kLds) {
                    numbers_of(first + 2 * kUnit);
                }
                Scores<TYPE, D, RT> s;
                if constexpr (kLds) { // queries do not move into registers ahead of the loop
                    asm volatile("" ::: "memory");
                }
                scores_of<TYPE, D, RT>(s, keys, queries, lanes);
                if constexpr (kLds) { // behind the reads from LDS, which would wait for these
                    __builtin_amdgcn_sched_barrier(0);
                    numbers_of(first + 2 * kUnit);
                    __builtin_amdgcn_sched_barrier(0);
                }
                softmax_step<TYPE, D, RT>(s, acc, run, keys, p.scale, first, lanes, edge, there);
                segment.load_keys(keys, tiles);
                if (edge) {
                    settle_values<TYPE, D, RT>(values, run, shape.tokens, first, lanes, there);
                }
                scale_weights<TYPE, D, RT>(s, values);
                add_values<TYPE, D, RT>(acc, s, values);
                segment.load_values(values, tiles);
            }
        }
        // The wavefronts' parts, joined: 16 threads a row, 4 columns each and 64 further on.
        const bool whole = item.first == 0 && units == shape.units;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            __syncthreads(); // the rows before have been read
#pragma unroll
            for (int q = 0; q < F::kColumns / 4; ++q) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    *reinterpret_cast<float4*>(
                        &joined[wave][lanes.row][column_at<TYPE, D>(lanes.quad, r, q)]) =
                        make_float4(acc[rt][4 * q][r], acc[rt][4 * q + 1][r],
                                    acc[rt][4 * q + 2][r], acc[rt][4 * q + 3][r]);
                }
            }
            const float sum = row_sum(run[rt].sum);
            if (lanes.quad == 0) {
                stats[wave][lanes.row][0] = run[rt].top;
                stats[wave][lanes.row][1] = sum;
            }
            __syncthreads();
            const int row = threadIdx.x / 16;
            const int32_t rr = row0 + 16 * rt + row;
            if (rr < rows) {
                float top = stats[0][row][0];
#pragma unroll
                for (int i = 1; i < kWaves; ++i) {
                    top = fmaxf(top, stats[i][row][0]);
                }
                float weight[kWaves], total = 0.0f;
#pragma unroll
                for (int i = 0; i < kWaves; ++i) {
                    weight[i] = dev::part_weight(stats[i][row][0], top);
                    total = fmaf(weight[i], stats[i][row][1], total);
                }
                const int32_t i = rr / p.work.group;
                const int32_t head = item.head * p.work.group + (rr - i * p.work.group);
                const int64_t part = mfr::kv::part_of(index, place.chunk, item.begin) * (16 * RT) +
                                     16 * rt + row;
#pragma unroll
                for (int c0 = 0; c0 < D; c0 += 64) {
                    const int c = c0 + 4 * (threadIdx.x % 16);
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int w = 0; w < kWaves; ++w) {
                        v = dev::add_scaled(v, *reinterpret_cast<const float4*>(&joined[w][row][c]),
                                            weight[w]);
                    }
                    if (whole) {
                        dev::finish(p, shape.span.first + static_cast<int64_t>(i), head, c, v, top,
                                    total);
                    } else {
                        *reinterpret_cast<float4*>(p.parts.values + part * D + c) = v;
                        if (c == 0) {
                            *reinterpret_cast<float2*>(p.parts.stats + 2 * part) =
                                make_float2(top, total);
                        }
                    }
                }
            }
        }
        at += units;
    }
}

// Joins the parts of the items that were cut, rows 8 y .. 8 y + 7 of one a workgroup: of item x, where the
// items are those of the prefix and no more than chunks, otherwise of the one that began in chunk x and goes
// on behind it (if there is one). 32 lanes
// hold a part's row; they take a row's parts in order, or, where an item has few rows, share them (a part in
// `split`) and join through LDS. Workgroups go to the chip's dies in turn. Items of many rows that begin in
// every 8th or 16th chunk would all go to one die: each takes neighbouring ones instead (16 items of 128
// rows in 16 parts each: 5.6 us, 22 from one die). Items of few rows go where their first part was written
// and may still be in a cache (256 sequences in 512 chunks: 6.4 us, 8.3 elsewhere).
constexpr int kJoinRows = 8;
constexpr int kDies = 8;

__global__ __launch_bounds__(kThreads) void attention_paged_join_kernel(Params p, uint32_t count,
                                                                       bool by_item) {
    __shared__ float4 values[kJoinRows][32];
    __shared__ float2 stats[kJoinRows];
    const uint32_t pieces = static_cast<uint32_t>(p.work.tile_rows + kJoinRows - 1) / kJoinRows;
    uint32_t x, y;
    if (p.work.tile_rows == kManyRows) {
        const uint32_t per_die = (count * pieces + kDies - 1) / kDies;
        const uint32_t at = blockIdx.x % kDies * per_die + blockIdx.x / kDies;
        x = at / pieces;
        y = at - x * pieces;
    } else {
        y = blockIdx.x / count;
        x = blockIdx.x - y * count;
    }
    if (x >= count || y >= pieces) {
        return;
    }
    int64_t index = x, chunk;
    Shape shape;
    Item item;
    if (by_item) {
        shape = mfr::kv::shape_of(p.work, 0);
        chunk = mfr::kv::chunk_of(shape.count, p.groups);
        item = mfr::kv::item_of(shape, 0, index * shape.units);
        index = mfr::kv::quotient(item.begin, chunk);
    } else {
        const dev::Place place = dev::find(p.work, p.groups, [&](int64_t total, int64_t length) {
            // The last unit of a chunk that another one follows.
            return (index + 1) * length < total ? (index + 1) * length - 1 : int64_t{-1};
        });
        if (place.seq < 0) {
            return;
        }
        chunk = place.chunk;
        shape = mfr::kv::shape_of(p.work, place.seq);
        item = mfr::kv::item_of(shape, place.base, (index + 1) * chunk - 1);
    }
    const int64_t end = item.begin + shape.units;
    if (item.begin < index * chunk || end <= (index + 1) * chunk) {
        return;
    }
    const int32_t rows = shape.span.count * p.work.group;
    const int32_t row0 = item.tile * p.work.tile_rows + kJoinRows * static_cast<int32_t>(y);
    const int32_t here = min(kJoinRows, min((item.tile + 1) * p.work.tile_rows, rows) - row0);
    if (here <= 0) {
        return;
    }
    const int64_t last = mfr::kv::quotient(end - 1, chunk); // the chunk of its last unit
    const int parts = static_cast<int>(last - index) + 1;
    const int split = here <= 1 ? 8 : here <= 2 ? 4 : here <= 4 ? 2 : 1;
    const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
    const int32_t r = group / split;
    const int c = 4 * lane;
    const int64_t first = mfr::kv::part_of(index, chunk, item.begin); // the others' are 2 apart
    const int64_t row = row0 - item.tile * p.work.tile_rows + r;
    float top = -INFINITY, sum = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r < here) {
        constexpr int kAtOnce = 8;
        for (int i0 = group % split; i0 < parts; i0 += kAtOnce * split) {
            float2 stat[kAtOnce];
            float4 value[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const int i = i0 + k * split;
                stat[k] = make_float2(-INFINITY, 0.0f);
                value[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (i < parts) {
                    const int64_t part = (i == 0 ? first : 2 * (index + i)) * p.work.tile_rows + row;
                    stat[k] = *reinterpret_cast<const float2*>(p.parts.stats + 2 * part);
                    if (c < p.depth) {
                        value[k] = *reinterpret_cast<const float4*>(p.parts.values + part * p.depth + c);
                    }
                }
            }
            float most = top;
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                most = fmaxf(most, stat[k].x);
            }
            const float a = dev::part_weight(top, most);
            sum *= a;
            v = dev::scaled(v, a);
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const float b = dev::part_weight(stat[k].x, most);
                sum = fmaf(b, stat[k].y, sum);
                v = dev::add_scaled(v, value[k], b);
            }
            top = most;
        }
    }
    if (split > 1) { // the whole workgroup
        values[group][lane] = v;
        if (lane == 0) {
            stats[group] = make_float2(top, sum);
        }
        __syncthreads();
        if (group % split != 0) {
            return;
        }
#pragma unroll 1
        for (int k = 1; k < split; ++k) {
            const float2 other = stats[group + k];
            const float most = fmaxf(top, other.x);
            const float a = dev::part_weight(top, most), b = dev::part_weight(other.x, most);
            sum = fmaf(b, other.y, a * sum);
            v = dev::add_scaled(dev::scaled(v, a), values[group + k][lane], b);
            top = most;
        }
    }
    if (r < here && c < p.depth) {
        const int32_t i = (row0 + r) / p.work.group;
        dev::finish(p, shape.span.first + static_cast<int64_t>(i),
                    item.head * p.work.group + (row0 + r - i * p.work.group), c, v, top, sum);
    }
}

template <int TYPE, int D> void launch_rows(const Params& p, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(p.groups);
    if (p.work.tile_rows == 16) {
        if (p.cache.d == D) {
            attention_paged_few_kernel<TYPE, D, 1, true><<<grid, kThreads, 0, stream>>>(p);
        } else {
            attention_paged_few_kernel<TYPE, D, 1, false><<<grid, kThreads, 0, stream>>>(p);
        }
    } else {
        if (p.cache.d == D) {
            attention_paged_few_kernel<TYPE, D, 2, true><<<grid, kThreads, 0, stream>>>(p);
        } else {
            attention_paged_few_kernel<TYPE, D, 2, false><<<grid, kThreads, 0, stream>>>(p);
        }
    }
    mfr::check_launch("attention_paged_few_kernel");
}

template <int TYPE> void launch_depth(const Params& p, hipStream_t stream) {
    if (p.depth == 64) {
        launch_rows<TYPE, 64>(p, stream);
    } else {
        launch_rows<TYPE, 128>(p, stream);
    }
}

} // namespace

namespace mfr::paged {

void launch_few(const Params& p, int32_t type, hipStream_t stream) {
    switch (type) {
    case MFR_KV_F32: launch_depth<MFR_KV_F32>(p, stream); break;
    case MFR_KV_BF16: launch_depth<MFR_KV_BF16>(p, stream); break;
    default: launch_depth<MFR_KV_F8>(p, stream); break;
    }
}

void launch_join(const Params& p, hipStream_t stream) {
    int64_t count = p.groups;
    bool by_item = false;
    if (p.work.shared != 0) { // known here
        const int64_t items = static_cast<int64_t>(kv::shape_of(p.work, 0).tiles) * p.work.heads;
        by_item = items <= count;
        count = by_item ? items : count;
    }
    const int64_t pieces = (p.work.tile_rows + kJoinRows - 1) / kJoinRows;
    const unsigned blocks = static_cast<unsigned>((count * pieces + kDies - 1) / kDies * kDies);
    attention_paged_join_kernel<<<blocks, kThreads, 0, stream>>>(p, static_cast<uint32_t>(count),
                                                              by_item);
    check_launch("attention_paged_join_kernel");
}

} // namespace mfr::paged
