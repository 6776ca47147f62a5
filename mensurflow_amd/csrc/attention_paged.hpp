// What the kernels of mfr_attention_paged share: their parameters, the search for a workgroup's place in
// the work (kv_work.hpp), and how results are written and joined.
#pragma once

#include "kv.hpp"
#include "kv_work.hpp"

namespace mfr::paged {

using kv::Batch;
using kv::Cache;
using kv::Heads;
using kv::Item;
using kv::Shape;
using kv::Work;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
template <int TYPE> constexpr int kBytes = TYPE == MFR_KV_F32 ? 4 : TYPE == MFR_KV_BF16 ? 2 : 1;

// Unnormalised results of rows: weighted values [row][depth], and the reference (of base-2 scores: a
// weight is 2 to a score less it) and sum of the weights [row][2].
struct Parts {
    float* values;
    float* stats;
};

struct Params {
    Work work;
    Cache cache;
    Heads q;
    float* out;
    int64_t out_ts, out_hs;
    int32_t q_heads;
    int32_t causal;
    float scale;    // times log2 e
    int32_t groups; // workgroups that share the work
    int32_t depth;  // of parts: d rounded up to 64 or 128
    Parts parts;    // [2 groups][tile_rows]
    // What the prefix gave each row and query head, [rows][q_heads]: written by the launch over the
    // prefix, read where rows are finished by the one over the sequences. Null: no prefix.
    Parts prefix;
};

// The forms: tiles of 16 or 32 rows (attention_paged_few.hip), and of 128 rows, not in fp32
// (attention_paged_tiles.hip).
constexpr int32_t kManyRows = 128;

// Workgroups that a compute unit holds at once, by the registers of the forms. (One tile of rows of 128 in 8
// bits, its queries in LDS, fits three times into 168 registers with 21 spilled: 64 sequences on up to 8191
// tokens 144 us, 122 twice.)
constexpr int per_unit(int32_t type, int depth, int32_t tile_rows) {
    if (tile_rows == kManyRows) {
        return 1;
    }
    if (tile_rows == 32) {
        return type == MFR_KV_F32 && depth == 128 ? 1 : 2;
    }
    return depth == 64 ? 3 : 2;
}

void launch_few(const Params& p, int32_t type, hipStream_t stream);
void launch_tiles(const Params& p, int32_t type, hipStream_t stream);
void launch_join(const Params& p, hipStream_t stream);

} // namespace mfr::paged

namespace mfr::paged::dev {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float exp2_native(float x) { return __builtin_amdgcn_exp2f(x); }

// Two floats cut into three bf16 parts each (the leading 8 bits of what is left, so that no part
// overflows), packed with x in the low half.
__device__ __forceinline__ void cut_pair(float x, float y, uint32_t& p0, uint32_t& p1,
                                         uint32_t& p2) {
    const auto high = [](float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); };
    const auto pack = [](float u, float v) {
        return __builtin_amdgcn_perm(__float_as_uint(v), __float_as_uint(u), 0x07060302u);
    };
    p0 = pack(x, y);
    x -= high(x);
    y -= high(y);
    p1 = pack(x, y);
    x -= high(x);
    y -= high(y);
    p2 = pack(x, y);
}

// Two e4m3 numbers of a half of w as bf16.
template <bool HIGH> __device__ __forceinline__ uint32_t widen(uint32_t w) {
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH));
}

// The largest of v over the four lanes of one row (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float row_max(float v) {
    float a, b;
    mfr::dev::swap_pair<true>(v, a, b);
    v = fmaxf(a, b);
    mfr::dev::swap_pair<false>(v, a, b);
    return fmaxf(a, b);
}

// Over two lanes, l and l ^ 32.
__device__ __forceinline__ float max_halves(float v) {
    float a, b;
    mfr::dev::swap_pair<true>(v, a, b);
    return fmaxf(a, b);
}

__device__ __forceinline__ float sum_halves(float v) {
    float a, b;
    mfr::dev::swap_pair<true>(v, a, b);
    return a + b;
}

__device__ __forceinline__ float row_sum(float v) {
    float a, b;
    mfr::dev::swap_pair<true>(v, a, b);
    v = a + b;
    mfr::dev::swap_pair<false>(v, a, b);
    return a + b;
}

// A workgroup barrier that waits for this wavefront's LDS accesses only: loads from memory stay under way.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The running softmax of a lane's row.
struct Running {
    float top = -INFINITY; // the weights' reference: near the maximum so far
    float sum = 0.0f; // this lane's share
    int32_t seen;     // tokens that the row sees
};

// The weights of a tile of rows as B operands of bf16 products.
struct Cut {
    bf16x8 part[3];
};
__device__ __forceinline__ Cut cut_weights(const floatx4& a, const floatx4& b) {
    uint4 cut[3];
    cut_pair(a[0], a[1], cut[0].x, cut[1].x, cut[2].x);
    cut_pair(a[2], a[3], cut[0].y, cut[1].y, cut[2].y);
    cut_pair(b[0], b[1], cut[0].z, cut[1].z, cut[2].z);
    cut_pair(b[2], b[3], cut[0].w, cut[1].w, cut[2].w);
    return {__builtin_bit_cast(bf16x8, cut[0]), __builtin_bit_cast(bf16x8, cut[1]),
            __builtin_bit_cast(bf16x8, cut[2])};
}

// sums + the products of one column, the smallest parts first.
__device__ __forceinline__ floatx4 add_column(floatx4 sums, bf16x8 column, const Cut& w) {
#pragma unroll
    for (int i = 2; i >= 0; --i) {
        sums = __builtin_amdgcn_mfma_f32_16x16x32_bf16(column, w.part[i], sums, 0, 0, 0);
    }
    return sums;
}

// Whether any of the numbers of a cache in a word is an infinity or NaN, and the word with zeros for
// those: values that some rows do not see must not meet their weights of 0. (Rows that see one are made
// NaN through their sum.)
template <int TYPE> __device__ __forceinline__ bool is_odd(uint32_t w) {
    if constexpr (TYPE == MFR_KV_F32) {
        return (w & 0x7f800000u) == 0x7f800000u;
    } else if constexpr (TYPE == MFR_KV_BF16) {
        return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
    } else { // a byte of 0x7f or 0xff: 0x01 is carried into its top bit
        return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
    }
}
template <int TYPE> __device__ __forceinline__ uint32_t without_odd(uint32_t w) {
    if constexpr (TYPE == MFR_KV_F32) {
        return is_odd<TYPE>(w) ? 0u : w;
    } else if constexpr (TYPE == MFR_KV_BF16) {
        return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) |
               ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
    } else {
        const uint32_t tops = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        return w & ~((tops >> 7) * 0xffu);
    }
}

struct Scan {
    int64_t total, before;
};

// The sum of v over the wavefront, and over the lanes before this one.
__device__ inline Scan wave_scan(int64_t v) {
    const int lane = threadIdx.x % 64;
    int64_t upto = v;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const int64_t other = __shfl_up(static_cast<long long>(upto), step, 64);
        upto += lane >= step ? other : 0;
    }
    return {__shfl(static_cast<long long>(upto), 63, 64), upto - v};
}

// The same over the workgroup.
__device__ inline Scan scan_of(int64_t v, int64_t* waves) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const Scan own = wave_scan(v);
    __syncthreads(); // `waves` of a call before has been read
    if (lane == 63) {
        waves[wave] = own.total;
    }
    __syncthreads();
    Scan s{0, own.before};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        s.before += i < wave ? waves[i] : 0;
        s.total += waves[i];
    }
    return s;
}

// A number at a uniform address in memory that this launch does not write, through the scalar cache: its
// wait is not one for the loads of keys and values that are under way.
__device__ __forceinline__ int32_t uniform_load(const int32_t* p) {
    return *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(
        reinterpret_cast<uintptr_t>(p));
}

// A lane's address in memory (and not anywhere: a flat load counts as one from LDS too, and every wait for
// LDS would wait for it), which the compiler takes as it is: a load's uniform offset is added to it in one
// instruction then, instead of all its terms one by one.
typedef const __attribute__((address_space(1))) uint8_t* GlobalBytes;
__device__ __forceinline__ GlobalBytes lane_address(const void* p, uint32_t lane_offset) {
    uint64_t at = reinterpret_cast<uintptr_t>(p) + lane_offset;
    asm volatile("" : "+v"(at));
    return reinterpret_cast<GlobalBytes>(at);
}
// T from `offset` bytes behind it, aligned to its size.
template <typename T> __device__ __forceinline__ T load_at(GlobalBytes base, int64_t offset) {
    typedef uint32_t Words __attribute__((ext_vector_type(sizeof(T) / 4)));
    const Words w = *reinterpret_cast<const __attribute__((address_space(1))) Words*>(base + offset);
    return __builtin_bit_cast(T, w);
}

// Where 16 tokens lie: in bytes from a head's first row, and from the first scale.
struct TileAt {
    int64_t at;
    int64_t scale_at;
    bool there; // their page is one of the cache's; another one's place is given otherwise
};

// The pages of a sequence (or the prefix), and one head of them, for the tokens in front of `last`: loads that
// run ahead of the work's end get the last 16 of those again, from a cache (one query against 4096 tokens
// read 32 MiB of 16 without this).
struct Pages {
    const int32_t* table;
    int32_t most; // the first token of the last 16
    int32_t head;

    __device__ __forceinline__ Pages(const Params& p, int32_t last, int32_t seq, int32_t head)
        : table(p.work.shared != 0 ? p.work.batch.prefix_pages
                                   : p.work.batch.table + seq * p.work.batch.table_rs),
          most((last - 1) & ~15), head(head) {}

    // The number of the page of 16 tokens; ones behind the last are taken as the last.
    __device__ __forceinline__ int32_t page(const Params& p, int32_t token) const {
        return uniform_load(table + (min(token, most) >> p.work.batch.page_log2));
    }
    __device__ __forceinline__ TileAt at(const Params& p, int32_t token, int32_t page) const {
        // (kv::page_checked without a branch.)
        const bool there = static_cast<uint32_t>(page) < static_cast<uint32_t>(p.work.batch.pages);
        const int64_t number = there ? page : 0;
        const int32_t slot = min(token, most) & ((1 << p.cache.page_log2) - 1);
        return {number * p.cache.page_stride + static_cast<int64_t>(slot) * p.cache.token_stride,
                4 * (((number * p.cache.heads + head) << p.cache.page_log2) + slot), there};
    }
};

// Where in the work a workgroup starts.
struct Place {
    int64_t total, chunk;
    int32_t seq;
    int64_t base; // of the sequence, in the list of units
};

// A number that is the same in all lanes, known to be so: what is found from it is in scalar registers.
__device__ __forceinline__ int32_t uniform(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    const uint32_t low = uniform(static_cast<int32_t>(v));
    const uint32_t high = uniform(static_cast<int32_t>(v >> 32));
    return static_cast<int64_t>(static_cast<uint64_t>(high) << 32 | low);
}

// Finds the sequence that holds unit `at(total, chunk)` of the list, for all threads; seq -1 where `at`
// gives a negative place. Up to 64 sequences are each wavefront's own matter, a lane each; more are a
// thread's each, in rounds.
template <typename At>
__device__ inline Place find_any(const Work& w, int32_t groups, At at) {
    const int32_t sequences = kv::sequences_of(w);
    Place p{};
    p.seq = -1;
    if (sequences <= 64) {
        int64_t mine = 0;
        Scan scan;
        if (sequences == 1) {
            mine = kv::shape_of(w, 0).count;
            scan = {mine, 0};
        } else {
            const int32_t lane = threadIdx.x % 64;
            mine = lane < sequences ? kv::shape_of(w, lane).count : 0;
            scan = wave_scan(mine);
        }
        p.total = scan.total;
        p.chunk = kv::chunk_of(p.total, groups);
        const int64_t target = at(p.total, p.chunk);
        if (target >= 0) {
            const uint64_t here = __ballot(scan.before <= target && target < scan.before + mine);
            p.seq = sequences == 1 ? 0 : static_cast<int32_t>(__builtin_ctzll(here));
            p.base = sequences == 1 ? 0 : __shfl(static_cast<long long>(scan.before), p.seq, 64);
        }
        return p;
    }
    __shared__ int64_t waves[kWaves];
    __shared__ int64_t found[2];
    Scan first{};
    int64_t mine = 0;
    for (int32_t s0 = 0; s0 < sequences; s0 += kThreads) {
        const int32_t s = s0 + static_cast<int32_t>(threadIdx.x);
        const int64_t v = s < sequences ? kv::shape_of(w, s).count : 0;
        const Scan scan = scan_of(v, waves);
        if (s0 == 0) {
            first = scan;
            mine = v;
        }
        p.total += scan.total;
    }
    p.chunk = kv::chunk_of(p.total, groups);
    const int64_t target = at(p.total, p.chunk);
    if (target < 0) {
        return p;
    }
    int64_t base = 0;
    for (int32_t s0 = 0; s0 < sequences; s0 += kThreads) {
        Scan scan = first;
        if (s0 > 0) {
            const int32_t s = s0 + static_cast<int32_t>(threadIdx.x);
            mine = s < sequences ? kv::shape_of(w, s).count : 0;
            scan = scan_of(mine, waves);
        }
        const int64_t here = base + scan.before;
        if (here <= target && target < here + mine) {
            found[0] = s0 + static_cast<int32_t>(threadIdx.x);
            found[1] = here;
        }
        base += scan.total;
        if (target < base) {
            break; // all threads alike
        }
    }
    __syncthreads();
    p.seq = static_cast<int32_t>(found[0]);
    p.base = found[1];
    return p;
}
template <typename At>
__device__ inline Place find(const Work& w, int32_t groups, At at) {
    const Place p = find_any(w, groups, at);
    return {uniform(p.total), uniform(p.chunk), uniform(p.seq), uniform(p.base)};
}

// Moves on to the next sequence that has units; false where there is none. Those that follow without rows (a
// batch of slots may hold many) are passed 64 at a time.
__device__ inline bool advance(const Work& w, int32_t& seq, Shape& shape) {
    if (++seq >= kv::sequences_of(w)) {
        return false;
    }
    shape = kv::shape_of(w, seq);
    while (shape.count == 0) {
        const int32_t s = seq + 1 + static_cast<int32_t>(threadIdx.x % 64);
        const uint64_t found =
            __ballot(s < kv::sequences_of(w) && kv::shape_of(w, s).count > 0);
        seq += found != 0 ? 1 + __builtin_ctzll(found) : 64;
        if (seq >= kv::sequences_of(w) - 1 && found == 0) {
            return false;
        }
        if (found != 0) {
            shape = kv::shape_of(w, seq);
        }
    }
    return true;
}

// exp2(m - top), 0 for a part that saw nothing (m = -inf, also where every part did).
__device__ inline float part_weight(float m, float top) {
    return m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
}

__device__ inline float4 scaled(float4 v, float by) {
    return make_float4(v.x * by, v.y * by, v.z * by, v.w * by);
}

__device__ inline float4 add_scaled(float4 a, float4 v, float by) {
    return make_float4(fmaf(v.x, by, a.x), fmaf(v.y, by, a.y), fmaf(v.z, by, a.z),
                       fmaf(v.w, by, a.w));
}

// Four columns from c on of a row's whole result: to the prefix's parts, or joined with them,
// divided by the sum and written out.
__device__ inline void finish(const Params& p, int64_t row, int32_t head, int c, float4 v, float top,
                              float sum) {
    const int64_t at = row * p.q_heads + head;
    if (p.work.shared != 0) {
        *reinterpret_cast<float4*>(p.prefix.values + at * p.depth + c) = v;
        if (c == 0) {
            *reinterpret_cast<float2*>(p.prefix.stats + 2 * at) = make_float2(top, sum);
        }
        return;
    }
    if (c >= p.cache.d) {
        return;
    }
    if (p.prefix.values != nullptr) {
        const float2 stats = *reinterpret_cast<const float2*>(p.prefix.stats + 2 * at);
        const float4 other = *reinterpret_cast<const float4*>(p.prefix.values + at * p.depth + c);
        const float most = fmaxf(top, stats.x);
        const float a = part_weight(top, most), b = part_weight(stats.x, most);
        sum = fmaf(b, stats.y, a * sum);
        v = add_scaled(scaled(v, a), other, b);
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    mfr::dev::store_loose(p.out + row * p.out_ts + head * p.out_hs + c, scaled(v, inv));
}

} // namespace mfr::paged::dev
