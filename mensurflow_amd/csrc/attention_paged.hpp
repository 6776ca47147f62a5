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
constexpr float kLog2e = 1.4426950408889634f;

// Unnormalised results of rows: weighted values [row][depth], and the running maximum (of base-2
// scores) and sum [row][2].
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

// The launches (attention_paged_few.hip, attention_paged_tiles.hip): `p` filled but for nothing.
void launch_few(const Params& p, int32_t type, hipStream_t stream);
void launch_join(const Params& p, hipStream_t stream);

} // namespace mfr::paged

namespace mfr::paged::dev {

// The sum of v over the workgroup, and over the threads before this one.
struct Scan {
    int64_t total, before;
};

__device__ inline Scan scan_of(int64_t v, int64_t* waves) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    int64_t upto = v;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
        const int64_t other = __shfl_up(static_cast<long long>(upto), step, 64);
        upto += lane >= step ? other : 0;
    }
    __syncthreads(); // `waves` of a call before has been read
    if (lane == 63) {
        waves[wave] = upto;
    }
    __syncthreads();
    Scan s{0, upto - v};
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        s.before += i < wave ? waves[i] : 0;
        s.total += waves[i];
    }
    return s;
}

// Where in the work a workgroup starts.
struct Place {
    int64_t total, chunk;
    int32_t seq;
    int64_t base; // of the sequence, in the list of units
};

// Finds the sequence that holds unit `at(total, chunk)` of the list, for all threads; seq -1 where `at`
// gives a negative place. A sequence a thread, in rounds.
template <typename At>
__device__ inline Place find(const Work& w, int32_t groups, At at) {
    __shared__ int64_t waves[kWaves];
    __shared__ int64_t found[2];
    const int32_t sequences = kv::sequences_of(w);
    Place p{};
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
    p.seq = -1;
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
    p.seq = __builtin_amdgcn_readfirstlane(static_cast<int>(found[0]));
    p.base = found[1];
    return p;
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
