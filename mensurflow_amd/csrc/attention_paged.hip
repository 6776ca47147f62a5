// mfr_attention_paged: attention of a step's rows against a paged cache (kv.hpp).
//
// The plain form: a workgroup per row and query head; 32 lanes hold a token's row, 4 columns each, so 8
// tokens go at a time, each lane group with its own running softmax; they are joined through LDS.
#include "kv.hpp"

#include <algorithm>
#include <cmath>

namespace {

using mfr::kv::Batch;
using mfr::kv::Cache;
using mfr::kv::Heads;

struct PagedParams {
    Cache cache;
    Batch batch;
    Heads q;
    float* out;
    int64_t out_ts, out_hs;
    int32_t q_heads, group;
    float scale;
    int32_t causal;
};

constexpr float kLog2e = 1.4426950408889634f;

template <int TYPE>
__device__ inline float4 load_row(const uint8_t* row, const float* scale, int c) {
    if constexpr (TYPE == MFR_KV_F32) {
        return *reinterpret_cast<const float4*>(row + 4 * c);
    } else if constexpr (TYPE == MFR_KV_BF16) {
        const uint2 w = *reinterpret_cast<const uint2*>(row + 2 * c);
        return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u),
                           __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
    } else {
        const int w = *reinterpret_cast<const int*>(row + c);
        const float s = *scale;
        return make_float4(__builtin_amdgcn_cvt_f32_fp8(w, 0) * s,
                           __builtin_amdgcn_cvt_f32_fp8(w, 1) * s,
                           __builtin_amdgcn_cvt_f32_fp8(w, 2) * s,
                           __builtin_amdgcn_cvt_f32_fp8(w, 3) * s);
    }
}

template <int TYPE> __global__ __launch_bounds__(256) void attention_paged_kernel(PagedParams p) {
    __shared__ float4 values[8][32];
    __shared__ float tops[8], sums[8];
    const int64_t blocks = static_cast<int64_t>(p.batch.rows) * p.q_heads;
    const int lane = threadIdx.x % 32, part = threadIdx.x / 32;
    const int c = 4 * lane;
    const bool live = c < p.cache.d;
    for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
        const int32_t row = static_cast<int32_t>(b / p.q_heads);
        const int32_t head = static_cast<int32_t>(b - static_cast<int64_t>(row) * p.q_heads);
        const int32_t seq = mfr::kv::sequence_of(p.batch, row);
        if (seq < 0) {
            continue;
        }
        const mfr::kv::Span span = mfr::kv::span_of(p.batch, seq);
        int64_t seen = mfr::kv::length_of(p.batch, seq);
        if (p.causal != 0) {
            const int64_t place =
                mfr::kv::first_place(p.batch, seq, span.count) + (row - span.first);
            seen = place + 1 < seen ? (place < 0 ? 0 : place + 1) : seen;
        }
        const int64_t kv_head = head / p.group;
        float4 q = make_float4(0.f, 0.f, 0.f, 0.f), acc = q;
        if (live) {
            q = mfr::dev::load_loose(p.q.p + row * p.q.ts + head * p.q.hs + c);
        }
        float top = -INFINITY, sum = 0.0f;
        const int64_t prefix = p.batch.prefix;
        for (int64_t j = part; j < prefix + seen; j += 8) {
            const int64_t place = j < prefix ? j : j - prefix;
            const int32_t page = j < prefix
                                     ? mfr::kv::prefix_page_of(p.batch, static_cast<int32_t>(j))
                                     : mfr::kv::page_of(p.batch, seq, place);
            if (page < 0) {
                continue;
            }
            const int64_t slot = place & ((1 << p.cache.page_log2) - 1);
            const int64_t at = page * p.cache.page_stride + slot * p.cache.token_stride +
                               kv_head * p.cache.head_stride;
            const int64_t scale_at =
                ((page * p.cache.heads + kv_head) << p.cache.page_log2) + slot;
            float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
            if (live) {
                k = load_row<TYPE>(p.cache.k + at, p.cache.k_scales + scale_at, c);
                v = load_row<TYPE>(p.cache.v + at, p.cache.v_scales + scale_at, c);
            }
            float s = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, q.w * k.w)));
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) {
                s += __shfl_xor(s, m, 64);
            }
            s = p.scale * s * kLog2e;
            const float most = fmaxf(top, s);
            const float reference = most == -INFINITY ? 0.0f : most;
            const float shrink = __builtin_amdgcn_exp2f(top - reference);
            const float w = __builtin_amdgcn_exp2f(s - reference);
            top = most;
            sum = fmaf(sum, shrink, w);
            acc.x = fmaf(acc.x, shrink, w * v.x);
            acc.y = fmaf(acc.y, shrink, w * v.y);
            acc.z = fmaf(acc.z, shrink, w * v.z);
            acc.w = fmaf(acc.w, shrink, w * v.w);
        }
        values[part][lane] = acc;
        if (lane == 0) {
            tops[part] = top;
            sums[part] = sum;
        }
        __syncthreads();
        if (part == 0 && live) {
            float most = -INFINITY;
            for (int i = 0; i < 8; ++i) {
                most = fmaxf(most, tops[i]);
            }
            float total = 0.0f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = 0; i < 8; ++i) {
                const float w = tops[i] == -INFINITY ? 0.0f
                                                     : __builtin_amdgcn_exp2f(tops[i] - most);
                total = fmaf(w, sums[i], total);
                v.x = fmaf(w, values[i][lane].x, v.x);
                v.y = fmaf(w, values[i][lane].y, v.y);
                v.z = fmaf(w, values[i][lane].z, v.z);
                v.w = fmaf(w, values[i][lane].w, v.w);
            }
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            mfr::dev::store_loose(p.out + row * p.out_ts + head * p.out_hs + c,
                                  make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
        }
        __syncthreads();
    }
}

// The descriptor's checks (of shapes, layouts and pointers: no device is needed).
PagedParams checked(const mfr_attention_paged_desc* desc) {
    using mfr::require;
    require(desc != nullptr, "attention_paged: null descriptor");
    const mfr_attention_paged_desc& d = *desc;
    PagedParams p{};
    p.cache = mfr::kv::checked(d.cache, false, "attention_paged");
    p.batch = mfr::kv::checked(d.batch, d.cache, "attention_paged");
    require(d.q_heads >= 1 && d.q_heads % d.cache.heads == 0,
            "attention_paged: q's heads are no multiple of the cache's");
    mfr::kv::supported(d.q_heads <= mfr::kv::kMostHeads, "attention_paged: too many heads");
    require(std::isfinite(d.scale), "attention_paged: scale is not finite");
    if (p.batch.rows > 0) {
        mfr::kv::check_heads(d.q, d.q_ts, d.q_hs, d.batch.rows, d.q_heads, d.cache.d, false,
                             "attention_paged: q");
        mfr::kv::check_heads(d.out, d.out_ts, d.out_hs, d.batch.rows, d.q_heads, d.cache.d, true,
                             "attention_paged: out");
    }
    p.q = {d.q, d.q_ts, d.q_hs};
    p.out = d.out;
    p.out_ts = d.out_ts;
    p.out_hs = d.out_hs;
    p.q_heads = static_cast<int32_t>(d.q_heads);
    p.group = static_cast<int32_t>(d.q_heads / d.cache.heads);
    p.scale = d.scale != 0.0f ? d.scale
                              : static_cast<float>(1.0 / std::sqrt(static_cast<double>(d.cache.d)));
    p.causal = d.causal;
    return p;
}

} // namespace

extern "C" {

int mfr_attention_paged(mfr_stream_t stream, const mfr_attention_paged_desc* desc) {
    return mfr::guarded([&] {
        const PagedParams p = checked(desc);
        auto& s = mfr::stream_of(stream);
        if (p.batch.rows == 0) {
            return;
        }
        const unsigned grid = static_cast<unsigned>(
            std::min<int64_t>(static_cast<int64_t>(p.batch.rows) * p.q_heads, 1 << 20));
        switch (desc->cache.type) {
        case MFR_KV_F32: attention_paged_kernel<MFR_KV_F32><<<grid, 256, 0, s.stream>>>(p); break;
        case MFR_KV_BF16: attention_paged_kernel<MFR_KV_BF16><<<grid, 256, 0, s.stream>>>(p); break;
        default: attention_paged_kernel<MFR_KV_F8><<<grid, 256, 0, s.stream>>>(p); break;
        }
        mfr::check_launch("attention_paged_kernel");
    });
}

int mfr_attention_paged_workspace(int device, const mfr_attention_paged_desc* desc, size_t* bytes) {
    return mfr::guarded([&] {
        (void)device;
        (void)checked(desc);
        mfr::require(bytes != nullptr, "attention_paged: null result");
        *bytes = 0;
    });
}

} // extern "C"
