// The paged cache (mfr_kv_cache, mfr_kv_batch): what the kernels that write and read it share.
#pragma once

#include "common.hpp"
#include "kv_places.hpp"

#include <string>

namespace mfr::kv {

// Strides are bytes here.
struct Cache {
    uint8_t* k;
    uint8_t* v;
    int64_t page_stride, head_stride;
    uint32_t token_stride;
    int32_t heads, d;
    int32_t page_log2;
    float* k_scales; // [pages, heads, page]
    float* v_scales;
};

constexpr int64_t kMostDepth = 128;
constexpr int64_t kMostTokens = int64_t{1} << 30;
constexpr int64_t kMostRows = int64_t{1} << 30;
constexpr int64_t kMostSequences = int64_t{1} << 24;
constexpr int64_t kMostHeads = int64_t{1} << 20;
constexpr int64_t kMostPages = (int64_t{1} << 31) - 1;
constexpr int64_t kMostTokenStride = int64_t{1} << 24; // bytes: a page's 32768 rows have 2^39
constexpr int64_t kMostStride = int64_t{1} << 40;

// Whether `count` steps of a stride stay inside 2^56 elements, and so inside 64 bits.
inline bool reaches(int64_t stride, int64_t count) {
    return stride == 0 || count - 1 <= (int64_t{1} << 56) / stride;
}

inline int64_t type_bytes(int32_t type) {
    return type == MFR_KV_F32 ? 4 : type == MFR_KV_BF16 ? 2 : 1;
}

inline void supported(bool condition, const std::string& message) {
    if (!condition) {
        throw Error(MFR_E_UNSUPPORTED, message);
    }
}

// Checks a cache and takes it over. `written`: no two of its rows may be one place.
inline Cache checked(const mfr_kv_cache& d, bool written, const char* what) {
    const std::string at = std::string(what) + ": the cache ";
    require(d.type == MFR_KV_F32 || d.type == MFR_KV_BF16 || d.type == MFR_KV_F8,
            at + "has an unknown type");
    require(d.pages >= 0 && d.heads >= 1 && d.d >= 1, at + "has no heads or a negative size");
    supported(d.d % 16 == 0 && d.d <= kMostDepth,
              at + "needs rows of 16, 32, ..., 128 (a multiple of 16)");
    supported(d.page_size >= 16 && d.page_size <= 32768 && (d.page_size & (d.page_size - 1)) == 0,
              at + "needs pages of a power of two of tokens, 16 to 32768");
    supported(d.pages <= kMostPages && d.heads <= kMostHeads, at + "has too many pages or heads");
    const int64_t bytes = type_bytes(d.type);
    require(d.page_stride >= 0 && d.token_stride >= 0 && d.head_stride >= 0,
            at + "has negative strides");
    supported(d.token_stride <= kMostTokenStride / bytes && d.page_stride <= kMostStride / bytes &&
                  d.head_stride <= kMostStride / bytes,
              at + "has strides that are too long");
    supported(reaches(d.page_stride, d.pages) && reaches(d.head_stride, d.heads),
              at + "reaches further than memory");
    require(d.pages == 0 || (d.k != nullptr && d.v != nullptr), at + "has a null pointer");
    supported(aligned16(d.k) && aligned16(d.v) && d.page_stride * bytes % 16 == 0 &&
                  d.token_stride * bytes % 16 == 0 && d.head_stride * bytes % 16 == 0,
              at + "needs 16-byte aligned rows");
    if (d.type == MFR_KV_F8) {
        require(d.pages == 0 || (d.k_scales != nullptr && d.v_scales != nullptr),
                at + "needs scales in 8 bits");
        supported(aligned16(d.k_scales) && aligned16(d.v_scales),
                  at + "needs 16-byte aligned scales");
    }
    if (written && d.pages > 0) {
        // The dimensions by stride: each steps past all of the ones inside it.
        int64_t stride[3] = {d.page_stride, d.token_stride, d.head_stride};
        int64_t count[3] = {d.pages, d.page_size, d.heads};
        for (int i = 0; i < 2; ++i) {
            for (int j = 0; j < 2 - i; ++j) {
                if (stride[j] > stride[j + 1]) {
                    std::swap(stride[j], stride[j + 1]);
                    std::swap(count[j], count[j + 1]);
                }
            }
        }
        int64_t reach = d.d; // elements that the dimensions so far span
        for (int i = 0; i < 3; ++i) {
            if (count[i] > 1) {
                require(stride[i] >= reach, at + "has rows that overlap");
                reach += stride[i] * (count[i] - 1);
            }
        }
        require(d.k != d.v, at + "holds keys and values in one place");
    }
    int log2 = 0;
    while ((1 << log2) < d.page_size) {
        ++log2;
    }
    return {static_cast<uint8_t*>(d.k),
            static_cast<uint8_t*>(d.v),
            d.page_stride * bytes,
            d.head_stride * bytes,
            static_cast<uint32_t>(d.token_stride * bytes),
            static_cast<int32_t>(d.heads),
            static_cast<int32_t>(d.d),
            log2,
            d.k_scales,
            d.v_scales};
}

inline Batch checked(const mfr_kv_batch& d, const mfr_kv_cache& cache, const char* what) {
    const std::string at = std::string(what) + ": the batch ";
    require(d.rows >= 0 && d.sequences >= 0 && d.width >= 0 && d.prefix >= 0,
            at + "has a negative size");
    supported(d.rows <= kMostRows && d.sequences <= kMostSequences, at + "is too large");
    supported(d.width <= kMostTokens / cache.page_size && d.prefix <= kMostTokens,
              at + "has too many tokens a sequence");
    Batch b{};
    if (d.rows == 0 || d.sequences == 0) {
        return b;
    }
    require(d.lengths != nullptr, at + "has no lengths");
    require(d.width == 0 || d.table != nullptr, at + "has no table");
    require(d.width == 0 || d.sequences == 1 || (d.table_rs >= 0 && d.table_rs <= kMostStride),
            at + "has a bad table stride");
    require(d.prefix == 0 || d.prefix_pages != nullptr, at + "has no pages for its prefix");
    if (d.starts == nullptr) {
        require(d.rows % d.sequences == 0,
                at + "has no starts, and rows that are not whole for each sequence");
    }
    b.rows = static_cast<int32_t>(d.rows);
    b.sequences = static_cast<int32_t>(d.sequences);
    b.each = static_cast<int32_t>(d.rows / d.sequences);
    b.starts = d.starts;
    b.lengths = d.lengths;
    b.table = d.table;
    b.table_rs = d.sequences == 1 ? 0 : d.table_rs;
    b.width = static_cast<int32_t>(d.width);
    b.pages = static_cast<int32_t>(cache.pages);
    b.prefix_pages = d.prefix_pages;
    b.prefix = static_cast<int32_t>(d.prefix);
    while ((1 << b.page_log2) < cache.page_size) {
        ++b.page_log2;
    }
    return b;
}

// Heads [rows, heads, d] in fp32.
struct Heads {
    const float* p;
    int64_t ts, hs;
};

// Strides are 0 or more and short enough that offsets stay in 64 bits.
inline void check_heads(const float* p, int64_t ts, int64_t hs, int64_t rows, int64_t heads, int64_t d,
                        bool written, const std::string& at) {
    require(p != nullptr, at + " is null");
    require(ts >= 0 && hs >= 0, at + " has negative strides");
    supported(ts <= kMostStride && hs <= kMostStride, at + " has strides that are too long");
    supported(reaches(ts, rows) && reaches(hs, heads), at + " reaches further than memory");
    if (written) {
        const auto apart = [&](int64_t inner, int64_t count, int64_t outer, int64_t others) {
            return (count == 1 || inner >= d) &&
                   (others == 1 || outer >= inner * (count - 1) + d);
        };
        require(apart(hs, heads, ts, rows) || apart(ts, rows, hs, heads), at + " overlaps itself");
    }
}

#if defined(__HIPCC__)
namespace dev {

// standing_of for a row that a whole wavefront has, 64 starts at a time: one step for up to 64 sequences.
__device__ inline Standing standing_of_wave(const Batch& b, int32_t row) {
    return standing_of(b, row, [&](int32_t low, int32_t step, int32_t count) -> int32_t {
        const int32_t at = static_cast<int32_t>(threadIdx.x % 64) * step; // 64 * 2^18 at most
        const uint64_t after = ~__ballot(at < count && b.starts[low + at] <= row);
        return after != 0 ? __builtin_ctzll(after) : 64;
    });
}

} // namespace dev
#endif

} // namespace mfr::kv
