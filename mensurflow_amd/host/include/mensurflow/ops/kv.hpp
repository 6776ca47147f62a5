// Rotary positions, a paged cache of keys and values, and attention against it: what a decoder's
// attention needs for prompts and for single tokens. mensurflow has no counterpart of these; the
// semantics are those of mfr_rope, mfr_kv_append and mfr_attention_paged (include/mfr_rocm.h). Only
// the rocm device has kernels for them: NotImplemented elsewhere.
#pragma once

#include "mensurflow/execution.hpp"
#include "mensurflow/tensor.hpp"

#include <array>
#include <cstdint>

namespace mensurflow {

// Which columns of a head turn together: i and columns / 2 + i, or 2 i and 2 i + 1.
enum class RotaryLayout { Halves, Pairs };

// A rotation of the first `columns` columns of a head (even, at most 256; 0: none): pair i turns by
// position * steps[i] radians and is multiplied by the amplitude.
struct Rotary {
    int columns = 0;
    RotaryLayout layout = RotaryLayout::Halves;
    float amplitude = 1.0f;
    std::array<double, 128> steps{};
};

// Steps base^(-2 i / columns), divided by `factor` for longer contexts; where `original`, the context
// that a model learned, is given, only pairs that turn less than `fast` times in it, and those below
// `slow` turns in full.
Rotary rotary(int columns, double base = 10000.0, RotaryLayout layout = RotaryLayout::Halves,
              double amplitude = 1.0, double factor = 1.0, double original = 0.0, double slow = 1.0,
              double fast = 32.0);

// x [rows, heads, d] turned by each row's position: positions[row] (I32), or first + row. backward
// turns by the negative angles: the gradient of x from the result's.
Tensor rope(const Tensor& x, const Rotary& rotary, const Tensor* positions = nullptr,
            std::int64_t first = 0, bool backward = false, Execution execution = Execution::Auto);

// A cache of `pages` pages of `page` tokens (a power of two from 16 on): k and v are contiguous
// [pages, heads, page, d], F32, BF16, or U8 (e4m3 codes) with a scale for each row of d.
struct KvCache {
    Tensor k, v;
    Tensor k_scales, v_scales; // F32 [pages, heads, page] beside U8, undefined otherwise

    // Undefined contents.
    static KvCache empty(std::int64_t pages, std::int64_t page, std::int64_t heads, std::int64_t d,
                         DType dtype = DType::F32, Device device = {});
};

// The sequences of a step, I32 tensors: `lengths` [sequences], tokens of each with this step's; `pages`
// [sequences, width], the pages that hold them; `starts` [sequences + 1], the rows of each (undefined:
// the same number each); `prefix` tokens in `prefix_pages` that all sequences share, in front.
struct KvBatch {
    Tensor lengths, pages, starts;
    std::int64_t prefix = 0;
    Tensor prefix_pages;
};

// Writes the step's keys and values [rows, heads, d] to their places in the cache, the keys turned if a
// rotation is given, and returns q [rows, q_heads, d] turned alike (undefined without q). Rows of no
// sequence of it are undefined. The cache's tensors are on one GPU, and so are the others.
Tensor kv_append(const KvCache& cache, const KvBatch& batch, const Tensor& k, const Tensor& v,
                 const Rotary* rotary = nullptr, const Tensor* q = nullptr,
                 const Tensor* positions = nullptr);

// softmax(scale q k^T) v of each row's queries [rows, q_heads, d] against the prefix and its sequence's
// tokens up to the row's own (all of them unless causal). scale 0: 1 / sqrt(d).
Tensor attention_paged(const Tensor& q, const KvCache& cache, const KvBatch& batch, float scale = 0.0f,
                       bool causal = true);

} // namespace mensurflow
