// What Rope, KvAppend and AttentionPaged take beside their tensors (OpArgs::kv), and which of the
// optional tensors are there. Inputs, in this order: Rope x; KvAppend k, v; AttentionPaged q, then the
// cache's k, v and scales; then of a batch lengths, pages, starts, prefix_pages; q; positions. Outputs:
// KvAppend the cache's k, v and scales, and q turned; the others their result.
#pragma once

#include "mensurflow/ops/kv.hpp"

namespace mensurflow::detail {

struct KvArgs {
    Rotary rotary;
    bool has_scales = false;
    bool has_starts = false;
    bool has_q = false;
    bool has_positions = false;
    bool backward = false;
    bool causal = true;
    std::int64_t first = 0;
    std::int64_t prefix = 0; // prefix_pages are there where it is not 0
    float scale = 0.0f;
};

} // namespace mensurflow::detail
