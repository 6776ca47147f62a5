// Rotary positions and the paged cache: validation and dispatch (see mensurflow/ops/kv.hpp).
#include "mensurflow/ops/kv.hpp"

#include "core/dispatcher.hpp"
#include "core/kv_args.hpp"
#include "ops/checks.hpp"

#include <string>

namespace mensurflow {

namespace {

using detail::KvArgs;
using detail::OpArgs;
using detail::OpCheck;
using detail::OpId;

void check_type(const OpCheck& check, const Tensor& t, const char* name, int rank, DType dtype) {
    check.operand(t, name, rank);
    if (t.dtype() != dtype) {
        check.fail(std::string(name) + " must be " + dtype_name(dtype) + ", got " +
                   dtype_name(t.dtype()));
    }
}

void check_shape(const OpCheck& check, const Tensor& t, const char* name, const Shape& shape) {
    if (t.shape() != shape) {
        check.fail(std::string(name) + " must have shape " + to_string(shape) + ", got " +
                   to_string(t.shape()));
    }
}

// Heads as the kernels take them: unit stride along d.
Tensor heads(const Tensor& t) { return t.size(2) <= 1 || t.strides()[2] == 1 ? t : t.contiguous(); }

void add_positions(const OpCheck& check, OpArgs& args, KvArgs& kv, const Tensor* positions,
                   std::int64_t rows) {
    if (positions != nullptr) {
        check_type(check, *positions, "positions", 1, DType::I32);
        check_shape(check, *positions, "positions", {rows});
        args.inputs.push_back(positions->contiguous());
        kv.has_positions = true;
    }
}

// The cache's tensors, to inputs or outputs.
void add_cache(const OpCheck& check, std::vector<Tensor>& to, KvArgs& kv, const KvCache& cache) {
    check.operand(cache.k, "cache.k", 4).operand(cache.v, "cache.v", 4);
    const DType dtype = cache.k.dtype();
    if (dtype != DType::F32 && dtype != DType::BF16 && dtype != DType::U8) {
        check.fail(std::string("cache.k must be f32, bf16 or u8, got ") + dtype_name(dtype));
    }
    check.same_dtype(cache.k, cache.v);
    check_shape(check, cache.v, "cache.v", cache.k.shape());
    const auto add = [&](const Tensor& t, const char* name) {
        if (!t.is_contiguous()) {
            check.fail(std::string(name) + " must be contiguous");
        }
        to.push_back(t);
    };
    add(cache.k, "cache.k");
    add(cache.v, "cache.v");
    if (dtype == DType::U8) {
        const Shape shape{cache.k.size(0), cache.k.size(1), cache.k.size(2)};
        for (const Tensor* t : {&cache.k_scales, &cache.v_scales}) {
            check_type(check, *t, "the cache's scales", 3, DType::F32);
            check_shape(check, *t, "the cache's scales", shape);
            add(*t, "the cache's scales");
        }
        kv.has_scales = true;
    }
}

void add_batch(const OpCheck& check, OpArgs& args, KvArgs& kv, const KvBatch& batch,
               std::int64_t rows, std::int64_t page) {
    check_type(check, batch.lengths, "lengths", 1, DType::I32);
    check_type(check, batch.pages, "pages", 2, DType::I32);
    const std::int64_t sequences = batch.lengths.size(0);
    check_shape(check, batch.pages, "pages", {sequences, batch.pages.size(1)});
    args.inputs.push_back(batch.lengths.contiguous());
    args.inputs.push_back(batch.pages.contiguous());
    if (batch.starts.defined()) {
        check_type(check, batch.starts, "starts", 1, DType::I32);
        check_shape(check, batch.starts, "starts", {sequences + 1});
        args.inputs.push_back(batch.starts.contiguous());
        kv.has_starts = true;
    } else if (sequences > 0 && rows % sequences != 0) {
        check.fail(std::to_string(rows) + " rows are not whole for each of " +
                   std::to_string(sequences) + " sequences");
    }
    if (batch.prefix < 0) {
        check.fail("negative prefix");
    }
    if (batch.prefix > 0) {
        check_type(check, batch.prefix_pages, "prefix_pages", 1, DType::I32);
        if (page < 1 || (batch.prefix - 1) / page >= batch.prefix_pages.size(0)) {
            check.fail("prefix_pages are too few for a prefix of " + std::to_string(batch.prefix));
        }
        args.inputs.push_back(batch.prefix_pages.contiguous());
        kv.prefix = batch.prefix;
    }
}

// Where the cache is: another device's copy of it would take nothing and give nothing back.
Execution execution_of(const KvCache& cache) {
    return cache.k.device().type == DeviceType::CPU ? Execution::CPU : Execution::GPU;
}

} // namespace

Tensor rope(const Tensor& x, const Rotary& rotary, const Tensor* positions, std::int64_t first,
            bool backward, Execution execution) {
    const OpCheck check("rope");
    check_type(check, x, "x", 3, DType::F32);
    KvArgs kv;
    kv.rotary = rotary;
    kv.first = first;
    kv.backward = backward;
    Tensor out = Tensor::empty(x.shape(), DType::F32, x.device());
    OpArgs args{{heads(x)}, {out}};
    add_positions(check, args, kv, positions, x.size(0));
    args.kv = &kv;
    detail::dispatch(OpId::Rope, args, execution);
    return out;
}

KvCache KvCache::empty(std::int64_t pages, std::int64_t page, std::int64_t heads, std::int64_t d,
                       DType dtype, Device device) {
    const OpCheck check("KvCache");
    if (dtype != DType::F32 && dtype != DType::BF16 && dtype != DType::U8) {
        check.fail(std::string("f32, bf16 or u8, got ") + dtype_name(dtype));
    }
    if (pages < 0 || page < 0 || heads < 0 || d < 0) {
        check.fail("negative dimension in " + to_string(Shape{pages, page, heads, d}));
    }
    KvCache out;
    out.k = Tensor::empty({pages, heads, page, d}, dtype, device);
    out.v = Tensor::empty({pages, heads, page, d}, dtype, device);
    if (dtype == DType::U8) {
        out.k_scales = Tensor::empty({pages, heads, page}, DType::F32, device);
        out.v_scales = Tensor::empty({pages, heads, page}, DType::F32, device);
    }
    return out;
}

Tensor kv_append(const KvCache& cache, const KvBatch& batch, const Tensor& k, const Tensor& v,
                 const Rotary* rotary, const Tensor* q, const Tensor* positions) {
    const OpCheck check("kv_append");
    KvArgs kv;
    OpArgs args;
    add_cache(check, args.outputs, kv, cache);
    check_type(check, k, "k", 3, DType::F32);
    check_type(check, v, "v", 3, DType::F32);
    const Shape shape{k.size(0), cache.k.size(1), cache.k.size(3)};
    check_shape(check, k, "k", shape);
    check_shape(check, v, "v", shape);
    args.inputs = {heads(k), heads(v)};
    add_batch(check, args, kv, batch, k.size(0), cache.k.size(2));
    Tensor turned;
    if (q != nullptr) {
        check_type(check, *q, "q", 3, DType::F32);
        check_shape(check, *q, "q", {k.size(0), q->size(1), cache.k.size(3)});
        if (q->size(1) < 1) {
            check.fail("q has no heads");
        }
        args.inputs.push_back(heads(*q));
        turned = Tensor::empty(q->shape(), DType::F32, cache.k.device());
        args.outputs.push_back(turned);
        kv.has_q = true;
    }
    add_positions(check, args, kv, positions, k.size(0));
    if (rotary != nullptr) {
        kv.rotary = *rotary;
    }
    args.kv = &kv;
    detail::dispatch(OpId::KvAppend, args, execution_of(cache));
    return turned;
}

Tensor attention_paged(const Tensor& q, const KvCache& cache, const KvBatch& batch, float scale,
                       bool causal) {
    const OpCheck check("attention_paged");
    KvArgs kv;
    kv.scale = scale;
    kv.causal = causal;
    check_type(check, q, "q", 3, DType::F32);
    OpArgs args;
    args.inputs = {heads(q)};
    add_cache(check, args.inputs, kv, cache);
    check_shape(check, q, "q", {q.size(0), q.size(1), cache.k.size(3)});
    add_batch(check, args, kv, batch, q.size(0), cache.k.size(2));
    Tensor out = Tensor::empty(q.shape(), DType::F32, cache.k.device());
    args.outputs = {out};
    args.kv = &kv;
    detail::dispatch(OpId::AttentionPaged, args, execution_of(cache));
    return out;
}

} // namespace mensurflow
