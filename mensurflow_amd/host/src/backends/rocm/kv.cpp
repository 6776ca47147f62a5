// Rotary positions and the paged cache on the ROCm device (OpId::Rope, KvAppend, AttentionPaged):
// adapters onto mfr_rope, mfr_kv_append and mfr_attention_paged. In a file of their own because
// mensurflow has no such ops: backend.cpp alone is what drops into its tree.
#include "core/kv_args.hpp"

#include "backends/backend.hpp"
#include "core/dispatcher.hpp"
#include "core/registry.hpp"
#include "core/tensor_access.hpp"
#include "mfr_rocm.h"

#include <algorithm>
#include <stdexcept>
#include <string>

namespace mensurflow::detail {

mfr_stream_t rocm_stream(Stream& stream); // backend.cpp

namespace {

void check(int status) {
    if (status == MFR_OK) {
        return;
    }
    const std::string message = mfr_last_error();
    if (status == MFR_E_INVALID) {
        throw std::invalid_argument(message);
    }
    if (status == MFR_E_UNSUPPORTED) {
        throw NotImplemented(message);
    }
    throw std::runtime_error(message);
}

float* floats(const Tensor& t) { return TensorAccess::data<float>(t); }
const std::int32_t* indices(const Tensor& t) { return TensorAccess::data<std::int32_t>(t); }

mfr_rotary rotary_of(const Rotary& rotary) {
    mfr_rotary r{};
    r.rot = rotary.columns;
    r.layout = rotary.layout == RotaryLayout::Pairs ? MFR_ROTARY_PAIRS : MFR_ROTARY_HALVES;
    r.amplitude = rotary.amplitude;
    std::copy(rotary.steps.begin(), rotary.steps.end(), r.steps);
    return r;
}

// The cache whose tensors begin at `at`, which is moved behind them.
mfr_kv_cache cache_of(const std::vector<Tensor>& tensors, std::size_t& at, const KvArgs& kv) {
    const Tensor &k = tensors[at], &v = tensors[at + 1];
    mfr_kv_cache c{};
    c.type = k.dtype() == DType::F32 ? MFR_KV_F32 : k.dtype() == DType::BF16 ? MFR_KV_BF16 : MFR_KV_F8;
    c.pages = k.size(0);
    c.heads = k.size(1);
    c.page_size = static_cast<std::int32_t>(std::min<std::int64_t>(k.size(2), INT32_MAX));
    c.d = k.size(3);
    // The offset is in elements of the tensor's type.
    const auto bytes = [](const Tensor& t) {
        return TensorAccess::data<std::uint8_t>(t) +
               static_cast<std::size_t>(t.offset()) * (t.itemsize() - 1);
    };
    c.k = bytes(k);
    c.v = bytes(v);
    c.token_stride = c.d;
    c.head_stride = c.page_size * c.d;
    c.page_stride = c.heads * c.head_stride;
    at += 2;
    if (kv.has_scales) {
        c.k_scales = floats(tensors[at++]);
        c.v_scales = floats(tensors[at++]);
    }
    return c;
}

mfr_kv_batch batch_of(const std::vector<Tensor>& inputs, std::size_t& at, const KvArgs& kv,
                      std::int64_t rows) {
    const Tensor &lengths = inputs[at], &pages = inputs[at + 1];
    at += 2;
    mfr_kv_batch b{};
    b.rows = rows;
    b.sequences = lengths.size(0);
    b.lengths = indices(lengths);
    b.table = indices(pages);
    b.width = pages.size(1);
    b.table_rs = b.width;
    if (kv.has_starts) {
        b.starts = indices(inputs[at++]);
    }
    b.prefix = kv.prefix;
    if (kv.prefix > 0) {
        b.prefix_pages = indices(inputs[at++]);
    }
    return b;
}

void rope_kernel(const OpArgs& args, Stream& stream) {
    const KvArgs& kv = *args.kv;
    const Tensor &x = args.inputs[0], &out = args.outputs[0];
    mfr_rope_desc d{};
    d.rows = x.size(0);
    d.heads = x.size(1);
    d.d = x.size(2);
    d.x = floats(x);
    d.x_ts = x.strides()[0];
    d.x_hs = x.strides()[1];
    d.out = floats(out);
    d.out_ts = out.strides()[0];
    d.out_hs = out.strides()[1];
    d.positions = kv.has_positions ? indices(args.inputs[1]) : nullptr;
    d.first = kv.first;
    d.backward = kv.backward ? 1 : 0;
    d.rotary = rotary_of(kv.rotary);
    check(mfr_rope(rocm_stream(stream), &d));
}

void append_kernel(const OpArgs& args, Stream& stream) {
    const KvArgs& kv = *args.kv;
    const Tensor &k = args.inputs[0], &v = args.inputs[1];
    mfr_kv_append_desc d{};
    std::size_t in = 2, out = 0;
    d.cache = cache_of(args.outputs, out, kv);
    d.batch = batch_of(args.inputs, in, kv, k.size(0));
    d.k = floats(k);
    d.k_ts = k.strides()[0];
    d.k_hs = k.strides()[1];
    d.v = floats(v);
    d.v_ts = v.strides()[0];
    d.v_hs = v.strides()[1];
    if (kv.has_q) {
        const Tensor &q = args.inputs[in++], &turned = args.outputs[out];
        d.q = floats(q);
        d.q_ts = q.strides()[0];
        d.q_hs = q.strides()[1];
        d.q_out = floats(turned);
        d.q_out_ts = turned.strides()[0];
        d.q_out_hs = turned.strides()[1];
        d.q_heads = q.size(1);
    }
    d.positions = kv.has_positions ? indices(args.inputs[in]) : nullptr;
    d.rotary = rotary_of(kv.rotary);
    check(mfr_kv_append(rocm_stream(stream), &d));
}

void attention_kernel(const OpArgs& args, Stream& stream) {
    const KvArgs& kv = *args.kv;
    const Tensor &q = args.inputs[0], &out = args.outputs[0];
    mfr_attention_paged_desc d{};
    std::size_t in = 1;
    d.cache = cache_of(args.inputs, in, kv);
    d.batch = batch_of(args.inputs, in, kv, q.size(0));
    d.q = floats(q);
    d.q_ts = q.strides()[0];
    d.q_hs = q.strides()[1];
    d.out = floats(out);
    d.out_ts = out.strides()[0];
    d.out_hs = out.strides()[1];
    d.q_heads = q.size(1);
    d.scale = kv.scale;
    d.causal = kv.causal ? 1 : 0;
    check(mfr_attention_paged(rocm_stream(stream), &d));
}

} // namespace

void register_rocm_kv(Registry& registry) {
    if (registry.find(DeviceType::ROCm) == nullptr) {
        return;
    }
    Dispatcher& dispatcher = registry.dispatcher();
    dispatcher.register_kernel({OpId::Rope, DeviceType::ROCm, DType::F32}, rope_kernel);
    dispatcher.register_kernel({OpId::KvAppend, DeviceType::ROCm, DType::F32}, append_kernel);
    dispatcher.register_kernel({OpId::AttentionPaged, DeviceType::ROCm, DType::F32}, attention_kernel);
}

} // namespace mensurflow::detail

namespace mensurflow {

Rotary rotary(int columns, double base, RotaryLayout layout, double amplitude, double factor,
              double original, double slow, double fast) {
    mfr_rotary r{};
    detail::check(mfr_rotary_init(
        &r, columns, layout == RotaryLayout::Pairs ? MFR_ROTARY_PAIRS : MFR_ROTARY_HALVES, base,
        amplitude, factor, original, slow, fast));
    Rotary out;
    out.columns = columns;
    out.layout = layout;
    out.amplitude = r.amplitude;
    std::copy(r.steps, r.steps + out.steps.size(), out.steps.begin());
    return out;
}

} // namespace mensurflow
