// The 8-bit ops of the ROCm device (OpId::RmsNorm, QuantizeF8, GemmF8): adapters onto
// mfr_rms_norm, mfr_f8_quantize and mfr_f8gemm. In a file of their own because mensurflow has no
// such ops: backend.cpp alone is what drops into its tree.
#include "backends/backend.hpp"
#include "core/dispatcher.hpp"
#include "core/registry.hpp"
#include "core/tensor_access.hpp"
#include "mfr_rocm.h"

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

// Values and scales as the ops lay them out (F8Tensor): rows of a pitch of 16 bytes' multiples,
// the scales of rows as [blocks, rows].
mfr_f8_matrix matrix(const Tensor& values, const Tensor& scales, int block_rows) {
    mfr_f8_matrix m{};
    m.values = TensorAccess::data<std::uint8_t>(values);
    m.rs = values.size(1);
    m.scales = floats(scales);
    m.scales_rs = block_rows == 1 ? 1 : scales.size(1);
    m.scales_cs = block_rows == 1 ? scales.size(1) : 1;
    m.block_rows = block_rows;
    return m;
}

void quantize_kernel(const OpArgs& args, Stream& stream) {
    const Tensor& x = args.inputs[0];
    const mfr_f8_matrix out = matrix(args.outputs[0], args.outputs[1], args.block_rows);
    check(mfr_f8_quantize(rocm_stream(stream), x.size(0), x.size(1), floats(x), x.size(1), &out));
}

// Inputs: x, weight and residual where given. Outputs: the sum where asked for, then the result.
void rms_norm_kernel(const OpArgs& args, Stream& stream) {
    const Tensor& x = args.inputs[0];
    std::size_t next = 1;
    mfr_rms_norm_desc d{};
    d.rows = x.size(0);
    d.cols = x.size(1);
    d.x = floats(x);
    d.x_rs = d.cols;
    if (args.has_weight) {
        d.weight = floats(args.inputs[next++]);
    }
    if (args.has_residual) {
        d.residual = floats(args.inputs[next]);
        d.residual_rs = d.cols;
    }
    next = 0;
    if (args.has_sum) {
        d.sum = floats(args.outputs[next++]);
        d.sum_rs = d.cols;
    }
    if (args.f8_out) {
        d.out_f8 = matrix(args.outputs[next], args.outputs[next + 1], 1);
    } else {
        d.out = floats(args.outputs[next]);
        d.out_rs = d.cols;
    }
    d.eps = args.alpha;
    check(mfr_rms_norm(rocm_stream(stream), &d));
}

// Inputs: a, b (values, scales each), then c and bias where given, or the second weight.
void gemm_kernel(const OpArgs& args, Stream& stream) {
    mfr_f8gemm_desc d{};
    d.m = args.inputs[0].size(0);
    d.n = args.inputs[2].size(0);
    d.k = args.columns;
    d.a = matrix(args.inputs[0], args.inputs[1], 1);
    d.b = matrix(args.inputs[2], args.inputs[3], 128);
    std::size_t next = 4;
    if (args.gated) {
        d.up = matrix(args.inputs[4], args.inputs[5], 128);
    }
    if (args.has_c) {
        d.c0 = floats(args.inputs[next++]);
        d.c0_rs = d.n;
        d.beta = args.beta;
    }
    if (args.has_bias) {
        d.bias = floats(args.inputs[next]);
    }
    if (args.f8_out) {
        d.out_f8 = matrix(args.outputs[0], args.outputs[1], 1);
    } else {
        d.c = floats(args.outputs[0]);
        d.c_rs = d.n;
    }
    d.act = args.activation;
    check(mfr_f8gemm(rocm_stream(stream), &d));
}

} // namespace

void register_rocm_f8(Registry& registry) {
    if (registry.find(DeviceType::ROCm) == nullptr) {
        return;
    }
    Dispatcher& dispatcher = registry.dispatcher();
    dispatcher.register_kernel({OpId::QuantizeF8, DeviceType::ROCm, DType::F32}, quantize_kernel);
    dispatcher.register_kernel({OpId::RmsNorm, DeviceType::ROCm, DType::F32}, rms_norm_kernel);
    dispatcher.register_kernel({OpId::GemmF8, DeviceType::ROCm, DType::U8}, gemm_kernel);
}

} // namespace mensurflow::detail
