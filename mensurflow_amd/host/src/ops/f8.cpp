// The 8-bit ops: validation and dispatch (see mensurflow/ops/f8.hpp).
#include "mensurflow/ops/f8.hpp"

#include "core/dispatcher.hpp"
#include "ops/checks.hpp"

#include <string>

namespace mensurflow {

namespace {

using detail::OpArgs;
using detail::OpCheck;
using detail::OpId;

constexpr std::int64_t kBlock = 128;

std::int64_t blocks_of(std::int64_t n) { return (n + kBlock - 1) / kBlock; }

void check_f32(const OpCheck& check, const Tensor& t, const char* name, int rank) {
    check.operand(t, name, rank);
    if (t.dtype() != DType::F32) {
        check.fail(std::string(name) + " must be F32, got " + dtype_name(t.dtype()));
    }
}

void check_shape(const OpCheck& check, const Tensor& t, const char* name, const Shape& shape) {
    if (t.shape() != shape) {
        check.fail(std::string(name) + " must have shape " + to_string(shape) + ", got " +
                   to_string(t.shape()));
    }
}

void check_f8(const OpCheck& check, const F8Tensor& t, const char* name, int block_rows) {
    check.operand(t.values, name, 2).operand(t.scales, name, 2);
    if (t.block_rows != block_rows) {
        check.fail(std::string(name) + " needs block_rows " + std::to_string(block_rows) +
                   ", got " + std::to_string(t.block_rows));
    }
    if (t.values.dtype() != DType::U8 || t.scales.dtype() != DType::F32) {
        check.fail(std::string(name) + " must be U8 values with F32 scales");
    }
    if (t.cols < 0 || t.values.size(1) < t.cols || t.values.size(1) % 16 != 0) {
        check.fail(std::string(name) + " has rows of " + std::to_string(t.values.size(1)) +
                   " bytes for " + std::to_string(t.cols) + " columns");
    }
    const std::int64_t rows = t.values.size(0);
    const Shape scales = block_rows == 1 ? Shape{blocks_of(t.cols), rows}
                                         : Shape{blocks_of(rows), blocks_of(t.cols)};
    check_shape(check, t.scales, name, scales);
    if (!t.values.is_contiguous() || !t.scales.is_contiguous()) {
        check.fail(std::string(name) + " must be contiguous");
    }
    check.same_device(t.values, t.scales);
}

// Inputs and outputs of a norm but for its result.
OpArgs norm_args(const OpCheck& check, const Tensor& x, const Tensor* weight,
                 const Tensor* residual, Tensor* sum, float eps) {
    check_f32(check, x, "x", 2);
    OpArgs args;
    args.inputs = {x.contiguous()};
    if (weight != nullptr) {
        check_f32(check, *weight, "weight", 1);
        check_shape(check, *weight, "weight", {x.size(1)});
        args.inputs.push_back(weight->contiguous());
        args.has_weight = true;
    }
    if (residual != nullptr) {
        check_f32(check, *residual, "residual", 2);
        check_shape(check, *residual, "residual", x.shape());
        args.inputs.push_back(residual->contiguous());
        args.has_residual = true;
    }
    if (sum != nullptr) {
        check_f32(check, *sum, "sum", 2);
        check_shape(check, *sum, "sum", x.shape());
        if (!sum->is_contiguous()) {
            check.fail("sum must be contiguous");
        }
        args.outputs = {*sum};
        args.has_sum = true;
    }
    args.alpha = eps;
    args.columns = x.size(1);
    return args;
}

OpArgs product_args(const OpCheck& check, const F8Tensor& a, const F8Tensor& b, const char* name,
                    F8Activation activation) {
    check_f8(check, a, "a", 1);
    check_f8(check, b, name, 128);
    if (a.cols != b.cols) {
        check.fail("inner dimensions differ (" + std::to_string(a.cols) + " and " +
                   std::to_string(b.cols) + ")");
    }
    OpArgs args;
    args.inputs = {a.values, a.scales, b.values, b.scales};
    args.activation = static_cast<int>(activation);
    args.columns = a.cols;
    return args;
}

} // namespace

F8Tensor F8Tensor::empty(std::int64_t rows, std::int64_t cols, int block_rows, Device device) {
    if (block_rows != 1 && block_rows != 128) {
        OpCheck("F8Tensor").fail("block_rows must be 1 or 128, got " + std::to_string(block_rows));
    }
    if (rows < 0 || cols < 0) {
        OpCheck("F8Tensor").fail("negative dimension in " + to_string(Shape{rows, cols}));
    }
    F8Tensor out;
    const std::int64_t unit = cols >= 1024 ? 128 : 16;
    out.values = Tensor::empty({rows, (cols + unit - 1) / unit * unit}, DType::U8, device);
    out.scales = Tensor::empty(block_rows == 1 ? Shape{blocks_of(cols), rows}
                                               : Shape{blocks_of(rows), blocks_of(cols)},
                               DType::F32, device);
    out.cols = cols;
    out.block_rows = block_rows;
    return out;
}

F8Tensor F8Tensor::to(Device device) const {
    F8Tensor out = *this;
    out.values = values.to(device);
    out.scales = scales.to(device);
    return out;
}

F8Tensor quantize_f8(const Tensor& x, int block_rows, Execution execution) {
    check_f32(OpCheck("quantize_f8"), x, "x", 2);
    F8Tensor out = F8Tensor::empty(x.size(0), x.size(1), block_rows, x.device());
    OpArgs args{{x.contiguous()}, {out.values, out.scales}};
    args.block_rows = block_rows;
    args.columns = x.size(1);
    detail::dispatch(OpId::QuantizeF8, args, execution);
    return out;
}

Tensor rms_norm(const Tensor& x, const Tensor* weight, const Tensor* residual, Tensor* sum,
                float eps, Execution execution) {
    OpArgs args = norm_args(OpCheck("rms_norm"), x, weight, residual, sum, eps);
    Tensor out = Tensor::empty(x.shape(), DType::F32, x.device());
    args.outputs.push_back(out);
    detail::dispatch(OpId::RmsNorm, args, execution);
    return out;
}

F8Tensor rms_norm_f8(const Tensor& x, const Tensor* weight, const Tensor* residual, Tensor* sum,
                     float eps, Execution execution) {
    OpArgs args = norm_args(OpCheck("rms_norm_f8"), x, weight, residual, sum, eps);
    F8Tensor out = F8Tensor::empty(x.size(0), x.size(1), 1, x.device());
    args.outputs.push_back(out.values);
    args.outputs.push_back(out.scales);
    args.f8_out = true;
    detail::dispatch(OpId::RmsNorm, args, execution);
    return out;
}

Tensor gemm_f8(const F8Tensor& a, const F8Tensor& b, const Tensor* bias, F8Activation activation,
               const Tensor* c, float beta, Execution execution) {
    const OpCheck check("gemm_f8");
    OpArgs args = product_args(check, a, b, "b", activation);
    const Shape shape{a.rows(), b.rows()};
    if (beta != 0.0f && c == nullptr) {
        check.fail("beta requires an output matrix");
    }
    if (c != nullptr && beta != 0.0f) {
        check_f32(check, *c, "c", 2);
        check_shape(check, *c, "c", shape);
        args.inputs.push_back(c->contiguous());
        args.has_c = true;
    }
    if (bias != nullptr) {
        check_f32(check, *bias, "bias", 1);
        check_shape(check, *bias, "bias", {shape[1]});
        args.inputs.push_back(bias->contiguous());
        args.has_bias = true;
    }
    args.beta = beta;
    Tensor out = Tensor::empty(shape, DType::F32, a.values.device());
    args.outputs = {out};
    detail::dispatch(OpId::GemmF8, args, execution);
    return out;
}

F8Tensor gemm_f8_gated(const F8Tensor& a, const F8Tensor& gate, const F8Tensor& up,
                       F8Activation activation, Execution execution) {
    const OpCheck check("gemm_f8_gated");
    OpArgs args = product_args(check, a, gate, "gate", activation);
    check_f8(check, up, "up", 128);
    if (up.rows() != gate.rows() || up.cols != gate.cols) {
        check.fail("gate and up differ in shape");
    }
    args.inputs.push_back(up.values);
    args.inputs.push_back(up.scales);
    args.gated = true;
    args.beta = 0.0f;
    F8Tensor out = F8Tensor::empty(a.rows(), gate.rows(), 1, a.values.device());
    args.outputs = {out.values, out.scales};
    args.f8_out = true;
    detail::dispatch(OpId::GemmF8, args, execution);
    return out;
}

} // namespace mensurflow
