// 8-bit matrices and the ops of a feed-forward block on them: conversion, root-mean-square norm,
// products with block scales and the gated pair of projections. mensurflow has no counterpart of
// these; the semantics are those of mfr_f8_quantize, mfr_rms_norm and mfr_f8gemm
// (include/mfr_rocm.h). Only the rocm device has kernels for them: NotImplemented elsewhere.
#pragma once

#include "mensurflow/execution.hpp"
#include "mensurflow/tensor.hpp"

#include <cstdint>

namespace mensurflow {

// A matrix of e4m3 values with a scale per block of block_rows x 128: element (r, c) stands for
// value * scale.
struct F8Tensor {
    Tensor values; // U8 [rows, pitch], pitch a multiple of 16, at least cols
    Tensor scales; // F32: [ceil(cols / 128), rows] for block_rows 1, else one row per 128 rows
    std::int64_t cols = 0;
    int block_rows = 1; // 1 (activations) or 128 (weights)

    std::int64_t rows() const { return values.size(0); }
    // Undefined contents. Rows are padded to 16 bytes, from 1024 columns on to 128: a block's bytes
    // are a cache line then.
    static F8Tensor empty(std::int64_t rows, std::int64_t cols, int block_rows = 1,
                          Device device = {});
    // A copy on `device`, or *this when it lives there.
    F8Tensor to(Device device) const;
};

// x [rows, cols] in 8 bits.
F8Tensor quantize_f8(const Tensor& x, int block_rows = 1, Execution execution = Execution::Auto);

// t = x + residual; t / sqrt(mean(t^2) + eps) * weight over the last dimension of a matrix. weight
// [cols] and residual may be null; t is written to *sum (which may be *residual, or x) if given.
Tensor rms_norm(const Tensor& x, const Tensor* weight = nullptr, const Tensor* residual = nullptr,
                Tensor* sum = nullptr, float eps = 1e-6f, Execution execution = Execution::Auto);

// rms_norm with its result in 8 bits, a scale per row and 128 columns.
F8Tensor rms_norm_f8(const Tensor& x, const Tensor* weight = nullptr,
                     const Tensor* residual = nullptr, Tensor* sum = nullptr, float eps = 1e-6f,
                     Execution execution = Execution::Auto);

enum class F8Activation { None, GeluTanh, Gelu, Silu };

// act(a b^T + beta * c + bias): a [m, k] with block_rows 1, b [n, k] with block_rows 128 (a weight
// as it is stored), c [m, n] and bias [n] or null.
Tensor gemm_f8(const F8Tensor& a, const F8Tensor& b, const Tensor* bias = nullptr,
               F8Activation activation = F8Activation::None, const Tensor* c = nullptr,
               float beta = 0.0f, Execution execution = Execution::Auto);

// act(a gate^T) * (a up^T) in 8 bits, for the next product.
F8Tensor gemm_f8_gated(const F8Tensor& a, const F8Tensor& gate, const F8Tensor& up,
                       F8Activation activation = F8Activation::Silu,
                       Execution execution = Execution::Auto);

} // namespace mensurflow
