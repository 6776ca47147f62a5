// The 8-bit ops through the public API: a feed-forward block on the rocm device against doubles,
// device-resident and from host tensors; what the CPU has no kernel for; the checks of arguments.
#include "core/dispatcher.hpp"
#include "oracle_cpu.hpp"
#include "test_util.hpp"

#include <algorithm>
#include <cstdint>

using namespace mensurflow;

namespace {

double e4m3(std::uint8_t code) {
    const int exponent = (code >> 3) & 15, mantissa = code & 7;
    const double v = exponent != 0 ? std::ldexp(8 + mantissa, exponent - 10)
                                   : std::ldexp(mantissa, -9);
    return (code & 0x80) != 0 ? -v : v;
}

// What an 8-bit matrix stands for, and a bound of what the conversion of `of` may be off: half a
// step of e4m3, 2^-4 of the value or 2^-10 of the scale.
struct Plain {
    std::vector<double> v, scale;
};

Plain plain(const F8Tensor& t) {
    const auto codes = t.values.to_vector<std::uint8_t>();
    const auto scales = t.scales.to_vector<float>();
    const std::int64_t rows = t.rows(), pitch = t.values.size(1);
    Plain out;
    for (std::int64_t r = 0; r < rows; ++r) {
        for (std::int64_t c = 0; c < t.cols; ++c) {
            const std::int64_t at = t.block_rows == 1
                                        ? c / 128 * rows + r
                                        : r / 128 * t.scales.size(1) + c / 128;
            out.scale.push_back(scales[static_cast<std::size_t>(at)]);
            out.v.push_back(e4m3(codes[static_cast<std::size_t>(r * pitch + c)]) *
                            out.scale.back());
        }
    }
    return out;
}

void require_quantized(const Plain& got, const std::vector<double>& want, double slack,
                       const std::string& what) {
    test::require(got.v.size() == want.size(), what + ": size");
    for (std::size_t i = 0; i < want.size(); ++i) {
        const double half = std::max(std::ldexp(std::fabs(want[i]), -4), std::ldexp(got.scale[i], -10));
        test::require(std::fabs(got.v[i] - want[i]) <= 1.001 * half + slack,
                      what + " at " + std::to_string(i));
    }
}

std::vector<double> doubles(const Tensor& t) {
    const auto v = t.to_vector<float>();
    return std::vector<double>(v.begin(), v.end());
}

std::vector<double> product(const Plain& a, const Plain& b, std::int64_t m, std::int64_t n,
                            std::int64_t k) {
    std::vector<double> out(static_cast<std::size_t>(m * n), 0.0);
    for (std::int64_t i = 0; i < m; ++i) {
        for (std::int64_t j = 0; j < n; ++j) {
            for (std::int64_t p = 0; p < k; ++p) {
                out[static_cast<std::size_t>(i * n + j)] +=
                    a.v[static_cast<std::size_t>(i * k + p)] * b.v[static_cast<std::size_t>(j * k + p)];
            }
        }
    }
    return out;
}

// data: where the tensors live; the ops run on the GPU.
void test_block(Device data) {
    const Execution gpu = Execution::GPU;
    const std::int64_t tokens = 21, hidden = 200, inner = 330;
    const Tensor x = normal({tokens, hidden}, 0.0f, 1.0f, 1, 0).to(data);
    Tensor residual = normal({tokens, hidden}, 0.0f, 2.0f, 2, 0).to(data);
    const Tensor weight = uniform({hidden}, 0.5f, 1.5f, 3, 0).to(data);
    const Tensor bias = uniform({hidden}, -1.0f, 1.0f, 4, 0).to(data);
    const auto weights = [&](std::int64_t n, std::int64_t k, std::uint64_t seed) {
        return quantize_f8(normal({n, k}, 0.0f, 0.05f, seed, 0).to(data), 128, gpu);
    };
    const F8Tensor gate = weights(inner, hidden, 5), up = weights(inner, hidden, 6),
                   down = weights(hidden, inner, 7);
    const auto xv = doubles(x), rv = doubles(residual), wv = doubles(weight), bv = doubles(bias);

    Tensor sum = Tensor::empty({tokens, hidden}, DType::F32, data);
    const Tensor normed = rms_norm(x, &weight, &residual, &sum, 1e-5f, gpu);
    const F8Tensor q = rms_norm_f8(x, &weight, &residual, &residual, 1e-5f, gpu); // in place
    test::require(test::same_bits(sum.to_vector<float>(), residual.to_vector<float>()), "sum");
    std::vector<double> want(xv.size());
    for (std::int64_t r = 0; r < tokens; ++r) {
        double squares = 0.0;
        for (std::int64_t c = 0; c < hidden; ++c) {
            const std::size_t at = static_cast<std::size_t>(r * hidden + c);
            want[at] = static_cast<float>(static_cast<float>(xv[at]) + static_cast<float>(rv[at]));
            squares += want[at] * want[at];
        }
        for (std::int64_t c = 0; c < hidden; ++c) {
            const std::size_t at = static_cast<std::size_t>(r * hidden + c);
            test::require(doubles(sum)[at] == want[at], "x + residual");
            want[at] *= wv[static_cast<std::size_t>(c)] /
                        std::sqrt(squares / static_cast<double>(hidden) + 1e-5f);
        }
    }
    const auto nv = doubles(normed);
    for (std::size_t i = 0; i < want.size(); ++i) {
        test::require(std::fabs(nv[i] - want[i]) <= std::ldexp(1.001 * std::fabs(want[i]), -24),
                      "rms_norm at " + std::to_string(i));
    }
    require_quantized(plain(q), want, 0.0, "rms_norm_f8");

    // Sums of at most 330 products, each within 2^-24 of the magnitudes' sum (below 200 here).
    const double slack = 330 * 200 * std::ldexp(1.0, -24);
    const F8Tensor h = gemm_f8_gated(q, gate, up, F8Activation::Silu, gpu);
    auto g = product(plain(q), plain(gate), tokens, inner, hidden);
    const auto u = product(plain(q), plain(up), tokens, inner, hidden);
    for (std::size_t i = 0; i < g.size(); ++i) {
        g[i] = g[i] / (1 + std::exp(-g[i])) * u[i];
    }
    require_quantized(plain(h), g, slack, "gemm_f8_gated");

    const Tensor y = gemm_f8(h, down, &bias, F8Activation::None, &sum, 0.5f, gpu);
    const auto p = product(plain(h), plain(down), tokens, hidden, inner);
    const auto yv = doubles(y), sv = doubles(sum);
    for (std::size_t i = 0; i < p.size(); ++i) {
        const double exact = p[i] + 0.5 * sv[i] + bv[i % static_cast<std::size_t>(hidden)];
        test::require(std::fabs(yv[i] - exact) <= slack, "gemm_f8 at " + std::to_string(i));
    }
    test::require(y.device() == data && h.values.device() == data, "results live with their inputs");
}

void test_cpu_has_no_kernels() {
    const Tensor x = Tensor::ones({3, 20});
    test::require_throws<detail::NotImplemented>([&] { rms_norm(x); }, "rms_norm on the CPU");
    test::require_throws<detail::NotImplemented>([&] { quantize_f8(x); }, "quantize_f8 on the CPU");
    const F8Tensor a = F8Tensor::empty(3, 20), b = F8Tensor::empty(5, 20, 128);
    test::require_throws<detail::NotImplemented>([&] { gemm_f8(a, b); }, "gemm_f8 on the CPU");
}

void test_checks() {
    using Invalid = std::invalid_argument;
    const Tensor x = Tensor::ones({3, 20});
    const Tensor w = Tensor::ones({19});
    const Tensor whole = Tensor::ones({3, 20}, DType::I32);
    test::require_throws<Invalid>([&] { rms_norm(x, &w); }, "weight's length");
    test::require_throws<Invalid>([&] { rms_norm(w); }, "rank");
    test::require_throws<Invalid>([&] { rms_norm(whole); }, "dtype");
    test::require_throws<Invalid>([&] { rms_norm(x, nullptr, &whole); }, "residual's dtype");
    Tensor view = Tensor::ones({20, 3}).transpose(0, 1);
    test::require_throws<Invalid>([&] { rms_norm(x, nullptr, nullptr, &view); }, "sum is a view");
    test::require_throws<Invalid>([&] { quantize_f8(x, 2); }, "block_rows");
    test::require_throws<Invalid>([&] { quantize_f8(Tensor()); }, "undefined");
    const F8Tensor a = F8Tensor::empty(3, 20), b = F8Tensor::empty(5, 20, 128),
                   other = F8Tensor::empty(5, 21, 128), more = F8Tensor::empty(6, 20, 128);
    test::require_throws<Invalid>([&] { gemm_f8(b, b); }, "a in blocks of 128 rows");
    test::require_throws<Invalid>([&] { gemm_f8(a, a); }, "b with a scale per row");
    test::require_throws<Invalid>([&] { gemm_f8(a, other); }, "depths");
    test::require_throws<Invalid>(
        [&] { gemm_f8(a, b, nullptr, F8Activation::None, nullptr, 1.0f); }, "beta without c");
    test::require_throws<Invalid>([&] { gemm_f8(a, b, &w); }, "bias's length");
    test::require_throws<Invalid>([&] { gemm_f8_gated(a, b, more); }, "gate and up differ");
    F8Tensor torn = b;
    torn.scales = Tensor::ones({2, 1});
    test::require_throws<Invalid>([&] { gemm_f8(a, torn); }, "scales' shape");
    const DType bytes = b.values.dtype();
    for (const std::int64_t pitch : {16, 24, 33}) {
        torn = b;
        torn.values = Tensor::empty({5, pitch}, bytes);
        test::require_throws<Invalid>([&] { gemm_f8(a, torn); }, "rows of " + std::to_string(pitch));
    }
    torn.values = Tensor::empty({5, 64}, bytes); // wider than it need be
    test::require_throws<detail::NotImplemented>([&] { gemm_f8(a, torn); }, "no kernel on the CPU");
    test::require(F8Tensor::empty(2, 1023).values.size(1) == 1024 &&
                      F8Tensor::empty(2, 1030).values.size(1) == 1152 &&
                      F8Tensor::empty(2, 17).values.size(1) == 32,
                  "pitches");
}

} // namespace

int main(int argc, char** argv) {
    return test::run("f8_test", argc, argv, [] {
        test::register_oracle_cpu_kernels(); // normal and uniform
        test_checks();
        test_cpu_has_no_kernels();
        for (const Device device : test::devices()) {
            if (device.type == DeviceType::ROCm) {
                test_block(device);
                test_block(Device{}); // host tensors, moved there and back
            }
        }
    });
}
