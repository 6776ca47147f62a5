// Rotary positions and the paged cache through the public API: a step of a decoder on the rocm device
// against doubles, a cache of each type; what the CPU has no kernel for; the checks of arguments.
#include "core/dispatcher.hpp"
#include "oracle_cpu.hpp"
#include "test_util.hpp"

#include <algorithm>
#include <cstdint>
#include <limits>

using namespace mensurflow;

namespace {

std::size_t at(std::int64_t i) { return static_cast<std::size_t>(i); }

std::vector<double> doubles(const Tensor& t) {
    const auto v = t.to_vector<float>();
    return std::vector<double>(v.begin(), v.end());
}

Tensor whole(std::vector<std::int32_t> v, Shape shape, Device device) {
    return Tensor::from_vector(v, std::move(shape), device);
}

// One head turned, from the formula.
std::vector<double> turned(const double* x, std::int64_t d, double position, int columns, bool pairs,
                           double base) {
    std::vector<double> out(x, x + d);
    for (int i = 0; i < columns / 2; ++i) {
        const double w = position * std::pow(base, -2.0 * i / columns);
        const int a = pairs ? 2 * i : i, b = pairs ? 2 * i + 1 : columns / 2 + i;
        out[at(a)] = x[a] * std::cos(w) - x[b] * std::sin(w);
        out[at(b)] = x[b] * std::cos(w) + x[a] * std::sin(w);
    }
    return out;
}

void require_near(double got, double want, double bound, const std::string& what) {
    test::require(std::fabs(got - want) <= bound,
                  what + ": " + std::to_string(got) + ", not " + std::to_string(want));
}

// data: where x lives; the op runs on the GPU.
void test_rope(Device data) {
    const std::int64_t rows = 7, heads = 3, d = 40;
    const Tensor x = normal({rows, heads, d}, 0.0f, 1.0f, 1, 0).to(data);
    const auto xv = doubles(x);
    std::vector<std::int32_t> places;
    for (std::int64_t r = 0; r < rows; ++r) {
        places.push_back(static_cast<std::int32_t>(1000 * r + 3));
    }
    const Tensor positions = whole(places, {rows}, data);
    for (const bool pairs : {false, true}) {
        const Rotary r = rotary(24, 500.0, pairs ? RotaryLayout::Pairs : RotaryLayout::Halves);
        const Tensor y = rope(x, r, &positions, 0, false, Execution::GPU);
        test::require(y.device() == data, "the result lives with its input");
        const auto yv = doubles(y), back = doubles(rope(y, r, &positions, 0, true, Execution::GPU));
        const auto from = doubles(rope(x, r, nullptr, 5, false, Execution::GPU));
        for (std::int64_t i = 0; i < rows * heads; ++i) {
            const auto want = turned(&xv[at(i * d)], d, places[at(i / heads)], 24, pairs, 500.0);
            const auto other = turned(&xv[at(i * d)], d, 5.0 + double(i / heads), 24, pairs, 500.0);
            for (std::int64_t c = 0; c < d; ++c) {
                // Two columns below 5, 1e-7 of a cosine's and sine's own error, four roundings.
                const double bound = 10.0 * (1e-7 + 4 * std::ldexp(1.0, -24));
                require_near(yv[at(i * d + c)], want[at(c)], bound, "rope");
                require_near(from[at(i * d + c)], other[at(c)], bound, "rope from 5");
                require_near(back[at(i * d + c)], xv[at(i * d + c)], 3 * bound, "rope back");
            }
        }
    }
}

// Keys or values of the cache in doubles, [pages, heads, page, d].
std::vector<double> held(const Tensor& t, const Tensor& scales) {
    std::vector<double> out;
    if (t.dtype() == DType::F32) {
        return doubles(t);
    }
    if (t.dtype() == DType::BF16) {
        std::vector<std::uint16_t> bits(at(t.numel()));
        t.copy_to_host(bits.data());
        for (const std::uint16_t b : bits) {
            const std::uint32_t word = static_cast<std::uint32_t>(b) << 16;
            float v;
            std::memcpy(&v, &word, 4);
            out.push_back(v);
        }
        return out;
    }
    const auto codes = t.to_vector<std::uint8_t>();
    const auto s = scales.to_vector<float>();
    for (std::size_t i = 0; i < codes.size(); ++i) {
        const int exponent = (codes[i] >> 3) & 15, mantissa = codes[i] & 7;
        const double v = exponent != 0 ? std::ldexp(8 + mantissa, exponent - 10)
                                       : std::ldexp(mantissa, -9);
        out.push_back(((codes[i] & 0x80) != 0 ? -v : v) * s[i / at(t.size(3))]);
    }
    return out;
}

void test_steps(Device device, DType dtype) {
    const std::int64_t heads = 2, group = 3, d = 32, page = 16, prefix = 20;
    const std::string name = dtype_name(dtype);
    KvCache cache = KvCache::empty(9, page, heads, d, dtype, device);
    const Rotary r = rotary(32);
    const Tensor shared = whole({8, 2}, {2}, device);
    KvBatch first;
    first.lengths = whole({static_cast<std::int32_t>(prefix)}, {1}, device);
    first.pages = shared.view({1, 2});
    const Tensor pk = normal({prefix, heads, d}, 0.0f, 1.0f, 3, 0).to(device),
                 pv = normal({prefix, heads, d}, 0.0f, 1.0f, 4, 0).to(device);
    test::require(!kv_append(cache, first, pk, pv, &r).defined(), "no queries, no result");
    // Sequence 0 in pages 0 and 5 with 17 rows, sequence 1 in page 3 with 2.
    KvBatch batch;
    batch.lengths = whole({17, 2}, {2}, device);
    batch.pages = whole({0, 5, 3, -1}, {2, 2}, device);
    batch.starts = whole({0, 17, 19}, {3}, device);
    batch.prefix = prefix;
    batch.prefix_pages = shared;
    const std::int64_t rows = 19;
    const Tensor k = normal({rows, heads, d}, 0.0f, 1.0f, 5, 0).to(device),
                 v = normal({rows, heads, d}, 0.0f, 1.0f, 6, 0).to(device),
                 q = normal({rows, heads * group, d}, 0.0f, 1.0f, 7, 0).to(device);
    const Tensor tq = kv_append(cache, batch, k, v, &r, &q);
    const auto keys = held(cache.k, cache.k_scales), values = held(cache.v, cache.v_scales);
    const auto kv = doubles(k), vv = doubles(v), qv = doubles(q), tv = doubles(tq);
    const double half = dtype == DType::F32 ? std::ldexp(1.0, -24)
                        : dtype == DType::BF16 ? std::ldexp(1.0, -8) : std::ldexp(1.0, -4);
    const auto place_of = [&](std::int64_t seq, std::int64_t token, std::int64_t head) {
        const std::int64_t pages[2][2] = {{0, 5}, {3, -1}}, own[2] = {8, 2};
        const std::int64_t in = token < prefix ? own[token / page]
                                               : pages[seq][(token - prefix) / page];
        return ((in * heads + head) * page + (token < prefix ? token : token - prefix) % page) * d;
    };
    for (std::int64_t row = 0; row < rows; ++row) {
        const std::int64_t seq = row < 17 ? 0 : 1, token = prefix + (seq == 0 ? row : row - 17);
        for (std::int64_t h = 0; h < heads; ++h) {
            const auto want = turned(&kv[at((row * heads + h) * d)], d, double(token), 32, false, 1e4);
            for (std::int64_t c = 0; c < d; ++c) {
                // Half a step of the type, in 8 bits also of the scale (below 6 / 448).
                const std::int64_t in = place_of(seq, token, h) + c;
                const double more = 1e-5 + (dtype == DType::U8 ? std::ldexp(6.0 / 448, -10) : 0.0);
                require_near(keys[at(in)], want[at(c)], 1.001 * half * std::fabs(want[at(c)]) + more,
                             name + " key");
                const double plain = vv[at((row * heads + h) * d + c)];
                require_near(values[at(in)], plain, 1.001 * half * std::fabs(plain) + more,
                             name + " value");
            }
        }
        for (std::int64_t h = 0; h < heads * group; ++h) {
            const std::int64_t in = (row * heads * group + h) * d;
            const auto want = turned(&qv[at(in)], d, double(token), 32, false, 1e4);
            for (std::int64_t c = 0; c < d; ++c) {
                require_near(tv[at(in + c)], want[at(c)], 1e-5, name + " query");
            }
        }
    }
    for (const bool causal : {true, false}) {
        const auto got = doubles(attention_paged(tq, cache, batch, 0.0f, causal));
        for (std::int64_t row = 0; row < rows; ++row) {
            const std::int64_t seq = row < 17 ? 0 : 1, own = seq == 0 ? 17 : 2;
            const std::int64_t place = seq == 0 ? row : row - 17;
            const std::int64_t sees = prefix + (causal ? place + 1 : own);
            for (std::int64_t h = 0; h < heads * group; ++h) {
                std::vector<double> score;
                double top = -std::numeric_limits<double>::infinity(), wide = 0.0, sum = 0.0;
                for (std::int64_t t = 0; t < sees; ++t) {
                    double s = 0.0, w = 0.0;
                    for (std::int64_t c = 0; c < d; ++c) {
                        const double p = tv[at((row * heads * group + h) * d + c)] *
                                         keys[at(place_of(seq, t, h / group) + c)];
                        s += p;
                        w += std::fabs(p);
                    }
                    score.push_back(s / std::sqrt(double(d)));
                    top = std::max(top, score.back());
                    wide = std::max(wide, w / std::sqrt(double(d)));
                }
                for (double& s : score) {
                    s = std::exp(s - top);
                    sum += s;
                }
                // What fp32 sums of d products, and of as many terms as tokens, may be off.
                const double eps = std::ldexp(1.0, -24), off = 2 * eps * ((d + 8) * wide + 4);
                for (std::int64_t c = 0; c < d; ++c) {
                    double want = 0.0, all = 0.0;
                    for (std::int64_t t = 0; t < sees; ++t) {
                        const double p =
                            score[at(t)] / sum * values[at(place_of(seq, t, h / group) + c)];
                        want += p;
                        all += std::fabs(p);
                    }
                    require_near(got[at((row * heads * group + h) * d + c)], want,
                                 (std::expm1(2 * off) + (2 * double(sees) + 16) * eps) * all,
                                 name + " attention");
                }
            }
        }
    }
}

KvBatch batch_of(std::int64_t sequences, std::int64_t width) {
    KvBatch b;
    b.lengths = Tensor::zeros({sequences}, DType::I32);
    b.pages = Tensor::zeros({sequences, width}, DType::I32);
    return b;
}

void test_cpu_has_no_kernels() {
    using None = detail::NotImplemented;
    const Tensor x = Tensor::ones({3, 2, 16});
    test::require_throws<None>([&] { rope(x, rotary(16)); }, "rope on the CPU");
    const KvCache cache = KvCache::empty(2, 16, 2, 16);
    const KvBatch batch = batch_of(3, 1);
    test::require_throws<None>([&] { kv_append(cache, batch, x, x); }, "kv_append on the CPU");
    test::require_throws<None>([&] { attention_paged(x, cache, batch); }, "attention on the CPU");
}

void test_checks() {
    using Invalid = std::invalid_argument;
    const auto refused = [](const auto& f, const char* what) { test::require_throws<Invalid>(f, what); };
    const Tensor x = Tensor::ones({3, 2, 16}), flat = Tensor::ones({3, 32});
    const Tensor ints = Tensor::ones({3, 2, 16}, DType::I32);
    const Tensor places = Tensor::zeros({3}, DType::I32), few = Tensor::zeros({2}, DType::I32);
    const Rotary r = rotary(16);
    refused([] { rotary(15); }, "odd columns");
    refused([] { rotary(300); }, "too many columns");
    refused([] { rotary(16, 0.5); }, "base");
    refused([&] { rope(flat, r); }, "rank");
    refused([&] { rope(ints, r); }, "dtype");
    refused([&] { rope(x, r, &few); }, "too few positions");
    refused([&] { rope(x, r, &x); }, "positions' dtype");
    refused([&] { rope(Tensor(), r); }, "undefined");
    refused([] { KvCache::empty(1, 16, 1, 16, DType::I32); }, "the cache's type");
    refused([] { KvCache::empty(-1, 16, 1, 16); }, "negative size");
    const KvCache cache = KvCache::empty(2, 16, 2, 16), codes = KvCache::empty(2, 16, 2, 16, DType::U8);
    const KvBatch batch = batch_of(3, 1);
    refused([&] { kv_append(cache, batch, x, flat); }, "v's rank");
    refused([&] { kv_append(cache, batch, x, Tensor::ones({3, 1, 16})); }, "v's heads");
    refused([&] { kv_append(cache, batch, ints, x); }, "k's dtype");
    refused([&] { kv_append(cache, batch, x, x, &r, &ints); }, "q's dtype");
    const Tensor none = Tensor::ones({3, 0, 16}), short_q = Tensor::ones({2, 2, 16});
    refused([&] { kv_append(cache, batch, x, x, &r, &none); }, "no heads of q");
    refused([&] { kv_append(cache, batch, x, x, &r, &short_q); }, "q's rows");
    refused([&] { kv_append(cache, batch, x, x, &r, nullptr, &few); }, "positions");
    refused([&] { attention_paged(ints, cache, batch); }, "q's dtype");
    refused([&] { attention_paged(Tensor::ones({3, 2, 8}), cache, batch); }, "q's depth");
    refused([&] { attention_paged(Tensor::ones({4, 2, 16}), cache, batch); }, "rows that are not whole");
    KvCache torn = codes;
    torn.k_scales = Tensor();
    refused([&] { attention_paged(x, torn, batch); }, "no scales");
    torn.k_scales = Tensor::ones({2, 2, 8});
    refused([&] { attention_paged(x, torn, batch); }, "the scales' shape");
    torn = cache;
    torn.v = Tensor::ones({2, 2, 8, 16});
    refused([&] { kv_append(torn, batch, x, x); }, "v's shape");
    torn.v = codes.v;
    refused([&] { kv_append(torn, batch, x, x); }, "two types");
    torn.v = Tensor::ones({2, 16, 2, 16}).transpose(1, 2);
    refused([&] { kv_append(torn, batch, x, x); }, "a view");
    KvBatch bad = batch;
    bad.starts = places;
    refused([&] { attention_paged(x, cache, bad); }, "too few starts");
    bad = batch;
    bad.lengths = Tensor::ones({3});
    refused([&] { attention_paged(x, cache, bad); }, "lengths' dtype");
    bad = batch_of(2, 1);
    bad.lengths = places;
    refused([&] { attention_paged(x, cache, bad); }, "pages' rows");
    bad = batch;
    bad.prefix = 5;
    refused([&] { attention_paged(x, cache, bad); }, "no pages of the prefix");
    bad.prefix = 33;
    bad.prefix_pages = few;
    refused([&] { attention_paged(x, cache, bad); }, "too few pages of the prefix");
    bad.prefix = -1;
    refused([&] { attention_paged(x, cache, bad); }, "negative prefix");
}

} // namespace

int main(int argc, char** argv) {
    return test::run("kv_test", argc, argv, [] {
        test::register_oracle_cpu_kernels(); // normal
        test_checks();
        test_cpu_has_no_kernels();
        for (const Device device : test::devices()) {
            if (device.type == DeviceType::ROCm) {
                test_rope(device);
                test_rope(Device{}); // host tensors, moved there and back
                for (const DType dtype : {DType::F32, DType::BF16, DType::U8}) {
                    test_steps(device, dtype);
                }
            }
        }
    });
}
