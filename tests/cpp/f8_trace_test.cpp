// The trace spans of the 8-bit ops: an op's checks allocate nothing, so the only allocations that a
// collector sees are those of its results.
#include "core/dispatcher.hpp"
#include "mensurflow/trace.hpp"
#include "test_util.hpp"

#include <string>
#include <vector>

using namespace mensurflow;

namespace {

std::vector<trace::Event>& recorded() {
    static std::vector<trace::Event> events;
    return events;
}

void record(const trace::Event& event) { recorded().push_back(event); }

// The allocations that `call` makes on the CPU, which has no kernel for it.
template <typename Call> std::size_t allocations(Call call) {
    recorded().clear();
    trace::hook.store(&record);
    test::require_throws<detail::NotImplemented>(call, "an 8-bit op on the CPU");
    trace::hook.store(nullptr);
    std::size_t count = 0;
    for (const trace::Event& e : recorded()) {
        count += std::string(e.name) == "Tensor::empty" ? 1 : 0;
    }
    return count;
}

void test_allocations() {
    constexpr Execution on = Execution::CPU;
    const F8Tensor a = F8Tensor::empty(3, 200), gate = F8Tensor::empty(5, 200, 128),
                   up = F8Tensor::empty(5, 200, 128);
    const Tensor x = Tensor::empty({3, 200}, DType::F32);
    const auto product = [&] {
        (void)gemm_f8(a, gate, nullptr, F8Activation::None, nullptr, 0.0f, on);
    };
    test::require(allocations(product) == 1, "gemm_f8 allocates its result alone");
    const auto gated = [&] { (void)gemm_f8_gated(a, gate, up, F8Activation::Silu, on); };
    test::require(allocations(gated) == 2, "gemm_f8_gated allocates values and scales alone");
    test::require(allocations([&] { (void)quantize_f8(x, 1, on); }) == 2,
                  "quantize_f8 allocates values and scales alone");
    const auto norm = [&] { (void)rms_norm(x, nullptr, nullptr, nullptr, 1e-6f, on); };
    test::require(allocations(norm) == 1, "rms_norm allocates its result alone");
}

} // namespace

int main(int argc, char** argv) {
    return test::run("f8_trace_test", argc, argv, test_allocations);
}
