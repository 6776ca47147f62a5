// F8Tensor::empty at sizes that no matrix has, and at empty ones.
#include "test_util.hpp"

using namespace mensurflow;

namespace {

void test_sizes() {
    for (const int block_rows : {1, 128}) {
        for (const std::int64_t cols : {-1, -5, -15, -16, -1000}) {
            test::require_throws<std::invalid_argument>(
                [&] { F8Tensor::empty(4, cols, block_rows); }, std::to_string(cols) + " columns");
        }
        test::require_throws<std::invalid_argument>([&] { F8Tensor::empty(-1, 4, block_rows); },
                                                    "-1 rows");
        test::require(F8Tensor::empty(0, 0, block_rows).rows() == 0 &&
                          F8Tensor::empty(3, 0, block_rows).values.numel() == 0,
                      "empty matrices");
    }
}

} // namespace

int main(int argc, char** argv) { return test::run("f8_sizes_test", argc, argv, test_sizes); }
