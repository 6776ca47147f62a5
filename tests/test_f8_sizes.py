"""Runs the C++ test of F8Tensor::empty's sizes (tests/cpp/f8_sizes_test.cpp), on the CPU."""
from test_cpp_host import run


def test_sizes_that_no_matrix_has_are_refused():
    run("f8_sizes_test")
