"""Runs the C++ test of the 8-bit ops' trace spans (tests/cpp/f8_trace_test.cpp), on the CPU."""
from test_cpp_host import run


def test_the_checks_of_the_8_bit_ops_allocate_nothing():
    run("f8_trace_test")
