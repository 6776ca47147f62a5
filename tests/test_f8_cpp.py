"""Runs the C++ test of the 8-bit ops (tests/cpp/f8_test.cpp): argument checks on the CPU, the ops
on the rocm device under -m gpu."""
import pytest

from test_cpp_host import run


def test_f8_host_layer_cpu():
    run("f8_test", "--cpu-only")


@pytest.mark.gpu
def test_f8_host_layer_rocm():
    run("f8_test", "--require-gpu")
