"""Runs the C++ test of rotary positions and the paged cache (tests/cpp/kv_test.cpp): argument checks on
the CPU, the ops on the rocm device under -m gpu."""
import pytest

from test_cpp_host import run


def test_kv_host_layer_cpu():
    run("kv_test", "--cpu-only")


@pytest.mark.gpu
def test_kv_host_layer_rocm():
    run("kv_test", "--require-gpu")
