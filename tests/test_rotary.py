"""The angles of rotary positions without a GPU."""
from test_cpp_host import run as run_cpp


def test_angles():
    run_cpp("rotary_angle_test")
