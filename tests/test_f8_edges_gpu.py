"""Calls at the edges of what the 8-bit ops allow."""
import numpy as np
import pytest

import mensurflow_amd as mf
from helpers import same_bits
from mensurflow_amd import abi
from test_f8_gpu import Held, assert_f8, dev, pitched

pytestmark = pytest.mark.gpu

# ---- products of depth 0 ------------------------------------------------------------------------

WILD = [0, 7, -16, 1 << 31, -(1 << 40)]


def empty_operand(stride, block_rows):
    """An operand without columns: nothing of it but block_rows means anything."""
    return abi.F8Desc(None, stride, None, stride, -stride, block_rows, 0)


# The last two are more rows than the form for few rows takes, which leaves them to a ring of slices.
@pytest.mark.parametrize("stride", WILD)
@pytest.mark.parametrize("m,n", [(1, 5), (3, 700), (300, 700), (70000, 130), (4194305, 64)])
def test_products_of_depth_0_read_nothing(stream, m, n, stride):
    rng = np.random.default_rng(n)
    bias = rng.standard_normal(n).astype(np.float32)
    out, added = mf.DeviceArray.empty((m, n), stream), dev(bias, stream)
    mf.fill(out, 7.0)
    d = abi.F8GemmDesc()
    d.m, d.n = m, n
    d.a, d.b = empty_operand(stride, 1), empty_operand(stride, 128)
    d.c, d.c_rs, d.bias = out.ptr, n, added.ptr
    mf.f8gemm(stream, d)
    got = out.numpy()
    assert all(same_bits(got[i:i + 65536], np.tile(bias, (min(65536, m - i), 1)))
               for i in range(0, m, 65536))
    out.close()


@pytest.mark.parametrize("stride", WILD)
def test_gated_products_of_depth_0(stream, stride):
    m, n = 40, 300
    for pointer in (None, 1 << 20):
        held, out = Held(m, n, stream), pitched(np.ones((m, n), np.float32), stream, 3)
        d = mf.f8gemm_desc(mf.F8Matrix.empty(m, 0, stream), mf.F8Matrix.empty(n, 0, stream, 128),
                           up=mf.F8Matrix.empty(n, 0, stream, 128), act=mf.ACT_SILU, out=out,
                           out_f8=held.matrix)
        d.a, d.b, d.up = (empty_operand(stride, r) for r in (1, 128, 128))
        d.up.values = pointer
        mf.f8gemm(stream, d)
        assert not np.any(out.numpy())
        assert_f8(held, np.zeros((m, n), np.float32))
