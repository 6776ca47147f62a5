"""Calls at the edges of what the 8-bit ops allow."""
import numpy as np
import pytest

import f8_reference as ref
import mensurflow_amd as mf
from helpers import same_bits
from mensurflow_amd import abi
from test_f8_forms_gpu import Graph
from test_f8_gpu import (Held, assert_f8, dev, held_of, pitched, random_operands, same_codes)

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


# ---- the silu where e^-x leaves fp32 ------------------------------------------------------------

# Few rows, rings of slices, tiles of 64 and 128 rows, and a depth in ranges.
FAR = [(1, 300, 300), (40, 400, 300), (64, 2048, 512), (32, 4096, 1024), (128, 4100, 1100),
       (300, 1000, 900), (155, 3457, 2499), (17, 2816, 8567), (1349, 2945, 130), (2305, 1818, 972)]


def one_product(value, m, n, k, stream):
    """Operands of the product value(i), exactly, throughout row i, and a weight that doubles it 100
    times."""
    a, b = np.zeros((m, k), np.uint8), np.zeros((n, k), np.uint8)
    a[:, 0] = b[:, 0] = ref.encode(1.0)
    sa = np.ones((m, ref.blocks(k)), np.float32)
    sa[:, 0] = value
    sb = np.ones((-(-n // 128), ref.blocks(k)), np.float32)
    return (held_of(a, sa, stream, 1), held_of(b, sb, stream, 128),
            held_of(b, sb * np.float32(2.0 ** 100), stream, 128))


@pytest.mark.parametrize("m,n,k", FAR)
def test_silu_far_below_zero(stream, m, n, k):
    """Two exponentials within 2^-23 each, two products and the last one, and what a result below the
    normal numbers is rounded by."""
    value = np.linspace(-87.5, -104.5, m) if m > 1 else np.full(1, -89.25)
    value = value.astype(np.float32)
    value[m // 2] = -88.75
    a, gate, up = one_product(value, m, n, k, stream)
    other = value.astype(np.float64)[:, None] * 2.0 ** 100
    want = ref.silu(value)[:, None] * other
    y = mf.gemm_f8_gated(a.matrix, gate.matrix, up.matrix,
                         out=pitched(np.zeros((m, n), np.float32), stream, 1)).numpy()
    assert np.all(want > 0)
    assert np.all(np.abs(y - want) <=
                  (7 + 2.0 ** -10) * ref.EPS32 * want + 2.0 ** -150 * np.abs(other))
    y = mf.gemm_f8(a.matrix, gate.matrix, act=mf.ACT_SILU).numpy()
    want = ref.silu(value)[:, None]
    assert np.all(np.abs(y - want) <= (6 + 2.0 ** -10) * ref.EPS32 * np.abs(want) + 2.0 ** -150)


def test_silu_of_the_ends(stream):
    """Nothing is left of the far negative numbers; infinity stays, and minus infinity is the
    formula's NaN."""
    value = np.float32([-300, -1e4, -3e38, -np.inf, np.inf, np.nan, 0.0, 3e38])
    a, b, _ = one_product(np.where(np.isfinite(value), value, 1), 8, 20, 3, stream)
    bias = np.zeros((8, 20), np.float32)
    bias[~np.isfinite(value)] = value[~np.isfinite(value), None]
    y = mf.gemm_f8(a.matrix, b.matrix, c0=dev(bias, stream), beta=1.0, act=mf.ACT_SILU).numpy()
    want = np.float32([0, 0, 0, np.nan, np.inf, np.nan, 0, 3e38])
    assert np.array_equal(y, np.repeat(want[:, None], 20, 1), equal_nan=True)


# ---- few rows with both outputs, captured -------------------------------------------------------

# Deep and narrow: where the depth in ranges, through the workspace, would be the faster plan.
DEEP = [(1, 1021, 7891), (1, 6675, 5631), (1, 6731, 7816), (39, 4097, 3153), (64, 1176, 8236),
        (35, 1510, 8992)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", DEEP)
def test_captured_few_deep_rows_with_both_outputs_run_as_they_do_eagerly(m, n, k, gated):
    """Real values, whose sums tell the order of summation: the same bits, replayed between eager calls."""
    rng = np.random.default_rng(m + n)
    with mf.Stream(0) as own:
        a = held_of(*random_operands(rng, m, k, 1), own, 1)
        gate, up = (held_of(*random_operands(rng, n, k, 128), own, 128) for _ in range(2))
        out, q = mf.DeviceArray.empty((m, n), own), Held(m, n, own)

        def body():
            if gated:
                mf.gemm_f8_gated(a.matrix, gate.matrix, up.matrix, out=out, out_f8=q.matrix)
            else:
                mf.gemm_f8(a.matrix, gate.matrix, out=out, out_f8=q.matrix)

        body()
        want, codes = out.numpy(), q.read()[0].copy()
        graph = Graph(own, body)
        for call in (graph.launch, graph.launch, body, graph.launch):
            mf.fill(out, 3.0)
            call()
            assert same_bits(out.numpy(), want) and same_codes(q.read()[0], codes)
        graph.close()
