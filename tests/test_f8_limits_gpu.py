"""The 8-bit entry points at the ends of what they take: more rows than a grid holds, outputs and
inputs whose offsets pass 32 bits, one-element problems, every activation in the gated form, outputs
that share arrays with inputs where that is allowed."""
import numpy as np
import pytest

import f8_reference as ref
import mensurflow_amd as mf
from helpers import same_bits
from mensurflow_amd import abi
from test_f8_gpu import (TINY, Held, assert_f8, assert_norm, assert_norm_f8, dev, exact_operands, held_of, pitched,
                         same_codes, sample)

pytestmark = pytest.mark.gpu


def equal(got, want):
    """Bit for bit but for the sign of zeros."""
    return same_bits(got + np.float32(0), want.astype(np.float32) + np.float32(0))


@pytest.mark.parametrize("rows,cols", [((1 << 21) + 5, 5), ((1 << 20) + 7, 3)])
def test_more_rows_than_a_launch(stream, rows, cols):
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    dx = dev(x, stream)
    out, held = mf.DeviceArray.empty(x.shape, stream), Held(rows, cols, stream)
    mf.rms_norm_run(stream, mf.rms_norm_desc(dx, out=out, out_f8=held.matrix))
    assert_norm(out.numpy(), x, None, 1e-6)
    assert_norm_f8(held, x, None, 1e-6)
    q = mf.F8Matrix.empty(rows, cols, stream)
    mf.quantize_f8(dx, out=q)
    codes, scales = ref.quantize(x)
    assert same_codes(q.values.numpy(), codes) and np.array_equal(q.scales.numpy(), scales)


@pytest.mark.parametrize("m,n,k", [(1_200_000, 20, 40), (2, 300_000, 64), (70_001, 130, 16)])
def test_long_sides(stream, m, n, k):
    rng = np.random.default_rng(n)
    a, sa = exact_operands(rng, m, k, 1)
    b, sb = exact_operands(rng, n, k, 128)
    p = ref.product(a, sa, b, sb)[0].astype(np.float32)
    ha, hb = held_of(a, sa, stream, 1), held_of(b, sb, stream, 128)
    q = mf.F8Matrix.empty(m, n, stream)
    out = mf.DeviceArray.empty((m, n), stream)
    mf.gemm_f8(ha.matrix, hb.matrix, out=out, out_f8=q)
    assert equal(out.numpy(), p)
    rows = rng.integers(0, m, 500)
    codes, scales = ref.quantize(p[rows])
    assert same_codes(q.values.numpy()[rows], codes)
    assert np.array_equal(q.scales.numpy()[rows], scales)


def test_output_offsets_past_32_bits(stream):
    """70000 x 32768 outputs: 9.2 GB, offsets past 2^31 elements."""
    rng = np.random.default_rng(3)
    m, n, k = 70000, 32768, 32
    a, sa = exact_operands(rng, m, k, 1)
    b, sb = exact_operands(rng, n, k, 128)
    out = mf.DeviceArray.empty((m, n), stream)
    mf.gemm_f8(held_of(a, sa, stream, 1).matrix, held_of(b, sb, stream, 128).matrix, out=out)
    for r in (0, 65535, 65536, m - 129, m - 1):
        want = ref.product(a[r:r + 1], sa[r:r + 1], b, sb)[0]
        assert equal(out.slice(0, r, r + 1).numpy(), want), r
    out.close()


@pytest.mark.parametrize("cols", [100, 1500, 9000])
def test_row_offsets_past_32_bits(stream, cols):
    """Rows 2^24 floats apart: 160 of them are 10.7 GB, 2.7e9 elements."""
    rng = np.random.default_rng(4)
    rows, pitch = 160, 1 << 24
    x = sample(rng, rows, cols)
    far = mf.DeviceArray.empty((rows, pitch), stream)
    near = dev(x, stream)
    for r in range(rows):
        abi.check(abi.load().mfr_memcpy_d2d(stream.handle, far.ptr + 4 * r * pitch,
                                            near.ptr + 4 * r * cols, 4 * cols))
    view = far.slice(1, 0, cols)
    for block_rows in (1, 128):
        q = mf.quantize_f8(view, block_rows)
        codes, scales = ref.quantize(x, block_rows)
        assert same_codes(q.values.numpy(), codes) and np.array_equal(q.scales.numpy(), scales)
    out = far.slice(1, cols, 2 * cols)
    held = Held(rows, cols, stream)
    mf.rms_norm_run(stream, mf.rms_norm_desc(view, eps=1e-5, out=out, out_f8=held.matrix))
    assert_norm(out.numpy(), x, None, 1e-5)
    assert_norm_f8(held, x, None, 1e-5)
    far.close()


@pytest.mark.parametrize("act", [mf.ACT_NONE, mf.ACT_GELU_TANH, mf.ACT_GELU_ERF, mf.ACT_SILU])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (5, 300, 200), (30, 200, 700), (100, 2000, 900),
                                   (257, 900, 300), (1300, 1500, 200), (65, 4122, 2921)])
def test_gated_activations(stream, m, n, k, act):
    """act(P) times the other projection, the gelus bit for bit mfr_bias_act's with one rounding of
    the product."""
    rng = np.random.default_rng(m + act)
    a, sa = exact_operands(rng, m, k, 1)
    g, sg = exact_operands(rng, n, k, 128)
    u, su = exact_operands(rng, n, k, 128)
    sg = sg / 128
    pg, pu = (ref.product(a, sa, *w)[0].astype(np.float32) for w in ((g, sg), (u, su)))
    ha, hg, hu = (held_of(c, s, stream, r) for c, s, r in ((a, sa, 1), (g, sg, 128), (u, su, 128)))
    held, out = Held(m, n, stream), mf.DeviceArray.empty((m, n), stream)
    mf.gemm_f8_gated(ha.matrix, hg.matrix, hu.matrix, act=act, out=out, out_f8=held.matrix)
    y = out.numpy()
    if act == mf.ACT_SILU:
        want = ref.silu(pg) * pu
        assert np.all(np.abs(y - want) <= 6 * ref.EPS32 * np.abs(want) + TINY * np.abs(pu))
    else:
        first = pg if act == mf.ACT_NONE else mf.bias_act(dev(pg, stream), None, act).numpy()
        assert equal(y, first * pu)
    assert_f8(held, y)


@pytest.mark.parametrize("m,n,k", [(4, 512, 512), (200, 512, 512), (1000, 2048, 640)])
def test_one_array_in_two_places(stream, m, n, k):
    """The weight as both projections, x as its own residual, c0 in place of c with 8 bits too."""
    rng = np.random.default_rng(m)
    a, sa = exact_operands(rng, m, k, 1)
    b, sb = exact_operands(rng, n, k, 128)
    p = ref.product(a, sa, b, sb)[0].astype(np.float32)
    ha, hb = held_of(a, sa, stream, 1), held_of(b, sb, stream, 128)
    out = mf.DeviceArray.empty((m, n), stream)
    mf.gemm_f8_gated(ha.matrix, hb.matrix, hb.matrix, act=mf.ACT_NONE, out=out)
    assert equal(out.numpy(), p * p)
    c0 = rng.standard_normal((m, n)).astype(np.float32)
    c, held = pitched(c0, stream, 4), Held(m, n, stream)
    mf.gemm_f8(ha.matrix, hb.matrix, c0=c, beta=-2.0, out=c, out_f8=held.matrix)
    want = p + np.float32(-2) * c0
    assert same_bits(c.numpy(), want)
    assert_f8(held, want)
    x = dev(c0, stream)
    y = mf.rms_norm(x, residual=x, summed=x, eps=1e-5)
    assert same_bits(x.numpy(), c0 + c0)
    assert_norm(y.numpy(), c0 + c0, None, 1e-5)


def test_infinities_in_weights_and_sums(stream):
    """Sums that overflow and infinite c0 and bias follow the formula; other columns are untouched."""
    for m in (1, 40, 300, 1500):
        a = np.full((m, 256), 0x7E, np.uint8)          # 448
        b = np.full((300, 256), 0x7E, np.uint8)
        sa, sb = np.ones((m, 2), np.float32), np.ones((3, 2), np.float32)
        sa[0], sb[1] = 2.0 ** 100, 2.0 ** 27           # 2^127 * 448^2 * 256 overflows
        bias = np.zeros(300, np.float32)
        bias[7], bias[8] = np.inf, np.nan
        got = mf.gemm_f8(held_of(a, sa, stream, 1).matrix, held_of(b, sb, stream, 128).matrix,
                         bias=dev(bias, stream)).numpy()
        with np.errstate(over="ignore"):
            want = (ref.product(a, sa, b, sb)[0].astype(np.float32) + bias).astype(np.float32)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(want)])


@pytest.mark.parametrize("cols,pitch", [(17, 32), (1023, 1024), (1024, 1024), (1030, 1152)])
def test_rows_are_padded(stream, cols, pitch):
    for block_rows in (1, 128):
        m = mf.F8Matrix.empty(3, cols, stream, block_rows)
        assert m.values.strides[0] == pitch and m.shape == (3, cols)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_values_next_to_the_borders_between_codes(stream, block_rows):
    """Blocks of random tops (over all of fp32's range) whose other values are the floats nearest to
    the borders between two codes, and the next floats to either side."""
    rng = np.random.default_rng(21)
    rows = 4096
    tops = np.exp2(rng.uniform(-148, 127, rows // block_rows))
    tops[::3] *= 448 * 2.0 ** -126 / 2.0 ** -117  # some of them near the least scale
    tops = np.minimum(tops, np.finfo(np.float32).max).astype(np.float32)
    by_row = np.repeat(tops, block_rows).astype(np.float64)
    x = np.empty((rows, 128), np.float32)
    with np.errstate(over="ignore", under="ignore"):
        borders = rng.choice(ref._MIDDLE, (rows, 127)) * rng.choice([-1.0, 1.0], (rows, 127))
        near = (borders * np.maximum(by_row / 448, 2.0 ** -126)[:, None]).astype(np.float32)
        step = rng.integers(-1, 2, near.shape)
        near = np.where(step < 0, np.nextafter(near, np.float32(-np.inf)),
                        np.where(step > 0, np.nextafter(near, np.float32(np.inf)), near))
    x[:, 1:] = np.clip(near, -by_row[:, None], by_row[:, None])
    x[:, 0] = by_row
    codes, scales = ref.quantize(x, block_rows)
    got = mf.quantize_f8(dev(x, stream), block_rows)
    assert np.array_equal(got.scales.numpy(), scales)
    assert same_codes(got.values.numpy(), codes)
