"""mfr_f8_quantize, mfr_rms_norm and mfr_f8gemm on the device against the definitions in numpy
(f8_reference.py): conversions bit for bit, norms to the one rounding they make, products bit for bit
where every sum is exact and within the fp32 bound of their sums elsewhere."""
import ctypes

import numpy as np
import pytest

import f8_reference as ref
import mensurflow_amd as mf
from helpers import same_bits
from mensurflow_amd import abi

pytestmark = pytest.mark.gpu

# What the silu's fp32 form loses where exp(-x) overflows: there exp(-x) > 2^128 (1 - 2^-25), x is
# below -88.72, and |x| exp(x) <= 88.73 * 2^-128 (falling from there on), under 2^-121.
TINY = 2.0 ** -121
POISON = np.float32(123.5)
NAN_BYTE = 0x7F


def dev(x, stream):
    return mf.DeviceArray.from_numpy(np.ascontiguousarray(x), stream)


def pitched(x, stream, extra):
    """x on the device with `extra` poisoned columns behind each row, as a view."""
    wide = np.full((x.shape[0], x.shape[1] + extra), POISON, np.float32)
    wide[:, :x.shape[1]] = x
    return dev(wide, stream).slice(1, 0, x.shape[1])


class Held:
    """An F8Matrix on the device with guard bytes: NaN codes behind each row (at most 16 bytes
    behind k are read, none may count) and two guard rows; scales poisoned where nothing belongs."""

    def __init__(self, rows, cols, stream, block_rows=1, codes=None, scales=None, extra=16,
                 by_row=False):
        pitch = -(-cols // 16) * 16 + extra
        self.host = np.full((rows + 2, pitch), NAN_BYTE, np.uint8)
        if codes is not None:
            self.host[:rows, :cols] = codes
        self.bytes = dev(self.host, stream)
        mb, nb = -(-rows // block_rows), ref.blocks(cols)
        self.rows, self.cols, self.mb, self.nb = rows, cols, mb, nb
        # by_row: scales [mb, nb] with a pitch; else [nb, mb], as F8Matrix.empty lays them out.
        shape = (mb, nb + 3) if by_row else (nb, mb + 3)
        self.host_scales = np.full(shape, POISON, np.float32)
        if scales is not None:
            self.host_scales[:, :nb if by_row else mb] = scales if by_row else scales.T
        self.store = dev(self.host_scales, stream)
        view = self.store.slice(1, 0, nb if by_row else mb)
        self.matrix = mf.F8Matrix(self.bytes.slice(0, 0, rows).slice(1, 0, cols),
                                  view if by_row else view.T, block_rows)
        self.by_row = by_row

    def read(self):
        """(codes, scales), after checking that nothing else was written."""
        got = self.bytes.numpy()
        assert np.all(got[self.rows:] == NAN_BYTE) and np.all(got[:, self.cols:] == NAN_BYTE)
        scales = self.store.numpy()
        used = self.nb if self.by_row else self.mb
        assert np.all(scales[:, used:] == POISON)
        scales = scales[:, :used] if self.by_row else scales[:, :used].T
        return got[:self.rows, :self.cols], np.ascontiguousarray(scales)


def same_codes(got, want):
    nan = np.isnan(ref.VALUES[want])
    return np.array_equal(np.isnan(ref.VALUES[got]), nan) and np.array_equal(got[~nan], want[~nan])


def assert_f8(held, y, block_rows=1):
    """`held` is y (float32, as the kernel made it) in 8 bits."""
    codes, scales = held.read()
    want_codes, want_scales = ref.quantize(y, block_rows)
    assert np.array_equal(scales, want_scales, equal_nan=True)
    assert same_codes(codes, want_codes)


def assert_norm_f8(held, t, weight, eps):
    """`held` is the norm in 8 bits, from the 64-bit value: the codes are the nearest ones, the scales
    rounded once."""
    codes, scales = held.read()
    want, sure, exact = ref.quantize_exact(ref.rms_norm(t, weight, eps))
    nan = np.isnan(exact)
    assert np.array_equal(np.isnan(scales), nan)
    with np.errstate(invalid="ignore"):
        off = np.abs(scales - exact) > ref.EPS32 * (1 + 2.0 ** -10) * exact + 2.0 ** -149
    assert not np.any(off[~nan])
    assert same_codes(np.where(sure, codes, 0), np.where(sure, want, 0))
    values = ref.VALUES[codes[~sure]], ref.VALUES[want[~sure]]
    assert np.all(np.abs(values[0] - values[1]) <= 0.125 * np.abs(values[1]) + 2.0 ** -9)


def sample(rng, rows, cols):
    """Values of widely differing size, rows and blocks of zeros among them."""
    x = rng.standard_normal((rows, cols)) * np.exp(2 * rng.standard_normal((rows, 1)))
    x[rng.random((rows, cols)) < 0.05] *= 60
    if rows > 2:
        x[rows // 2] = 0
    return x.astype(np.float32)


# ---- conversion -----------------------------------------------------------------------------------

SIZES = [(1, 1), (1, 3), (2, 128), (3, 127), (5, 129), (129, 260), (128, 128), (257, 1023), (7, 4100)]


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantize(stream, rows, cols, block_rows):
    rng = np.random.default_rng(rows * 1000 + cols + block_rows)
    x = sample(rng, rows, cols)
    for extra, by_row in ((0, False), (5, True)):
        held = Held(rows, cols, stream, block_rows, by_row=by_row)
        mf.quantize_f8(pitched(x, stream, extra), block_rows, out=held.matrix)
        assert_f8(held, x, block_rows)
    made = mf.quantize_f8(dev(x, stream), block_rows)
    codes, scales = ref.quantize(x, block_rows)
    assert same_codes(made.values.numpy(), codes) and np.array_equal(made.scales.numpy(), scales)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_extremes(stream, block_rows):
    """Every e4m3 value and midpoint under the scale 1, tiny and huge blocks, infinities, NaN."""
    rows = np.zeros((6, 640), np.float32)
    rows[0, :126], rows[0, 126] = ref._MIDDLE, 448
    rows[0, 128:254], rows[0, 254] = -ref._MIDDLE, -448
    rows[0, 256:383] = ref._FINITE
    rows[1, 5], rows[1, 6], rows[1, 200] = 1e-44, 1e-38, np.finfo(np.float32).max
    rows[1, 201] = -np.finfo(np.float32).max / 3
    rows[2, 0], rows[2, 1] = np.inf, 3
    rows[3, 300], rows[3, 301] = np.nan, 5
    rows[4, 639] = -np.inf
    held = Held(6, 640, stream, block_rows)
    mf.quantize_f8(dev(rows, stream), block_rows, out=held.matrix)
    assert_f8(held, rows, block_rows)


def test_empty_matrices(stream):
    for rows, cols in ((0, 5), (5, 0), (0, 0)):
        x = mf.DeviceArray.empty((rows, cols), stream)
        for block_rows in (1, 128):
            assert mf.quantize_f8(x, block_rows).shape == (rows, cols)
        assert mf.rms_norm(x).shape == (rows, cols)
    a = mf.quantize_f8(mf.DeviceArray.empty((0, 40), stream))
    b = mf.quantize_f8(dev(np.ones((9, 40), np.float32), stream), 128)
    assert mf.gemm_f8(a, b).shape == (0, 9)
    assert mf.gemm_f8_gated(a, b, b).shape == (0, 9)
    none = mf.quantize_f8(mf.DeviceArray.empty((0, 40), stream), 128)
    assert mf.gemm_f8(mf.quantize_f8(dev(np.ones((3, 40), np.float32), stream)), none).shape == (3, 0)


# ---- norm -----------------------------------------------------------------------------------------

NORM_SIZES = SIZES + [(3, 1024), (2, 1025), (9, 2048), (2, 4096), (2, 4097), (3, 8192), (2, 8193),
                      (1, 16384), (2, 16385), (1, 40001), (300, 64),
                      (600, 300), (513, 1100), (520, 2100), (515, 4100), (514, 8200)]


def assert_norm(y, t, weight, eps):
    """One rounding of the 64-bit value (and the 64-bit steps before it, far below 2^-40 of it)."""
    want = ref.rms_norm(t, weight, eps)
    assert np.all(np.abs(y - want) <= ref.EPS32 * (1 + 2.0 ** -10) * np.abs(want) + 2.0 ** -149)


@pytest.mark.parametrize("rows,cols", NORM_SIZES)
def test_rms_norm(stream, rows, cols):
    rng = np.random.default_rng(rows * 77 + cols)
    x, r = sample(rng, rows, cols), sample(rng, rows, cols)
    w = (1 + 0.3 * rng.standard_normal(cols)).astype(np.float32)
    t = x + r
    dw = dev(w, stream)
    # fp32 alone, from pitched rows, no residual.
    out = pitched(np.zeros_like(x), stream, 3)
    mf.rms_norm(pitched(x, stream, 1), dw, eps=1e-5, out=out)
    assert_norm(out.numpy(), x, w, 1e-5)
    # Everything at once: the sum exactly, fp32, and 8 bits that are the fp32 result's.
    held, summed = Held(rows, cols, stream), pitched(np.zeros_like(x), stream, 2)
    out = pitched(np.zeros_like(x), stream, 5)
    dx, dr = pitched(x, stream, 3), dev(r, stream)
    mf.rms_norm_run(stream, mf.rms_norm_desc(dx, dw, residual=dr, eps=1e-6, summed=summed, out=out,
                                             out_f8=held.matrix))
    y = out.numpy()
    assert same_bits(summed.numpy(), t)
    assert_norm(y, t, w, 1e-6)
    assert_norm_f8(held, t, w, 1e-6)
    wide = mf.DeviceArray(out._base.shape, np.float32, stream, _base=out._base, _ptr=out._base._ptr)
    assert np.all(wide.numpy()[:, cols:] == POISON), "written behind the rows"
    # In place: the sum over the residual, the result over x; 8 bits from the sum alone; no weight.
    mf.rms_norm(dx, dw, residual=dr, summed=dr, out=dx)
    assert same_bits(dr.numpy(), t) and same_bits(dx.numpy(), y)
    again = Held(rows, cols, stream, by_row=True)
    mf.rms_norm_f8(dr, dw, out=again.matrix)
    assert_norm_f8(again, t, w, 1e-6)
    assert_norm(mf.rms_norm(dr, eps=0.5).numpy(), t, None, 0.5)


def test_rms_norm_residual_without_the_sum(stream):
    rng = np.random.default_rng(4)
    for cols in (100, 5000, 20000):
        x, r = sample(rng, 3, cols), sample(rng, 3, cols)
        assert_norm(mf.rms_norm(dev(x, stream), residual=dev(r, stream)).numpy(), x + r, None, 1e-6)


@pytest.mark.parametrize("cols", [130, 1500, 6000, 12000, 20000])
def test_rms_norm_extremes(stream, cols):
    """Rows whose squares leave fp32's range, rows of zeros, infinities, NaN, eps 0."""
    x = np.zeros((7, cols), np.float32)
    x[0] = 1e30
    x[1] = 1e-30
    x[2, 3] = 1e-40
    x[4, cols - 1] = np.inf
    x[5, 0] = np.nan
    x[6] = np.linspace(-1, 1, cols)
    for eps in (1e-6, 0.0):
        held, out = Held(7, cols, stream), mf.DeviceArray.empty((7, cols), stream)
        mf.rms_norm_run(stream, mf.rms_norm_desc(dev(x, stream), eps=eps, out=out,
                                                 out_f8=held.matrix))
        y = out.numpy()
        want = ref.rms_norm(x, None, eps)
        fine = np.isfinite(want)
        assert np.array_equal(np.isnan(want), np.isnan(y))
        assert np.all(np.abs(y - want)[fine] <= ref.EPS32 * (1 + 2.0 ** -10) * np.abs(want[fine])
                      + 2.0 ** -149)
        assert_norm_f8(held, x, None, eps)


def test_many_rows(stream):
    rng = np.random.default_rng(8)
    x = rng.standard_normal((70001, 33)).astype(np.float32)
    held, out = Held(70001, 33, stream), mf.DeviceArray.empty(x.shape, stream)
    mf.rms_norm_run(stream, mf.rms_norm_desc(dev(x, stream), out=out, out_f8=held.matrix))
    assert_norm(out.numpy(), x, None, 1e-6)
    assert_norm_f8(held, x, None, 1e-6)


# ---- products -------------------------------------------------------------------------------------

_WHOLE = np.array([c for c in range(256) if np.isfinite(ref.VALUES[c]) and ref.VALUES[c] ==
                   np.round(ref.VALUES[c]) and abs(ref.VALUES[c]) <= 16], np.uint8)
_POWERS = np.array([c for c in range(256) if np.isfinite(ref.VALUES[c]) and
                    abs(ref.VALUES[c]) in [2.0 ** e for e in range(9)]], np.uint8)


def exact_operands(rng, rows, k, block_rows, powers=False):
    """Whole values up to 16 (or powers of two from 1 to 256 in a tenth of the places) under scales
    1/2, 1 and 2: every sum of products is a multiple of 1/4 below 2^22, exact in fp32."""
    if powers:
        codes = np.where(rng.random((rows, k)) < 0.1, rng.choice(_POWERS, (rows, k)), 0)
        codes = codes.astype(np.uint8)
    else:
        codes = rng.choice(_WHOLE, (rows, k))
    scales = rng.choice(np.float32([0.5, 1, 2]), (-(-rows // block_rows), ref.blocks(k)))
    return codes, scales


def random_operands(rng, rows, k, block_rows):
    return ref.quantize(sample(rng, rows, k), block_rows)


def held_of(codes, scales, stream, block_rows, **kw):
    return Held(codes.shape[0], codes.shape[1], stream, block_rows, codes, scales, **kw)


GEMM_SIZES = [(1, 1, 1), (1, 128, 128), (1, 300, 1000), (2, 3, 17), (3, 130, 15), (8, 100, 256),
              (9, 129, 129), (16, 257, 127), (17, 64, 300), (31, 500, 640), (32, 128, 2049),
              (33, 127, 128), (48, 200, 513), (64, 384, 384), (65, 129, 143), (100, 40, 1030),
              (127, 255, 260), (128, 256, 512), (129, 257, 385), (200, 1100, 130), (257, 513, 700),
              (520, 260, 255), (1000, 30, 64), (2100, 2200, 300), (2049, 2305, 129),
              (512, 1024, 4096), (600, 1300, 2100), (260, 4100, 900), (40, 8300, 1000),
              (100, 9000, 300), (700, 700, 3100)]


@pytest.mark.parametrize("m,n,k", GEMM_SIZES)
def test_f8gemm_exact(stream, m, n, k):
    """Sums that fp32 holds exactly, so every bit is known: the product, alpha-free epilogue with c0
    and bias in their roundings, the 8-bit result, in place, and layouts with guards."""
    rng = np.random.default_rng(m * 10007 + n * 101 + k)
    for powers in (False, True):
        a, sa = exact_operands(rng, m, k, 1, powers)
        b, sb = exact_operands(rng, n, k, 128, powers)
        p, magnitude = ref.product(a, sa, b, sb)
        assert magnitude.max() < 2 ** 22
        ha = held_of(a, sa, stream, 1, by_row=powers, extra=0 if powers else 32)
        hb = held_of(b, sb, stream, 128, by_row=not powers)
        out = pitched(np.zeros((m, n), np.float32), stream, 3)
        assert mf.gemm_f8(ha.matrix, hb.matrix, out=out) is out
        assert same_bits(out.numpy() + np.float32(0), p.astype(np.float32) + np.float32(0))
        wide = mf.DeviceArray(out._base.shape, np.float32, stream, _base=out._base,
                              _ptr=out._base._ptr)
        assert np.all(wide.numpy()[:, n:] == POISON), "written behind the rows"
        # c0, bias and 8 bits.
        c0 = rng.standard_normal((m, n)).astype(np.float32)
        bias = rng.standard_normal(n).astype(np.float32)
        want = (p.astype(np.float32) + np.float32(0.3) * c0) + bias
        held = Held(m, n, stream, by_row=powers)
        c = pitched(c0, stream, 2)
        mf.gemm_f8(ha.matrix, hb.matrix, c0=c, beta=0.3, bias=dev(bias, stream), out=c,
                   out_f8=held.matrix)
        assert same_bits(c.numpy(), want.astype(np.float32))
        assert_f8(held, want.astype(np.float32))
        only = Held(m, n, stream)
        assert mf.gemm_f8(ha.matrix, hb.matrix, out_f8=only.matrix) is only.matrix
        assert_f8(only, p.astype(np.float32))


@pytest.mark.parametrize("m,n,k", GEMM_SIZES)
def test_f8gemm_gated_exact_projections(stream, m, n, k):
    """Projections that fp32 holds exactly; the silu, in fp32, is 1 / (1 + exp(-x)) with an
    exponential within 2^-23, three more roundings and the product's, and nothing where exp
    overflows (below 2^-121 of the other projection)."""
    rng = np.random.default_rng(m * 10009 + n * 103 + k)
    a, sa = exact_operands(rng, m, k, 1)
    g, sg = exact_operands(rng, n, k, 128)
    u, su = exact_operands(rng, n, k, 128)
    sg = sg / 64  # gates within the activation's range
    pg, pu = ref.product(a, sa, g, sg)[0], ref.product(a, sa, u, su)[0]
    ha, hg, hu = (held_of(c, s, stream, r) for c, s, r in ((a, sa, 1), (g, sg, 128), (u, su, 128)))
    held, out = Held(m, n, stream), pitched(np.zeros((m, n), np.float32), stream, 1)
    assert mf.gemm_f8_gated(ha.matrix, hg.matrix, hu.matrix, out=out, out_f8=held.matrix) \
        is held.matrix
    y = out.numpy()
    want = ref.silu(pg) * pu
    assert np.all(np.abs(y - want) <= 6 * ref.EPS32 * np.abs(want) + TINY * np.abs(pu))
    assert_f8(held, y)
    # Without an activation the gate is a product, with one rounding.
    plain = mf.gemm_f8_gated(ha.matrix, hg.matrix, hu.matrix, act=mf.ACT_NONE, out=out)
    assert plain is out
    assert same_bits(out.numpy() + np.float32(0), (pg * pu).astype(np.float32) + np.float32(0))
    made = mf.gemm_f8_gated(ha.matrix, hg.matrix, hu.matrix)
    codes, scales = ref.quantize(y)
    assert same_codes(made.values.numpy(), codes) and np.array_equal(made.scales.numpy(), scales)


@pytest.mark.parametrize("act", [mf.ACT_GELU_TANH, mf.ACT_GELU_ERF, mf.ACT_SILU])
@pytest.mark.parametrize("m", [5, 150])
def test_f8gemm_activations(stream, oracle, act, m):
    """The gelus are mfr_bias_act's, bit for bit."""
    rng = np.random.default_rng(act)
    a, sa = exact_operands(rng, m, 200, 1)
    b, sb = exact_operands(rng, 140, 200, 128)
    sb = sb / 256
    bias = rng.standard_normal(140).astype(np.float32)
    before = ref.product(a, sa, b, sb)[0].astype(np.float32) + bias
    ha, hb = held_of(a, sa, stream, 1), held_of(b, sb, stream, 128)
    y = mf.gemm_f8(ha.matrix, hb.matrix, bias=dev(bias, stream), act=act).numpy()
    if act == mf.ACT_SILU:
        want = ref.silu(before)
        assert np.all(np.abs(y - want) <= 5 * ref.EPS32 * np.abs(want) + TINY)
    else:
        assert same_bits(y, mf.bias_act(dev(before, stream), None, act).numpy())


@pytest.mark.parametrize("m,n,k", GEMM_SIZES + [(1, 4096, 4096), (24, 700, 4100), (300, 256, 4224)])
def test_f8gemm_random(stream, m, n, k):
    rng = np.random.default_rng(m * 31 + n * 7 + k)
    a, sa = random_operands(rng, m, k, 1)
    b, sb = random_operands(rng, n, k, 128)
    ha, hb = held_of(a, sa, stream, 1), held_of(b, sb, stream, 128)
    p, magnitude = ref.product(a, sa, b, sb)
    got = mf.gemm_f8(ha.matrix, hb.matrix).numpy()
    assert np.all(np.abs(got - p) <= ref.product_bound(magnitude, k) + ref.EPS32 * np.abs(p))
    assert same_bits(got, mf.gemm_f8(ha.matrix, hb.matrix).numpy()), "two calls differ"


def test_f8gemm_nothing_to_sum(stream):
    """k == 0: c0 and bias alone."""
    c0, bias = np.arange(12, dtype=np.float32).reshape(3, 4), np.float32([1, 2, 3, 4])
    a = mf.F8Matrix.empty(3, 0, stream)
    b = mf.F8Matrix.empty(4, 0, stream, 128)
    got = mf.gemm_f8(a, b, c0=dev(c0, stream), beta=2.0, bias=dev(bias, stream)).numpy()
    assert same_bits(got, 2 * c0 + bias)
    assert np.all(mf.gemm_f8(a, b).numpy() == 0)
    codes = mf.gemm_f8_gated(a, b, b)
    assert np.all(ref.VALUES[codes.values.numpy()] == 0)


@pytest.mark.parametrize("m", [1, 20, 150])
def test_f8gemm_nan_and_infinite_scales_stay_in_their_rows(stream, m):
    rng = np.random.default_rng(m)
    n, k = 140, 300
    a, sa = exact_operands(rng, m, k, 1)
    b, sb = exact_operands(rng, n, k, 128)
    p = ref.product(a, sa, b, sb)[0].astype(np.float32)
    b[130, 299] = 0xFF            # NaN in one output's row
    if m > 1:
        a[m - 1, 40] = NAN_BYTE   # and in the last activation's
    want = p.copy()
    want[:, 130] = np.nan
    if m > 1:
        want[m - 1] = np.nan
    held, out = Held(m, n, stream), mf.DeviceArray.empty((m, n), stream)
    mf.gemm_f8(held_of(a, sa, stream, 1).matrix, held_of(b, sb, stream, 128).matrix, out=out,
               out_f8=held.matrix)
    got = out.numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~np.isnan(got)], want[~np.isnan(got)])
    assert_f8(held, got)


def test_a_feed_forward_block(stream):
    """Norm, gated pair and second product in a row, as a decoder's block runs them, each against its
    definition on the device's own inputs; the second product adds the residual stream in place."""
    rng = np.random.default_rng(11)
    hidden, inner = 640, 1100
    wg, wu = (rng.standard_normal((inner, hidden)).astype(np.float32) / 25 for _ in range(2))
    wd = rng.standard_normal((hidden, inner)).astype(np.float32) / 33
    gate, up, down = (mf.quantize_f8(dev(w, stream), 128) for w in (wg, wu, wd))
    qw = [ref.quantize(w, 128) for w in (wg, wu, wd)]
    norm = dev((1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32), stream)
    for tokens in (1, 7, 33, 300):
        x, r = (rng.standard_normal((tokens, hidden)).astype(np.float32) for _ in range(2))
        dx, dr = dev(x, stream), dev(r, stream)
        q = mf.rms_norm_f8(dx, norm, residual=dr, summed=dr)
        t = dr.numpy()
        h = mf.gemm_f8_gated(q, gate, up)
        mf.gemm_f8(h, down, c0=dr, beta=1.0, out=dr)
        assert same_bits(t, x + r)
        a, sa = q.values.numpy(), q.scales.numpy()
        y = ref.rms_norm(t, norm.numpy())
        # Half a step of e4m3 (2^-4, or 2^-10 of the scale below the normal numbers).
        step = np.repeat(sa.astype(np.float64), 128, 1)[:, :hidden]
        assert np.all(np.abs(ref.dequantize(a, sa) - y) <=
                      1.001 * np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * step))
        (pg, mg), (pu, mu) = (ref.product(a, sa, *w) for w in qw[:2])
        eg, eu = ref.product_bound(mg, hidden), ref.product_bound(mu, hidden)
        want = ref.silu(pg) * pu
        # |silu'| < 1.1; then the activation's roundings.
        off = 1.1 * eg * np.abs(pu) + np.abs(ref.silu(pg)) * eu + 8 * ref.EPS32 * np.abs(want)
        hc, hs = h.values.numpy(), h.scales.numpy()
        step = np.repeat(hs.astype(np.float64), 128, 1)[:, :inner]
        assert np.all(np.abs(ref.dequantize(hc, hs) - want) <=
                      1.001 * np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * step) + 1.1 * off)
        p, magnitude = ref.product(hc, hs, *qw[2])
        got = dr.numpy()
        assert np.all(np.abs(got - (t + p)) <= ref.product_bound(magnitude, inner) +
                      2 * ref.EPS32 * (np.abs(p) + np.abs(t)))


def test_wrapped_stream_and_memory(stream):
    """Stream.wrap and DeviceArray.wrap: the same HIP stream and another owner's memory."""
    rng = np.random.default_rng(12)
    x = dev(rng.standard_normal((5, 200)).astype(np.float32), stream)
    with mf.Stream.wrap(stream.hip_stream(), stream.device) as wrapped:
        view = mf.DeviceArray.wrap(x.ptr, (5, 100), wrapped, strides=(200, 1))
        y = mf.rms_norm(view).numpy()
        view.close()
    assert_norm(y, x.numpy()[:, :100], None, 1e-6)
    assert same_bits(mf.rms_norm(x.slice(1, 0, 100)).numpy(), y)


def test_captured_and_replayed(stream):
    """The block in a graph, replayed with other inputs after eager calls on the same stream."""
    hip = ctypes.CDLL("libamdhip64.so.7")  # the runtime that the library has loaded

    def hip_call(name, *args):
        assert getattr(hip, name)(*args) == 0, name

    rng = np.random.default_rng(13)
    for tokens in (1, 40, 260):
        with mf.Stream(0) as own:
            x = dev(rng.standard_normal((tokens, 512)).astype(np.float32), own)
            gate, up = (mf.quantize_f8(dev(rng.standard_normal((384, 512)).astype(np.float32), own),
                                       128) for _ in range(2))
            down = mf.quantize_f8(dev(rng.standard_normal((512, 384)).astype(np.float32), own), 128)
            q, h = mf.F8Matrix.empty(tokens, 512, own), mf.F8Matrix.empty(tokens, 384, own)
            out = mf.DeviceArray.empty((tokens, 512), own)

            def block():
                mf.rms_norm_f8(x, out=q)
                mf.gemm_f8_gated(q, gate, up, out_f8=h)
                mf.gemm_f8(h, down, c0=x, beta=1.0, out=out)

            block()
            handle = ctypes.c_void_p(own.hip_stream())
            graph, run = ctypes.c_void_p(), ctypes.c_void_p()
            hip_call("hipStreamBeginCapture", handle, ctypes.c_int(1))  # thread local
            block()
            hip_call("hipStreamEndCapture", handle, ctypes.byref(graph))
            hip_call("hipGraphInstantiate", ctypes.byref(run), graph, None, None, ctypes.c_size_t(0))
            for _ in range(3):
                host = rng.standard_normal((tokens, 512)).astype(np.float32)
                x.upload(host)
                block()
                codes = h.values.numpy()
                for launched in (False, True):
                    if launched:
                        mf.fill(out, 7.0)
                        hip_call("hipGraphLaunch", run, handle)
                    # A captured product may add its ranges of depth in another order, so that a
                    # code next to a border is another: each is held to its own codes.
                    again = h.values.numpy()
                    assert np.mean(again != codes) < 0.01
                    p, magnitude = ref.product(again, h.scales.numpy(), down.values.numpy(),
                                               down.scales.numpy())
                    assert np.all(np.abs(out.numpy() - (host + p)) <=
                                  ref.product_bound(magnitude, 384) +
                                  2 * ref.EPS32 * (np.abs(p) + np.abs(host)))
            hip_call("hipGraphExecDestroy", run)
            hip_call("hipGraphDestroy", graph)


def test_the_other_entry_points_refuse_the_silu(stream):
    x = dev(np.ones((2, 4), np.float32), stream)
    with pytest.raises(ValueError):
        mf.bias_act(x, None, abi.ACT_SILU)
    with pytest.raises(ValueError):
        mf.gemm(x, x, trans_b=True, act=abi.ACT_SILU)


def test_offsets_past_32_bits(stream):
    """Rows that lie more than 4 GiB apart in all: the last rows' values and scales are found."""
    rng = np.random.default_rng(14)
    m, n, k, pitch = 280, 129, 200, 1 << 24  # 280 rows of 16 MiB: 4.4 GiB
    a, sa = exact_operands(rng, m, k, 1)
    b, sb = exact_operands(rng, n, k, 128)
    far = mf.DeviceArray.empty((m, pitch), stream, np.uint8)
    near = dev(a, stream)
    for r in range(m):
        abi.check(abi.load().mfr_memcpy_d2d(stream.handle, far.ptr + r * pitch, near.ptr + r * k, k))
    held = held_of(a, sa, stream, 1)
    wide = mf.F8Matrix(far.slice(1, 0, k), held.matrix.scales, 1)
    hb = held_of(b, sb, stream, 128)
    p = ref.product(a, sa, b, sb)[0].astype(np.float32)
    assert same_bits(mf.gemm_f8(wide, hb.matrix).numpy() + np.float32(0), p + np.float32(0))
    y = mf.DeviceArray.empty((m, n), stream)
    q = mf.F8Matrix(far.slice(1, k, k + 144).slice(1, 8, 8 + n), mf.F8Matrix.empty(m, n, stream).scales)
    assert (q.values.ptr - far.ptr) % 16 == 0
    mf.gemm_f8(wide, hb.matrix, out=y, out_f8=q)
    codes, scales = ref.quantize(y.numpy())
    assert same_codes(q.values.numpy(), codes) and np.array_equal(q.scales.numpy(), scales)
    far.close()
