"""8-bit matrices without a GPU: the numpy reference against torch's own e4m3, and what the entry
points refuse (the descriptors are checked before the stream is looked at)."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import f8_reference as ref
import mensurflow_amd as mf
from mensurflow_amd import abi

STREAM = SimpleNamespace(device=0, handle=None)


def array(shape, dtype=np.float32, strides=None, ptr=1 << 20):
    return mf.DeviceArray.wrap(ptr, shape, STREAM, dtype, strides)


def matrix(rows, cols, block_rows=1, ptr=1 << 20):
    pitch = -(-max(cols, 1) // 16) * 16
    return mf.F8Matrix(array((rows, cols), np.uint8, (pitch, 1), ptr),
                       array((-(-rows // block_rows), ref.blocks(cols))), block_rows)


def test_reference_codes_are_torchs():
    codes = np.arange(256, dtype=np.uint8)
    theirs = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(theirs, ref.VALUES, equal_nan=True)
    rng = np.random.default_rng(1)
    x = np.concatenate([rng.uniform(-448, 448, 20000), rng.standard_normal(20000) * 2.0 ** -8,
                        ref._MIDDLE, -ref._MIDDLE, ref._FINITE]).astype(np.float32)
    theirs = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ref.encode(x), theirs)


def test_reference_scales():
    x = np.zeros((130, 200), np.float32)
    x[3, 7], x[129, 150] = -448 * 3, 1e-44
    codes, scales = ref.quantize(x, 128)
    assert scales.shape == (2, 2) and scales[0, 0] == 3 and scales[1, 1] == np.float32(2.0 ** -126)
    assert codes[3, 7] == 0xFE and np.all(ref.dequantize(codes, scales, 128)[:129] == x[:129])


def call(entry, desc):
    return getattr(abi.load(), entry)(None, ctypes.byref(desc)), abi.last_error()


def good_norm(**kw):
    args = dict(residual=None, summed=None, out=array((4, 100)), out_f8=matrix(4, 100))
    args.update(kw)
    return mf.rms_norm_desc(array((4, 100), ptr=1 << 24), array((100,)), **args)


def good_gemm(gated=False, **kw):
    args = dict(up=matrix(200, 100, 128) if gated else None, out=array((4, 200)),
                out_f8=matrix(4, 200))
    args.update(kw)
    return mf.f8gemm_desc(matrix(4, 100), matrix(200, 100, 128), **args)


@pytest.mark.parametrize("entry,desc", [("mfr_rms_norm", good_norm()), ("mfr_f8gemm", good_gemm()),
                                        ("mfr_f8gemm", good_gemm(gated=True, act=mf.ACT_SILU))])
def test_a_good_descriptor_comes_as_far_as_the_stream(entry, desc):
    assert call(entry, desc) == (abi.MFR_E_INVALID, "null stream")


NORM = [
    (dict(rows=-1), abi.MFR_E_INVALID, "negative dimension"),
    (dict(eps=-1e-3), abi.MFR_E_INVALID, "eps"),
    (dict(eps=float("nan")), abi.MFR_E_INVALID, "eps"),
    (dict(x=None), abi.MFR_E_INVALID, "null input"),
    (dict(x_rs=99), abi.MFR_E_INVALID, "overlap"),
    (dict(out_rs=-100), abi.MFR_E_INVALID, "overlap"),
    (dict(residual=1 << 25, residual_rs=0), abi.MFR_E_INVALID, "overlap"),
    (dict(sum=1 << 20, sum_rs=100), abi.MFR_E_INVALID, "one array"),
    (dict(sum=1 << 24, sum_rs=101), abi.MFR_E_INVALID, "in place"),
    (dict(out=1 << 24, out_rs=200), abi.MFR_E_INVALID, "in place"),
]


@pytest.mark.parametrize("change,status,message", NORM)
def test_rms_norm_refuses(change, status, message):
    d = good_norm()
    for name, value in change.items():
        setattr(d, name, value)
    got = call("mfr_rms_norm", d)
    assert got[0] == status and message in got[1], got


def test_rms_norm_needs_an_output():
    status, message = call("mfr_rms_norm", good_norm(out=None, out_f8=None))
    assert status == abi.MFR_E_INVALID and "neither" in message


F8 = [
    (dict(block_rows=2), abi.MFR_E_INVALID, "block_rows 1 or 128"),
    (dict(values=(1 << 20) + 8), abi.MFR_E_UNSUPPORTED, "16-byte aligned"),
    (dict(rs=232), abi.MFR_E_UNSUPPORTED, "16-byte aligned"),
    (dict(rs=96), abi.MFR_E_INVALID, "overlap"),
    (dict(rs=-208), abi.MFR_E_INVALID, "overlap"),
    (dict(rs=(1 << 24) + 16), abi.MFR_E_UNSUPPORTED, "too far apart"),
    (dict(scales_rs=(1 << 23) + 1), abi.MFR_E_UNSUPPORTED, "too far apart"),
    (dict(scales_cs=(1 << 40) + 1), abi.MFR_E_UNSUPPORTED, "too far apart"),
    (dict(scales=None), abi.MFR_E_INVALID, "null pointer"),
    (dict(scales_rs=-1), abi.MFR_E_INVALID, "negative scale strides"),
]
SCALES_OVERLAP = [dict(scales_rs=0), dict(scales_cs=0), dict(scales_rs=1, scales_cs=3),
                  dict(scales_rs=1, scales_cs=1)]


@pytest.mark.parametrize("which", ["a", "b", "up", "out_f8"])
@pytest.mark.parametrize("change,status,message", F8)
def test_f8gemm_refuses_matrices(which, change, status, message):
    d = good_gemm(gated=True)
    for name, value in change.items():
        setattr(getattr(d, which), name, value)
    got = call("mfr_f8gemm", d)
    assert got[0] == status and message in got[1] and which in got[1], got


@pytest.mark.parametrize("which,block_rows", [("a", 128), ("b", 1), ("up", 1), ("out_f8", 128)])
def test_f8gemm_refuses_the_other_blocks(which, block_rows):
    d = good_gemm(gated=True)
    getattr(d, which).block_rows = block_rows
    got = call("mfr_f8gemm", d)
    assert got[0] == abi.MFR_E_UNSUPPORTED and which in got[1], got


@pytest.mark.parametrize("change", SCALES_OVERLAP)
def test_outputs_with_overlapping_scales_are_refused(change):
    for entry, d in (("mfr_f8gemm", good_gemm()), ("mfr_rms_norm", mf.rms_norm_desc(
            array((4, 200), ptr=1 << 24), out_f8=matrix(4, 200)))):
        for name, value in change.items():
            setattr(d.out_f8, name, value)
        got = call(entry, d)
        assert got[0] == abi.MFR_E_INVALID and "scales that overlap" in got[1], got


GEMM = [
    (dict(k=-1), "negative dimension"), (dict(act=4), "activation"), (dict(act=-1), "activation"),
    (dict(beta=1.0), "beta requires c0"), (dict(c_rs=199), "overlap"),
    (dict(c0=1 << 24, c0_rs=0, beta=0.5), "overlap"),
    (dict(c0=1 << 20, c0_rs=208, beta=0.5), "row stride"),
]


@pytest.mark.parametrize("change,message", GEMM)
def test_f8gemm_refuses(change, message):
    d = good_gemm()
    for name, value in change.items():
        setattr(d, name, value)
    got = call("mfr_f8gemm", d)
    assert got[0] == abi.MFR_E_INVALID and message in got[1], got


def test_f8gemm_gated_refuses_c0_and_bias_and_needs_an_output():
    for kw in (dict(c0=array((4, 200))), dict(bias=array((200,)))):
        status, message = call("mfr_f8gemm", good_gemm(gated=True, **kw))
        assert status == abi.MFR_E_INVALID and "gated" in message
    status, message = call("mfr_f8gemm", good_gemm(out=None, out_f8=None))
    assert status == abi.MFR_E_INVALID and "neither" in message


def test_quantize_needs_an_output():
    lib = abi.load()
    assert lib.mfr_f8_quantize(None, 1, 1, None, 1, None) == abi.MFR_E_INVALID
    assert "null output" in abi.last_error()


def test_quantize_refuses():
    lib = abi.load()
    d = mf._f8_desc(matrix(4, 100), "x")
    for rows, x, x_rs, message in ((-1, 1 << 24, 100, "negative"), (4, None, 100, "null input"),
                                   (4, 1 << 24, 99, "overlap"), (4, 1 << 24, 100, "null stream")):
        assert lib.mfr_f8_quantize(None, rows, 100, x, x_rs, ctypes.byref(d)) == abi.MFR_E_INVALID
        assert message in abi.last_error()


def test_python_refuses_shapes_that_disagree():
    x, w = array((4, 100)), array((100,))
    with pytest.raises(ValueError):
        mf.rms_norm_desc(x, array((99,)), out=x)
    with pytest.raises(ValueError):
        mf.rms_norm_desc(x, w, out=array((4, 99)))
    with pytest.raises(ValueError):
        mf.rms_norm_desc(x, w, residual=array((4, 100), np.int64), out=x)
    with pytest.raises(ValueError):
        mf.rms_norm_desc(array((4, 100), strides=(1, 4)), w, out=x)
    with pytest.raises(ValueError):
        mf.rms_norm_desc(x, w, out_f8=matrix(4, 99))
    with pytest.raises(ValueError):
        mf.f8gemm_desc(matrix(4, 100), matrix(200, 99, 128), out=array((4, 200)))
    with pytest.raises(ValueError):
        mf.f8gemm_desc(matrix(4, 100), matrix(200, 100, 128), up=matrix(201, 100, 128),
                       out=array((4, 200)))
    with pytest.raises(ValueError):
        mf.f8gemm_desc(matrix(4, 100), matrix(200, 100, 128), out=array((5, 200)))
    with pytest.raises(ValueError):
        mf.f8gemm_desc(matrix(4, 100), matrix(200, 100, 128), out_f8=matrix(4, 199))
    bad = matrix(4, 300)
    bad.scales = array((4, 2))
    with pytest.raises(ValueError):
        mf.f8gemm_desc(bad, matrix(200, 300, 128), out=array((4, 200)))
    with pytest.raises(ValueError):
        mf.quantize_f8(x, 128, out=matrix(4, 100, 1))


def test_sizes_past_64_bits_are_refused():
    """Products of sizes that would leave 64 bits: refused by the sizes, before any launch."""
    for change in (dict(m=1 << 41), dict(n=1 << 41), dict(m=1 << 30, n=1 << 20)):
        d = good_gemm(out_f8=None)
        d.c_rs = 1 << 50
        for name, value in change.items():
            setattr(d, name, value)
        status, message = call("mfr_f8gemm", d)
        assert status == abi.MFR_E_INVALID and ("too many rows" in message or
                                                "too large" in message), message
    lib = abi.load()
    for block_rows in (1, 128):
        d = mf._f8_desc(matrix(4, 100, block_rows), "x")
        assert lib.mfr_f8_quantize(None, 1 << 41, 100, 1 << 24, 100,
                                   ctypes.byref(d)) == abi.MFR_E_INVALID
        assert "too many rows" in abi.last_error()


def test_a_single_row_has_any_stride():
    row = array((1, 100), strides=(1, 1))
    d = mf.rms_norm_desc(row, residual=row, summed=row, out_f8=matrix(1, 100))
    assert (d.x_rs, d.residual_rs, d.sum_rs) == (100, 100, 100)
    q = matrix(1, 100)
    q.values = array((1, 100), np.uint8, (1, 1))
    assert mf.f8gemm_desc(q, matrix(20, 100, 128), out=array((1, 20))).a.rs == 112
    for entry, desc in (("mfr_rms_norm", d),
                        ("mfr_f8gemm", mf.f8gemm_desc(q, matrix(20, 100, 128),
                                                      out=array((1, 20))))):
        assert call(entry, desc) == (abi.MFR_E_INVALID, "null stream")


def test_python_refuses_operands_of_two_devices():
    other = SimpleNamespace(device=1, handle=None)
    x = array((4, 100))
    far = mf.DeviceArray.wrap(1 << 20, (4, 100), other)
    far_f8 = mf.F8Matrix(mf.DeviceArray.wrap(1 << 20, (200, 100), other, np.uint8, (112, 1)),
                         mf.DeviceArray.wrap(1 << 20, (2, 1), other), 128)
    with pytest.raises(ValueError, match="devices"):
        mf.rms_norm_desc(x, residual=far, out=x)
    with pytest.raises(ValueError, match="devices"):
        mf.quantize_f8(far, out=matrix(4, 100))
    with pytest.raises(ValueError, match="devices"):
        mf.f8gemm_desc(matrix(4, 100), far_f8, out=array((4, 200)))
