"""Which form of mfr_f8gemm a size takes (mfr_f8gemm_plan): that the sizes of the tests reach every form
with every kind of output, that plans without a workspace are what captured calls need, and what the
query refuses."""
import ctypes

import pytest

import mensurflow_amd as mf
from mensurflow_amd import abi
from test_f8 import array, good_gemm, matrix
from test_f8_edges_gpu import DEEP
from test_f8_forms_gpu import FORMS
from test_f8_forms_gpu import test_forms as check_forms
from test_f8_forms_gpu import test_gated_forms as check_gated_forms

pytestmark = pytest.mark.gpu

# Few rows against a gated pair, 64 a workgroup, without and with an 8-bit output; 64-row tiles with
# the whole depth and fp32 alone.
MORE = [(17, 2060, 80), (64, 2048, 512), (34, 8339, 546)]


@pytest.mark.parametrize("m,n,k", MORE)
def test_more_forms(stream, m, n, k):
    check_forms(stream, m, n, k)


@pytest.mark.parametrize("m,n,k", MORE)
def test_more_gated_forms(stream, m, n, k):
    check_gated_forms(stream, m, n, k)


OUTPUTS = {"c": (True, False), "q": (False, True), "both": (True, True)}


def descriptor(m, n, k, gated, outputs):
    c, q = OUTPUTS[outputs]
    return mf.f8gemm_desc(matrix(m, k), matrix(n, k, 128), up=matrix(n, k, 128) if gated else None,
                          out=array((m, n)) if c else None, out_f8=matrix(m, n) if q else None)


RINGS_AND_TILES = {abi.F8_RING_32, abi.F8_RING_64, abi.F8_RING_64_PAIR, abi.F8_RING_128,
                   abi.F8_TILE_64, abi.F8_TILE_128}
PLAIN = RINGS_AND_TILES | {abi.F8_FEW_16, abi.F8_FEW_32, abi.F8_FEW_32_WIDE, abi.F8_FEW_64,
                           abi.F8_RING_32_WIDE}
GATED = RINGS_AND_TILES | {abi.F8_FEW_16, abi.F8_FEW_32, abi.F8_FEW_64}


@pytest.mark.parametrize("outputs", OUTPUTS)
@pytest.mark.parametrize("gated", [False, True])
def test_the_sizes_of_the_tests_reach_every_form(stream, gated, outputs):
    if mf.device_info(0).compute_units != 256:
        pytest.skip("the sizes are for 256 compute units")
    plans = [mf.f8gemm_plan(stream, descriptor(*size, gated, outputs)) for size in FORMS + MORE]
    # A part of the outputs that runs by itself takes its own form; the main part's is named.
    whole = {form for form, splits, _, _ in plans if splits == 1}
    assert whole == (GATED if gated else PLAIN)
    ranges = {form for form, splits, _, _ in plans if splits > 1}
    assert ranges == {abi.F8_TILE_64, abi.F8_TILE_128}
    assert {regions for _, _, regions, _ in plans} == {1, 2, 3}


def test_up_to_64_rows_with_both_outputs_take_no_workspace(stream):
    for gated in (False, True):
        for m, n, k in FORMS + MORE + DEEP:
            m = 1 + m % 64
            form, splits, _, workspace = mf.f8gemm_plan(stream, descriptor(m, n, k, gated, "both"))
            assert form and splits == 1 and workspace == 0


def test_what_takes_the_workspace(stream):
    """Ranges, and the sums of the forms whose 8-bit output is a second launch's; nothing else."""
    tiles = {abi.F8_TILE_64, abi.F8_TILE_128}
    for gated in (False, True):
        for outputs in OUTPUTS:
            for m, n, k in FORMS + MORE + DEEP:
                form, splits, regions, workspace = mf.f8gemm_plan(
                    stream, descriptor(m, n, k, gated, outputs))
                if regions > 1:
                    continue
                if splits > 1:
                    assert form in tiles and workspace >= (1 + gated) * splits * 4 * m * n
                elif outputs == "q" and form not in tiles | {abi.F8_RING_128}:
                    assert workspace == 4 * m * n
                else:
                    assert workspace == 0


def test_a_plan_of_nothing(stream):
    for m, n in ((0, 5), (5, 0)):
        assert mf.f8gemm_plan(stream, descriptor(m, n, 100, False, "c")) == (0, 0, 0, 0)
    assert mf.f8gemm_plan(stream, descriptor(5, 5, 0, False, "c"))[0] == abi.F8_FEW_16


def test_the_plan_refuses_what_the_call_does(stream):
    d = good_gemm()
    d.act = 4
    with pytest.raises(ValueError, match="activation"):
        mf.f8gemm_plan(stream, d)
    d = good_gemm()
    d.a.rs = 232
    with pytest.raises(NotImplementedError, match="aligned"):
        mf.f8gemm_plan(stream, d)
    lib = abi.load()
    out = [ctypes.c_int32() for _ in range(3)] + [ctypes.c_size_t()]
    for missing in range(4):
        given = [None if i == missing else ctypes.byref(o) for i, o in enumerate(out)]
        status = lib.mfr_f8gemm_plan(0, ctypes.byref(good_gemm()), *given)
        assert status == abi.MFR_E_INVALID and "null argument" in abi.last_error()
    status = lib.mfr_f8gemm_plan(0, None, *map(ctypes.byref, out))
    assert status == abi.MFR_E_INVALID and "null descriptor" in abi.last_error()
    assert lib.mfr_f8gemm_plan(mf.device_count(), ctypes.byref(good_gemm()),
                               *map(ctypes.byref, out)) != abi.MFR_OK
