"""What the Python entry points of the 8-bit ops do with their arguments, without a GPU."""
import weakref
from types import SimpleNamespace

import pytest

import mensurflow_amd as mf
from test_f8 import STREAM, array, call, good_gemm, good_norm, matrix


def owners(operand):
    """The arrays of an operand, and what owns their memory."""
    arrays = ([operand.values, operand.scales] if isinstance(operand, mf.F8Matrix) else [operand])
    return [weakref.ref(x) for a in arrays for x in (a, a._base) if x is not None]


def norm(**operands):
    return mf.rms_norm_desc(operands.pop("x"), **operands)


def gemm(**operands):
    return mf.f8gemm_desc(operands.pop("a"), operands.pop("b"), **operands)


NORM = dict(x=lambda: array((4, 100), ptr=1 << 24), weight=lambda: array((100,)),
            residual=lambda: array((4, 100), ptr=1 << 25), summed=lambda: array((4, 100), ptr=1 << 26),
            out=lambda: array((4, 100)), out_f8=lambda: matrix(4, 100))
GEMM = dict(a=lambda: matrix(4, 100), b=lambda: matrix(200, 100, 128),
            c0=lambda: array((4, 200)), bias=lambda: array((200,)), out=lambda: array((4, 200)),
            out_f8=lambda: matrix(4, 200))
GATED = dict(a=GEMM["a"], b=GEMM["b"], up=GEMM["b"], out=GEMM["out"], out_f8=GEMM["out_f8"])


@pytest.mark.parametrize("make,operands", [(norm, NORM), (gemm, GEMM), (gemm, GATED)])
def test_a_descriptor_keeps_its_arrays(make, operands):
    """Arrays that were made for the descriptor alone live as long as it does, and no longer."""
    given = {name: f() for name, f in operands.items()}
    of = {name: owners(v) for name, v in given.items()}
    desc = make(**given)
    for operand in given.values():
        if isinstance(operand, mf.F8Matrix):  # another matrix from now on
            operand.values = operand.scales = None
    del given, operand
    assert {n for n, refs in of.items() if any(r() is None for r in refs)} == set()
    assert call("mfr_rms_norm" if make is norm else "mfr_f8gemm", desc)[1] == "null stream"
    del desc
    assert {n for n, refs in of.items() if any(r() is not None for r in refs)} == set()


@pytest.mark.parametrize("run,desc", [(mf.rms_norm_run, good_norm()), (mf.f8gemm, good_gemm()),
                                      (mf.f8gemm, good_gemm(gated=True))])
def test_a_descriptor_is_refused_by_a_stream_of_another_device(run, desc):
    with pytest.raises(ValueError, match="another device"):
        run(SimpleNamespace(device=1, handle=None), desc)
    with pytest.raises(ValueError, match="null stream"):
        run(SimpleNamespace(device=0, handle=None), desc)


@pytest.mark.parametrize("block_rows", [0, 2, -128])
def test_room_for_other_blocks_is_refused(block_rows):
    with pytest.raises(ValueError, match="block_rows"):
        mf.F8Matrix.empty(4, 100, STREAM, block_rows)
    with pytest.raises(ValueError, match="block_rows"):
        mf.quantize_f8(array((4, 100)), block_rows)


@pytest.mark.parametrize("rows,cols", [(4, -5), (4, -16), (4, -1000), (-1, 5)])
def test_room_for_negative_sizes_is_refused(rows, cols):
    for block_rows in (1, 128):
        with pytest.raises(ValueError, match="negative"):
            mf.F8Matrix.empty(rows, cols, STREAM, block_rows)
