"""mfr_rope on the device against the rotation in 64 bits."""
import numpy as np
import pytest

import kv_reference as ref
import mensurflow_amd as mf
from helpers import same_bits
from kv_reference import dev

pytestmark = pytest.mark.gpu
LAYOUTS = [mf.ROTARY_HALVES, mf.ROTARY_PAIRS]


def check(got, want, off, what):
    bad = ~(np.abs(got - want) <= off + np.abs(want) * 0)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3], got[bad][:3], want[bad][:3])


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("rows,heads,d,rot", [
    (1, 1, 2, 2), (1, 1, 128, 128), (3, 40, 128, 128), (700, 3, 64, 64), (5, 7, 80, 48),
    (33, 5, 80, 46), (2, 3, 7, 6), (9, 2, 33, 10), (4, 1, 300, 256), (6, 2, 515, 254), (1, 100, 96, 2),
    (2000, 17, 16, 8), (3, 2, 5, 0)])
def test_turns(stream, layout, rows, heads, d, rot):
    rng = np.random.default_rng(rows + d)
    print(f"rope {rows}x{heads}x{d} rot {rot} layout {layout}", flush=True)
    x = rng.standard_normal((rows, heads, d)).astype(np.float32)
    positions = rng.integers(0, 131072, rows).astype(np.int32)
    r = mf.rotary(rot, layout=layout)
    for backward in (False, True):
        want, off = ref.turn(x, positions, ref.steps(rot), layout, backward=backward)
        dx = dev(x, stream)
        got = mf.rope(dx, r, positions=dev(positions, stream), backward=backward).numpy()
        check(got, want, off, (backward, "new"))
        assert same_bits(got[..., rot:], x[..., rot:])
        assert same_bits(dx.numpy(), x)
        assert same_bits(mf.rope(dx, r, positions=dev(positions, stream), backward=backward,
                                 out=dx).numpy(), got), "in place"


@pytest.mark.parametrize("layout", LAYOUTS)
def test_positions_without_an_array(stream, layout):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((50, 3, 32)).astype(np.float32)
    r = mf.rotary(32, layout=layout)
    for first in (0, 7, -20, (1 << 31) - 50, -(1 << 31)):
        want, off = ref.turn(x, first + np.arange(50), ref.steps(32), layout)
        check(mf.rope(dev(x, stream), r, first=first).numpy(), want, off, first)


def test_far_and_negative_positions(stream):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((400, 2, 64)).astype(np.float32)
    positions = rng.integers(-(1 << 31), 1 << 31, 400).astype(np.int32)
    want, off = ref.turn(x, positions, ref.steps(64), mf.ROTARY_HALVES)
    check(mf.rope(dev(x, stream), mf.rotary(64), positions=dev(positions, stream)).numpy(), want, off,
          "far")


@pytest.mark.parametrize("scaling", [dict(factor=4.0), dict(factor=8.0, original=4096.0),
                                     dict(factor=32.0, original=8192.0, slow=1.0, fast=4.0),
                                     dict(base=500000.0)])
def test_scaled_steps(stream, scaling):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((64, 2, 128)).astype(np.float32)
    positions = rng.integers(0, 131072, 64).astype(np.int32)
    want, off = ref.turn(x, positions, ref.steps(128, **scaling), mf.ROTARY_HALVES, 1.25)
    got = mf.rope(dev(x, stream), mf.rotary(128, amplitude=1.25, **scaling),
                  positions=dev(positions, stream)).numpy()
    check(got, want, off, scaling)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("rot", [64, 42])
def test_strides(stream, layout, rot):
    """Heads inside wider rows at any 4-byte alignment, heads in front of rows, one row for all."""
    rng = np.random.default_rng(5)
    rows, heads, d = 37, 5, 64
    r = mf.rotary(rot, layout=layout)
    wide = rng.standard_normal((rows, heads + 2, d + 3)).astype(np.float32)
    positions = rng.integers(0, 9999, rows).astype(np.int32)
    dp = dev(positions, stream)
    dw = dev(wide, stream)
    view = dw.slice(1, 1, 1 + heads).slice(2, 1, 1 + d)
    x = wide[:, 1:1 + heads, 1:1 + d]
    want, off = ref.turn(x, positions, ref.steps(rot), layout)
    check(mf.rope(view, r, positions=dp).numpy(), want, off, "wide rows")
    turned = mf.DeviceArray.empty((heads, rows, d), stream)
    mf.rope(view, r, positions=dp, out=turned.transpose(0, 1))
    check(turned.numpy().transpose(1, 0, 2), want, off, "heads first")
    mf.rope(view, r, positions=dp, out=view)
    after = dw.numpy()
    check(after[:, 1:1 + heads, 1:1 + d], want, off, "in place")
    after[:, 1:1 + heads, 1:1 + d] = x
    assert same_bits(after, wide), "columns around the heads were written"
    one = dev(x[:1], stream).expand((rows, heads, d))
    want, off = ref.turn(np.broadcast_to(x[:1], x.shape), positions, ref.steps(rot), layout)
    check(mf.rope(one, r, positions=dp).numpy(), want, off, "one row for all")


def test_gradient_against_differences(stream):
    """The backward pass is the transposed map: sum(g * turn(x)) changes with x[j] by backward(g)[j]."""
    rng = np.random.default_rng(6)
    r = mf.rotary(12, layout=mf.ROTARY_PAIRS, amplitude=1.5, factor=2.0)
    x = rng.standard_normal((3, 2, 16)).astype(np.float32)
    g = rng.standard_normal(x.shape).astype(np.float32)
    p = dev(np.array([5, 0, 60000], np.int32), stream)
    grad = mf.rope(dev(g, stream), r, positions=p, backward=True).numpy()

    def loss(y):
        return float(np.sum(mf.rope(dev(y, stream), r, positions=p).numpy().astype(np.float64) * g))

    for _ in range(24):
        at = tuple(rng.integers(0, n) for n in x.shape)
        hi, lo = x.copy(), x.copy()
        hi[at] += 0.5
        lo[at] -= 0.5
        step = float(hi[at]) - float(lo[at])
        # Linear: the difference is exact but for the outputs' rounding, each 3e-7 of at most 1.5 |x| |g|.
        off = 3e-7 * 1.5 * 2 * 2 * (np.abs(hi).max() + 0.5) * np.abs(g).sum() / step
        assert abs((loss(hi) - loss(lo)) / step - grad[at]) <= off


def test_empty(stream):
    r = mf.rotary(8)
    for shape in ((0, 3, 16), (4, 0, 16)):
        out = mf.rope(mf.DeviceArray.empty(shape, stream), r)
        assert out.shape == shape


def test_offsets_past_32_bits(stream):
    """Rows 2^24 + 4 floats apart: 140 of them pass 2^31 elements."""
    rng = np.random.default_rng(7)
    rows, pitch, heads, d = 140, (1 << 24) + 4, 3, 64
    x = rng.standard_normal((rows, heads, d)).astype(np.float32)
    far = mf.DeviceArray.empty((rows, pitch), stream)
    view = far._view((rows, heads, d), (pitch, d, 1), 0)
    near = dev(x, stream)
    for i in range(rows):
        mf.abi.check(mf.abi.load().mfr_memcpy_d2d(stream.handle, far.ptr + 4 * i * pitch,
                                                  near.ptr + 4 * i * heads * d, 4 * heads * d))
    want, off = ref.turn(x, np.arange(rows), ref.steps(64), mf.ROTARY_HALVES)
    mf.rope(view, mf.rotary(64), out=view)
    check(view.numpy(), want, off, "far rows")
    far.close()


def test_many_rows(stream):
    """More tokens than a launch has workgroups."""
    rng = np.random.default_rng(8)
    rows = (1 << 20) + 77
    x = rng.standard_normal((rows, 1, 8)).astype(np.float32)
    want, off = ref.turn(x, np.arange(rows), ref.steps(8), mf.ROTARY_PAIRS)
    check(mf.rope(dev(x, stream), mf.rotary(8, layout=mf.ROTARY_PAIRS)).numpy(), want, off, "many")


def test_many_heads(stream):
    """So many heads of a token that few tokens are taken at once."""
    rng = np.random.default_rng(9)
    x = rng.standard_normal((40, 1 << 18, 8)).astype(np.float32)
    got = mf.rope(dev(x, stream), mf.rotary(8), first=5).numpy()
    for h in (0, 1, 70000, (1 << 18) - 1):
        want, off = ref.turn(x[:, h:h + 1], np.arange(40) + 5, ref.steps(8), mf.ROTARY_HALVES)
        check(got[:, h:h + 1], want, off, h)
    one = rng.standard_normal((300, 1, 8)).astype(np.float32)
    wide = dev(one, stream).expand((300, 1 << 17, 8))
    got = mf.rope(wide, mf.rotary(8)).numpy()
    want, off = ref.turn(one, np.arange(300), ref.steps(8), mf.ROTARY_HALVES)
    check(got, np.broadcast_to(want, got.shape), np.broadcast_to(off, got.shape), "one for all")
