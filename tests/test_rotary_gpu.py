"""What a rotation multiplies by, and its roundings, on the device."""
import numpy as np
import pytest

import mensurflow_amd as mf
from helpers import same_bits
from kv_reference import Paged, dev, rows_to_held

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("amplitude", [1.0, -0.75, 1.2079441547393799])
@pytest.mark.parametrize("far", [100, 131072, 1 << 31])
def test_cosines_and_sines(stream, far, amplitude):
    """Columns (1, 0) turn to (cosine, sine): the nearest fp32 numbers, but for what double leaves of a far
    angle."""
    rng = np.random.default_rng(far)
    rot, rows = 128, 4000
    r = mf.rotary(rot, amplitude=amplitude)
    x = np.zeros((rows, 1, rot), np.float32)
    x[..., :rot // 2] = 1
    positions = rng.integers(-far, far, rows).astype(np.int32)
    got = mf.rope(dev(x, stream), r, positions=dev(positions, stream)).numpy()[:, 0]
    w = positions.astype(np.longdouble)[:, None] * np.array(r.steps[:rot // 2], np.longdouble)
    off = abs(r.amplitude) * (2.0 ** -25 + 1e-11 + 1.8e-16 * np.abs(w))
    if amplitude != 1.0:
        off = off + 2.0 ** -25      # numbers above 1 are twice as far apart
    assert np.all(np.abs(got[:, :rot // 2] - r.amplitude * np.cos(w)) <= off)
    assert np.all(np.abs(got[:, rot // 2:] - r.amplitude * np.sin(w)) <= off)


def formula(x, cos, sin, layout):
    """The rotation of x [rows, heads, d] in fp32, each product and sum rounded, by cos and sin [rows, pairs]."""
    half = cos.shape[1]
    first = slice(0, half) if layout == mf.ROTARY_HALVES else slice(0, 2 * half, 2)
    second = slice(half, 2 * half) if layout == mf.ROTARY_HALVES else slice(1, 2 * half, 2)
    out, a, b = x.copy(), x[..., first], x[..., second]
    cos, sin = cos[:, None], sin[:, None]
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    return out


def cosines_and_sines(stream, r, positions, backward=False):
    half = r.rot // 2
    x = np.zeros((len(positions), 1, r.rot), np.float32)
    x[..., :half] = 1
    unit = mf.rotary(r.rot)
    unit.steps, unit.amplitude = r.steps, r.amplitude
    got = mf.rope(dev(x, stream), unit, positions=dev(positions, stream), backward=backward).numpy()[:, 0]
    return got[:, :half], got[:, half:]


@pytest.mark.parametrize("layout", [mf.ROTARY_HALVES, mf.ROTARY_PAIRS])
@pytest.mark.parametrize("d,rot", [(128, 128), (80, 48), (96, 46)])
@pytest.mark.parametrize("backward", [False, True])
def test_roundings_of_the_formula(stream, layout, d, rot, backward):
    """Bit for bit the formula in fp32 with the device's own cosines and sines."""
    rng = np.random.default_rng(d)
    r = mf.rotary(rot, layout=layout, amplitude=1.25)
    x = rng.standard_normal((300, 5, d)).astype(np.float32)
    positions = rng.integers(0, 131072, 300).astype(np.int32)
    got = mf.rope(dev(x, stream), r, positions=dev(positions, stream), backward=backward).numpy()
    assert same_bits(got, formula(x, *cosines_and_sines(stream, r, positions, backward), layout))


@pytest.mark.parametrize("layout", [mf.ROTARY_HALVES, mf.ROTARY_PAIRS])
@pytest.mark.parametrize("d,rot", [(128, 128), (80, 48), (96, 46)])
@pytest.mark.parametrize("held", ["f32", "bf16", "e4m3"])
def test_roundings_of_what_a_cache_holds(stream, layout, d, rot, held):
    """Keys, queries and the codes of keys in 8 bits are those of the formula in fp32."""
    rng = np.random.default_rng(d)
    r = mf.rotary(rot, layout=layout)
    p = Paged(rng, stream, [(700, 700)], 4, d, held, page=64)
    k, v = (rng.standard_normal((p.rows, 4, d)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((p.rows, 8, d)).astype(np.float32)
    cache = p.cache()
    got_q = mf.kv_append(cache, p.batch(), dev(k, stream), dev(v, stream), rotary=r, q=dev(q, stream)).numpy()
    angles = cosines_and_sines(stream, r, np.arange(700, dtype=np.int32))
    assert same_bits(got_q, formula(q, *angles, layout))
    place = np.arange(700)
    at = p.table[0, place // 64], slice(None), place % 64
    for x, numbers, scales in ((formula(k, *angles, layout), cache.k, cache.k_scales),
                               (v, cache.v, cache.v_scales)):
        want, want_scales = rows_to_held(x, held)
        assert np.array_equal(numbers.numpy()[at], want)
        if scales is not None:
            assert np.array_equal(scales.numpy()[at], want_scales)
