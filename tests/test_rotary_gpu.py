"""What a rotation multiplies by, and its roundings, on the device."""
import numpy as np
import pytest

import mensurflow_amd as mf
from kv_reference import dev, steps

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
