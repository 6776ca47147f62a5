"""mfr_attention_paged where numbers are near the ends of fp32's range but the results are not, in the forms
for few rows and for many."""
import numpy as np
import pytest

from test_attention_paged_gpu import case, check, run

pytestmark = pytest.mark.gpu
MANY = [(150, 200), (40, 64), (1, 300)]     # rows enough for tiles of many
FEW = [(1, 300), (3, 40)]


@pytest.mark.parametrize("counts,power", [(MANY, 90), (MANY, 98), (MANY, 110), (MANY, 120), (FEW, 90), (FEW, 100)])
@pytest.mark.parametrize("d", [64, 128])
def test_large_keys_under_small_queries(stream, counts, power, d):
    """Scales of keys up to 2^120 under queries as small: ordinary scores."""
    rng = np.random.default_rng(power)
    p, q = case(rng, stream, counts, 2, 2, d, "e4m3", prefix=40)
    p.ks *= np.float32(2.0 ** power)
    q *= np.float32(2.0 ** -power)
    check(p, q, run(p, q), norm=False)


@pytest.mark.parametrize("counts,power", [(MANY, 60), (MANY, 84), (FEW, 60), (FEW, 84)])
def test_small_keys_under_large_queries(stream, counts, power):
    rng = np.random.default_rng(power)
    p, q = case(rng, stream, counts, 2, 2, 128, "e4m3", prefix=40)
    p.ks *= np.float32(2.0 ** -power)
    q *= np.float32(2.0 ** power)
    check(p, q, run(p, q), norm=False)
