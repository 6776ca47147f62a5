"""mfr_attention_paged where numbers are near the ends of fp32's range but the results are not, in the forms
for few rows and for many."""
import numpy as np
import pytest

import f8_reference as f8
import kv_reference as ref
from kv_reference import Paged
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


@pytest.mark.parametrize("d", [64, 128])
def test_queries_keep_their_bits(stream, d):
    """Two tokens, each of one column: the weights say what the queries of many rows in 8 bits were taken as."""
    rng = np.random.default_rng(d)
    p = Paged(rng, stream, [(220, 2)] * 3, 2, d, "e4m3")
    one = f8.VALUES.tolist().index(1.0)
    for s in range(3):
        for token in range(2):
            at = p.table[s, 0], slice(None), token
            p.k[at], p.v[at] = 0, 0
            p.k[at][:, token], p.v[at][:, token] = one, one
            p.ks[at], p.vs[at] = 1, 1
    size = 2000.0                       # of the scores
    q = np.zeros((p.rows, 4, d), np.float32)
    q[..., 0] = size * (1 + rng.random(q.shape[:2]))
    q[..., 1] = np.float32(q[..., 0].astype(np.float16))    # as it is in one part
    got = run(p, q, scale=1.0, causal=False)
    want, _ = p.attend(q, scale=1.0, causal=False)
    # A last place of the number (2^-23 of up to 2 size), the difference's rounding, and those behind it.
    off = 0.25 * (2.0 ** -23 + 2.0 ** -24) * 2 * size + 2.0 ** -21
    error = got[..., 0].astype(np.float64) - want[..., 0]
    assert np.abs(error).max() <= off
    # Of either sign.
    assert abs(error.mean()) <= off / 8


def test_weights_keep_their_bits(stream):
    """Rows that see one token give its value: off by the weight's parts, a product and a division."""
    rng = np.random.default_rng(3)
    p = Paged(rng, stream, [(110, 1)] * 40, 2, 64, "e4m3")
    q = rng.standard_normal((p.rows, 4, 64)).astype(np.float32)
    got = run(p, q, causal=False)
    want, _ = p.attend(q, causal=False)
    assert np.all(np.abs(got - want) <= (2.0 ** -23 + 4 * 2.0 ** -24) * np.abs(want))
    # Each of 17600 weights off by up to a last place, of either sign; parts cut towards zero are 2e-8 below.
    there = want != 0
    assert abs(np.mean(got[there] / want[there] - 1)) <= 2.0 ** -24 / 6


@pytest.mark.parametrize("held", ["f32", "bf16", "e4m3"])
@pytest.mark.parametrize("counts", [MANY, FEW])
@pytest.mark.parametrize("power", [16, 20, 24, 26, 28, 30, 32, 36, 60, 100])
@pytest.mark.parametrize("small", [1.0, 2.0 ** -90])
def test_far_scores(stream, held, counts, power, small):
    """Scores far from 0: rows whose largest one is apart from the next give its value."""
    if small != 1.0 and held != "e4m3":
        pytest.skip("no scales")
    rng = np.random.default_rng(power)
    p, q = case(rng, stream, counts, 2, 2, 64, held, prefix=40)
    q *= np.float32(2.0 ** power)
    if held == "e4m3":
        p.vs *= np.float32(small) ** rng.integers(0, 2, p.vs.shape).astype(np.float32)
    got = run(p, q)
    looked = wrong = 0
    for s, (n, tokens) in enumerate(p.counts):
        k, v = p.tokens_of(s)
        for i in range(n):
            row, seen = p.starts[s] + i, p.prefix + max(0, min(tokens, tokens - n + i + 1))
            for h in range(q.shape[1]):
                kk, x = k[:seen, h // 2], q[row, h].astype(np.float64)
                score = kk @ x / 8
                # What fp32 may be off by (kv_reference.Paged.attend), for each of two scores.
                off = 4 * ref.EPS32 * (72 * (np.abs(kk) @ np.abs(x)).max() / 8 + 4)
                second, first = np.sort(score)[-2:]
                if first - second > off + 90:       # and 2^-126 of another one's values
                    want = v[score.argmax(), h // 2]
                    wrong += not np.all(np.abs(got[row, h] - want) <= 2.0 ** -21 * np.abs(want) + 1e-37)
                    looked += 1
    assert looked > 0.5 * p.rows * q.shape[1] and wrong == 0, (looked, wrong)


@pytest.mark.parametrize("held", ["f32", "bf16", "e4m3"])
@pytest.mark.parametrize("counts", [[(110, 300)], [(1, 300)], [(20, 300)]])
@pytest.mark.parametrize("rise", [0.0, 3.0, 7.5, 20.0])
def test_large_values_under_rising_scores(stream, held, counts, rise):
    """Values near 2^119 of 300 tokens, the later two thirds with 2^rise times the weight of the first."""
    p = Paged(np.random.default_rng(5), stream, counts, 1, 64, held)
    rng = np.random.default_rng(6)
    k = np.zeros((300, 1, 64))
    k[100:, 0, 0] = rise
    v = 2.0 ** 119 * rng.uniform(0.5, 1.0, (300, 1, 64))
    for numbers, scales, x in ((p.k, p.ks, k), (p.v, p.vs, v)):
        p.fill(numbers, scales, x, p.table[0], 300)
    q = np.zeros((p.rows, 2, 64), np.float32)
    q[..., 0] = 8 * np.log(2)           # scale 1 / 8
    got = run(p, q, causal=False)
    want, bound = p.attend(q, causal=False)
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("held", ["f32", "bf16", "e4m3"])
@pytest.mark.parametrize("rows", [1, 30])
def test_large_values_under_rising_scores_in_several_steps(stream, held, rows):
    """The same with so many tokens that each workgroup of a card of 256 compute units takes several steps."""
    sequences, tokens, heads = 64, 3200, 4
    p = Paged(np.random.default_rng(7), stream, [(rows, 1)] * sequences, heads, 64, held, page=64)
    pages = tokens // 64
    rng = np.random.default_rng(8)
    k = np.zeros((pages, heads, 64, 64))
    k[..., 0] = np.arange(tokens).reshape(pages, 1, 64) % 256 / 256 * 7.5
    v = 2.0 ** 118 * rng.uniform(0.5, 1.0, (pages, heads, 64, 64))
    (p.k, p.ks), (p.v, p.vs) = (ref.rows_to_held(x, held) for x in (k, v))
    p.pages, p.width = pages, pages
    p.table = np.tile(np.arange(pages, dtype=np.int32), (sequences, 1))
    p.lengths[:] = tokens
    q = np.zeros((p.rows, heads, 64), np.float32)
    q[..., 0] = 8 * np.log(2)
    got = run(p, q, causal=False)
    p.counts = [(rows, tokens)]             # every sequence and row is the same
    want, bound = p.attend(q[:rows], causal=False)
    got = got.reshape(sequences, rows, heads, 64)
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("counts", [[(150, 200), (40, 64), (110, 600)], FEW])
@pytest.mark.parametrize("large", [2.0 ** 10, 2.0 ** 40, 2.0 ** 100])
@pytest.mark.parametrize("zeros", ["front", "behind", "prefix", "own", "all", "mixed"])
@pytest.mark.parametrize("scale", [0.0, 2.0 ** -126])
def test_zeros_beside_large_values(stream, counts, large, zeros, scale):
    """Tokens whose values are zeros under the least scale take their weight from others of large values."""
    rng = np.random.default_rng(11)
    p, q = case(rng, stream, counts, 2, 2, 64, "e4m3", prefix=140)

    def empty(pages, tokens):
        for t in tokens:
            at = pages[t // 16], slice(None), t % 16
            p.v[at], p.vs[at] = 0, scale

    p.vs[np.isfinite(p.vs)] = large
    for s, (_, tokens) in enumerate(counts):
        if zeros != "prefix":
            empty(p.table[s], {"front": range(tokens // 2), "behind": range(tokens // 2, tokens),
                               "mixed": range(0, tokens, 3)}.get(zeros, range(tokens)))
    if zeros in ("prefix", "all", "mixed"):
        empty(p.prefix_pages, range(0, 140, 2 if zeros == "mixed" else 1))
    check(p, q, run(p, q), norm=False)


@pytest.mark.parametrize("power", [-126, -118, -110, -100, -97, -95])
@pytest.mark.parametrize("counts", [MANY, [(64, 900), (64, 700)]])
def test_small_values_of_many_rows(stream, counts, power):
    """Values under scales as small as there are, and zeros among them, keep their bits."""
    rng = np.random.default_rng(-power)
    p, q = case(rng, stream, counts, 2, 2, 64, "e4m3", prefix=40)
    seen = np.isfinite(p.vs)
    p.vs[seen] = np.float32(2.0 ** power) * rng.choice(np.float32([1, 1.25, 1.9]), p.vs[seen].shape)
    p.v[np.logical_and(seen, rng.random(seen.shape) < 0.2)] = 0
    got = run(p, q)
    want, bound = p.attend(q)
    there = ~np.isnan(want)
    # In place of what `bound` allows for numbers next to fp32's least: sums of up to 940 of those.
    off = bound - 1e-37 + 1000 * 448 * 2.0 ** -149
    assert np.all(np.abs(got - want)[there] <= off[there])
    assert np.count_nonzero(got[there]) > 0.9 * np.count_nonzero(want[there])


@pytest.mark.parametrize("power", [-112, -108, -104, -100])
def test_small_values_of_few_rows(stream, power):
    """Of a weight times its value's scale, what lies below 2^-126 is lost, and no more."""
    rng = np.random.default_rng(-power)
    p, q = case(rng, stream, FEW, 2, 2, 64, "e4m3")
    p.vs[np.isfinite(p.vs)] = np.float32(2.0 ** power)
    got = run(p, q)
    want, bound = p.attend(q)
    for s, (n, tokens) in enumerate(p.counts):
        k, v = p.tokens_of(s)
        for i in range(n):
            row, seen = p.starts[s] + i, tokens - n + i + 1
            for h in range(q.shape[1]):
                score = k[:seen, h // 2] @ q[row, h].astype(np.float64) / 8
                weight = np.exp(score - score.max())
                # Weights against the largest's 2^-7 at least.
                lost = np.minimum(weight / weight.sum() * 2.0 ** power, 2.0 ** -126 / (weight.sum() * 2.0 ** -7))
                off = bound[row, h] + lost @ np.abs(v[:seen, h // 2]) / 2.0 ** power
                assert np.all(np.abs(got[row, h] - want[row, h]) <= off)
                assert got[row, h].any()
