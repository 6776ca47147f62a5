"""mfr_kv_append on the device: every number of the cache and of the queries against the definition,
and nothing else written."""
import numpy as np
import pytest

import f8_reference as f8
import kv_reference as ref
import mensurflow_amd as mf
from helpers import same_bits
from kv_reference import Paged, dev

pytestmark = pytest.mark.gpu


def check_append(p, rot, layout, rng, q_heads=0, positions=None, in_place=False, **rotary):
    """Appends new rows to a copy of p's cache and compares all of it."""
    heads, d = p.heads, p.d
    k, v = (rng.standard_normal((p.rows, heads, d)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((p.rows, max(q_heads, 1), d)).astype(np.float32)
    before = [x.copy() for x in (p.k, p.v)]
    cache, batch = p.cache(), p.batch()
    q_out = None
    if q_heads:
        dq = dev(q, p.stream)
        q_out = dq if in_place else dev(np.full(q.shape, 7.0, np.float32), p.stream)
    mf.kv_append(cache, batch, dev(k, p.stream), dev(v, p.stream),
                 rotary=mf.rotary(rot, layout=layout, **rotary) if rot else None,
                 q=dq if q_heads else None, q_out=q_out,
                 positions=None if positions is None else dev(positions, p.stream))
    got_k, got_v = cache.k.numpy(), cache.v.numpy()
    scales = [None if s is None else s.numpy() for s in (cache.k_scales, cache.v_scales)]
    step = ref.steps(rot)
    places = np.zeros(p.rows, np.int64)
    real = np.zeros(p.rows, bool)
    written = np.zeros((p.pages, p.page), bool)
    for s, (n, tokens) in enumerate(p.counts):
        for i in range(n):
            row, place = p.starts[s] + i, int(p.lengths[s]) - n + i
            places[row], real[row] = p.prefix + place, True
            if not 0 <= place < p.width * p.page:
                continue
            page = p.table[s, place // p.page]
            if not 0 <= page < p.pages:
                continue
            at = page, slice(None), place % p.page
            written[page, place % p.page] = True
            position = [p.prefix + place if positions is None else positions[row]]
            wk, off_k = ref.turn(k[row][None], position, step, layout)
            for numbers, sc, want, off in ((got_k, scales[0], wk[0], off_k[0]),
                                           (got_v, scales[1], v[row], 0.0)):
                if p.held == "e4m3":
                    top = np.abs(want).max(-1)
                    scale = np.maximum(top / 448, 2.0 ** -126)
                    assert np.all(np.abs(sc[at] - scale) <= 4 * ref.EPS32 * scale + np.max(off) / 448)
                    if not np.any(off):
                        codes, exact = f8.quantize(np.asarray(want, np.float32))
                        assert np.array_equal(numbers[at] & 0x7F, codes & 0x7F)
                        assert np.array_equal(sc[at], exact[:, 0])
                    there = ref.held_to_rows(numbers[at], sc[at])
                    # Half a step of 8 bits, and the scale's own error.
                    assert np.all(np.abs(there - want) <= (2.0 ** -4 + 2.0 ** -20) * np.abs(want) +
                                  2.0 ** -10 * scale[:, None] + 2 * off)
                elif p.held == "bf16":
                    there = ref.bf16_values(numbers[at])
                    assert np.all(np.abs(there - want) <= 2.0 ** -8 * np.abs(want) + 2 * off)
                    if not np.any(off):
                        assert np.array_equal(numbers[at], ref.bf16_bits(want))
                else:
                    assert np.all(np.abs(numbers[at] - want) <= off)
    for got, was in ((got_k, before[0]), (got_v, before[1])):
        rest = np.broadcast_to(~written[:, None, :, None], got.shape)
        assert same_bits(got[rest], was[rest]), "places of no row were written"
    if q_heads:
        got = q_out.numpy()
        want, off = ref.turn(q, places if positions is None else positions, step, layout)
        assert np.all(np.abs(got - want)[real] <= off[real])
        assert same_bits(got[~real], q[~real] if in_place else np.full_like(got[~real], 7.0))


HELD = ["f32", "bf16", "e4m3"]


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("counts,heads,d,rot,q_heads", [
    ([(1, 1)], 1, 16, 16, 1), ([(1, 40)] * 5, 8, 128, 128, 32),
    ([(3, 3), (0, 9), (17, 40), (1, 17), (0, 0), (33, 33)], 3, 80, 48, 6),
    ([(70, 75)], 5, 112, 0, 0), ([(5, 64), (40, 64)], 2, 64, 22, 3), ([(2, 31)] * 9, 9, 96, 96, 0)])
@pytest.mark.parametrize("layout", [mf.ROTARY_HALVES, mf.ROTARY_PAIRS])
def test_appends(stream, held, counts, heads, d, rot, q_heads, layout):
    rng = np.random.default_rng(heads * d + rot)
    print(f"append {counts} {heads}x{d} {held} rot {rot}", flush=True)
    p = Paged(rng, stream, counts, heads, d, held, front=2, behind=3)
    check_append(p, rot, layout, rng, q_heads)


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("cache_layout", ["heads", "tokens", "apart"])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_layouts_and_pages(stream, held, cache_layout, page):
    rng = np.random.default_rng(page)
    p = Paged(rng, stream, [(4, 20), (30, 200), (1, page), (1, page + 1)], 3, 48, held, page=page,
              layout=cache_layout, prefix=21)
    check_append(p, 32, mf.ROTARY_HALVES, rng, q_heads=3, in_place=True)


@pytest.mark.parametrize("held", HELD)
def test_rows_each(stream, held):
    rng = np.random.default_rng(1)
    check_append(Paged(rng, stream, [(3, 10), (3, 3), (3, 50)], 2, 64, held, even=True), 64,
                 mf.ROTARY_HALVES, rng, q_heads=4)


@pytest.mark.parametrize("held", HELD)
def test_places_and_pages_that_there_are_not(stream, held):
    """Fewer tokens than rows, tokens past the table, and pages out of range: nothing is written for
    those rows, and the others are."""
    rng = np.random.default_rng(2)
    p = Paged(rng, stream, [(5, 3), (40, 40), (4, 64), (2, 30)], 2, 32, held, width=4)
    p.lengths = np.array([3, 40, 66, 30], np.int32)     # of 66, two past the table
    p.table[1, 1], p.table[3, 1] = -7, p.pages
    check_append(p, 32, mf.ROTARY_PAIRS, rng, q_heads=2)


def test_positions_of_their_own(stream):
    rng = np.random.default_rng(3)
    p = Paged(rng, stream, [(5, 30), (6, 6)], 2, 64, "f32")
    check_append(p, 64, mf.ROTARY_HALVES, rng, 2,
                 positions=rng.integers(0, 100000, p.rows).astype(np.int32))


@pytest.mark.parametrize("held", HELD)
def test_odd_numbers(stream, held):
    """Zeros, the least and the largest numbers, infinities and NaN, without a rotation."""
    rng = np.random.default_rng(4)
    p = Paged(rng, stream, [(6, 6)], 1, 16, held)
    x = rng.standard_normal((6, 1, 16)).astype(np.float32)
    x[0], x[1, 0, :3] = 0, (1e-42, -1e-40, 3e-39)
    x[1, 0, 3:] = 0
    x[2, 0, :2] = (np.float32(3.4e38), -3.4e38)
    x[3, 0, 5], x[4, 0, 6], x[5, 0, 7] = np.nan, np.inf, -np.inf
    cache, batch = p.cache(), p.batch()
    mf.kv_append(cache, batch, dev(x, stream), dev(-x, stream))
    page = p.table[0, 0]
    got = cache.k.numpy()[page, 0, :6]
    if held == "f32":
        assert same_bits(got, x[:, 0])
    elif held == "bf16":
        want = ref.bf16_values(ref.bf16_bits(x[:, 0]))
        with np.errstate(invalid="ignore"):
            assert np.array_equal(ref.bf16_values(got), want, equal_nan=True)
    else:
        codes, scales = f8.quantize(x[:, 0])
        nan = codes & 0x7F == 0x7F
        assert np.array_equal(got[~nan] & 0x7F, codes[~nan] & 0x7F)
        assert np.all(got[nan] & 0x7F == 0x7F)
        assert np.array_equal(cache.k_scales.numpy()[page, 0, :6], scales[:, 0], equal_nan=True)


def test_many_rows_and_far_pages(stream):
    """A long prompt over many sequences, a cache past 2^31 elements whose last pages are used."""
    rng = np.random.default_rng(5)
    heads, d, page, pages = 8, 128, 64, 40000              # 2.6e9 elements of each of k and v
    cache = mf.KvCache.empty(pages, page, heads, d, stream, np.uint8)
    counts = [(300, 300), (1, 64), (500, 512)]
    rows = sum(n for n, _ in counts)
    table = rng.choice(np.arange(pages - 64, pages), 24, False).astype(np.int32).reshape(3, 8)
    starts = np.concatenate(([0], np.cumsum([n for n, _ in counts]))).astype(np.int32)
    batch = mf.KvBatch(dev(np.array([t for _, t in counts], np.int32), stream), dev(table, stream),
                       starts=dev(starts, stream))
    k, v = (rng.standard_normal((rows, heads, d)).astype(np.float32) for _ in range(2))
    mf.kv_append(cache, batch, dev(k, stream), dev(v, stream))
    for s, (n, tokens) in enumerate(counts):
        for i in (0, n // 2, n - 1):
            place = tokens - n + i
            at = int(table[s, place // page])
            got = cache.v.slice(0, at, at + 1).numpy()
            codes, _ = f8.quantize(v[starts[s] + i])
            assert np.array_equal(got[0, :, place % page] & 0x7F, codes & 0x7F)
    cache.k.close()
    cache.v.close()
