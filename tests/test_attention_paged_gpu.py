"""mfr_attention_paged on the device against the formula in 64 bits. Unused parts of the caches hold
NaN, unused entries of the tables name pages that there are not (kv_reference.Paged)."""
import numpy as np
import pytest

import kv_reference as ref
import mensurflow_amd as mf
from helpers import same_bits
from kv_reference import Paged, dev

pytestmark = pytest.mark.gpu
HELD = ["f32", "bf16", "e4m3"]


def run(p, q, out=None, **kw):
    out = dev(np.full(q.shape, 7.0, np.float32), p.stream) if out is None else out
    mf.attention_paged(dev(q, p.stream), p.cache(), p.batch(), out=out, **kw)
    return out.numpy()


def check(p, q, got, norm=True, **kw):
    want, bound = p.attend(q, **kw)
    there = ~np.isnan(want)
    assert np.all(got[~there] == 7.0), "rows of no sequence were written"
    off = np.abs(got.astype(np.float64) - want)[there]
    bad = ~(off <= bound[there])
    assert not bad.any(), (int(bad.sum()), np.argwhere(there)[bad][:4], got[there][bad][:4],
                           want[there][bad][:4])
    if norm and there.any() and np.any(want[there]):
        # Roundings that add up like a random walk: a score's d products, a sum's tokens in steps of 32.
        tokens = max([t for _, t in p.counts]) + p.prefix
        error = ref.attention_error(got, want)
        limit = ref.EPS32 * (2 * np.sqrt(p.d) + 2 * np.sqrt(tokens / 32) + 8)
        print(f"error {error:.2e} of {limit:.2e}", flush=True)
        assert error <= limit


def case(rng, stream, counts, heads, group, d, held, **kw):
    print(f"attend {counts if len(counts) < 8 else len(counts)} {heads}x{group}x{d} {held} {kw}",
          flush=True)
    p = Paged(rng, stream, counts, heads, d, held, **kw)
    return p, rng.standard_normal((p.rows, heads * group, d)).astype(np.float32)


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("tokens", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 1000])
def test_one_query(stream, held, tokens):
    rng = np.random.default_rng(tokens)
    p, q = case(rng, stream, [(1, tokens)], 2, 4, 128, held)
    check(p, q, run(p, q))


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("group", [1, 3, 8])
def test_depths_and_groups(stream, held, d, group):
    rng = np.random.default_rng(d + group)
    p, q = case(rng, stream, [(1, 70), (2, 33), (1, 1)], 3, group, d, held, front=1, behind=2)
    check(p, q, run(p, q))


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("counts", [
    [(5, 5), (1, 200), (0, 0), (7, 100), (1, 0), (3, 1), (16, 17)],
    [(40, 40), (33, 130), (1, 1)], [(130, 200), (17, 64), (64, 64)], [(2, 90)] * 20,
    [(0, 0), (0, 5)], [(300, 300)]])
@pytest.mark.parametrize("causal", [True, False])
def test_ragged(stream, held, counts, causal):
    rng = np.random.default_rng(len(counts))
    p, q = case(rng, stream, counts, 2, 4, 64, held, front=3, behind=2)
    check(p, q, run(p, q, causal=causal), causal=causal)


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("prefix", [1, 16, 31, 100, 700])
@pytest.mark.parametrize("counts", [[(1, 50), (1, 1), (1, 0), (1, 333)], [(9, 9), (0, 3), (20, 70)],
                                    [(1, 20)] * 40])
def test_shared_prefix(stream, held, prefix, counts):
    rng = np.random.default_rng(prefix)
    p, q = case(rng, stream, counts, 2, 4, 128, held, prefix=prefix, behind=1)
    check(p, q, run(p, q))


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("cache_layout", ["heads", "tokens", "apart"])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_layouts_and_pages(stream, held, cache_layout, page):
    rng = np.random.default_rng(page)
    p, q = case(rng, stream, [(1, 20), (3, 300), (2, page), (1, page + 1)], 3, 2, 80, held, page=page,
                layout=cache_layout, prefix=37)
    check(p, q, run(p, q))


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("each", [1, 4])
def test_rows_each(stream, held, each):
    rng = np.random.default_rng(each)
    p, q = case(rng, stream, [(each, 10 + 50 * i) for i in range(6)], 2, 2, 64, held, even=True)
    check(p, q, run(p, q))


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("scale", [1.0, 0.01, 3.0, -0.5])
def test_scales(stream, held, scale):
    rng = np.random.default_rng(3)
    p, q = case(rng, stream, [(1, 300), (6, 50)], 2, 2, 32, held)
    check(p, q, run(p, q, scale=scale), norm=False, scale=scale)


@pytest.mark.parametrize("held", HELD)
def test_strides(stream, held):
    """Queries and outputs inside wider rows, heads in front of rows, one query for all rows."""
    rng = np.random.default_rng(4)
    p = Paged(rng, stream, [(1, 100), (5, 40)], 2, 64, held)
    wide = rng.standard_normal((p.rows, 10, 70)).astype(np.float32)
    q = wide[:, 1:9, 3:67]
    dq = dev(wide, stream).slice(1, 1, 9).slice(2, 3, 67)
    out = dev(np.full((8, p.rows, 65), 7.0, np.float32), stream)
    mf.attention_paged(dq, p.cache(), p.batch(), out=out.slice(2, 1, 65).transpose(0, 1))
    got = out.numpy()
    assert np.all(got[..., 0] == 7.0)
    check(p, q, got[..., 1:].transpose(1, 0, 2))
    one = dev(q[:1], stream).expand(q.shape)
    got = mf.attention_paged(one, p.cache(), p.batch()).numpy()
    check(p, np.broadcast_to(q[:1], q.shape), got)


@pytest.mark.parametrize("held", HELD)
def test_bad_pages_count_as_absent(stream, held):
    rng = np.random.default_rng(5)
    p, q = case(rng, stream, [(1, 100), (4, 64)], 2, 2, 64, held, prefix=40)
    absent = [(0, t) for t in range(32, 48)] + [(1, t) for t in range(16)]
    keep = p.table.copy()
    want, bound = p.attend(q, absent=absent)
    p.table[0, 2], p.table[1, 0] = -1, p.pages
    got = run(p, q)
    p.table = keep
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("held", HELD)
def test_lengths_out_of_range(stream, held):
    """A length below 0 is none, one past the table is the table's."""
    rng = np.random.default_rng(6)
    p, q = case(rng, stream, [(1, 0), (1, 64), (3, 0)], 2, 2, 32, held, width=4)
    want, bound = p.attend(q)
    p.lengths = np.array([-5, 64, np.iinfo(np.int32).min], np.int32)
    assert np.all(np.abs(run(p, q) - want) <= bound)
    p.lengths[1] = 1000
    assert np.all(np.abs(run(p, q) - want) <= bound)


@pytest.mark.parametrize("held", HELD)
def test_large_and_small_scores(stream, held):
    """One token outweighs all; scores far below the first; equal scores."""
    rng = np.random.default_rng(7)
    p, q = case(rng, stream, [(1, 500), (2, 70)], 1, 4, 64, held)
    q[0] *= 40
    q[1] = 0
    q[2] *= 1e-6
    check(p, q, run(p, q), norm=False)


@pytest.mark.parametrize("held", HELD)
def test_nan_where_it_is_not_seen(stream, held):
    """Tokens behind a row's place hold NaN and infinities: the rows before are as without."""
    rng = np.random.default_rng(8)
    p, q = case(rng, stream, [(20, 60), (40, 40)], 2, 3, 64, held)
    want, bound = p.attend(q)
    for s, n in ((0, 60), (1, 40)):
        place = n - 7                              # seen by the last 7 rows alone
        at = p.table[s, place // 16], slice(None), place % 16
        for numbers, scales in ((p.k, p.ks), (p.v, p.vs)):
            if held == "e4m3":
                scales[at] = np.inf
                numbers[at][..., 3] = 0x7F
            else:
                bits = np.float32([np.inf, -np.inf, np.nan])
                numbers[at][..., 1:4] = bits if held == "f32" else ref.bf16_bits(bits)
    got = run(p, q)
    sees = np.zeros(p.rows, bool)
    for s in (0, 1):
        sees[p.starts[s + 1] - 7:p.starts[s + 1]] = True
    assert np.all(np.abs(got - want)[~sees] <= bound[~sees])
    assert not np.isfinite(got[sees]).all(axis=-1).any()


@pytest.mark.parametrize("held", HELD)
def test_nan_queries_stay_in_their_rows(stream, held):
    rng = np.random.default_rng(9)
    p, q = case(rng, stream, [(5, 60), (1, 10)], 2, 2, 64, held, prefix=20)
    want, bound = p.attend(q)
    q[2, 1, 5], q[4, 3, 0] = np.nan, np.inf
    got = run(p, q)
    bad = np.zeros(q.shape[:2], bool)
    bad[2, 1] = bad[4, 3] = True
    assert np.all(np.abs(got - want)[~bad] <= bound[~bad])
    assert not np.isfinite(got[bad]).all(axis=-1).any()


@pytest.mark.parametrize("held", HELD)
def test_the_same_call_gives_the_same_bits(stream, held):
    rng = np.random.default_rng(10)
    p, q = case(rng, stream, [(1, 2000), (3, 900), (1, 17)] * 5, 4, 4, 128, held, prefix=500)
    first = run(p, q)
    check(p, q, first)
    assert same_bits(run(p, q), first)


@pytest.mark.parametrize("held", HELD)
def test_a_decoding_loop(stream, held):
    """Append with the rotation, then attend, step by step: a prompt, then single tokens, against
    attention over the turned rows of the whole sequence."""
    rng = np.random.default_rng(11)
    heads, group, d, page, seqs = 2, 3, 64, 16, 3
    rot = mf.rotary(d)
    cache = mf.KvCache.empty(24, page, heads, d, stream, ref.HELD[held])
    p = Paged(rng, stream, [(0, 0)] * seqs, heads, d, held, width=8, spare=24)
    p.table = rng.permutation(24).astype(np.int32).reshape(seqs, 8)
    lengths = np.zeros(seqs, np.int32)
    for new in ([5, 40, 1], [1, 1, 1], [1, 1, 1], [3, 0, 20], [1, 1, 1]):
        new = np.array(new)
        lengths = (lengths + new).astype(np.int32)
        p.lengths, p.counts = lengths, list(zip(new.tolist(), lengths.tolist()))
        p.starts = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
        p.rows = int(new.sum())
        k, v = (rng.standard_normal((p.rows, heads, d)).astype(np.float32) for _ in range(2))
        q = rng.standard_normal((p.rows, heads * group, d)).astype(np.float32)
        batch = p.batch()
        dq = mf.kv_append(cache, batch, dev(k, stream), dev(v, stream), rotary=rot, q=dev(q, stream))
        got = mf.attention_paged(dq, cache, batch).numpy()
        # What the cache now holds was checked by the tests of kv_append.
        p.k, p.v = cache.k.numpy(), cache.v.numpy()
        if held == "e4m3":
            p.ks, p.vs = cache.k_scales.numpy(), cache.v_scales.numpy()
        check(p, dq.numpy(), got)
