"""mfr_attention_paged where every workgroup has much to do: several steps of tokens, items cut inside, several
items one after the other. What a workgroup gets is computed here as the library cuts it (csrc/kv_work.hpp,
attention_paged.hip), so that the sizes are known to reach it."""
import numpy as np
import pytest

import kv_reference as ref
import mensurflow_amd as mf
from test_attention_paged_gpu import case, run

pytestmark = pytest.mark.gpu


def cut(p, group, held, shared=False):
    """(rows of a tile, units of a workgroup, items, workgroups) of the launch over the prefix or the
    sequences' own tokens."""
    sequences = 1 if shared else len(p.counts)
    rows = p.rows * group
    many = held != "f32" and rows > 96 * sequences
    tile = 128 if many else 16 if rows <= 16 * sequences else 32
    unit = 64 if many or held == "f32" else 128
    depth = 64 if p.d <= 64 else 128
    each = 1 if many else (1 if held == "f32" and depth == 128 else 2) if tile == 32 else 3 if depth == 64 else 2
    groups = mf.device_info(0).compute_units * each
    tokens = p.prefix if shared else p.width * p.page
    most = max(1, -(-tokens // unit))
    items = (rows // tile + sequences) * p.heads
    groups = groups if items >= groups else min(groups, items * most)
    lists = [(p.rows, p.prefix)] if shared else p.counts
    items = sum(-(-n * group // tile) * p.heads for n, _ in lists)
    total = sum(-(-n * group // tile) * p.heads * max(1, -(-t // unit)) for n, t in lists)
    return tile, -(-total // groups), items, groups


def rising(p, rng, q, by):
    """Scores that rise by `by` along each sequence's tokens, beside what they are at random."""
    for s, (_, tokens) in enumerate(p.counts):
        x = rng.standard_normal((tokens, p.heads, p.d)) * p.size
        x[..., 0] = np.linspace(0, by, tokens)[:, None]
        p.fill(p.k, p.ks, x, p.table[s], tokens)
    q[..., 0] = np.sqrt(p.d)


def compare(p, q, got, **kw):
    want, bound = p.attend(q, **kw)
    there = ~np.isnan(want)
    assert np.all(got[~there] == 7.0), "rows of no sequence were written"
    bad = ~(np.abs(got - want) <= bound) & there
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])


@pytest.mark.parametrize("held", ["bf16", "e4m3"])
@pytest.mark.parametrize("d,rise", [(64, 0), (64, 40), (128, 40)])
def test_many_rows_on_many_tokens(stream, held, d, rise):
    """Tiles of 128 rows, several of 64 tokens a workgroup, items cut inside; pages that there are not in the
    middle, edges of what a row sees in middle tiles of items, tokens of NaN behind."""
    rng = np.random.default_rng(d + rise)
    p, q = case(rng, stream, [(70, 2100), (40, 40), (33, 3000)], 8, 4, d, held, front=1, behind=2)
    tile, chunk, items, groups = cut(p, 4, held)
    assert tile == 128 and chunk >= 4 and items < groups
    if rise:
        rising(p, rng, q, rise)
    gone = [(0, 3), (0, 20), (0, 21), (0, 22), (0, 23), (0, 130), (2, 0), (2, 77), (2, 186)]
    keep = p.table.copy()
    for i, (s, page) in enumerate(gone):
        p.table[s, page] = ref.BAD[i % len(ref.BAD)]
    got = run(p, q)
    p.table = keep
    compare(p, q, got, absent=[(s, t) for s, g in gone for t in range(16 * g, 16 * g + 16)])


@pytest.mark.parametrize("held", ["bf16", "e4m3"])
@pytest.mark.parametrize("causal", [True, False])
def test_many_short_items_of_many_rows(stream, held, causal):
    """Several items of tiles of 128 rows in a workgroup, one after the other, of one step and of more."""
    rng = np.random.default_rng(3)
    counts = [(25 + 3 * (i % 7), (1, 30, 64, 65, 200, 300, 129, 0)[i % 8] + 40 * (i % 3)) for i in range(48)]
    p, q = case(rng, stream, counts, 8, 4, 64, held, page=32)
    tile, chunk, items, groups = cut(p, 4, held)
    assert tile == 128 and chunk >= 4 and items >= 2 * groups
    compare(p, q, run(p, q, causal=causal), causal=causal)


@pytest.mark.parametrize("held", ["f32", "bf16", "e4m3"])
@pytest.mark.parametrize("d,rows,rise", [(64, 1, 0), (128, 1, 40), (64, 6, 40), (128, 6, 0)])
def test_few_rows_on_many_tokens(stream, held, d, rows, rise):
    """Tiles of 16 and 32 rows: several steps a wavefront, items cut inside and several of them, lengths of all
    sizes, pages that there are not, NaN behind."""
    rng = np.random.default_rng(d + rows + rise)
    counts = [(rows, 17 + (i * 389) % 1700) for i in range(64)]
    p, q = case(rng, stream, counts, 8, 4, d, held, page=64, front=1, behind=1)
    tile, chunk, _, _ = cut(p, 4, held)
    assert tile == (16 if rows == 1 else 32) and chunk >= 4
    if rise:
        rising(p, rng, q, rise)
    gone = [(5, 1), (6, 0), (7, 2), (7, 3), (40, 5)]
    gone = [(s, g) for s, g in gone if g < counts[s][1] // 64]
    keep = p.table.copy()
    for i, (s, page) in enumerate(gone):
        p.table[s, page] = ref.BAD[i % len(ref.BAD)]
    got = run(p, q)
    p.table = keep
    compare(p, q, got, absent=[(s, t) for s, g in gone for t in range(64 * g, 64 * g + 64)])


@pytest.mark.parametrize("held", ["bf16", "e4m3"])
@pytest.mark.parametrize("prefix", [300, 1000])
def test_more_items_of_a_prefix_than_workgroups(stream, held, prefix):
    rng = np.random.default_rng(prefix)
    p, q = case(rng, stream, [(2, 3 + i % 40) for i in range(272)], 8, 8, 64, held, prefix=prefix, behind=1)
    tile, chunk, items, groups = cut(p, 8, held, shared=True)
    assert tile == 128 and chunk >= 4 and items > groups
    compare(p, q, run(p, q))


@pytest.mark.parametrize("held", ["f32", "bf16", "e4m3"])
def test_more_items_of_a_prefix_than_workgroups_of_few_rows(stream, held):
    rng = np.random.default_rng(9)
    p, q = case(rng, stream, [(3, 20), (25, 30), (12, 12)], 400, 1, 32, held, prefix=600)
    tile, chunk, items, groups = cut(p, 1, held, shared=True)
    assert tile == 32 and chunk >= 4 and items > groups
    compare(p, q, run(p, q))
