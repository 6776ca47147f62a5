"""Appending to a paged cache and attention against it where many rows share an item, in captured
graphs, on streams and threads side by side, and in caches past 32 bits of offsets."""
import numpy as np
import pytest

import kv_reference as ref
import mensurflow_amd as mf
from helpers import same_bits
from kv_reference import Paged, dev
from test_attention_paged_gpu import case, check, run
from test_f8_forms_gpu import Graph, in_threads

pytestmark = pytest.mark.gpu
HELD = ["f32", "bf16", "e4m3"]
MANY = [(150, 200), (40, 64), (1, 300)]     # rows enough for tiles of many


# ---- many rows ------------------------------------------------------------------------------------


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("d", [16, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("scale", [0.0, -0.5])
def test_many_rows_of_each_depth(stream, held, d, scale):
    rng = np.random.default_rng(d)
    p, q = case(rng, stream, MANY, 2, 3, d, held, prefix=70, front=1, behind=1)
    kw = {"scale": scale} if scale else {}
    check(p, q, run(p, q, **kw), norm=False, **kw)


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("tokens", [0, 1, 15, 16, 63, 64, 65, 127, 128, 129, 192, 193, 257])
@pytest.mark.parametrize("causal", [True, False])
def test_many_rows_on_few_tokens(stream, held, tokens, causal):
    rng = np.random.default_rng(tokens)
    p, q = case(rng, stream, [(60, tokens), (33, 64)], 1, 3, 64, held)
    check(p, q, run(p, q, causal=causal), causal=causal)


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("prefix", [1, 63, 64, 65, 333])
def test_many_rows_on_a_prefix_seen_whole(stream, held, prefix):
    rng = np.random.default_rng(prefix)
    p, q = case(rng, stream, [(2, 20), (1, 0), (3, 40)] * 30, 2, 2, 128, held, prefix=prefix)
    check(p, q, run(p, q, causal=False), causal=False)


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("gone", [[1], [5], [0, 3, 12], [2, 6, 7, 11], [4, 5, 6, 7], list(range(13))])
@pytest.mark.parametrize("prefix", [False, True])
def test_many_rows_with_bad_pages(stream, held, gone, prefix):
    """Pages that there are not, at each place of a tile of 64 tokens: their tokens are absent, and what
    an earlier tile held is not taken for theirs. Every row sees all tokens."""
    rng = np.random.default_rng(len(gone))
    counts = [(40, 0), (60, 0)] if prefix else [(60, 13 * 16), (40, 13 * 16)]
    p, q = case(rng, stream, counts, 2, 2, 64, held, prefix=13 * 16 if prefix else 0)
    seqs = [0, 1] if prefix else [1]
    at = [(s, (t if not prefix else t - p.prefix)) for s in seqs for g in gone
          for t in range(16 * g, 16 * g + 16)]
    want, bound = p.attend(q, causal=False, absent=at)
    kept = p.prefix_pages.copy(), p.table.copy()
    for i, g in enumerate(gone):
        bad = ref.BAD[i % len(ref.BAD)]
        if prefix:
            p.prefix_pages[g] = bad
        else:
            p.table[1, g] = bad
    got = run(p, q, causal=False)
    p.prefix_pages, p.table = kept
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("held", ["bf16", "e4m3"])
@pytest.mark.parametrize("which", ["scale", "number"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("in_values", [False, True])
def test_many_rows_before_a_token_of_no_number(stream, held, which, bad, in_values):
    """One token's key or value is no number: rows in front of it are as without, rows that see it
    are no numbers."""
    if which == "scale" and held != "e4m3":
        pytest.skip("no scales")
    rng = np.random.default_rng(12)
    p, q = case(rng, stream, [(100, 150)], 1, 2, 64, held)
    want, bound = p.attend(q)
    place = 97
    numbers, scales = (p.v, p.vs) if in_values else (p.k, p.ks)
    at = p.table[0, place // 16], slice(None), place % 16
    if which == "scale":
        scales[at] = bad
    elif held == "e4m3":
        numbers[at][..., 5] = 0x7F if np.isnan(bad) else 0xFF
    else:
        numbers[at][..., 5] = ref.bf16_bits(np.float32([bad]))[0]
    got = run(p, q)
    sees = np.arange(100) + 50 >= place
    assert np.all(np.abs(got - want)[~sees] <= bound[~sees])
    if np.isnan(bad) or in_values:
        assert not np.isfinite(got[sees]).all(axis=-1).any()


@pytest.mark.parametrize("counts", [MANY, [(1, 300), (3, 40)]])
def test_scales_of_any_sign(stream, counts):
    """A cache that another program filled may have scales below 0, and rows of zeros a scale of 0."""
    rng = np.random.default_rng(22)
    p, q = case(rng, stream, counts, 2, 2, 64, "e4m3", prefix=40)
    for scales in (p.ks, p.vs):
        scales *= rng.choice(np.float32([-1, 1, 1, 0]), scales.shape)
    check(p, q, run(p, q))


@pytest.mark.parametrize("scale", [2.0 ** -126, 2.0 ** -90, 2.0 ** 100])
@pytest.mark.parametrize("counts", [MANY, [(1, 300), (3, 40)]])
def test_small_and_large_values(stream, counts, scale):
    """Values under one small or large scale, some rows of zeros among them."""
    rng = np.random.default_rng(23)
    p, q = case(rng, stream, counts, 2, 2, 64, "e4m3", prefix=40)
    seen = np.isfinite(p.vs)
    p.vs[seen] = scale
    p.v[np.logical_and(seen, rng.random(seen.shape) < 0.2)] = 0
    if scale < 2.0 ** -96:      # parts of weights under fp16's least number: those values lose bits
        got, (want, _) = run(p, q), p.attend(q)
        there = ~np.isnan(want)
        assert np.all(np.abs(got[there]) <= 448 * scale)
        return
    check(p, q, run(p, q))


@pytest.mark.parametrize("held", HELD)
def test_many_sequences(stream, held):
    """More sequences than a workgroup looks at together, most of them empty, and one long one."""
    rng = np.random.default_rng(13)
    counts = [(int(n), int(n + t)) for n, t in zip(rng.integers(0, 3, 700), rng.integers(0, 9, 700))]
    counts[300], counts[650] = (1, 1500), (20, 40)
    p, q = case(rng, stream, counts, 1, 2, 32, held, prefix=33, front=2, behind=2)
    check(p, q, run(p, q))


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("rows", [1, 150])
def test_slots_without_rows(stream, held, rows):
    """Thousands of slots, of which few have rows."""
    rng = np.random.default_rng(24)
    counts = [(0, 0)] * 5000
    for s in (0, 1, 70, 2500, 2565, 4999):
        counts[s] = (rows, rows + 20)
    p, q = case(rng, stream, counts, 1, 2, 32, held, front=1, behind=1)
    check(p, q, run(p, q))
    k, v = (rng.standard_normal((p.rows, 1, 32)).astype(np.float32) for _ in range(2))
    cache, batch = p.cache(), p.batch()
    mf.kv_append(cache, batch, dev(k, stream), dev(v, stream))
    got = cache.v.numpy()
    values, _ = ref.rows_to_held(v, held)
    for s in (0, 1, 70, 2500, 2565, 4999):
        for i in (0, rows - 1):
            place = 20 + i
            assert np.array_equal(got[p.table[s, place // 16], :, place % 16], values[p.starts[s] + i])


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("pages", [0, 3])
def test_no_room(stream, held, pages):
    """No pages, or tables without entries: nothing is written, nothing is seen, queries are turned."""
    rng = np.random.default_rng(25)
    cache = mf.KvCache.empty(pages, 16, 2, 32, stream, ref.HELD[held])
    batch = mf.KvBatch(dev(np.array([3, 9], np.int32), stream),
                       mf.DeviceArray.empty((2, 0 if pages else 1), stream, np.int32),
                       starts=dev(np.array([0, 3, 200], np.int32), stream))
    k, v = (rng.standard_normal((200, 2, 32)).astype(np.float32) for _ in range(2))
    q = rng.standard_normal((200, 4, 32)).astype(np.float32)
    rot = mf.rotary(32)
    turned = mf.kv_append(cache, batch, dev(k, stream), dev(v, stream), rotary=rot, q=dev(q, stream))
    places = np.concatenate((np.arange(3), 9 - 197 + np.arange(197)))
    want, off = ref.turn(q, places, ref.steps(32), mf.ROTARY_HALVES)
    assert np.all(np.abs(turned.numpy() - want) <= off)
    assert not mf.attention_paged(turned, cache, batch).numpy().any()


@pytest.mark.parametrize("held", HELD)
def test_a_page_of_several_sequences(stream, held):
    """Tables may name a page more than once, in one sequence and in several."""
    rng = np.random.default_rng(14)
    p, q = case(rng, stream, [(1, 64), (5, 60), (2, 33)], 2, 2, 64, held)
    p.table[1, :4] = p.table[0, [1, 1, 0, 3]]
    p.table[2, 0] = p.table[0, 2]
    check(p, q, run(p, q))


# ---- captured -------------------------------------------------------------------------------------


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_captured_steps(held, rows):
    """An append and the attention behind it, captured once and replayed for one step after another as
    the lengths on the device grow, with eager calls between that use the stream's own workspace: each
    replay gives the bits of the eager calls."""
    rng = np.random.default_rng(rows)
    heads, group, d, page, seqs, steps = 2, 2, 64, 16, 3, 4
    print(f"captured {held} {rows}", flush=True)
    with mf.Stream(0) as own:
        caches = [mf.KvCache.empty(40, page, heads, d, own, ref.HELD[held]) for _ in range(2)]
        table = dev(rng.permutation(40).astype(np.int32)[:36].reshape(seqs, 12), own)
        shared = dev(np.array([7, 30], np.int32), own)
        prefix_rows = [dev(rng.standard_normal((20, heads, d)), own, np.float32) for _ in range(2)]
        lengths = dev(np.zeros(seqs, np.int32), own)
        batch = mf.KvBatch(lengths, table, prefix=20, prefix_pages=shared)
        k, v = (dev(np.zeros((seqs * rows, heads, d), np.float32), own) for _ in range(2))
        q = dev(np.zeros((seqs * rows, heads * group, d), np.float32), own)
        outs = [mf.DeviceArray.empty(q.shape, own) for _ in range(2)]
        turned = [mf.DeviceArray.empty(q.shape, own) for _ in range(2)]
        rot = mf.rotary(d)
        for c in caches:
            one = mf.KvBatch(dev(np.array([20], np.int32), own), shared.view((1, 2)))
            mf.kv_append(c, one, *prefix_rows, rotary=rot)
        attends = [mf.attention_paged_desc(turned[i], caches[i], batch, out=outs[i]) for i in range(2)]
        need = mf.attention_paged_workspace(own, attends[0])
        work = mf.DeviceArray.empty((need,), own, np.uint8)
        attends[0] = mf.attention_paged_desc(turned[0], caches[0], batch, out=outs[0], workspace=work)

        def body(i):
            mf.kv_append(caches[i], batch, k, v, rotary=rot, q=q, q_out=turned[i])
            mf.attention_paged_run(own, attends[i])

        graph = Graph(own, lambda: body(0))
        for step in range(steps):
            lengths.upload(np.array([(step + 1) * rows, (step + 1) * rows, rows], np.int32))
            for a in (k, v, q):
                a.upload(rng.standard_normal(a.shape).astype(np.float32))
            for o in outs:
                mf.fill(o, 3.0)
            graph.launch()
            body(1)
            got, want = (o.numpy() for o in outs)
            assert same_bits(got, want), step
            graph.launch()
            assert same_bits(outs[0].numpy(), want), step
        graph.close()


@pytest.mark.parametrize("held", ["f32", "e4m3"])
def test_two_graphs_with_a_workspace_each(held):
    rng = np.random.default_rng(16)
    with mf.Stream(0) as own, mf.Stream(0) as other:
        cases, graphs = [], []
        for counts in ([(1, 900), (1, 30)], [(100, 300)]):
            p, q = case(rng, own, counts, 2, 2, 64, held, prefix=100)
            out = mf.DeviceArray.empty(q.shape, own)
            args = dev(q, own), p.cache(), p.batch()
            need = mf.attention_paged_workspace(own, mf.attention_paged_desc(*args, out=out))
            work = mf.DeviceArray.empty((need,), own, np.uint8)
            desc = mf.attention_paged_desc(*args, out=out, workspace=work)
            mf.attention_paged_run(own, desc)
            want = out.numpy()
            check(p, q, want)
            graphs.append(Graph(own, lambda desc=desc: mf.attention_paged_run(own, desc)))
            cases.append((out, want))
        for _ in range(3):
            for out, _ in cases:
                mf.fill(out, 5.0)
            own.synchronize()
            graphs[0].launch()
            graphs[1].launch(other)
            own.synchronize()
            other.synchronize()
            for out, want in cases:
                assert same_bits(out.numpy(), want)
        for g in graphs:
            g.close()


def test_a_captured_call_needs_a_workspace():
    """Without one the call is refused, nothing is captured, and the stream goes on."""
    rng = np.random.default_rng(17)
    with mf.Stream(0) as own:
        p, q = case(rng, own, [(1, 100)], 1, 1, 64, "f32")
        out = dev(np.zeros(q.shape, np.float32), own)
        desc = mf.attention_paged_desc(dev(q, own), p.cache(), p.batch(), out=out)

        def body():
            with pytest.raises(ValueError, match="captured call needs a workspace"):
                mf.attention_paged_run(own, desc)

        graph = Graph(own, body)
        graph.launch()
        assert not out.numpy().any()
        graph.close()
        check(p, q, run(p, q))


def test_a_workspace_too_small_or_misaligned_is_refused():
    rng = np.random.default_rng(18)
    with mf.Stream(0) as own:
        p, q = case(rng, own, [(1, 500), (2, 40)], 2, 2, 64, "bf16", prefix=40)
        out = dev(np.full(q.shape, 7.0, np.float32), own)
        args = dev(q, own), p.cache(), p.batch()
        need = mf.attention_paged_workspace(own, mf.attention_paged_desc(*args, out=out))
        work = mf.DeviceArray.empty((need + 256,), own, np.uint8)
        for first, count in ((0, need - 1), (8, need), (0, 0)):
            desc = mf.attention_paged_desc(*args, out=out, workspace=work.slice(0, first, first + count))
            with pytest.raises(ValueError, match="workspace is too small"):
                mf.attention_paged_run(own, desc)
        assert np.all(out.numpy() == 7.0)
        desc = mf.attention_paged_desc(*args, out=out, workspace=work.slice(0, 256, 256 + need))
        mf.attention_paged_run(own, desc)
        check(p, q, out.numpy())


# ---- streams and threads --------------------------------------------------------------------------


def test_streams_of_several_threads():
    rng = np.random.default_rng(19)
    with mf.Stream(0) as one, mf.Stream(0) as two:
        sets = []
        for s, counts in ((one, [(1, 800)] * 4), (two, [(90, 200), (1, 50)])):
            p, q = case(rng, s, counts, 2, 2, 64, "bf16", prefix=50)
            out = mf.DeviceArray.empty(q.shape, s)
            desc = mf.attention_paged_desc(dev(q, s), p.cache(), p.batch(), out=out)
            sets.append((p, q, s, desc, out))
        in_threads(*(lambda c=c: [mf.attention_paged_run(c[2], c[3]) for _ in range(20)] for c in sets))
        for p, q, _, _, out in sets:
            check(p, q, out.numpy())


def test_one_stream_of_two_threads():
    """Calls from two threads on one stream take its workspace one after the other."""
    rng = np.random.default_rng(20)
    with mf.Stream(0) as s:
        sets = []
        for counts in ([(1, 700)] * 3, [(80, 300)]):
            p, q = case(rng, s, counts, 2, 2, 64, "e4m3", prefix=50)
            out = mf.DeviceArray.empty(q.shape, s)
            sets.append((p, q, mf.attention_paged_desc(dev(q, s), p.cache(), p.batch(), out=out), out))
        in_threads(*(lambda c=c: [mf.attention_paged_run(s, c[2]) for _ in range(20)] for c in sets))
        for p, q, _, out in sets:
            check(p, q, out.numpy())


# ---- large ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("rows", [1, 50])
def test_caches_past_32_bits(stream, held, rows):
    """The last pages of a cache of more than 2^31 elements (its offsets pass 32 bits), one head."""
    rng = np.random.default_rng(21)
    d, page = 128, 64
    pages = (1 << 31) // (page * d) + 100
    cache = mf.KvCache.empty(pages, page, 1, d, stream, ref.HELD[held])
    p = Paged(rng, stream, [(rows, 300), (rows, 130)], 1, d, held, page=page)
    q = rng.standard_normal((p.rows, 4, d)).astype(np.float32)
    shift = pages - p.pages
    for here, there in ((p.k, cache.k), (p.v, cache.v), (p.ks, cache.k_scales), (p.vs, cache.v_scales)):
        if here is not None:
            there.slice(0, shift, pages).upload(here)
    batch = p.batch()
    used = np.where((p.table >= 0) & (p.table < p.pages), p.table + shift, -1).astype(np.int32)
    batch = mf.KvBatch(batch.lengths, dev(used, stream), starts=batch.starts)
    got = mf.attention_paged(dev(q, stream), cache, batch).numpy()
    check(p, q, got)
    for a in (cache.k, cache.v):
        a.close()
