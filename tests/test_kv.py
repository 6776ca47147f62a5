"""Rotary positions and the paged cache without a GPU: rotations and their steps, where rows and tokens
stand, and what the entry points refuse (descriptors are checked before the stream is looked at)."""
import ctypes
import weakref
from types import SimpleNamespace

import numpy as np
import pytest

import kv_reference as ref
import mensurflow_amd as mf
from mensurflow_amd import abi
from test_cpp_host import run as run_cpp

STREAM = SimpleNamespace(device=0, handle=None)


def array(shape, dtype=np.float32, strides=None, ptr=1 << 20):
    return mf.DeviceArray.wrap(ptr, shape, STREAM, dtype, strides)


def call(entry, desc):
    return getattr(abi.load(), entry)(None, ctypes.byref(desc)), abi.last_error()


@pytest.mark.parametrize("name", ["kv_places_test", "kv_work_test"])
def test_places_and_work(name):
    run_cpp(name)


# ---- rotations ------------------------------------------------------------------------------------


@pytest.mark.parametrize("rot", [0, 2, 64, 126, 256])
@pytest.mark.parametrize("scaling", [dict(), dict(base=500000.0), dict(factor=4.0),
                                     dict(factor=8.0, original=4096.0),
                                     dict(factor=32.0, original=8192.0, slow=1.0, fast=4.0)])
def test_steps(rot, scaling):
    r = mf.rotary(rot, **scaling)
    want = ref.steps(rot, **scaling)
    # pow in double, and three more roundings.
    assert np.all(np.abs(np.array(r.steps[:rot // 2]) - want) <= 8 * 2.0 ** -53 * want)
    assert not any(r.steps[rot // 2:])
    assert (r.rot, r.layout, r.amplitude) == (rot, mf.ROTARY_HALVES, 1.0)


@pytest.mark.parametrize("change,message", [
    (dict(rot=3), "even"), (dict(rot=-2), "even"), (dict(rot=258), "256"), (dict(layout=2), "layout"),
    (dict(base=0.5), "base"), (dict(base=float("nan")), "base"), (dict(amplitude=float("inf")), "amplitude"),
    (dict(amplitude=1e300), "amplitude"), (dict(factor=0.5), "factor"), (dict(factor=float("nan")), "factor"),
    (dict(original=-1.0), "original"), (dict(original=4096.0, slow=2.0, fast=2.0), "slow"),
    (dict(original=4096.0, fast=float("inf")), "slow")])
def test_rotations_that_are_refused(change, message):
    with pytest.raises(ValueError, match=message):
        mf.rotary(**{"rot": 64, **change})


# ---- descriptors ----------------------------------------------------------------------------------


def rope(**kw):
    args = dict(positions=array((4,), np.int32), out=array((4, 3, 64), ptr=1 << 22))
    args.update(kw)
    return mf.rope_desc(array((4, 3, 64)), mf.rotary(64), **args)


def cache(dtype=np.uint8, pages=10, page=16, heads=3, d=64):
    k, v = (array((pages, heads, page, d), dtype, ptr=p) for p in (1 << 24, 1 << 26))
    if dtype != np.uint8:
        return mf.KvCache(k, v)
    return mf.KvCache(k, v, *(array((pages, heads, page), ptr=p) for p in (1 << 27, 1 << 28)))


def batch(prefix=20, **kw):
    args = dict(starts=array((3,), np.int32), prefix=prefix,
                prefix_pages=array((2,), np.int32) if prefix else None)
    args.update(kw)
    return mf.KvBatch(array((2,), np.int32), array((2, 5), np.int32), **args)


def append(dtype=np.uint8, **kw):
    args = dict(rotary=mf.rotary(64), q=array((4, 6, 64)), q_out=array((4, 6, 64), ptr=1 << 22),
                positions=array((4,), np.int32))
    args.update(kw)
    return mf.kv_append_desc(cache(dtype), batch(), array((4, 3, 64)), array((4, 3, 64)), **args)


def attend(dtype=np.uint8, **kw):
    args = dict(out=array((4, 6, 64), ptr=1 << 22))
    args.update(kw)
    return mf.attention_paged_desc(array((4, 6, 64)), cache(dtype), batch(), **args)


MAKE = {"mfr_rope": rope, "mfr_kv_append": append, "mfr_attention_paged": attend}


@pytest.mark.parametrize("entry", list(MAKE))
def test_a_good_descriptor_comes_as_far_as_the_stream(entry):
    assert call(entry, MAKE[entry]()) == (abi.MFR_E_INVALID, "null stream")
    assert getattr(abi.load(), entry)(None, None) == abi.MFR_E_INVALID
    assert "null descriptor" in abi.last_error()


@pytest.mark.parametrize("entry", ["mfr_kv_append", "mfr_attention_paged"])
@pytest.mark.parametrize("dtype", [np.float32, np.uint16, np.uint8])
def test_good_descriptors_of_each_type(entry, dtype):
    assert call(entry, MAKE[entry](dtype)) == (abi.MFR_E_INVALID, "null stream")


ROPE = [
    (dict(rows=-1), abi.MFR_E_INVALID, "negative dimension"),
    (dict(d=62), abi.MFR_E_INVALID, "more columns"),
    (dict(x=None), abi.MFR_E_INVALID, "null"),
    (dict(out=None), abi.MFR_E_INVALID, "null"),
    (dict(x_ts=-1), abi.MFR_E_INVALID, "negative strides"),
    (dict(out_hs=63), abi.MFR_E_INVALID, "overlaps"),
    (dict(out_ts=0), abi.MFR_E_INVALID, "overlaps"),
    (dict(out=1 << 20, out_ts=1000), abi.MFR_E_INVALID, "in place"),
    (dict(x_ts=(1 << 40) + 1), abi.MFR_E_UNSUPPORTED, "too long"),
    (dict(d=1 << 21), abi.MFR_E_UNSUPPORTED, "too large"),
    (dict(rows=1 << 30, x_ts=1 << 40), abi.MFR_E_UNSUPPORTED, "further than memory"),
    (dict(rows=1 << 30, out_ts=1 << 40), abi.MFR_E_UNSUPPORTED, "further than memory"),
    (dict(positions=None, first=(1 << 31) - 3), abi.MFR_E_INVALID, "2^31"),
    (dict(positions=None, first=-(1 << 31) - 1), abi.MFR_E_INVALID, "2^31"),
]


@pytest.mark.parametrize("change,status,message", ROPE)
def test_rope_refuses(change, status, message):
    d = rope()
    for name, value in change.items():
        setattr(d, name, value)
    got = call("mfr_rope", d)
    assert got[0] == status and message in got[1], got


@pytest.mark.parametrize("entry", ["mfr_rope", "mfr_kv_append"])
@pytest.mark.parametrize("change,message", [
    (dict(rot=5), "even"), (dict(rot=-2), "even"), (dict(rot=66), "more columns"), (dict(rot=258), "256"),
    (dict(layout=-1), "layout"), (dict(amplitude=float("nan")), "amplitude"),
    (dict(steps=float("inf")), "steps"), (dict(steps=float("nan")), "steps"), (dict(steps=2e6), "steps")])
def test_bad_rotations_are_refused(entry, change, message):
    d = MAKE[entry]()
    for name, value in change.items():
        if name == "steps":
            d.rotary.steps[7] = value
        else:
            setattr(d.rotary, name, value)
    got = call(entry, d)
    assert got[0] == abi.MFR_E_INVALID and message in got[1], got


CACHE = [
    (dict(type=3), abi.MFR_E_INVALID, "type"), (dict(type=-1), abi.MFR_E_INVALID, "type"),
    (dict(d=0), abi.MFR_E_INVALID, "no heads"), (dict(heads=0), abi.MFR_E_INVALID, "no heads"),
    (dict(pages=-1), abi.MFR_E_INVALID, "no heads"),
    (dict(d=72), abi.MFR_E_UNSUPPORTED, "multiple of 16"),
    (dict(d=144), abi.MFR_E_UNSUPPORTED, "multiple of 16"),
    (dict(page_size=8), abi.MFR_E_UNSUPPORTED, "power of two"),
    (dict(page_size=24), abi.MFR_E_UNSUPPORTED, "power of two"),
    (dict(page_size=65536), abi.MFR_E_UNSUPPORTED, "power of two"),
    (dict(pages=1 << 31), abi.MFR_E_UNSUPPORTED, "too many"),
    (dict(page_stride=-1), abi.MFR_E_INVALID, "negative"),
    (dict(token_stride=(1 << 24) + 16), abi.MFR_E_UNSUPPORTED, "too long"),
    (dict(head_stride=(1 << 40) + 16), abi.MFR_E_UNSUPPORTED, "too long"),
    (dict(pages=1 << 30, page_stride=1 << 38), abi.MFR_E_UNSUPPORTED, "further than memory"),
    (dict(heads=1 << 20, head_stride=1 << 38), abi.MFR_E_UNSUPPORTED, "further than memory"),
    (dict(k=None), abi.MFR_E_INVALID, "null"), (dict(v=None), abi.MFR_E_INVALID, "null"),
    (dict(k=(1 << 24) + 8), abi.MFR_E_UNSUPPORTED, "16-byte aligned rows"),
    (dict(token_stride=72), abi.MFR_E_UNSUPPORTED, "16-byte aligned rows"),
    (dict(k_scales=None), abi.MFR_E_INVALID, "scales"),
    (dict(v_scales=(1 << 28) + 4), abi.MFR_E_UNSUPPORTED, "aligned scales"),
]


@pytest.mark.parametrize("entry", ["mfr_kv_append", "mfr_attention_paged"])
@pytest.mark.parametrize("change,status,message", CACHE)
def test_bad_caches_are_refused(entry, change, status, message):
    d = MAKE[entry]()
    if entry == "mfr_kv_append":
        d.rotary.rot = 0
    for name, value in change.items():
        setattr(d.cache, name, value)
    got = call(entry, d)
    assert got[0] == status and message in got[1], got


@pytest.mark.parametrize("change", [dict(token_stride=48), dict(head_stride=16 * 64 - 16),
                                    dict(page_stride=3 * 16 * 64 - 16), dict(page_stride=0),
                                    dict(head_stride=0), dict(token_stride=128)])
def test_an_append_refuses_rows_that_overlap(change):
    d = append()
    for name, value in change.items():
        setattr(d.cache, name, value)
    got = call("mfr_kv_append", d)
    assert got[0] == abi.MFR_E_INVALID and "overlap" in got[1], got


def test_an_append_refuses_one_place_for_keys_and_values():
    d = append()
    d.cache.v = d.cache.k
    assert "one place" in call("mfr_kv_append", d)[1]


BATCH = [
    (dict(rows=-1), abi.MFR_E_INVALID, "negative size"),
    (dict(sequences=-1), abi.MFR_E_INVALID, "negative size"),
    (dict(width=-1), abi.MFR_E_INVALID, "negative size"),
    (dict(prefix=-1), abi.MFR_E_INVALID, "negative size"),
    (dict(rows=(1 << 30) + 1), abi.MFR_E_UNSUPPORTED, "too large"),
    (dict(sequences=(1 << 24) + 1), abi.MFR_E_UNSUPPORTED, "too large"),
    (dict(width=(1 << 26) + 1), abi.MFR_E_UNSUPPORTED, "too many tokens"),
    (dict(prefix=(1 << 30) + 1), abi.MFR_E_UNSUPPORTED, "too many tokens"),
    (dict(lengths=None), abi.MFR_E_INVALID, "no lengths"),
    (dict(table=None), abi.MFR_E_INVALID, "no table"),
    (dict(table_rs=-1), abi.MFR_E_INVALID, "table stride"),
    (dict(prefix_pages=None), abi.MFR_E_INVALID, "no pages"),
    (dict(starts=None, sequences=3), abi.MFR_E_INVALID, "not whole"),
]


@pytest.mark.parametrize("entry", ["mfr_kv_append", "mfr_attention_paged"])
@pytest.mark.parametrize("change,status,message", BATCH)
def test_bad_batches_are_refused(entry, change, status, message):
    d = MAKE[entry]()
    for name, value in change.items():
        setattr(d.batch, name, value)
    got = call(entry, d)
    assert got[0] == status and message in got[1], got


@pytest.mark.parametrize("change,message", [
    (dict(k=None), "k is null"), (dict(v=None), "v is null"), (dict(q_out=None), "q_out is null"),
    (dict(q_heads=0), "number of heads"), (dict(q_out_hs=32), "q_out overlaps"),
    (dict(k_ts=-1), "negative strides"), (dict(q_out=1 << 20, q_out_ts=1000), "in place")])
def test_an_append_refuses_heads(change, message):
    d = append()
    for name, value in change.items():
        setattr(d, name, value)
    got = call("mfr_kv_append", d)
    assert got[0] == abi.MFR_E_INVALID and message in got[1], got


@pytest.mark.parametrize("change,message", [
    (dict(q=None), "q is null"), (dict(out=None), "out is null"), (dict(q_heads=4), "multiple"),
    (dict(q_heads=0), "multiple"), (dict(out_ts=64), "overlaps"), (dict(q_hs=-1), "negative strides"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale")])
def test_attention_refuses(change, message):
    d = attend()
    for name, value in change.items():
        setattr(d, name, value)
    got = call("mfr_attention_paged", d)
    assert got[0] == abi.MFR_E_INVALID and message in got[1], got


# ---- what the Python entry points do with their arguments -------------------------------------------


def test_python_refuses_arrays_of_other_types_and_shapes():
    with pytest.raises(ValueError, match="float32"):
        mf.rope_desc(array((4, 3, 64), np.uint16), mf.rotary(64))
    with pytest.raises(ValueError, match="unit stride"):
        mf.rope_desc(array((4, 3, 64), strides=(400, 130, 2)), mf.rotary(64))
    with pytest.raises(ValueError, match="positions"):
        rope(positions=array((5,), np.int32))
    with pytest.raises(ValueError, match="int32"):
        rope(positions=array((4,), np.int64))
    good = cache()
    for bad in (mf.KvCache(good.k, good.v), mf.KvCache(good.k, array((9, 3, 16, 64), np.uint8)),
                mf.KvCache(good.k, good.v, good.k_scales, array((10, 3, 15))),
                mf.KvCache(array((10, 3, 16, 64), np.int32), array((10, 3, 16, 64), np.int32)),
                mf.KvCache(*(array((10, 3, 16, 64)) for _ in range(2)), good.k_scales, good.v_scales),
                mf.KvCache(array((10, 3, 16, 64)), array((10, 3, 16, 64), strides=(4096, 1024, 64, 1)))):
        with pytest.raises(ValueError):
            mf.attention_paged_desc(array((4, 6, 64)), bad, batch(), out=array((4, 6, 64)))
    for bad in (batch(starts=array((2,), np.int32)), batch(prefix=40), batch(prefix_pages=None),
                mf.KvBatch(array((3,), np.int32), array((2, 5), np.int32)),
                mf.KvBatch(array((2,), np.int64), array((2, 5), np.int32)),
                mf.KvBatch(array((2,), np.int32), array((2, 5), np.int32, (10, 2)))):
        with pytest.raises(ValueError):
            mf.attention_paged_desc(array((4, 6, 64)), good, bad, out=array((4, 6, 64)))
    with pytest.raises(ValueError, match="without q"):
        append(q=None)
    with pytest.raises(ValueError, match="needed"):
        attend(out=array((4, 6, 32)))
    with pytest.raises(ValueError, match="float32, uint16"):
        mf.KvCache.empty(1, 16, 1, 64, STREAM, np.float64)
    with pytest.raises(ValueError, match="negative"):
        mf.KvCache.empty(-1, 16, 1, 64, STREAM)


@pytest.mark.parametrize("entry", list(MAKE))
def test_operands_of_two_devices_are_refused(entry):
    other = SimpleNamespace(device=1, handle=None)
    there = mf.DeviceArray.wrap(1 << 20, (4, 6, 64), other)
    with pytest.raises(ValueError, match="different devices"):
        if entry == "mfr_rope":
            rope(out=mf.DeviceArray.wrap(1 << 20, (4, 3, 64), other))
        elif entry == "mfr_kv_append":
            append(q=there)
        else:
            attend(out=there)


@pytest.mark.parametrize("run,desc", [(mf.rope_run, rope), (mf.kv_append_run, append),
                                      (mf.attention_paged_run, attend),
                                      (mf.attention_paged_workspace, attend)])
def test_a_descriptor_is_refused_by_a_stream_of_another_device(run, desc):
    with pytest.raises(ValueError, match="another device"):
        run(SimpleNamespace(device=1, handle=None), desc())


def test_descriptors_keep_their_arrays():
    kept = []
    for make in (rope, append, attend):
        out = array((4, 3, 64) if make is rope else (4, 6, 64), ptr=1 << 23)
        refs = [weakref.ref(out), weakref.ref(out._base)]
        d = make(**{"q_out" if make is append else "out": out})
        del out
        assert all(r() is not None for r in refs)
        kept.append((d, refs))
    for i in range(3):
        d, refs = kept[i]
        kept[i] = None
        del d
        assert all(r() is None for r in refs)
