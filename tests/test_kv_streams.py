"""Which stream an append to a paged cache runs on: without a GPU the choice and the refusals, on the device
what it orders."""
from types import SimpleNamespace

import numpy as np
import pytest

import kv_reference as ref
import mensurflow_amd as mf
from helpers import same_bits
from kv_reference import Paged, dev


def fake(handle, device=0):
    return SimpleNamespace(device=device, handle=handle, hip_stream=lambda: handle)


def arrays(**streams):
    """(cache, batch, k, v, q, q_out), the cache and the batch on a stream of their own."""
    far = fake(1)

    def array(shape, stream, dtype=np.float32):
        return mf.DeviceArray.wrap(1 << 20, shape, stream, dtype)

    cache = mf.KvCache(*(array((4, 2, 16, 64), far) for _ in range(2)))
    batch = mf.KvBatch(array((3,), far, np.int32), array((3, 1), far, np.int32))
    heads = {"k": 2, "v": 2, "q": 4, "q_out": 4}
    return cache, batch, {name: array((3, heads[name], 64), s) for name, s in streams.items()}


@pytest.mark.parametrize("given", [False, True])
def test_an_append_runs_on_its_keys_stream(monkeypatch, given):
    ran, made = [], []
    monkeypatch.setattr(mf, "kv_append_run", lambda stream, desc: ran.append(stream))
    monkeypatch.setattr(mf.DeviceArray, "empty", classmethod(
        lambda cls, shape, stream, dtype=np.float32: made.append(stream) or cls.wrap(1 << 22, shape, stream)))
    own = fake(2)
    cache, batch, a = arrays(k=own, v=own, q=own, q_out=own)
    out = a["q_out"] if given else None
    got = mf.kv_append(cache, batch, a["k"], a["v"], q=a["q"], q_out=out)
    assert ran == [own] and made == ([] if given else [own]) and got.stream is own


@pytest.mark.parametrize("name", ["v", "q", "q_out"])
def test_operands_of_another_stream_are_refused(monkeypatch, name):
    ran = []
    monkeypatch.setattr(mf, "kv_append_run", lambda stream, desc: ran.append(stream))
    own = fake(2)
    cache, batch, a = arrays(**{"k": own, "v": own, "q": own, "q_out": own, name: fake(3)})
    with pytest.raises(ValueError, match=f"{name} is on another stream"):
        mf.kv_append(cache, batch, a["k"], a["v"], q=a["q"], q_out=a["q_out"])
    assert not ran
    # Another Stream over the same HIP stream is the same.
    cache, batch, a = arrays(**{"k": own, "v": own, "q": own, "q_out": own, name: fake(2)})
    mf.kv_append(cache, batch, a["k"], a["v"], q=a["q"], q_out=a["q_out"])
    assert ran == [own]


@pytest.mark.parametrize("call", ["rope", "attention_paged"])
def test_a_result_on_another_stream_is_refused(monkeypatch, call):
    ran = []
    monkeypatch.setattr(mf, call + "_run", lambda stream, desc: ran.append(stream))
    own = fake(2)

    def run(out_stream):
        cache, batch, a = arrays(q=own, q_out=out_stream)
        if call == "rope":
            mf.rope(a["q"], mf.rotary(64), out=a["q_out"])
        else:
            mf.attention_paged(a["q"], cache, batch, out=a["q_out"])

    with pytest.raises(ValueError, match="out is on another stream"):
        run(fake(3))
    assert not ran
    run(own)
    assert ran == [own]


@pytest.mark.gpu
@pytest.mark.parametrize("held", ["f32", "bf16", "e4m3"])
def test_a_cache_of_another_stream(held):
    """A cache and a batch made on one stream, which is waited for once; steps on another one behind much
    work, an append and the attention that reads it."""
    rng = np.random.default_rng(1)
    with mf.Stream(0) as far, mf.Stream(0) as own:
        p = Paged(rng, far, [(1, 40), (5, 30), (2, 2)], 2, 64, held)
        k, v = (rng.standard_normal((p.rows, 2, 64)).astype(np.float32) for _ in range(2))
        q = rng.standard_normal((p.rows, 8, 64)).astype(np.float32)
        cache, batch = p.cache(), p.batch()
        far.synchronize()
        big = mf.DeviceArray.from_numpy(rng.standard_normal((4096, 4096)).astype(np.float32), own)
        ready = [dev(x, own) for x in (k, v, q)]
        late = [dev(np.zeros_like(x), own) for x in (k, v, q)]
        product = mf.gemm(big, big)
        own.synchronize()
        for _ in range(20):         # some 20 ms
            mf.gemm(big, big, out=product)
        none = mf.rotary(0)
        for x, y in zip(ready, late):
            mf.rope(x, none, out=y)
        turned = mf.kv_append(cache, batch, late[0], late[1], q=late[2])
        assert turned.stream is own
        got = mf.attention_paged(turned, cache, batch).numpy()
        assert same_bits(turned.numpy(), q)
        for s, (n, tokens) in enumerate(p.counts):
            for numbers, scales, x in ((p.k, p.ks, k), (p.v, p.vs, v)):
                values, sizes = ref.rows_to_held(x, held)
                for i in range(n):
                    at = p.table[s, (tokens - n + i) // 16], slice(None), (tokens - n + i) % 16
                    numbers[at] = values[p.starts[s] + i]
                    if scales is not None:
                        scales[at] = sizes[p.starts[s] + i]
        want, bound = p.attend(q)
        assert np.all(np.abs(got - want) <= bound)
