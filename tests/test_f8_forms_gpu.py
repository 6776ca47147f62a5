"""The forms of mfr_f8gemm that sizes choose between (few rows, rings of slices, tiles of 64 and 128
rows, the depth in ranges, strips past a multiple of 128 by themselves), each with every kind of output, and what is
queued around them: calls of two threads on one stream, on two streams, a workspace that grows,
graphs that are replayed between eager calls."""
import ctypes
import threading

import numpy as np
import pytest

import f8_reference as ref
import mensurflow_amd as mf
from helpers import same_bits
from test_f8_gpu import (TINY, Held, assert_f8, dev, exact_operands, held_of, pitched,
                         random_operands, same_codes)

pytestmark = pytest.mark.gpu

# Sums of 9000 products of whole values up to 16 under scales up to 4 stay below 2^22 on average by
# far; the tests assert it of the magnitudes' sums, which makes every partial sum exact.
FORMS = [(2, 4683, 454), (740, 125, 549), (35, 5759, 786), (105, 2437, 549),  # few rows
         (1, 6913, 5450), (3, 8300, 1000), (128, 4100, 1100), (99, 2559, 3360),  # rings
         (155, 3457, 2499), (258, 6145, 4260), (65, 4507, 4438), (200, 4096, 2048),
         (1792, 513, 1878), (30, 14200, 700), (8, 7424, 8399),
         (39, 4097, 3153), (201, 4674, 4375), (2051, 195, 5841),  # 64-row tiles in ranges
         (65, 4122, 2921), (268, 1664, 5874), (17, 2816, 8567),  # the gated ones
         (200, 4737, 8536), (210, 4112, 8909), (205, 4824, 6303), (2335, 385, 6024),  # 128-row tiles in ranges
         (2305, 19, 8334), (1025, 137, 8767),                     # the gated ones
         (1349, 2945, 130), (639, 3208, 271),                     # and whole
         (1883, 4353, 777), (1668, 4863, 642), (2304, 1802, 629),  # a strip of columns, of rows
         (2176, 3843, 1335), (2051, 3971, 1064),
         (1841, 4638, 1866), (2177, 3885, 3033), (2305, 1818, 972), (1667, 2481, 2445)]  # and both


def equal(got, want):
    """Bit for bit but for the sign of zeros."""
    return same_bits(got + np.float32(0), want.astype(np.float32) + np.float32(0))


@pytest.mark.parametrize("m,n,k", FORMS)
def test_forms(stream, m, n, k):
    rng = np.random.default_rng(m + n + k)
    a, sa = exact_operands(rng, m, k, 1)
    b, sb = exact_operands(rng, n, k, 128)
    p, magnitude = ref.product(a, sa, b, sb)
    assert magnitude.max() < 2 ** 22
    p = p.astype(np.float32)
    ha, hb = held_of(a, sa, stream, 1), held_of(b, sb, stream, 128)
    out = pitched(np.zeros((m, n), np.float32), stream, 3)
    mf.gemm_f8(ha.matrix, hb.matrix, out=out)
    assert equal(out.numpy(), p)
    by_row = held_of(a, sa, stream, 1, by_row=True, extra=0)
    out = pitched(np.ones((m, n), np.float32), stream, 3)
    mf.gemm_f8(by_row.matrix, held_of(b, sb, stream, 128, by_row=True).matrix, out=out)
    assert equal(out.numpy(), p)
    c0 = rng.standard_normal((m, n)).astype(np.float32)
    bias = rng.standard_normal(n).astype(np.float32)
    want = ((p + np.float32(0.3) * c0) + bias).astype(np.float32)
    held = Held(m, n, stream, by_row=True)
    c = pitched(c0, stream, 2)
    mf.gemm_f8(ha.matrix, hb.matrix, c0=c, beta=0.3, bias=dev(bias, stream), out=c,
               out_f8=held.matrix)
    assert same_bits(c.numpy(), want)
    assert_f8(held, want)
    only = Held(m, n, stream)
    mf.gemm_f8(ha.matrix, hb.matrix, c0=dev(c0, stream), beta=0.3, bias=dev(bias, stream),
               out_f8=only.matrix)
    assert_f8(only, want)
    wide = mf.DeviceArray(out._base.shape, np.float32, stream, _base=out._base, _ptr=out._base._ptr)
    assert np.all(wide.numpy()[:, n:] == np.float32(123.5)), "written behind the rows"


@pytest.mark.parametrize("m,n,k", FORMS)
def test_gated_forms(stream, m, n, k):
    rng = np.random.default_rng(m + n + k + 1)
    a, sa = exact_operands(rng, m, k, 1)
    g, sg = exact_operands(rng, n, k, 128)
    u, su = exact_operands(rng, n, k, 128)
    sg = sg / 64
    pg, pu = (ref.product(a, sa, *w)[0] for w in ((g, sg), (u, su)))
    ha, hg, hu = (held_of(c, s, stream, r) for c, s, r in ((a, sa, 1), (g, sg, 128), (u, su, 128)))
    held, out = Held(m, n, stream), pitched(np.zeros((m, n), np.float32), stream, 1)
    mf.gemm_f8_gated(ha.matrix, hg.matrix, hu.matrix, out=out, out_f8=held.matrix)
    y = out.numpy()
    want = ref.silu(pg) * pu
    # An exponential within 2^-23, three more roundings and the product's.
    assert np.all(np.abs(y - want) <= 6 * ref.EPS32 * np.abs(want) + TINY * np.abs(pu))
    assert_f8(held, y)
    only = Held(m, n, stream, by_row=True)
    mf.gemm_f8_gated(ha.matrix, hg.matrix, hu.matrix, out_f8=only.matrix)
    assert_f8(only, y)
    mf.gemm_f8_gated(ha.matrix, hg.matrix, hu.matrix, act=mf.ACT_NONE, out=out)
    assert equal(out.numpy(), pg * pu)


@pytest.mark.parametrize("act", [mf.ACT_GELU_TANH, mf.ACT_GELU_ERF, mf.ACT_SILU])
@pytest.mark.parametrize("m,n,k", [(1349, 2945, 130), (193, 4382, 7538), (1668, 4863, 642)])
def test_activations_in_the_large_forms(stream, m, n, k, act):
    rng = np.random.default_rng(m + act)
    a, sa = exact_operands(rng, m, k, 1)
    b, sb = exact_operands(rng, n, k, 128)
    sb = sb / 512
    before = ref.product(a, sa, b, sb)[0].astype(np.float32)
    y = mf.gemm_f8(held_of(a, sa, stream, 1).matrix, held_of(b, sb, stream, 128).matrix,
                   act=act).numpy()
    if act == mf.ACT_SILU:
        want = ref.silu(before)
        assert np.all(np.abs(y - want) <= 5 * ref.EPS32 * np.abs(want) + TINY)
    else:
        assert same_bits(y, mf.bias_act(dev(before, stream), None, act).numpy())


@pytest.mark.parametrize("m,n,k", [(3, 300, 700), (200, 300, 700), (600, 1300, 300)])
def test_scales_of_stride_zero(stream, m, n, k):
    """One scale for a row, for a block of depths, or for a whole operand: strides of 0."""
    rng = np.random.default_rng(m)
    a, _ = exact_operands(rng, m, k, 1)
    b, _ = exact_operands(rng, n, k, 128)
    mb, nb = -(-n // 128), ref.blocks(k)
    one = dev(np.float32([2]), stream)
    per_row = dev(rng.choice(np.float32([0.5, 1, 2]), m), stream)
    ha = held_of(a, np.ones((m, nb), np.float32), stream, 1).matrix
    hb = held_of(b, np.ones((mb, nb), np.float32), stream, 128).matrix
    hb.scales = mf.DeviceArray.wrap(one.ptr, (mb, nb), stream, strides=(0, 0))
    ha.scales = mf.DeviceArray.wrap(per_row.ptr, (m, nb), stream, strides=(1, 0))
    want = ref.product(a, np.repeat(per_row.numpy()[:, None], nb, 1), b,
                       np.full((mb, nb), 2, np.float32))[0]
    assert equal(mf.gemm_f8(ha, hb).numpy(), want)


# One of each kind that takes the workspace: a depth in ranges, few rows in 8 bits alone.
SHARED = [(39, 4097, 3153), (4, 4000, 4100), (210, 4112, 8909)]


def make_calls(stream, seed):
    """[(run, check)] of products that take the stream's workspace, in rising sizes of it."""
    rng = np.random.default_rng(seed)
    calls = []
    for m, n, k in SHARED:
        a, sa = exact_operands(rng, m, k, 1)
        b, sb = exact_operands(rng, n, k, 128)
        p = ref.product(a, sa, b, sb)[0].astype(np.float32)
        ha, hb = held_of(a, sa, stream, 1), held_of(b, sb, stream, 128)
        out, q = mf.DeviceArray.empty((m, n), stream), Held(m, n, stream)

        def run(ha=ha, hb=hb, out=out, q=q, few=m < 16):
            if few:
                mf.gemm_f8(ha.matrix, hb.matrix, out_f8=q.matrix)
            else:
                mf.gemm_f8(ha.matrix, hb.matrix, out=out, out_f8=q.matrix)

        def check(out=out, q=q, p=p, few=m < 16):
            assert few or equal(out.numpy(), p)
            assert_f8(q, p)

        calls.append((run, check))
    return calls


def in_threads(*work):
    """Runs each callable in a thread, then raises what one of them raised."""
    failed = []

    def body(f):
        try:
            f()
        except BaseException as e:  # noqa: BLE001 - handed on below
            failed.append(e)

    threads = [threading.Thread(target=body, args=(f,)) for f in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if failed:
        raise failed[0]


def test_two_threads_on_one_stream_share_its_workspace():
    with mf.Stream(0) as own:
        sets = [make_calls(own, seed) for seed in (1, 2)]
        orders = [(0, 1, 2, 0, 1, 2), (2, 0, 1, 1, 2, 0)]

        def work(calls, order):
            for i in order:
                calls[i][0]()

        in_threads(*(lambda c=c, o=o: work(c, o) for c, o in zip(sets, orders)))
        for calls in sets:
            for _, check in calls:
                check()


def test_two_streams_at_once():
    with mf.Stream(0) as one, mf.Stream(0) as two:
        sets = [make_calls(s, seed) for s, seed in ((one, 3), (two, 4))]
        in_threads(*(lambda c=c: [run() for _ in range(5) for run, _ in c] for c in sets))
        for calls in sets:
            for _, check in calls:
                check()


def hip_call(name, *args):
    hip = ctypes.CDLL("libamdhip64.so.7")  # the runtime that the library has loaded
    assert getattr(hip, name)(*args) == 0, name


class Graph:
    """What `body` queues on a stream, captured."""

    def __init__(self, stream, body):
        self.handle = ctypes.c_void_p(stream.hip_stream())
        self.graph, self.run = ctypes.c_void_p(), ctypes.c_void_p()
        hip_call("hipStreamBeginCapture", self.handle, ctypes.c_int(1))  # thread local
        body()
        hip_call("hipStreamEndCapture", self.handle, ctypes.byref(self.graph))
        hip_call("hipGraphInstantiate", ctypes.byref(self.run), self.graph, None, None,
                 ctypes.c_size_t(0))

    def launch(self, stream=None):
        to = self.handle if stream is None else ctypes.c_void_p(stream.hip_stream())
        hip_call("hipGraphLaunch", self.run, to)

    def close(self):
        hip_call("hipGraphExecDestroy", self.run)
        hip_call("hipGraphDestroy", self.graph)


def test_captured_before_the_workspace_exists_and_beside_calls_that_use_it():
    """Two graphs of calls that would take the workspace, captured on a new stream, replayed on two
    streams at once and between eager calls that allocate, use and grow it: exact sums throughout."""
    with mf.Stream(0) as own, mf.Stream(0) as other:
        first, second = make_calls(own, 5), make_calls(own, 6)
        graphs = [Graph(own, lambda c=c: [run() for run, _ in c]) for c in (first, second)]
        for _ in range(3):
            graphs[0].launch()
            graphs[1].launch(other)
            own.synchronize()
            other.synchronize()
            for _, check in first + second:
                check()
            for run, _ in first + second:
                run()
            own.synchronize()
            for _, check in first + second:
                check()
        for g in graphs:
            g.close()


@pytest.mark.parametrize("m,n,k", [(1, 4100, 2300), (30, 14200, 700), (70, 1000, 2300), (300, 1000, 900)])
def test_captured_8_bit_outputs_alone(m, n, k):
    """Without a workspace: exact sums, the plain and the gated product, replayed between eager calls."""
    rng = np.random.default_rng(m + 1)
    with mf.Stream(0) as own:
        a, sa = exact_operands(rng, m, k, 1)
        b, sb = exact_operands(rng, n, k, 128)
        p = ref.product(a, sa, b, sb)[0].astype(np.float32)
        ha, hb = held_of(a, sa, own, 1), held_of(b, sb, own, 128)
        q, gated = Held(m, n, own), Held(m, n, own)

        def body():
            mf.gemm_f8(ha.matrix, hb.matrix, out_f8=q.matrix)
            mf.gemm_f8_gated(ha.matrix, hb.matrix, hb.matrix, act=mf.ACT_NONE, out_f8=gated.matrix)

        graph = Graph(own, body)
        for _ in range(3):
            for call in (graph.launch, body):
                mf.fill(q.store, 1.0)
                mf.fill(gated.store, 1.0)
                call()
                codes, scales = ref.quantize(p)
                got = q.bytes.numpy()[:m, :n], q.store.numpy()[:, :m].T
                assert same_codes(got[0], codes) and np.array_equal(got[1], scales)
                codes, scales = ref.quantize(p * p)
                got = gated.bytes.numpy()[:m, :n], gated.store.numpy()[:, :m].T
                assert same_codes(got[0], codes) and np.array_equal(got[1], scales)
        graph.close()


@pytest.mark.parametrize("m", [1, 12, 40])
def test_captured_few_rows_with_both_outputs_run_as_they_do_eagerly(m):
    rng = np.random.default_rng(m)
    n, k = 1000, 2300
    with mf.Stream(0) as own:
        a, sa = random_operands(rng, m, k, 1)
        gate, up = (held_of(*random_operands(rng, n, k, 128), own, 128) for _ in range(2))
        ha = held_of(a, sa, own, 1)
        out, q = mf.DeviceArray.empty((m, n), own), Held(m, n, own)

        def body():
            mf.gemm_f8_gated(ha.matrix, gate.matrix, up.matrix, out=out, out_f8=q.matrix)

        body()
        want, codes = out.numpy(), q.read()[0]
        graph = Graph(own, body)
        for _ in range(3):
            mf.fill(out, 3.0)
            graph.launch()
            assert same_bits(out.numpy(), want) and same_codes(q.read()[0], codes)
        graph.close()


def test_calls_repeat_bit_for_bit(stream):
    """Real values (inexact sums): every form gives the same bits on every call."""
    for m, n, k in FORMS[::3]:
        rng = np.random.default_rng(k)
        a, b = (held_of(*random_operands(rng, r, k, x), stream, x) for r, x in ((m, 1), (n, 128)))
        first = mf.gemm_f8(a.matrix, b.matrix).numpy()
        for _ in range(3):
            assert same_bits(mf.gemm_f8(a.matrix, b.matrix).numpy(), first)
