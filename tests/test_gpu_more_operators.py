"""The recurrence, the grouped 4-bit products and the router by scores where their calls meet: recorded into graphs and replayed beside
eager calls on other streams, and on arrays whose rows lie gigabytes apart."""
import ctypes as C
import sys

import numpy as np
import pytest

from test_gpu_operators import HALF_ULP, TINY, store, values
from test_gpu_grouped import expected, matrices, packed, weights
from test_gpu_recurrence import plain as plain_recurrence
from test_gpu_score_router import plain as plain_routing

pytestmark = pytest.mark.gpu


def say(*a):
    print("[case]", *a)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def A():
    import acchip
    return acchip


@pytest.fixture(scope="module")
def hip():
    h = C.CDLL("libamdhip64.so")
    h.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    h.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    h.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    h.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    h.hipGraphExecDestroy.argtypes = h.hipGraphDestroy.argtypes = [C.c_void_p]
    h.hipMemcpy2D.argtypes = [C.c_void_p, C.c_size_t, C.c_void_p, C.c_size_t, C.c_size_t, C.c_size_t, C.c_int]
    return h


@pytest.mark.parametrize("tokens,n", ((5, 70), (90, 70), (1300, 70), (1300, 700)))
def test_routed_products_recorded_into_graphs(A, hip, tokens, n):
    """a router, products with the experts' 4-bit matrices through its order (each form of them, by the rows that an expert has), the
    router's gradient: two graphs replayed beside eager calls on a third stream"""
    ctx, rng = A.Context(0), np.random.default_rng(tokens)
    k, e, choose, elt = 200, 8, 2, "bfloat16"
    router, product = A.ScoreRouter(ctx, elt, choose, 4, 2), A.Grouped(ctx, elt, 64)
    q, scales, zeros = matrices(rng, e, n, k, 64, elt, True, False)
    codes, scales, zeros = ctx.array(packed(q)), ctx.array(store(scales, elt)), ctx.array(zeros)
    x, logits, dw, bias = ctx.empty((tokens, k), np.uint16), ctx.empty((tokens, e), np.uint16), ctx.empty((tokens, choose), np.float32), ctx.empty((e,), np.float32)

    def fill():
        x.set(store(rng.standard_normal((tokens, k)), elt))
        logits.set(store(rng.standard_normal((tokens, e)), elt))
        dw.set(rng.standard_normal((tokens, choose)).astype(np.float32))
        bias.set((rng.standard_normal(e) * 0.1).astype(np.float32))

    def arrays():
        made = dict(experts=ctx.empty((tokens, choose), np.int32), weights=ctx.empty((tokens, choose), np.float32), offsets=ctx.empty((e + 1,), np.int32), order=ctx.empty((tokens * choose,), np.int32),
                    place=ctx.empty((tokens, choose), np.int32), out=ctx.empty((tokens * choose, n), np.uint16), back=ctx.empty((tokens, e), np.uint16))
        for a in made.values():
            a.set(np.zeros(a.shape, a.dtype))
        return made

    def call(r, stream):
        router.route(logits, r["experts"], r["weights"], r["offsets"], r["order"], r["place"], bias=bias, stream=stream)
        product.rows(x, codes, scales, r["offsets"], r["out"], zeros=zeros, index=r["order"], per=choose, stream=stream)
        router.gradient(logits, r["experts"], dw, r["back"], stream=stream)
    streams = [ctx.stream() for _ in range(3)]
    made, graphs = [arrays() for _ in streams], []
    fill()
    for j, stream in enumerate(streams):
        call(made[j], stream)
        ctx.sync()
        if j == 2:
            break
        graph, graph_exec = C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        try:
            call(made[j], stream)
        finally:
            rc = hip.hipStreamEndCapture(stream, C.byref(graph))
        assert rc == 0 and graph.value and hip.hipGraphInstantiate(C.byref(graph_exec), graph, None, None, 0) == 0
        graphs.append((graph, graph_exec))
    w = weights(q, values(scales.get(), elt), zeros.get(), 64)
    largest = weights(np.full_like(q, 15), values(scales.get(), elt), None, 64) * (63.0 / 7.0)      # s (31 + 16 + z) and more
    for replay in range(5):
        say(tokens, "replay", replay)
        fill()
        ctx.sync()
        for j in (0, 1):
            assert hip.hipGraphLaunch(graphs[j][1], streams[j]) == 0
        call(made[2], streams[2])
        call(made[2], streams[2])
        ctx.sync()
        want = {name: a.get().copy() for name, a in made[2].items()}
        for j in (0, 1):
            for name, a in made[j].items():
                assert np.array_equal(a.get(), want[name]), (replay, j, name)
        experts, _, offsets, order, _ = plain_routing(values(logits.get(), elt), bias.get(), choose, 4, 2, True, 1.0)
        assert np.array_equal(want["experts"], experts) and np.array_equal(want["offsets"], offsets) and np.array_equal(want["order"], order)
        y, size = expected(values(x.get(), elt), w, offsets, tokens * choose, order, choose)
        got = values(want["out"], elt)
        # (half a unit of every weight, where many rows share a matrix; the groups' sums; the result's rounding)
        bound = 2.0 ** -24 * (k + 8) * expected(values(x.get(), elt), largest, offsets, tokens * choose, order, choose)[1] + HALF_ULP[elt] * 1.01 * size
        assert np.all(np.abs(got - y) <= bound + HALF_ULP[elt] * 1.001 * (np.abs(y) + bound))
    for graph, graph_exec in graphs:
        hip.hipGraphExecDestroy(graph_exec)
        hip.hipGraphDestroy(graph)
    router.destroy()
    product.destroy()
    ctx.close()


class Apart(object):
    """rows of a large allocation, `pitch` elements of `size` bytes apart, `at` bytes into it"""

    def __init__(self, A, hip, memory, host, pitch, at):
        self.hip, self.host = hip, np.ascontiguousarray(host)
        self.rows, self.width = self.host.shape[0], self.host.nbytes // self.host.shape[0]
        self.ptr, self.pitch = memory.ptr + at, pitch * self.host.itemsize
        assert at + (self.rows - 1) * self.pitch + self.width <= memory.shape[0]
        assert hip.hipMemcpy2D(self.ptr, self.pitch, self.host.ctypes.data, self.width, self.width, self.rows, 1) == 0
        strides = [pitch] + [int(np.prod(host.shape[d + 1:])) for d in range(1, host.ndim)]
        self.array = A.Strided(host.shape, strides, self.ptr, memory)

    def get(self):
        out = np.empty_like(self.host)
        assert self.hip.hipMemcpy2D(out.ctypes.data, self.width, self.ptr, self.pitch, self.width, self.rows, 2) == 0
        return out


@pytest.fixture(scope="module")
def apart(A, hip):
    ctx = A.Context(0)
    memory = ctx.empty((42 << 30,), np.uint8)
    yield ctx, lambda host, pitch, at: Apart(A, hip, memory, host, pitch, at)
    ctx.close()


@pytest.mark.parametrize("elt", ("float", "bfloat16"))
def test_a_recurrence_whose_rows_lie_gigabytes_apart(A, apart, elt):
    ctx, put = apart
    rng, rows, width = np.random.default_rng(1), 90, 40
    pitch = 180 * 2 ** 20 // (4 if elt == "float" else 2)                    # 90 rows: 15.8 GiB
    z, x = values(store(rng.standard_normal((rows, width)) + 1, elt), elt), values(store(rng.standard_normal((rows, width)), elt), elt)
    offsets, state = np.array([0, 30, 30, 90], np.int32), rng.standard_normal((3, width)).astype(np.float32)
    want, _ = plain_recurrence(z, x, offsets, state.astype(np.float64), "sigmoid")[:2]
    op = A.Recurrence(ctx, elt, "sigmoid")
    bz, bx, out = put(store(z, elt), pitch, 0), put(store(x, elt), pitch, 4096), put(store(np.zeros((rows, width)), elt), pitch, 8192)
    op.scan(bz.array, bx.array, ctx.array(offsets), out.array, state=ctx.array(state))
    ctx.sync()
    assert np.all(np.abs(values(out.get(), elt) - want) <= HALF_ULP[elt] * 1.01 * np.abs(want) + 200 * 2.0 ** -24 * np.abs(want).max())
    # the gradient of the same against the same of arrays that lie together
    dout, dz, dx = put(store(rng.standard_normal((rows, width)), elt), pitch, 12288), put(store(np.zeros((rows, width)), elt), pitch, 16384), put(store(np.zeros((rows, width)), elt), pitch, 20480)
    near = [ctx.array(a.host) for a in (bz, bx)] + [ctx.array(out.get()), ctx.array(dout.host), ctx.array(dz.host), ctx.array(dx.host)]
    op.gradient(bz.array, bx.array, ctx.array(offsets), out.array, dout.array, dz.array, dx.array, state=ctx.array(state))
    op.gradient(near[0], near[1], ctx.array(offsets), near[2], near[3], near[4], near[5], state=ctx.array(state))
    ctx.sync()
    assert np.array_equal(dz.get(), near[4].get()) and np.array_equal(dx.get(), near[5].get()) and np.any(dx.get() != 0)
    # one step of sequences whose states lie as far apart, the last first
    table = put(rng.standard_normal((rows, width)).astype(np.float32), 180 * 2 ** 18, 17 << 30)
    index = np.arange(rows)[::-1].astype(np.int32)
    op.step(bz.array, bx.array, table.array, table.array, out.array, index=ctx.array(index))
    ctx.sync()
    small = ctx.array(table.host), ctx.array(store(np.zeros((rows, width)), elt))
    op.step(near[0], near[1], small[0], small[0], small[1], index=ctx.array(index))
    ctx.sync()
    assert np.array_equal(table.get(), small[0].get()) and np.array_equal(out.get(), small[1].get())
    op.destroy()


def test_tall_products_whose_arrays_lie_gigabytes_apart(A, apart):
    """the same in tiles of 64 rows by 256 columns"""
    ctx, put = apart
    rng, rows, k, n, e, elt = np.random.default_rng(5), 1300, 300, 1500, 2, "half"
    q, scales, zeros = matrices(rng, e, n, k, 64, elt, True, True)
    x, offsets, pitch = rng.integers(-3, 4, (rows, k)).astype(np.float64), np.array([0, rows // 2, rows], np.int32), (6 << 30) // rows // 16 * 8
    want, _ = expected(x, weights(q, scales, zeros, 64), offsets, rows, None, 0)
    op = A.Grouped(ctx, elt, 64)
    bx, out = put(store(x, elt), pitch, 0), put(store(np.zeros((rows, n)), elt), pitch, 4096)
    op.rows(bx.array, put(packed(q), 5 << 30, 7 << 30).array, put(store(scales, elt), 5 << 29, 18 << 30).array, ctx.array(offsets), out.array, zeros=put(zeros, 5 << 30, 30 << 30).array)
    ctx.sync()
    assert np.array_equal(out.get(), store(want, elt))
    op.destroy()


@pytest.mark.parametrize("rows", (6, 700))
def test_products_whose_arrays_lie_gigabytes_apart(A, apart, rows):
    """matrices 5 GiB apart, rows of codes 250 MiB, rows of x and of the results over 6 GiB"""
    ctx, put = apart
    rng, k, n, e, elt = np.random.default_rng(2), 300, 20, 2, "bfloat16"
    q, scales, zeros = matrices(rng, e, n, k, 32, elt, True, True)
    x = rng.integers(-3, 4, (rows, k)).astype(np.float64)
    offsets = np.array([0, rows // 2, rows], np.int32)
    want, _ = expected(x, weights(q, scales, zeros, 32), offsets, rows, None, 0)
    op, p = A.Grouped(ctx, elt, 32), packed(q)
    pitch = (6 << 30) // rows // 16 * 8                                      # x and the results in the first 6 GiB
    for name, far in (("matrices", True), ("rows of codes", False)):
        say(rows, name)
        if far:
            codes = put(p, 5 << 30, 7 << 30).array
        else:
            a = put(p.reshape(e * n, -1), 250 << 20, 7 << 30)
            codes = A.Strided((e, n, p.shape[2]), (n * (250 << 20), 250 << 20, 1), a.ptr, a)
        bs = put(store(scales, elt), 5 << 29, 18 << 30)
        bx, out = put(store(x, elt), pitch, 0), put(store(np.zeros((rows, n)), elt), pitch, 4096)
        op.rows(bx.array, codes, bs.array, ctx.array(offsets), out.array, zeros=ctx.array(zeros))
        ctx.sync()
        assert np.array_equal(out.get(), store(want, elt))
    # and the matrices made again, and made into codes, that far apart
    made = put(store(np.zeros((e, n, k)), elt), 5 << 29, 24 << 30)
    op.values(put(p, 5 << 30, 7 << 30).array, bs.array, made.array, zeros=ctx.array(zeros))
    ctx.sync()
    assert np.array_equal(made.get(), store(weights(q, scales, zeros, 32), elt))
    to = [put(np.zeros_like(p), 5 << 30, 30 << 30), put(store(np.zeros(scales.shape), elt), 5 << 29, 36 << 30), ctx.empty(zeros.shape, np.uint8)]
    near = [ctx.empty(p.shape, np.uint8), ctx.empty(scales.shape, np.uint16), ctx.empty(zeros.shape, np.uint8)]
    op.quantise(made.array, to[0].array, to[1].array, zeros=to[2])
    op.quantise(ctx.array(made.host * 0 + made.get()), near[0], near[1], zeros=near[2])
    ctx.sync()
    for a, b in zip(to, near):
        assert np.array_equal(a.get(), b.get())
    op.destroy()


def test_a_router_whose_tokens_lie_gigabytes_apart(A, apart):
    ctx, put = apart
    rng, t, e = np.random.default_rng(3), 700, 64
    op = A.ScoreRouter(ctx, "float", 4, 8, 3)
    x = rng.standard_normal((t, e)).astype(np.float32)
    pitch = 5 * 2 ** 20
    bx, back = put(x, pitch, 0), put(np.zeros((t, e), np.float32), pitch, 4096)
    r = [ctx.empty((t, 4), np.int32), ctx.empty((t, 4), np.float32), ctx.empty((e + 1,), np.int32), ctx.empty((t * 4,), np.int32), ctx.empty((t, 4), np.int32)]
    op.route(bx.array, *r)
    dw, near = ctx.array(rng.standard_normal((t, 4)).astype(np.float32)), ctx.empty((t, e), np.float32)
    op.gradient(bx.array, r[0], dw, back.array)
    op.gradient(ctx.array(x), r[0], dw, near)
    ctx.sync()
    for a, b in zip(r, plain_routing(x.astype(np.float64), None, 4, 8, 3, True, 1.0)):
        assert np.array_equal(a.get(), b) if a.dtype == np.int32 else np.allclose(a.get(), b, rtol=1e-5)
    assert np.array_equal(back.get(), near.get()) and np.any(back.get() != 0)
    op.destroy()
