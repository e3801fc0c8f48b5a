"""The gated linear recurrence (include/acc_hip.h, section D) against its definition in 64 bits, row after row, through the C ABI.

Error bound.  h[t] is a sum over the rows s up to t of a product of t - s kept shares and what row s adds.  In Float32 every factor
carries the relative error of its gate, GATE units of 2^-24, and of its multiplication, one; a sum's rounding is one unit of every term
per row that it passes, and the halves in which a tile's map is put together and applied add no more than as many again.  So a
term's error is at most (t - s + 1) (GATE + 4) + 8 units of itself; the bound below adds these up beside the recurrence.  A gate by
1 / (1 + e^-z): the exponent's rounding shows in e^-z as up to |z| units, the exponential, the sum, the reciprocal and the product
as up to 6 together; gates here are up to 12, so GATE is 18.  A given gate has none.
"""
import sys

import numpy as np
import pytest

from test_gpu_operators import HALF_ULP, TINY, Boxed as Bits, store, values

pytestmark = pytest.mark.gpu
TYPES = ("float", "half", "bfloat16")
UNIT = 2.0 ** -24
GATE = {"given": 0, "sigmoid": 18}


def say(*a):
    print("[case]", *a)
    sys.stdout.flush()


def Boxed(A, ctx, v, elt, **more):
    """an array of values inside a larger one"""
    return Bits(A, ctx, store(v, elt), elt, **more)


@pytest.fixture(scope="module")
def A():
    import acchip
    return acchip


@pytest.fixture(scope="module")
def ctx(A):
    c = A.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def ops(A, ctx):
    made = {}

    def get(elt, gate):
        if (elt, gate) not in made:
            made[elt, gate] = A.Recurrence(ctx, elt, gate)
        return made[elt, gate]
    yield get
    for op in made.values():
        op.destroy()


def sequences_of(rng, rows, kind):
    if kind == "one":
        return np.array([0, rows], np.int32)
    if kind == "gaps":                                     # rows in front of the first and behind the last
        return np.sort(rng.integers(rows // 7, max(rows // 7, rows - rows // 9) + 1, 6)).astype(np.int32)
    if kind == "short":                                    # many of a few rows, some of none
        return np.concatenate([[0], np.cumsum(rng.multinomial(rows, np.full(max(1, rows // 2), 1.0 / max(1, rows // 2))))]).astype(np.int32)
    return np.concatenate([[0], np.cumsum(rng.multinomial(rows, rng.dirichlet(np.full(9, 0.5))))]).astype(np.int32)


def maps_of(gates, vals, gate):
    if gate == "given":
        return gates, vals
    keep = 1.0 / (1.0 + np.exp(-gates))
    return keep, vals / (1.0 + np.exp(gates))


def plain(gates, vals, offsets, state, gate, states=None):
    """(h, the states behind the last rows, bounds of both' errors) by rows; rows of no sequence are NaN"""
    keep, add = maps_of(gates, vals, gate)
    h, bound = np.full(gates.shape, np.nan), np.zeros(gates.shape)
    width, n = gates.shape[1], len(offsets) - 1
    last, last_bound = np.zeros((n, width)), np.zeros((n, width))
    each = GATE[gate] + 4
    for s in range(n):
        v = np.zeros(width) if state is None else state[s]
        size, paths = np.abs(v), np.zeros(width)
        for t in range(offsets[s], offsets[s + 1]):
            v = keep[t] * v + add[t]
            paths = np.abs(keep[t]) * (paths + each * size) + (each + 8) * np.abs(add[t])
            size = np.abs(keep[t]) * size + np.abs(add[t])
            h[t], bound[t] = v, (paths + 8 * size) * UNIT
        last[s], last_bound[s] = v, (paths + 8 * size) * UNIT
    return h, last, bound, last_bound


def inputs(rng, rows, width, elt, gate):
    z = rng.standard_normal((rows, width)) * 2.0 + 1.5 if gate == "sigmoid" else np.exp(-0.5 * np.exp(rng.standard_normal((rows, width)))) * np.where(rng.random((rows, width)) < 0.1, -1, 1)
    z = np.clip(z, -12, 12)
    return [values(store(v, elt), elt) for v in (z, rng.standard_normal((rows, width)))]


def near(got, want, bound, elt, what):
    off = np.abs(got - want)
    allowed = bound + np.abs(want) * HALF_ULP[elt] * 1.001 + TINY[elt]
    worst = np.max(off - allowed) if off.size else 0
    assert np.all(off <= allowed), "%s: %g over, at %s" % (what, worst, np.unravel_index(np.argmax(off - allowed), off.shape))


SHAPES = [(1, 1), (1, 200), (2, 3), (31, 64), (32, 2), (33, 129), (255, 65), (256, 128), (257, 127), (513, 300), (1000, 31), (3001, 130), (9000, 5)]


@pytest.mark.parametrize("gate", ("given", "sigmoid"))
@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("kind", ("one", "ragged", "gaps", "short"))
def test_recurrence_of_every_shape(A, ctx, ops, elt, gate, kind):
    rng = np.random.default_rng(len(kind) * 7 + len(elt))
    for rows, width in SHAPES:
        offsets = sequences_of(rng, rows, kind)
        say(elt, gate, kind, rows, width)
        z, x = inputs(rng, rows, width, elt, gate)
        n = len(offsets) - 1
        state = rng.standard_normal((n, width)).astype(np.float32) if rows % 2 else None
        h, last, bound, last_bound = plain(z, x, offsets, state, gate)
        loose = int(rng.integers(0, 3))
        gz, gx, out = Boxed(A, ctx, z, elt, lead=loose, extra=loose), Boxed(A, ctx, x, elt, extra=2 * loose), Boxed(A, ctx, np.full(z.shape, 7.0), elt, lead=loose, extra=1, fill=5.0)
        dlast = Boxed(A, ctx, np.zeros((n, width)), "float", extra=loose, fill=3.0)
        dstate = None if state is None else Boxed(A, ctx, state, "float", lead=1)
        ops(elt, gate).scan(gz.array, gx.array, ctx.array(offsets), out.array, state=None if state is None else dstate.array, last=dlast.array)
        ctx.sync()
        got = values(out.get(), elt)
        none = np.isnan(h)
        assert np.all(got[none] == 7.0), "rows of no sequence"
        near(got[~none], h[~none], bound[~none], elt, "h")
        near(dlast.get().astype(np.float64), last, last_bound, "float", "last")


@pytest.mark.parametrize("elt,gate", [("bfloat16", "sigmoid"), ("float", "given")])
def test_states_through_an_index_and_in_place(A, ctx, ops, elt, gate):
    """sequences enter and leave by rows of a table; an index that names none begins with zeros and is not kept; the same array"""
    rng = np.random.default_rng(5)
    for rows, width, n in ((700, 140, 9), (40, 3, 40), (9000, 66, 3)):
        say(elt, gate, rows, width, n)
        offsets = np.concatenate([[0], np.cumsum(rng.multinomial(rows, rng.dirichlet(np.full(n, 0.7))))]).astype(np.int32)
        index = rng.permutation(n + 4)[:n].astype(np.int32)
        index[::3] = [(-1, n + 4, 2 ** 31 - 1)[k % 3] for k in range(len(index[::3]))]
        table = rng.standard_normal((n + 4, width)).astype(np.float32)
        z, x = inputs(rng, rows, width, elt, gate)
        there = (index >= 0) & (index < n + 4)
        state = np.where(there[:, None], table[np.where(there, index, 0)], 0.0)
        h, last, bound, last_bound = plain(z, x, offsets, state, gate)
        d, out = ctx.array(table), Boxed(A, ctx, np.zeros(z.shape), elt)
        ops(elt, gate).scan(Boxed(A, ctx, z, elt).array, Boxed(A, ctx, x, elt).array, ctx.array(offsets), out.array, state=d, last=d, index=ctx.array(index))
        ctx.sync()
        near(values(out.get(), elt), h, bound, elt, "h")
        got = d.get().astype(np.float64)
        near(got[index[there]], last[there], last_bound[there], "float", "states")
        others = np.setdiff1d(np.arange(n + 4), index[there])
        assert np.array_equal(got[others], table[others].astype(np.float64))


def plain_gradient(z, x, offsets, h, dout, state, dlast, gate):
    """(dgates, dvalues, dstate, bounds of their errors), row after row from the last"""
    keep, _ = maps_of(z, x, gate)
    n, width = len(offsets) - 1, z.shape[1]
    dz, dx, bz, bx = (np.full(z.shape, np.nan) for _ in range(4))
    dstate, bstate = np.zeros((n, width)), np.zeros((n, width))
    each = GATE[gate] + 4
    for s in range(n):
        u = np.zeros(width) if dlast is None else dlast[s].astype(np.float64)
        size, paths = np.abs(u), np.zeros(width)
        for t in range(offsets[s + 1] - 1, offsets[s] - 1, -1):
            g, g_size, g_paths = dout[t] + u, np.abs(dout[t]) + size, paths + 8 * (np.abs(dout[t]) + size)
            before = h[t - 1] if t > offsets[s] else np.zeros(width) if state is None else state[s]
            if gate == "sigmoid":
                f, take = keep[t] * (1 - keep[t]), 1 - keep[t]
                dz[t], dx[t] = g * (before - x[t]) * f, g * take
                # (the difference is rounded once, each gate's share and the products as the bound says)
                bz[t] = UNIT * f * np.abs(before - x[t]) * (g_paths + (2 * each + 8) * g_size)
                bx[t] = UNIT * take * (g_paths + (each + 8) * g_size)
            else:
                dz[t], dx[t] = g * before, g
                bz[t], bx[t] = UNIT * np.abs(before) * (g_paths + 8 * g_size), UNIT * (g_paths + 8 * g_size)
            u = keep[t] * g
            paths = np.abs(keep[t]) * (g_paths + each * g_size)
            size = np.abs(keep[t]) * g_size
        dstate[s], bstate[s] = u, UNIT * (paths + 8 * size)
    return dz, dx, dstate, bz, bx, bstate


@pytest.mark.parametrize("gate", ("given", "sigmoid"))
@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("kind", ("one", "ragged", "gaps", "short"))
def test_gradient_of_every_shape(A, ctx, ops, elt, gate, kind):
    rng = np.random.default_rng(len(kind) * 11 + len(elt))
    for rows, width in SHAPES:
        offsets = sequences_of(rng, rows, kind)
        say(elt, gate, kind, rows, width)
        z, x = inputs(rng, rows, width, elt, gate)
        n = len(offsets) - 1
        state, dlast = (rng.standard_normal((n, width)).astype(np.float32) if rows % 2 == k else None for k in (1, 0))
        h = values(store(np.nan_to_num(plain(z, x, offsets, state, gate)[0]), elt), elt)
        dout = values(store(rng.standard_normal(z.shape), elt), elt)
        want = plain_gradient(z, x, offsets, h, dout, state, dlast, gate)
        loose = int(rng.integers(0, 3))
        dz, dx = (Boxed(A, ctx, np.full(z.shape, 7.0), elt, lead=loose, extra=1, fill=5.0) for _ in range(2))
        ds = Boxed(A, ctx, np.zeros((n, width)), "float", extra=loose, fill=3.0)
        box = lambda v, e=elt: None if v is None else Boxed(A, ctx, v, e, lead=loose, extra=loose).array
        keep = [box(z), None if gate == "given" else box(x), ctx.array(offsets), box(h), box(dout)]
        ops(elt, gate).gradient(*keep, dz.array, dx.array, state=box(state, "float"), dlast=box(dlast, "float"), dstate=ds.array)
        ctx.sync()
        none = np.isnan(want[0])
        for got, k, what in ((dz, 0, "dgates"), (dx, 1, "dvalues")):
            v = values(got.get(), elt)
            assert np.all(v[none] == 7.0), "rows of no sequence"
            near(v[~none], want[k][~none], want[3 + k][~none], elt, what)
        near(ds.get().astype(np.float64), want[2], want[5], "float", "dstate")


@pytest.mark.parametrize("gate", ("given", "sigmoid"))
def test_gradient_against_differences(A, ctx, ops, gate):
    """the loss <h, dh> + <last, dlast> in 64 bits, an input moved either way; Float32 results"""
    rng = np.random.default_rng(2)
    rows, width, offsets = 41, 3, np.array([0, 17, 17, 38, 41], np.int32)
    z, x = inputs(rng, rows, width, "float", gate)
    state, dlast = rng.standard_normal((4, width)).astype(np.float32), rng.standard_normal((4, width)).astype(np.float32)
    dout = values(store(rng.standard_normal(z.shape), "float"), "float")
    h = plain(z, x, offsets, state, gate)[0].astype(np.float32).astype(np.float64)
    dz, dx, ds = (Boxed(A, ctx, np.zeros(s), "float") for s in (z.shape, z.shape, state.shape))
    box = lambda v: Boxed(A, ctx, v, "float").array
    ops("float", gate).gradient(box(z), box(x), ctx.array(offsets), box(h), box(dout), dz.array, dx.array, state=box(state), dlast=box(dlast), dstate=ds.array)
    ctx.sync()

    def loss(z, x, state):
        h, last, _, _ = plain(z, x, offsets, state, gate)
        return np.sum(h * dout) + np.sum(last * dlast)
    given = {"z": z, "x": x, "state": state.astype(np.float64)}
    for name, got in (("z", dz), ("x", dx), ("state", ds)):
        got = got.get()
        for at in [(int(rng.integers(given[name].shape[0])), int(rng.integers(width))) for _ in range(12)]:
            moved = []
            for by in (1e-5, -1e-5):
                other = {k: v.copy() for k, v in given.items()}
                other[name][at] += by
                moved.append(loss(**other))
            slope = (moved[0] - moved[1]) / 2e-5
            # (h is rounded to Float32 for the gradient, 2^-24 of some units; differences of this step are good to 1e-8)
            assert abs(got[at] - slope) <= 1e-5 * (1 + abs(slope)), (name, at, got[at], slope)


@pytest.mark.parametrize("gate", ("given", "sigmoid"))
@pytest.mark.parametrize("elt", TYPES)
def test_one_step_of_many_sequences(A, ctx, ops, elt, gate):
    rng = np.random.default_rng(9)
    for rows, width, with_index in ((1, 1, False), (1, 4096, True), (3, 511, True), (64, 513, False), (257, 1000, True)):
        say(elt, gate, rows, width)
        z, x = inputs(rng, rows, width, elt, gate)
        n = rows + 5
        table = rng.standard_normal((n, width)).astype(np.float32)
        index = rng.permutation(n)[:rows].astype(np.int32)
        if with_index:
            index[::5] = -1
        at = index if with_index else np.arange(rows)
        there = at >= 0
        keep, add = maps_of(z, x, gate)
        want = keep * table[at] + add
        bound = UNIT * (GATE[gate] + 4) * (np.abs(keep * table[at]) + np.abs(add))
        for in_place in (False, True):
            d, out = ctx.array(table), Boxed(A, ctx, np.full(z.shape, 7.0), elt, extra=1)
            last = d if in_place else ctx.array(table)
            ops(elt, gate).step(Boxed(A, ctx, z, elt).array, Boxed(A, ctx, x, elt, lead=1).array, d, last, out.array, index=ctx.array(index) if with_index else None)
            ctx.sync()
            got = values(out.get(), elt)
            near(got[there], want[there], bound[there], elt, "h")
            assert np.all(got[~there] == 7.0)
            after = last.get().astype(np.float64)
            near(after[at[there]], want[there], bound[there], "float", "states")
            others = np.setdiff1d(np.arange(n), at[there])
            assert np.array_equal(after[others], table[others].astype(np.float64))


def test_nothing_passes_from_one_sequence_to_the_next(A, ctx, ops):
    """infinities and NaN stay in their sequence and channel; gates at the ends of their range; -inf and inf as logits"""
    rng = np.random.default_rng(3)
    rows, width, offsets = 2000, 70, np.array([0, 300, 700, 701, 1500, 2000], np.int32)
    for gate in ("given", "sigmoid"):
        z, x = inputs(rng, rows, width, "float", gate)
        clean = plain(z, x, offsets, None, gate)
        bad = x.copy()
        bad[299, 5], bad[450, 6], bad[700, 7], bad[1499, 8] = np.inf, np.nan, -np.inf, np.nan
        out = Boxed(A, ctx, np.zeros(z.shape), "float")
        ops("float", gate).scan(Boxed(A, ctx, z, "float").array, Boxed(A, ctx, bad, "float").array, ctx.array(offsets), out.array)
        ctx.sync()
        got = out.get().astype(np.float64)
        touched = np.zeros(z.shape, bool)
        touched[299:300, 5] = touched[450:700, 6] = touched[700:701, 7] = touched[1499:1500, 8] = True
        assert not np.any(np.isfinite(got[touched]))
        near(got[~touched], clean[0][~touched], clean[2][~touched], "float", gate)
    z = np.full((4, 6), np.inf)
    z[1], z[2], z[3] = -np.inf, 3e38, -3e38
    x = np.arange(24.0).reshape(4, 6) + 1
    out = Boxed(A, ctx, np.zeros(z.shape), "float")
    ops("float", "sigmoid").scan(Boxed(A, ctx, z, "float").array, Boxed(A, ctx, x, "float").array, ctx.array(np.array([0, 4], np.int32)), out.array, state=ctx.array(np.full((1, 6), 5, np.float32)))
    ctx.sync()
    assert np.array_equal(out.get(), np.stack([np.full(6, 5.0), x[1], x[1], x[3]]).astype(np.float32))


def test_the_same_bits_every_time_and_on_other_streams(A, ctx, ops):
    rng = np.random.default_rng(4)
    rows, width, offsets = 20000, 200, np.array([0, 15000, 20000], np.int32)
    z, x = inputs(rng, rows, width, "bfloat16", "sigmoid")
    gz, gx, off = Boxed(A, ctx, z, "bfloat16"), Boxed(A, ctx, x, "bfloat16"), ctx.array(offsets)
    first = None
    streams = [None, ctx.stream(), ctx.stream()]
    ctx.sync()
    outs = [Boxed(A, ctx, np.zeros(z.shape), "bfloat16") for _ in range(9)]
    for k, out in enumerate(outs):                         # (on three streams at once)
        ops("bfloat16", "sigmoid").scan(gz.array, gx.array, off, out.array, stream=streams[k % 3])
    ctx.sync()
    bits = [out.get().copy() for out in outs]
    want = plain(z, x, offsets, None, "sigmoid")
    near(values(bits[0], "bfloat16"), want[0], want[2], "bfloat16", "h")
    for b in bits[1:]:
        assert np.array_equal(b, bits[0])


def test_recorded_into_graphs_that_are_replayed_side_by_side(A):
    """two graphs on streams of their own, eager calls on a third at the same time, inputs that change between the replays"""
    import ctypes as C
    hip = C.CDLL("libamdhip64.so")
    hip.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    hip.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    hip.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    hip.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    hip.hipGraphExecDestroy.argtypes = hip.hipGraphDestroy.argtypes = [C.c_void_p]
    ctx, rng = A.Context(0), np.random.default_rng(8)
    rows, width, n = 30000, 300, 3
    op, off = A.Recurrence(ctx, "float", "sigmoid"), ctx.array(np.array([0, 20001, 20001, 29990], np.int32))
    z, x, dout = (ctx.empty((rows, width), np.float32) for _ in range(3))
    state = ctx.array(rng.standard_normal((n, width)).astype(np.float32))
    fill = lambda: [a.set(rng.standard_normal((rows, width)).astype(np.float32) + by) for a, by in ((z, 2), (x, 0), (dout, 0))]
    streams = [ctx.stream() for _ in range(3)]

    def arrays():
        made = {name: ctx.empty((rows, width), np.float32) for name in ("h", "dz", "dx", "again")}
        made.update({name: ctx.empty((n, width), np.float32) for name in ("last", "ds")})
        for a in made.values():
            a.set(np.zeros(a.shape, np.float32))
        return made

    def call(r, stream):
        op.scan(z, x, off, r["h"], state=state, last=r["last"], stream=stream)
        op.gradient(z, x, off, r["h"], dout, r["dz"], r["dx"], state=state, dstate=r["ds"], stream=stream)
        op.scan(z, r["h"], off, r["again"], stream=stream)
    made = [arrays() for _ in streams]
    fill()
    graphs = []
    for k, stream in enumerate(streams):
        call(made[k], stream)
        ctx.sync()
        if k == 2:
            break
        graph, graph_exec = C.c_void_p(), C.c_void_p()
        assert hip.hipStreamBeginCapture(stream, 2) == 0
        try:
            call(made[k], stream)
        finally:
            rc = hip.hipStreamEndCapture(stream, C.byref(graph))
        assert rc == 0 and graph.value and hip.hipGraphInstantiate(C.byref(graph_exec), graph, None, None, 0) == 0
        graphs.append((graph, graph_exec))
    for replay in range(5):
        say("replay", replay)
        fill()
        ctx.sync()
        for k in (0, 1):
            assert hip.hipGraphLaunch(graphs[k][1], streams[k]) == 0
        call(made[2], streams[2])
        call(made[2], streams[2])
        ctx.sync()
        want = {name: a.get().copy() for name, a in made[2].items()}
        for k in (0, 1):
            for name, a in made[k].items():
                assert np.array_equal(a.get(), want[name]), (replay, k, name)
    for graph, graph_exec in graphs:
        hip.hipGraphExecDestroy(graph_exec)
        hip.hipGraphDestroy(graph)
    op.destroy()
    ctx.close()


def test_recurrences_that_are_refused(A, ctx, ops):
    op = ops("float", "sigmoid")
    f = lambda *s: ctx.empty(s, np.float32)
    i = lambda *v: ctx.array(np.array(v, np.int32))
    z, x, out, off, st = f(8, 6), f(8, 6), f(8, 6), i(0, 3, 8), f(2, 6)
    wrong = [dict(gates=f(8, 5)), dict(values=f(7, 6)), dict(out=f(9, 6)), dict(out=z), dict(state=f(2, 5)), dict(last=f(2, 7)), dict(index=i(0)), dict(state=f(3, 6), last=st),
             dict(gates=A.Strided((8, 6), (1, 8), z.ptr)), dict(out=A.Strided((8, 6), (3, 1), out.ptr)), dict(offsets=f(3, 1)), dict(gates=None), dict(offsets=None), dict(out=None),
             dict(last=A.Strided((2, 6), (6, 1), z.ptr)), dict(state=A.Strided((2, 6), (6, 1), st.ptr), last=A.Strided((2, 6), (6, 1), st.ptr + 4))]
    for w in wrong:
        args = dict(gates=z, values=x, offsets=off, out=out, state=None, last=None, index=None)
        args.update(w)
        with pytest.raises((A.AccError, AttributeError)) as e:
            op.scan(**args)
        assert not isinstance(e.value, A.AccError) or e.value.code == A.ERR_INVALID
    base = dict(gates=z, values=x, offsets=off, h=f(8, 6), dout=f(8, 6), dgates=f(8, 6), dvalues=f(8, 6), state=st, dlast=None, dstate=None)
    for w in (dict(values=None), dict(h=f(8, 7)), dict(dgates=z), dict(dstate=st), dict(dstate=f(3, 6)), dict(dlast=f(1, 6)), dict(dvalues=f(7, 6))):
        with pytest.raises(A.AccError) as e:
            op.gradient(**dict(base, **w))
        assert e.value.code == A.ERR_INVALID
    same = f(8, 6)
    with pytest.raises(A.AccError):
        op.gradient(**dict(base, dgates=same, dvalues=same))
    for w in (dict(state=None), dict(last=None), dict(state=f(8, 5)), dict(index=i(0, 1)), dict(out=x)):
        with pytest.raises(A.AccError) as e:
            op.step(**dict(dict(gates=z, values=x, state=f(8, 6), last=f(8, 6), out=out, index=None), **w))
        assert e.value.code == A.ERR_INVALID
    # nothing to do
    op.scan(f(0, 6), f(0, 6), i(0), f(0, 6))
    op.scan(f(0, 6), f(0, 6), i(0, 0, 0), f(0, 6))
    op.step(f(0, 6), f(0, 6), st, f(2, 6), f(0, 6))
    last = ctx.array(np.zeros((2, 6), np.float32))
    op.scan(f(0, 6), f(0, 6), i(0, 0, 0), f(0, 6), state=ctx.array(np.full((2, 6), 4, np.float32)), last=last)
    ctx.sync()
    assert np.all(last.get() == 4)
