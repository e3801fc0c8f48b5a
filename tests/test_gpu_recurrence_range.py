"""The gated linear recurrence (include/acc_hip.h, section D) where products of gates, or states, leave Float32's range: against the
definition row after row in Float32, through the C ABI.

Gates are powers of two and values are 0 where results are compared bit by bit: every product is exact then, until it is beyond the
largest number, and infinite from there on, as it is in the definition.  Products stay above 2^-126, so nothing is rounded there either.
"""
import sys

import numpy as np
import pytest

from test_gpu_operators import Boxed as Bits, store, values
from test_gpu_recurrence import inputs, near, plain, sequences_of

pytestmark = pytest.mark.gpu
TYPES = ("float", "half", "bfloat16")


def say(*a):
    print("[case]", *a)
    sys.stdout.flush()


def Boxed(A, ctx, v, elt, **more):
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


def definition(keep, add, offsets, state):
    """(h, the states behind the last rows), a row at a time, in Float32"""
    h, last = np.zeros(keep.shape, np.float32), np.array(state, np.float32)
    keep, add = keep.astype(np.float32), add.astype(np.float32)
    with np.errstate(all="ignore"):
        for s in range(len(offsets) - 1):
            for t in range(offsets[s], offsets[s + 1]):
                last[s] = h[t] = keep[t] * last[s] + add[t]
    return h, last


def same(got, want):
    return np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])


def up_and_down(rng, offsets, width):
    """gates of 2 for a while, then of a half, so that a state of 2^-60 stays within 2^-110 .. 2^120 in every sequence: the products of a
    tile's gates do not"""
    gates = np.full((offsets[-1], width), 2.0)
    for begin, end in zip(offsets[:-1], offsets[1:]):
        for c in range(width):
            at, level = begin, -60
            while at < end:
                up = bool(rng.integers(0, 2)) if c % 3 else level <= 0
                n = min(int(rng.integers(1, 180)), (120 - level) if up else (level + 110), end - at)
                gates[at:at + n, c] = 2.0 if up else 0.5
                at, level = at + n, level + (n if up else -n)
    return gates


@pytest.mark.parametrize("kind", ("one", "ragged", "gaps"))
@pytest.mark.parametrize("elt", TYPES)
def test_products_of_gates_beyond_the_largest_number(A, ctx, ops, elt, kind):
    rng = np.random.default_rng(len(elt) + len(kind))
    for rows, width in ((40, 3), (700, 130), (5000, 70), (20000, 64)):
        offsets = sequences_of(rng, rows, kind)
        n = len(offsets) - 1
        say(elt, kind, rows, width)
        gates, x = np.full((rows, width), 2.0), np.zeros((rows, width))
        gates[:offsets[-1]] = up_and_down(rng, offsets, width)
        gates[:, ::5] = 16.0                                   # (these run beyond the largest number, or stay 0)
        state = np.full((n, width), 2.0 ** -60, np.float32)
        state[:, ::10] = 0.0
        want, want_last = definition(gates, x, offsets, state)
        here = np.zeros(rows, bool)
        here[offsets[0]:offsets[-1]] = True
        assert not np.isnan(want).any() and (rows < 300 or np.isinf(want).any())
        out, last = Boxed(A, ctx, np.full((rows, width), 3.0), elt), Bits(A, ctx, np.full((n, width), 3.0, np.float32), "float")
        ops(elt, "given").scan(Boxed(A, ctx, gates, elt).array, Boxed(A, ctx, x, elt).array, ctx.array(offsets), out.array, state=ctx.array(state), last=last.array)
        ctx.sync()
        got = values(out.get(), elt)
        with np.errstate(over="ignore"):
            assert same(got[here], values(store(want, elt), elt)[here]) and np.all(got[~here] == 3.0)
        assert same(last.get(), want_last)


@pytest.mark.parametrize("elt", TYPES)
def test_gradients_beyond_the_largest_number(A, ctx, ops, elt):
    """gates of 2 and gradients of 0 leave zeros; what goes on from the last row becomes infinite, and stays so"""
    rng = np.random.default_rng(3)
    for rows, width in ((700, 130), (6000, 67)):
        offsets = np.array([0, rows // 3, rows], np.int32)
        say(elt, rows, width)
        gates, zeros = np.full((rows, width), 2.0), np.zeros((rows, width))
        dlast = np.full((2, width), 2.0 ** -100, np.float32)
        dlast[:, ::2] = 0.0
        h = np.ones((rows, width))
        turned, back = np.array([0, rows - rows // 3, rows], np.int32), slice(None, None, -1)
        u, first = definition(gates, zeros, turned, dlast[back])
        g = np.empty((rows, width), np.float32)                # u[t + 1]: of the last rows dlast
        for s in range(2):
            b, e = turned[s], turned[s + 1]
            g[b], g[b + 1:e] = dlast[back][s], u[b:e - 1]
        g, dstate = g[back], first[back]
        dgates, dvalues = (Boxed(A, ctx, np.full((rows, width), 3.0), elt) for _ in range(2))
        ds = Bits(A, ctx, np.full((2, width), 3.0, np.float32), "float")
        ops(elt, "given").gradient(Boxed(A, ctx, gates, elt).array, None, ctx.array(offsets), Boxed(A, ctx, h, elt).array, Boxed(A, ctx, zeros, elt).array, dgates.array, dvalues.array,
                                   dlast=ctx.array(dlast), dstate=ds.array)
        ctx.sync()
        with np.errstate(all="ignore"):
            assert same(ds.get(), dstate) and same(values(dvalues.get(), elt), values(store(g, elt), elt))
            want = g * 1.0
            want[[0, rows // 3]] = g[[0, rows // 3]] * np.float32(0.0)         # (states of zeros come before first rows)
            assert same(values(dgates.get(), elt), values(store(want, elt), elt))


@pytest.mark.parametrize("gate", ("given", "sigmoid"))
@pytest.mark.parametrize("elt", TYPES)
def test_a_state_that_is_infinite_or_not_a_number(A, ctx, ops, elt, gate):
    """it stays what it is to the end of its sequence, however small the product of the gates is by then, and other sequences and channels do
    not notice"""
    rng, rows, width = np.random.default_rng(8), 4000, 90
    offsets = np.array([0, 1900, 2300, rows], np.int32)
    z, x = inputs(rng, rows, width, elt, gate)
    # (kept shares about a fifth, and none of 0: the product of a tile's is below the smallest number)
    z = values(store(z - 3.0 if gate == "sigmoid" else np.clip(0.4 * np.abs(z), 0.05, 0.4), elt), elt)
    state = rng.standard_normal((3, width)).astype(np.float32)
    want, want_last, bound, last_bound = plain(z, x, offsets, state.astype(np.float64), gate)
    odd = state.copy()
    odd[0, 3], odd[0, 40], odd[1, 7], odd[2, 50] = np.inf, -np.inf, np.nan, np.inf
    x = x.copy()
    x[1000, 60], x[2500, 61] = np.inf, np.nan                  # (and so a value that is)
    out, last = Boxed(A, ctx, np.zeros((rows, width)), elt), Bits(A, ctx, np.zeros((3, width), np.float32), "float")
    ops(elt, gate).scan(Boxed(A, ctx, z, elt).array, Boxed(A, ctx, x, elt).array, ctx.array(offsets), out.array, state=ctx.array(odd), last=last.array)
    ctx.sync()
    got, got_last = values(out.get(), elt), last.get().astype(np.float64)
    special = np.zeros((rows, width), bool)
    for s, c, v in ((0, 3, np.inf), (0, 40, -np.inf), (1, 7, np.nan), (2, 50, np.inf), (0, 60, np.inf), (2, 61, np.nan)):
        rows_of = slice(max(offsets[s], 1000 if c == 60 else 2500 if c == 61 else 0), offsets[s + 1])
        special[rows_of, c] = True
        assert same(got[rows_of, c], np.full(rows_of.stop - rows_of.start, v)) and same(got_last[s, c:c + 1], np.array([v])), (s, c)
        want_last[s, c] = got_last[s, c] = 0.0
    near(np.where(special, 0.0, got), np.where(special, 0.0, want), bound, elt, "h")
    near(got_last, want_last, last_bound, "float", "last")


def test_gates_beyond_one_beside_others(A, ctx, ops):
    """channels whose gates' products leave the range, beside channels whose do not: those are as near as ever"""
    rng, rows, width = np.random.default_rng(9), 9000, 200
    offsets = sequences_of(rng, rows, "ragged")
    z, x = inputs(rng, rows, width, "float", "given")
    wild = np.zeros(width, bool)
    wild[::7] = True
    z[:, wild], x[:, wild] = 4.0, 0.0
    n = len(offsets) - 1
    state = rng.standard_normal((n, width)).astype(np.float32)
    state[:, wild] = 0.0
    want, want_last, bound, last_bound = plain(z, x, offsets, state.astype(np.float64), "given")
    out, last = Boxed(A, ctx, np.zeros((rows, width)), "float"), Bits(A, ctx, np.zeros((n, width), np.float32), "float")
    ops("float", "given").scan(Boxed(A, ctx, z, "float").array, Boxed(A, ctx, x, "float").array, ctx.array(offsets), out.array, state=ctx.array(state), last=last.array)
    ctx.sync()
    assert np.all(out.get()[:, wild] == 0.0)
    near(out.get().astype(np.float64), want, bound, "float", "h")
    near(last.get().astype(np.float64), want_last, last_bound, "float", "last")
