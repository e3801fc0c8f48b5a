"""The operators of a layer of experts (include/acc_hip.h, section D) against plain numpy in 64 bits, through the C ABI.

Products are checked twice: on small whole numbers, whose sums are exact in Float32 whatever their order, so that the result is
the exact sum rounded once -- equal, not near; and on normal values, with the error bound of a sum of k products in Float32,
(k + 2) 2^-24 sum |x| |w|, and half a unit of the result's last place.
"""
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TYPES = ("float", "half", "bfloat16")
STORED = {"float": np.float32, "half": np.float16, "bfloat16": np.uint16}
HALF_ULP = {"float": 2.0 ** -24, "half": 2.0 ** -11, "bfloat16": 2.0 ** -8}      # of a rounding (bfloat16 keeps 8 bits)
TINY = {"float": 2.0 ** -149, "half": 2.0 ** -25, "bfloat16": 2.0 ** -133}


def say(*a):
    print("[case]", *a)
    sys.stdout.flush()


def to_bits(v):
    """Float64 values as bfloat16, nearest even, by way of Float32's bits (the values here are exact in Float32, or far from a tie)"""
    b = np.asarray(v, np.float32).view(np.uint32)
    nan = np.isnan(np.asarray(v, np.float32))
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(nan, np.uint16(0x7FC0), r)


def store(v, elt):
    return to_bits(v) if elt == "bfloat16" else np.asarray(v).astype(STORED[elt])


def values(a, elt):
    if elt == "bfloat16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


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

    def get(name, *args):
        if (name,) + args not in made:
            made[(name,) + args] = getattr(A, name)(ctx, *args)
        return made[(name,) + args]
    yield get
    for op in made.values():
        op.destroy()


class Boxed(object):
    """an array inside a larger one that is filled with `fill`: `lead` elements in front, rows `pitch` apart"""

    def __init__(self, A, ctx, host, elt, lead=0, extra=0, fill=0.0, swap=False):
        self.elt, self.swap = elt, swap
        host = np.asarray(host)
        if swap:
            host = np.ascontiguousarray(np.swapaxes(host, -1, -2))
        self.shape = host.shape
        pitch = host.shape[-1] + extra
        rows = int(np.prod(host.shape[:-1]))
        whole = np.zeros(lead + rows * pitch + 8, STORED[elt])
        whole[:] = store(np.full(whole.shape, fill), elt)
        whole[lead:lead + rows * pitch].reshape(rows, pitch)[:, :host.shape[-1]] = host.reshape(rows, host.shape[-1])
        self.lead, self.pitch, self.rows = lead, pitch, rows
        self.whole, self.dev = whole, ctx.array(whole)
        strides = [1]
        step = pitch
        for n in reversed(host.shape[:-1]):
            strides.insert(0, step)
            step *= n
        s = A.Strided(self.shape, strides, self.dev.ptr + lead * whole.itemsize, self.dev)
        self.array = s.swap() if swap else s

    def get(self):
        """the array's elements, after a check that nothing beside them has changed"""
        now = self.dev.get()
        mask = np.ones(now.shape, bool)
        n, whole = self.shape[-1], slice(self.lead, self.lead + self.rows * self.pitch)
        out = now[whole].reshape(self.rows, self.pitch)[:, :n]
        mask[whole].reshape(self.rows, self.pitch)[:, :n] = False
        assert np.array_equal(now[mask], self.whole[mask]), "written beside the result"
        out = out.reshape(self.shape)
        return np.swapaxes(out, -1, -2) if self.swap else out


def segments(rng, rows, experts, kind):
    """offsets: even shares, a skewed share with empty segments, or segments that leave rows out at either end"""
    if kind == "gaps":
        cuts = np.sort(rng.integers(rows // 5, max(rows // 5, rows - rows // 6) + 1, experts + 1))
        return cuts.astype(np.int32)
    p = np.full(experts, 1.0 / experts) if kind == "even" else rng.permutation((np.arange(experts) + 1.0) ** -1.5 * (np.arange(experts) < max(1, experts - 2)))
    return np.concatenate([[0], np.cumsum(rng.multinomial(rows, p / p.sum()))]).astype(np.int32)


def plain_rows(x, w, offsets, rows, index=None, per=0):
    r = np.arange(rows) if index is None else np.where(index < 0, -1, index // max(per, 1))
    out = np.zeros((rows, w.shape[1]))
    size = np.zeros((rows, w.shape[1]))
    for e in range(w.shape[0]):
        b, t = int(np.clip(offsets[e], 0, rows)), int(np.clip(offsets[e + 1], 0, rows))
        for m in range(b, t):
            if 0 <= r[m] < x.shape[0]:
                out[m] = w[e] @ x[r[m]]
                size[m] = np.abs(w[e]) @ np.abs(x[r[m]])
    return out, size


def plain_outer(a, b, offsets, experts, index=None, per=0):
    rows = a.shape[0]
    r = np.arange(rows) if index is None else np.where(index < 0, -1, index // max(per, 1))
    out, size = np.zeros((experts, a.shape[1], b.shape[1])), np.zeros((experts, a.shape[1], b.shape[1]))
    for e in range(experts):
        m = np.arange(int(np.clip(offsets[e], 0, rows)), int(np.clip(offsets[e + 1], 0, rows)))
        m = m[(r[m] >= 0) & (r[m] < b.shape[0])]
        out[e] = a[m].T @ b[r[m]]
        size[e] = np.abs(a[m]).T @ np.abs(b[r[m]])
    return out, size


def bound(want, size, k, elt):
    return (k + 2) * 2.0 ** -24 * size + HALF_ULP[elt] * np.abs(want) * (1 + 2.0 ** -10) + TINY[elt]


# rows, experts, n, k, segments, w's order, index (slots a token), elements in front of the arrays, elements between rows
ROWS = [
    (1, 1, 1, 1, "even", "nk", 0, 0, 0),
    (1, 3, 17, 33, "even", "kn", 0, 0, 0),
    (5, 8, 128, 64, "even", "nk", 2, 0, 0),
    (16, 8, 256, 512, "skewed", "nk", 0, 0, 0),
    (37, 70, 130, 96, "even", "kn", 0, 0, 8),
    (64, 4, 1024, 1000, "even", "nk", 1, 8, 16),
    (129, 5, 129, 127, "skewed", "nk", 3, 1, 3),
    (200, 3, 96, 200, "gaps", "kn", 2, 0, 0),
    (333, 2, 257, 65, "gaps", "nk", 0, 3, 1),
    (700, 6, 320, 136, "skewed", "kn", 0, 8, 8),
    (1500, 3, 264, 72, "even", "kn", 4, 0, 0),
    (2100, 2, 512, 200, "even", "nk", 0, 0, 0),
    (2100, 2, 300, 77, "gaps", "kn", 2, 5, 2),
    (3000, 1, 513, 130, "even", "nk", 2, 0, 8),
    # few rows and columns, long sums: in pieces
    (33, 3, 100, 2104, "even", "nk", 0, 0, 0),
    (70, 2, 33, 2101, "gaps", "kn", 2, 0, 1),
    (300, 1, 64, 1600, "even", "kn", 0, 0, 0),
    (19, 5, 7, 4099, "skewed", "nk", 0, 1, 0),
]


@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("rows,experts,n,k,kind,order,per,lead,extra", ROWS)
def test_products_of_rows(A, ctx, ops, elt, rows, experts, n, k, kind, order, per, lead, extra):
    say("rows", elt, rows, experts, n, k, kind, order, per, lead, extra)
    rng = np.random.default_rng(rows * 7 + n)
    offsets = segments(rng, rows, experts, kind)
    tokens = rows if not per else rows // per + 1
    index = rng.integers(0, tokens * per, rows).astype(np.int32) if per else None
    if per and rows > 4:
        index[rng.integers(0, rows, 3)] = (-1, tokens * per, 2 ** 31 - 1)
    for whole in (True, False):
        draw = (lambda s: rng.integers(-4, 5, s).astype(float)) if whole else rng.standard_normal
        x, w = store(draw((tokens, k)), elt), store(draw((experts, n, k)), elt)
        # what lies beside the arrays is not a number: none of it may get into a sum
        dx, dw = Boxed(A, ctx, x, elt, lead, extra, np.nan), Boxed(A, ctx, w, elt, lead, extra, np.nan, swap=order == "kn")
        out = Boxed(A, ctx, np.zeros((rows, n), STORED[elt]), elt, lead, extra, 7.0)
        ops("Product", elt).rows(dx.array, dw.array, ctx.array(offsets), out.array, index=None if index is None else ctx.array(index), per=per)
        want, size = plain_rows(values(x, elt), values(w, elt), offsets, rows, index, per)
        got = out.get()
        if whole:
            assert np.array_equal(values(got, elt), values(store(want, elt), elt))
        else:
            assert (np.abs(values(got, elt) - want) <= bound(want, size, k, elt)).all()


# rows, experts, i, j, segments, the result's order, index, elements in front, elements between rows
OUTER = [
    (1, 1, 1, 1, "even", "ij", 0, 0, 0),
    (0, 3, 40, 24, "even", "ij", 0, 0, 0),
    (7, 4, 64, 128, "skewed", "ij", 2, 0, 0),
    (65, 9, 33, 129, "even", "ji", 0, 0, 0),
    (300, 3, 136, 72, "gaps", "ij", 3, 8, 8),
    (301, 2, 131, 70, "gaps", "ji", 2, 1, 3),
    (1000, 5, 256, 128, "skewed", "ij", 0, 0, 0),
    (260, 130, 264, 256, "even", "ij", 0, 0, 0),
    (400, 131, 257, 259, "skewed", "ji", 1, 3, 0),
    # few results and long segments: sums in pieces
    (5000, 2, 70, 90, "even", "ij", 0, 0, 0),
    (3001, 3, 130, 264, "skewed", "ji", 2, 0, 0),
    (2777, 70, 33, 5, "skewed", "ij", 1, 1, 2),
    (4100, 1, 264, 256, "gaps", "ij", 2, 0, 0),
    (9000, 4, 256, 512, "gaps", "ji", 0, 0, 0),
]


@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("rows,experts,ni,nj,kind,order,per,lead,extra", OUTER)
def test_products_of_columns(A, ctx, ops, elt, rows, experts, ni, nj, kind, order, per, lead, extra):
    say("outer", elt, rows, experts, ni, nj, kind, order, per, lead, extra)
    rng = np.random.default_rng(rows * 5 + ni)
    offsets = segments(rng, rows, experts, kind)
    tokens = rows if not per else rows // per + 1
    index = rng.integers(0, tokens * per, rows).astype(np.int32) if per else None
    if per:
        index[0] = -3
    for whole in (True, False):
        draw = (lambda s: rng.integers(-4, 5, s).astype(float)) if whole else rng.standard_normal
        a, b = store(draw((rows, ni)), elt), store(draw((tokens, nj)), elt)
        da, db = Boxed(A, ctx, a, elt, lead, extra, np.nan), Boxed(A, ctx, b, elt, lead, extra, np.nan)
        out = Boxed(A, ctx, np.zeros((experts, ni, nj), STORED[elt]), elt, lead, extra, 7.0, swap=order == "ji")
        ops("Product", elt).outer(da.array, db.array, ctx.array(offsets), out.array, index=None if index is None else ctx.array(index), per=per)
        want, size = plain_outer(values(a, elt), values(b, elt), offsets, experts, index, per)
        got = out.get()
        if whole:
            assert np.array_equal(values(got, elt), values(store(want, elt), elt))
        else:
            assert (np.abs(values(got, elt) - want) <= bound(want, size, max(1, rows), elt)).all()


@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("rows,n,k", [(40, 24, 56), (300, 136, 264), (301, 70, 33)])
def test_gradients_of_the_products(A, ctx, ops, elt, rows, n, k):
    """<G, rows(x, w)> in whole numbers: the products' gradients are the formula's, and the loss moves by exactly as much
    as they say (it is linear in either operand)"""
    rng = np.random.default_rng(rows)
    experts, per = 4, 2
    tokens = rows // per + 1
    draw = lambda s: rng.integers(-1, 2, s).astype(float)
    offsets = segments(rng, rows, experts, "skewed")
    slots = rng.permutation(tokens * per)[:rows].astype(np.int32)
    x, w, g = draw((tokens, k)), draw((experts, n, k)), draw((rows, n))
    p = ops("Product", elt)
    do, di = ctx.array(offsets), ctx.array(slots)

    def forward(x, w):
        out = ctx.empty((rows, n), STORED[elt])
        p.rows(ctx.array(store(x, elt)), ctx.array(store(w, elt)), do, out, index=di, per=per)
        return values(out.get(), elt)
    dw, dxs = ctx.empty((experts, n, k), STORED[elt]), ctx.empty((rows, k), STORED[elt])
    p.outer(ctx.array(store(g, elt)), ctx.array(store(x, elt)), do, dw, index=di, per=per)
    # with respect to the rows as they were taken: the same product with the last dimensions of w exchanged
    p.rows(ctx.array(store(g, elt)), A.Strided.of(ctx.array(store(w, elt))).swap(), do, dxs)
    # ... and to the tokens they were taken from: the slots' rows summed
    place = np.full(tokens * per, -1, np.int32)
    place[slots] = np.arange(rows)
    dx = ctx.empty((tokens, k), STORED[elt])
    ops("Combiner", elt).combine(dxs, ctx.array(place.reshape(tokens, per)), None, dx)
    want_w, _ = plain_outer(g, x, offsets, experts, slots, per)
    want_s, _ = plain_rows(g, np.swapaxes(w, 1, 2), offsets, rows)
    want_x = np.zeros((tokens, k))
    np.add.at(want_x, slots // per, want_s)
    assert np.array_equal(values(dw.get(), elt), values(store(want_w, elt), elt))
    assert np.array_equal(values(dxs.get(), elt), values(store(want_s, elt), elt))
    assert np.array_equal(values(dx.get(), elt), values(store(want_x, elt), elt))
    # differences: a few elements move by one (sums of less than 256 stay exact in every type)
    if elt == "float":
        for _ in range(3):
            t, c = rng.integers(tokens), rng.integers(k)
            moved = x.copy()
            moved[t, c] += 1
            assert (g * (forward(moved, w) - forward(x, w))).sum() == want_x[t, c]
            e, i, c = rng.integers(experts), rng.integers(n), rng.integers(k)
            moved = w.copy()
            moved[e, i, c] += 1
            assert (g * (forward(x, moved) - forward(x, w))).sum() == want_w[e, i, c]


def test_segments_out_of_range_and_out_of_order_name_no_row_outside(A, ctx, ops):
    """offsets are looked at on the device: whatever they say, only rows of the arrays are read and written"""
    rng = np.random.default_rng(3)
    x, w = rng.integers(-4, 5, (50, 40)).astype(np.float32), rng.integers(-4, 5, (3, 30, 40)).astype(np.float32)
    for offsets in ([-5, 10, 20, 1000], [0, 0, 0, 0], [50, 50, 50, 50], [7, 7, 9, 9], [-2 ** 31, 0, 50, 2 ** 31 - 1]):
        offsets = np.array(offsets, np.int32)
        out = Boxed(A, ctx, np.full((50, 30), 5.0, np.float32), "float", 4, 4, 7.0)
        ops("Product", "float").rows(ctx.array(x), ctx.array(w), ctx.array(offsets), out.array)
        want, _ = plain_rows(x.astype(float), w.astype(float), offsets, 50)
        assert np.array_equal(out.get(), want)
        dw = Boxed(A, ctx, np.full((3, 30, 40), 5.0, np.float32), "float", 4, 4, 7.0)
        ops("Product", "float").outer(out.array, ctx.array(x), ctx.array(offsets), dw.array)
        assert np.array_equal(dw.get(), plain_outer(want, x.astype(float), offsets, 3)[0])
    # (starts that go back: the result is nothing in particular, but it stays where it belongs)
    out = Boxed(A, ctx, np.zeros((50, 30), np.float32), "float", 4, 4, 7.0)
    ops("Product", "float").rows(ctx.array(x), ctx.array(w), ctx.array(np.array([40, 3, 60, 5], np.int32)), out.array)
    out.get()


def test_values_that_are_no_numbers_stay_in_their_rows(A, ctx, ops):
    """an infinity or NaN in a row, in a neighbour's segment or in an expert without rows reaches the rows that use it and no other"""
    rng = np.random.default_rng(4)
    for rows, n, k in ((20, 40, 72), (600, 300, 136)):
        x, w = rng.integers(-2, 3, (rows, k)).astype(np.float32), rng.integers(-2, 3, (4, n, k)).astype(np.float32)
        offsets = np.array([0, rows // 2, rows // 2, rows - 3, rows], np.int32)
        w[1] = np.nan                                             # nobody's
        x[3, 5], x[rows - 1, 0], w[2, 7, 1] = np.nan, np.inf, np.inf
        x[rows // 2 + 1, 1] = 1.0
        out, dw = ctx.empty((rows, n), np.float32), ctx.empty((4, n, k), np.float32)
        ops("Product", "float").rows(ctx.array(x), ctx.array(w), ctx.array(offsets), out)
        with np.errstate(invalid="ignore"):
            want, _ = plain_rows(x.astype(float), w.astype(float), offsets, rows)
        got = out.get()
        clean = np.isfinite(want)
        assert np.array_equal(np.isfinite(got), clean) and np.array_equal(got[clean], want[clean])
        g = rng.integers(-2, 3, (rows, n)).astype(np.float32)
        ops("Product", "float").outer(ctx.array(g), ctx.array(x), ctx.array(offsets), dw)
        with np.errstate(invalid="ignore"):
            want, _ = plain_outer(g.astype(float), x.astype(float), offsets, 4)
        got = dw.get()
        clean = np.isfinite(want)
        assert np.array_equal(np.isfinite(got), clean) and np.array_equal(got[clean], want[clean])


def test_rows_whose_index_names_none_are_zero_whatever_they_would_meet(A, ctx, ops):
    """no row times a matrix of infinities is zeros, and a row without a partner adds nothing to a sum, not even its NaN"""
    for rows, n, k in ((10, 24, 40), (300, 264, 72)):
        x, w = np.ones((4, k), np.float32), np.full((2, n, k), np.inf, np.float32)
        w[0] = 1.0
        index = (np.arange(rows) % 4).astype(np.int32)
        index[[1, rows - 1]] = (-1, 4)
        offsets = np.array([0, rows // 2, rows], np.int32)
        out, dw = ctx.empty((rows, n), np.float32), ctx.empty((2, n, k), np.float32)
        ops("Product", "float").rows(ctx.array(x), ctx.array(w), ctx.array(offsets), out, index=ctx.array(index))
        got = out.get()
        assert (got[[1, rows - 1]] == 0).all() and np.isinf(got[rows // 2:rows - 1]).all() and (got[0] == k).all()
        g = np.ones((rows, n), np.float32)
        g[1], g[rows - 1] = np.nan, np.inf
        ops("Product", "float").outer(ctx.array(g), ctx.array(x), ctx.array(offsets), dw, index=ctx.array(index))
        got = dw.get()
        assert (got[0] == rows // 2 - 1).all() and (got[1] == rows - rows // 2 - 1).all()


def test_a_sum_of_no_products_is_zero(A, ctx, ops):
    out = ctx.array(np.full((6, 5), 3.0, np.float32))
    ops("Product", "float").rows(ctx.empty((6, 0), np.float32), ctx.empty((2, 5, 0), np.float32), ctx.array(np.array([0, 2, 6], np.int32)), out)
    assert np.array_equal(out.get(), np.zeros((6, 5)))
    out = ctx.array(np.full((6, 5), 3.0, np.float32))
    ops("Product", "float").rows(ctx.empty((6, 4), np.float32), ctx.empty((0, 5, 4), np.float32), ctx.array(np.array([0], np.int32)), out)
    assert np.array_equal(out.get(), np.zeros((6, 5)))


@pytest.mark.parametrize("elt,order,lead,extra", [("half", "nk", 0, 0), ("half", "kn", 1, 2), ("bfloat16", "nk", 3, 8), ("bfloat16", "kn", 0, 0)])
def test_large_products_of_rows_that_start_anywhere(A, ctx, ops, elt, order, lead, extra):
    """operands that are copied into whole chunks first; whole numbers, whose sums are exact"""
    rows, n, k = 2100, 1501, 1605
    say("packed", elt, order, lead, extra)
    rng = np.random.default_rng(k + lead)
    offsets, index = np.array([3, 1000, 1400, 2098], np.int32), rng.integers(-2, 2 * rows, rows).astype(np.int32)
    x, w = rng.integers(-3, 4, (rows, k)).astype(float), rng.integers(-3, 4, (3, n, k)).astype(float)
    dx, dw = Boxed(A, ctx, store(x, elt), elt, lead, extra, np.nan), Boxed(A, ctx, store(w, elt), elt, lead, extra, np.nan, swap=order == "kn")
    doff, dindex = ctx.array(offsets), ctx.array(index)
    named = np.where(index < 0, -1, index // 2)
    for use in (False, True):
        taken = np.where(named[:, None] >= 0, x[named], 0.0) if use else x
        want = np.zeros((rows, n))
        for e in range(3):
            want[offsets[e]:offsets[e + 1]] = taken[offsets[e]:offsets[e + 1]] @ w[e].T
        out = Boxed(A, ctx, np.ones((rows, n), STORED[elt]), elt, lead, extra, 7.0)
        ops("Product", elt).rows(dx.array, dw.array, doff, out.array, index=dindex if use else None, per=2 if use else 0)
        assert np.array_equal(values(out.get(), elt), values(store(want, elt), elt))
        g = rng.integers(-3, 4, (rows, n)).astype(float)
        dg = Boxed(A, ctx, store(g, elt), elt, lead, extra, np.nan)
        grad = Boxed(A, ctx, np.ones((3, n, k), STORED[elt]), elt, lead, extra, 7.0, swap=order == "kn")
        ops("Product", elt).outer(dg.array, dx.array, doff, grad.array, index=dindex if use else None, per=2 if use else 0)
        want = np.stack([g[offsets[e]:offsets[e + 1]].T @ taken[offsets[e]:offsets[e + 1]] for e in range(3)])
        assert np.array_equal(values(grad.get(), elt), values(store(want, elt), elt))


@pytest.mark.parametrize("order", ["ij", "ji"])
@pytest.mark.parametrize("elt,rows,ni,nj", [("float", 1049, 999, 131), ("bfloat16", 2086, 1005, 260), ("half", 17476, 60, 131)])
def test_no_row_behind_the_last_one_is_read(A, ctx, ops, elt, rows, ni, nj, order):
    """both operands end where an allocation of 2 MB pages does, but for less than a row; the last segment ends amid a step, and an
    index names the other operand's rows"""
    say("outer, at the end", elt, rows, ni, nj, order)
    rng = np.random.default_rng(rows)
    a = store(rng.integers(-4, 5, (rows, ni)).astype(float), elt)
    assert 0 <= -a.nbytes % (2 << 20) < a.nbytes // rows
    b = store(rng.integers(-4, 5, (rows // 2, nj)).astype(float), elt)
    offsets, index = np.array([0, 31, 900, rows], np.int32), rng.integers(0, rows, rows).astype(np.int32)
    out = Boxed(A, ctx, np.zeros((3, ni, nj), STORED[elt]), elt, 0, 0, 7.0, swap=order == "ji")
    ops("Product", elt).outer(ctx.array(a), ctx.array(b), ctx.array(offsets), out.array, index=ctx.array(index), per=2)
    want, _ = plain_outer(values(a, elt), values(b, elt), offsets, 3, index, 2)
    assert np.array_equal(values(out.get(), elt), values(store(want, elt), elt))


@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("n,k", [(40, 64), (37, 33), (300, 130), (3, 2)])
def test_an_index_of_an_operand_without_rows_names_none(A, ctx, ops, elt, n, k):
    say("no rows", elt, n, k)
    rows, offsets, index = 70, ctx.array(np.array([0, 30, 70], np.int32)), ctx.array(np.arange(70, dtype=np.int32))
    none = A.Strided((0, k), (k, 1), 0)
    out = Boxed(A, ctx, np.ones((rows, n), STORED[elt]), elt, 0, 0, 7.0)
    for order in ("nk", "kn"):
        w = Boxed(A, ctx, store(np.full((2, n, k), np.inf), elt), elt, swap=order == "kn")
        ops("Product", elt).rows(none, w.array, offsets, out.array, index=index)
        assert np.array_equal(values(out.get(), elt), np.zeros((rows, n)))
    for order in ("ij", "ji"):
        dw = Boxed(A, ctx, np.ones((2, n, k), STORED[elt]), elt, 0, 0, 7.0, swap=order == "ji")
        ops("Product", elt).outer(ctx.array(store(np.full((rows, n), np.inf), elt)), none, offsets, dw.array, index=index)
        assert np.array_equal(values(dw.get(), elt), np.zeros((2, n, k)))


# ------------------------------------------------------------------------------ the router

def plain_route(logits, choose, normalise):
    t, e = logits.shape
    x = np.where(np.isnan(logits), -np.inf, logits)
    experts, weights = np.full((t, choose), -1, np.int32), np.zeros((t, choose))
    if t > 2000:                                     # many tokens: by rows at a time, what the loop below does one by one
        top = np.max(x, axis=1, keepdims=True)
        with np.errstate(invalid="ignore"):
            power = np.where(x == top, 1.0, np.exp(np.where(x == top, 0.0, x - top)))
        power[x == -np.inf] = 0.0
        best = np.argsort(-x, axis=1, kind="stable")[:, :choose]
        there = np.take_along_axis(x, best, 1) > -np.inf
        experts[:] = np.where(there, best, -1)
        taken = np.take_along_axis(power, best, 1) * there
        total = (taken if normalise else power).sum(1, keepdims=True)
        weights[:] = np.divide(taken, total, out=np.zeros_like(taken), where=there)
    for r in range(t if t <= 2000 else 0):
        best = [i for i in np.argsort(-x[r], kind="stable") if x[r, i] > -np.inf]
        top = x[r, best[0]] if best else 0.0
        with np.errstate(invalid="ignore"):
            power = np.where(x[r] == top, 1.0, np.exp(np.where(x[r] == top, 0.0, x[r] - top)))
        power[x[r] == -np.inf] = 0.0
        best = best[:choose]
        experts[r, :len(best)] = best
        total = power[best].sum() if normalise else power.sum()
        weights[r, :len(best)] = power[best] / total if best else 0.0
    flat = experts.reshape(-1)
    order = [s for i in range(e) for s in np.nonzero(flat == i)[0]]
    offsets = np.concatenate([[0], np.cumsum([(flat == i).sum() for i in range(e)])])
    place = np.full(t * choose, -1)
    place[order] = np.arange(len(order))
    return experts, weights, offsets, np.concatenate([order, np.full(t * choose - len(order), -1)]).astype(int), place.reshape(t, choose)


def router_logits(rng, tokens, experts, elt):
    """normal values, many of them equal, with rows that have nothing, one or too few to choose from, and values of every odd kind"""
    x = np.round(rng.standard_normal((tokens, experts)) * 4) / 4 if tokens % 2 else rng.standard_normal((tokens, experts)) * 3
    x = values(store(x, elt), elt)
    lowest = -65504.0 if elt == "half" else -3.0e38
    odd = [np.full(experts, -np.inf), np.full(experts, np.nan), np.full(experts, values(store(np.array(lowest), elt), elt)), np.zeros(experts)]
    one = np.full(experts, -np.inf)
    one[experts // 2] = -2.0
    some = x[0].copy()
    some[::2] = np.nan
    top = x[0].copy()
    top[experts // 3] = np.inf
    signed = np.zeros(experts)
    signed[::2] = -0.0
    for k, row in enumerate(odd + [one, some, top, signed]):
        if k + 1 < tokens:
            x[k + 1] = row
    return x


ROUTE = [(1, 1, 1), (1, 4, 4), (8, 64, 4), (9, 7, 3), (12, 2, 1), (64, 8, 2), (255, 16, 2), (256, 60, 4), (257, 128, 8), (700, 33, 5), (1000, 256, 8), (300, 513, 6),
         (40, 2048, 16), (530, 100, 64), (16400, 72, 8), (16384, 37, 3), (20011, 8, 1),
         (32768, 72, 8), (32801, 128, 7), (65537, 40, 4), (65600, 8, 1), (100, 512, 8), (515, 300, 3)]


@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("tokens,experts,choose", ROUTE)
def test_routes(A, ctx, ops, elt, tokens, experts, choose):
    say("route", elt, tokens, experts, choose)
    rng = np.random.default_rng(tokens + experts)
    x = router_logits(rng, tokens, experts, elt)
    for normalise, lead, extra in ((True, 0, 0), (False, 3, 5)):
        logits = Boxed(A, ctx, store(x, elt), elt, lead, extra, 99.0)
        got = [ctx.array(np.full(s, -7, np.int32)) for s in ((tokens, choose), (experts + 1,), (tokens * choose,), (tokens, choose))]
        weights = ctx.array(np.full((tokens, choose), np.nan, np.float32))
        ops("Router", elt, choose, normalise).route(logits.array, got[0], weights, got[1], got[2], got[3])
        want = plain_route(x, choose, normalise)
        for g, w in zip(got, (want[0], want[2], want[3], want[4])):
            assert np.array_equal(g.get(), w)
        # a weight is a quotient of powers in Float32: an exponential (within 2 units of its last place, and 2^-24 |x - top| for
        # its rounded argument), a sum of `experts` of them, a division
        err = (experts + 8) * 2.0 ** -24 + 100 * 2.0 ** -23
        assert (np.abs(weights.get() - want[1]) <= err * want[1] + 2.0 ** -126).all()


@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("tokens,experts,choose", [(1, 4, 2), (33, 7, 3), (300, 64, 4), (100, 130, 8), (17, 600, 5)])
def test_gradient_of_the_router(A, ctx, ops, elt, tokens, experts, choose):
    """against the formula, and against differences of the weights in 64 bits"""
    rng = np.random.default_rng(tokens)
    x = values(store(rng.standard_normal((tokens, experts)), elt), elt)
    if tokens > 2:
        x[1] = -np.inf
        x[2, ::2] = -np.inf
    dw = rng.standard_normal((tokens, choose)).astype(np.float32)
    for normalise, lead, extra in ((True, 0, 0), (False, 1, 2)):
        chosen, weights, _, _, _ = plain_route(x, choose, normalise)
        out = Boxed(A, ctx, np.zeros((tokens, experts), STORED[elt]), elt, lead, extra, 7.0)
        logits = Boxed(A, ctx, store(x, elt), elt, lead, extra, 99.0)
        ops("Router", elt, choose, normalise).gradient(logits.array, ctx.array(chosen), ctx.array(weights.astype(np.float32)), ctx.array(dw), out.array)
        got = values(out.get(), elt)
        want, size = np.zeros((tokens, experts)), np.zeros((tokens, experts))
        for t in range(tokens):
            some = x[t] > -np.inf
            if not some.any():
                continue
            p = np.where(some, np.exp(np.where(some, x[t], 0.0)), 0.0)
            take = [e for e in chosen[t] if e >= 0]
            if normalise:
                p[[e for e in range(experts) if e not in take]] = 0.0
            p /= p.sum()
            d = np.zeros(experts)
            d[take] = dw[t, :len(take)]
            want[t] = p * (d - (p * d).sum())
            size[t] = p * (np.abs(d) + (p * np.abs(d)).sum())
        # weights and their products with dw are each off by the bound of the forward test, their differences by both
        err = 4 * ((experts + choose + 8) * 2.0 ** -24 + 100 * 2.0 ** -23)
        assert (np.abs(got - want) <= err * size + HALF_ULP[elt] * np.abs(want) * 1.001 + TINY[elt]).all()
        # differences: the chosen stay the chosen under a step this small (no two logits are that near, and the step's error is h^2)
        for t in (0, tokens - 1):
            for e in rng.integers(0, experts, 4):
                if x[t, e] == -np.inf:
                    continue
                h = 1e-5

                def loss(step):
                    z = x[t].copy()
                    z[e] += step
                    p = np.exp(z - z[z > -np.inf].max())
                    take = [i for i in chosen[t] if i >= 0]
                    return (p[take] / (p[take].sum() if normalise else p.sum()) * dw[t, :len(take)]).sum()
                assert abs((loss(h) - loss(-h)) / (2 * h) - want[t, e]) < 1e-8


# ------------------------------------------------------------------------------ the combination

@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("tokens,choose,width,lead,extra", [(1, 1, 1, 0, 0), (3, 2, 8, 0, 0), (50, 4, 264, 0, 8), (33, 6, 131, 1, 2), (130, 9, 72, 0, 0), (7, 3, 2048, 8, 0), (5, 2, 1501, 0, 0),
                                                               (6, 67, 40, 0, 0), (5, 130, 19, 1, 1), (4, 3, 5003, 0, 3), (9, 5, 7, 0, 0), (3, 64, 12, 0, 4)])
def test_combination_and_its_gradient(A, ctx, ops, elt, tokens, choose, width, lead, extra):
    say("combine", elt, tokens, choose, width, lead, extra)
    rng = np.random.default_rng(tokens + width)
    rows = tokens * choose + 3
    place = rng.permutation(rows)[:tokens * choose].astype(np.int32).reshape(tokens, choose)
    if tokens > 1:
        place[0] = -1
        place[1, 0] = rows
        place[-1, -1] = -5
    weights = rng.random((tokens, choose)).astype(np.float32)
    y, dout = store(rng.standard_normal((rows, width)), elt), store(rng.standard_normal((tokens, width)), elt)
    there = (place >= 0) & (place < rows)
    yv, dv = values(y, elt), values(dout, elt)
    taken = np.where(there[:, :, None], yv[np.where(there, place, 0)], 0.0)
    op = ops("Combiner", elt)
    by, bd = Boxed(A, ctx, y, elt, lead, extra, np.nan), Boxed(A, ctx, dout, elt, lead, extra, np.nan)
    dplace, dweights = ctx.array(place), ctx.array(weights)
    for w in (weights, None):
        out = Boxed(A, ctx, np.zeros((tokens, width), STORED[elt]), elt, lead, extra, 7.0)
        op.combine(by.array, dplace, None if w is None else dweights, out.array)
        f = np.ones((tokens, choose)) if w is None else w.astype(float)
        want, size = (taken * f[:, :, None]).sum(1), np.abs(taken * f[:, :, None]).sum(1)
        assert (np.abs(values(out.get(), elt) - want) <= bound(want, size, choose, elt)).all()
        # the gradient: rows that no slot has keep what they held
        dy, dw = Boxed(A, ctx, np.full((rows, width), 3, STORED[elt]), elt, lead, extra, 7.0), ctx.array(np.full((tokens, choose), np.nan, np.float32))
        op.gradient(bd.array, by.array, dplace, None if w is None else dweights, dy.array, dw)
        got = dy.get()
        want = np.full((rows, width), np.nan)
        for t in range(tokens):
            for j in range(choose):
                if there[t, j]:
                    want[place[t, j]] = f[t, j] * dv[t]
        written = ~np.isnan(want[:, 0])
        assert (np.abs(values(got, elt)[written] - want[written]) <= bound(want[written], np.abs(want[written]), 1, elt)).all()
        assert np.array_equal(got[~written], np.full((rows, width), 3, STORED[elt])[~written])
        wdw, sdw = (taken * dv[:, None, :]).sum(2), np.abs(taken * dv[:, None, :]).sum(2)
        assert (np.abs(dw.get() - wdw) <= (width + 2) * 2.0 ** -24 * sdw + 2.0 ** -126).all()
        # without the weights' gradient
        dy2 = Boxed(A, ctx, np.full((rows, width), 3, STORED[elt]), elt, lead, extra, 7.0)
        op.gradient(bd.array, None, dplace, None if w is None else dweights, dy2.array, None)
        assert np.array_equal(dy2.get(), got)
    # differences: the loss <dout, out> is linear in y and in the weights, and its slopes are what the gradient gave
    t, j, c = tokens - 1, 0, width // 2
    if there[t, j]:
        step = weights.astype(float).copy()
        step[t, j] += 0.5
        moved = (dv * (taken * step[:, :, None]).sum(1)).sum() - (dv * (taken * weights[:, :, None].astype(float)).sum(1)).sum()
        assert abs(moved / 0.5 - wdw[t, j]) <= 1e-9 * (1 + np.abs(dv).sum())


# ------------------------------------------------------------------------------ 4-bit numbers

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def plain_quantise(x):
    """(codes by element, scale bytes, values) of rows in 64 bits"""
    rows, k = x.shape
    b = (k + 31) // 32
    v = np.zeros((rows, b * 32))
    v[:, :k] = x
    v = v.reshape(rows, b, 32)
    most = np.abs(v).max(2)
    bad = ~np.isfinite(most)
    with np.errstate(divide="ignore", invalid="ignore"):
        power = np.where(most > 0, np.frexp(np.where(bad, 1.0, most))[1] - 1 - 2, -127)
    power = np.maximum(power, -127)
    a = np.abs(np.where(bad[:, :, None], 0.0, v)) / 2.0 ** power[:, :, None]
    off = np.abs(np.minimum(a, 6.0)[..., None] - GRID)
    near = off == off.min(-1, keepdims=True)
    code = np.where(near, np.where(np.arange(8) % 2 == 0, 2, 1), 0).argmax(-1)
    vals = np.where(bad[:, :, None], np.nan, np.copysign(GRID[code], v) * 2.0 ** power[:, :, None])
    code = np.where(bad[:, :, None], 0, code + 8 * np.signbit(v))
    return code.reshape(rows, -1), np.where(bad, 255, power + 127).astype(np.uint8), vals.reshape(rows, -1)[:, :k]


def packed(code):
    return (code[:, 0::2] + 16 * code[:, 1::2]).astype(np.uint8)


def micro_values(rng, rows, k, elt):
    x = rng.standard_normal((rows, k)) * 2.0 ** rng.integers(-8, 9, (rows, 1))
    x[0] = np.resize([0.0, -0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -7.5, 0.2499, 0.2501, 4.99, 5.01], k)
    if rows > 1:
        x[1] = 0.0
    if rows > 2:
        x[2] = np.resize([-0.0, 6.0e-8, 1.0e-7], k) if elt == "half" else np.resize([1e-39, -3e-39, 1.2e-38, 0.0], k)
    if rows > 3:
        x[3] = np.resize([6.0e4, -3.0e4] if elt == "half" else [3.0e38, -1.0e38, 2.9e38], k)
    if rows > 4:
        x[4, k // 2] = np.nan
    if rows > 5:
        x[5, 0] = -np.inf
    return store(x, elt)


@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("rows,k,lead,extra", [(1, 1, 0, 0), (3, 32, 0, 0), (9, 100, 0, 0), (70, 256, 8, 8), (33, 77, 1, 3), (257, 1000, 0, 0)])
def test_four_bit_numbers(A, ctx, ops, elt, rows, k, lead, extra):
    say("micro", elt, rows, k, lead, extra)
    x = micro_values(np.random.default_rng(rows), rows, k, elt)
    b = (k + 31) // 32
    codes, scales = ctx.array(np.full((rows, 16 * b), 0xAB, np.uint8)), ctx.array(np.full((rows, b), 0xAB, np.uint8))
    op = ops("Microscale", elt)
    op.quantise(Boxed(A, ctx, x, elt, lead, extra, 99.0).array, codes, scales)
    want_codes, want_scales, want = plain_quantise(values(x, elt))
    assert np.array_equal(scales.get(), want_scales)
    assert np.array_equal(codes.get(), packed(want_codes))
    out = Boxed(A, ctx, np.zeros((rows, k), STORED[elt]), elt, lead, extra, 7.0)
    op.values(codes, scales, out.array)
    got = out.get()
    assert np.array_equal(values(got, elt), values(store(want, elt), elt), equal_nan=True)
    # what has been rounded is rounded to itself
    again = ctx.empty((rows, 16 * b), np.uint8), ctx.empty((rows, b), np.uint8)
    fine = np.isfinite(values(got, elt)).all(1)
    if elt == "float":
        op.quantise(ctx.array(np.ascontiguousarray(got)), *again)
        out2 = ctx.empty((rows, k), STORED[elt])
        op.values(again[0], again[1], out2)
        assert np.array_equal(out2.get()[fine], got[fine])


@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("rows,experts,n,k,kind,per", [(60, 3, 130, 4000, "gaps", 0), (100, 2, 64, 4096, "even", 2), (1, 1, 1, 1, "even", 0), (5, 3, 40, 70, "even", 2), (33, 8, 256, 128, "skewed", 0), (90, 2, 129, 544, "gaps", 3),
                                                       (300, 4, 300, 1000, "skewed", 0), (1100, 2, 520, 256, "even", 2), (600, 1, 256, 1040, "gaps", 0)])
def test_products_of_four_bit_numbers(A, ctx, ops, elt, rows, experts, n, k, kind, per):
    say("micro rows", elt, rows, experts, n, k, kind, per)
    rng = np.random.default_rng(n + k)
    offsets = segments(rng, rows, experts, kind)
    tokens = rows if not per else rows // per + 1
    index = rng.integers(0, tokens * per, rows).astype(np.int32) if per else None
    if per and rows > 4:
        index[rng.integers(0, rows, 3)] = (-1, tokens * per, 2 ** 31 - 1)
    xc, xs, xv = plain_quantise(rng.standard_normal((tokens, k)) * 2.0 ** rng.integers(-3, 4, (tokens, 1)))
    wc, ws, wv = plain_quantise(rng.standard_normal((experts * n, k)) * 2.0 ** rng.integers(-3, 4, (experts * n, 1)))
    b = (k + 31) // 32
    out = Boxed(A, ctx, np.zeros((rows, n), STORED[elt]), elt, 8, 8, 7.0)
    ops("Microscale", elt).rows(ctx.array(packed(xc)), ctx.array(xs), ctx.array(packed(wc).reshape(experts, n, 16 * b)), ctx.array(ws.reshape(experts, n, b)),
                                ctx.array(offsets), out.array, index=None if index is None else ctx.array(index), per=per)
    want, size = plain_rows(xv, wv.reshape(experts, n, k), offsets, rows, index, per)
    assert (np.abs(values(out.get(), elt) - want) <= bound(want, size, k, elt)).all()
    # a block that is not a number reaches its row and its column
    xs[0, 0], ws[1 % ws.shape[0], 0] = 255, 255
    ops("Microscale", elt).rows(ctx.array(packed(xc)), ctx.array(xs), ctx.array(packed(wc).reshape(experts, n, 16 * b)), ctx.array(ws.reshape(experts, n, b)),
                                ctx.array(offsets), out.array, index=None if index is None else ctx.array(index), per=per)
    r = np.arange(rows) if index is None else np.where(index < 0, -1, index // max(per, 1))
    got = np.isnan(values(out.get(), elt))
    inside = np.zeros((rows, n), bool)
    for e in range(experts):
        for m in range(offsets[e], offsets[e + 1]):
            if 0 <= r[m] < tokens:
                inside[m] = r[m] == 0
                if e == 0:
                    inside[m, 1 % ws.shape[0]:1 % ws.shape[0] + 1] = True
    if n > 1:
        assert np.array_equal(got, inside)


# ------------------------------------------------------------------------------ streams, loops, refusals

def test_operators_on_a_stream_of_their_own_and_under_a_guard(A, ctx, ops):
    rng = np.random.default_rng(8)
    x, w = rng.integers(-4, 5, (40, 64)).astype(np.float32), rng.integers(-4, 5, (2, 48, 64)).astype(np.float32)
    offsets = np.array([0, 13, 40], np.int32)
    want, _ = plain_rows(x.astype(float), w.astype(float), offsets, 40)
    stream, guard = ctx.stream(), A.Guard(ctx)
    dx, dw, do = ctx.array(x), ctx.array(w), ctx.array(offsets)
    out = ctx.array(np.full((40, 48), 3.0, np.float32))
    guard.attach(stream)
    guard.reset(stream)
    p = ops("Product", "float")
    p.rows(dx, dw, do, out, stream=stream)
    A.check(A.lib().acc_stream_sync(ctx.handle, stream))
    assert np.array_equal(out.get(), want)
    # the guard goes down: nothing is written any more, by any of them
    guard.latch(ctx.empty((), np.uint8).set(np.zeros((), np.uint8)), stream)
    held = {}

    def kept(name, shape, dtype):
        held[name] = (ctx.array(np.full(shape, 3, dtype)), np.full(shape, 3, dtype))
        return held[name][0]
    c, o = ctx.array(np.zeros((4, 32), np.uint8)), np.float32
    place = ctx.array(np.zeros((2, 1), np.int32))
    p.rows(dx, dw, do, kept("rows", (40, 48), o), stream=stream)
    p.outer(dx, dx, do, kept("outer", (2, 64, 64), o), stream=stream)
    ops("Router", "float", 2, True).route(dx, kept("e", (40, 2), np.int32), kept("w", (40, 2), o), kept("o", (65,), np.int32), kept("r", (80,), np.int32),
                                          kept("p", (40, 2), np.int32), stream=stream)
    ops("Router", "float", 2, True).gradient(dx, ctx.array(np.zeros((40, 2), np.int32)), ctx.array(np.zeros((40, 2), o)), ctx.array(np.zeros((40, 2), o)),
                                             kept("g", (40, 64), o), stream=stream)
    ops("Combiner", "float").combine(dx, place, None, kept("c", (2, 64), o), stream=stream)
    ops("Combiner", "float").gradient(ctx.array(np.zeros((2, 64), o)), dx, place, None, kept("dy", (40, 64), o), kept("dw", (2, 1), o), stream=stream)
    ops("Microscale", "float").quantise(dx, kept("q", (40, 32), np.uint8), kept("s", (40, 2), np.uint8), stream=stream)
    ops("Microscale", "float").values(c, ctx.array(np.zeros((4, 2), np.uint8)), kept("v", (4, 64), o), stream=stream)
    ops("Microscale", "float").rows(c, ctx.array(np.zeros((4, 2), np.uint8)), ctx.array(np.zeros((1, 5, 32), np.uint8)), ctx.array(np.zeros((1, 5, 2), np.uint8)),
                                    ctx.array(np.array([0, 4], np.int32)), kept("m", (4, 5), o), stream=stream)
    A.check(A.lib().acc_stream_sync(ctx.handle, stream))
    for name, (dev, was) in held.items():
        assert np.array_equal(dev.get(), was), name
    guard.detach(stream)
    guard.destroy()
    A.check(A.lib().acc_stream_destroy(ctx.handle, stream))


def test_calls_that_are_refused(A, ctx, ops):
    f, i = (lambda *s: ctx.empty(s, np.float32)), (lambda *s: ctx.empty(s, np.int32))
    u = lambda *s: ctx.empty(s, np.uint8)
    p, r, c, m = ops("Product", "float"), ops("Router", "float", 2, True), ops("Combiner", "float"), ops("Microscale", "float")
    x = f(6, 8)
    S = A.Strided

    def refused(call, *args, **kw):
        with pytest.raises(A.AccError) as e:
            call(*args, **kw)
        assert e.value.code == A.ERR_INVALID and e.value.message
    refused(p.rows, f(6, 8), f(2, 5, 9), i(3), f(6, 5))                          # another k
    refused(p.rows, f(6, 8), f(2, 5, 8), i(4), f(6, 5))                          # too many offsets
    refused(p.rows, f(7, 8), f(2, 5, 8), i(3), f(6, 5))                          # other rows
    refused(p.rows, f(6, 8), f(2, 5, 8), i(3), f(6, 4))                          # another n
    refused(p.rows, f(6, 8), f(5, 8), i(3), f(6, 5))                             # w of rank 2
    refused(p.rows, f(9, 8), f(2, 5, 8), i(3), f(6, 5), index=i(5))              # too short an index
    refused(p.rows, f(6, 8), f(2, 5, 8), i(3), f(6, 5), per=-1)
    refused(p.rows, None, f(2, 5, 8), i(3), f(6, 5))
    refused(p.rows, S((6, 8), (8, 1), 0), f(2, 5, 8), i(3), f(6, 5))             # NULL
    refused(p.rows, S((6, 8), (1, 6), x.ptr, x), f(2, 5, 8), i(3), f(6, 5))      # columns in memory
    refused(p.rows, S((6, 8), (-8, 1), x.ptr, x), f(2, 5, 8), i(3), f(6, 5))
    refused(p.rows, x, f(2, 8, 8), i(3), x)                                      # in place
    refused(p.rows, x, S((2, 2, 8), (4, 2, 3), x.ptr, x), i(3), f(6, 2))         # neither way contiguous
    refused(p.rows, f(6, 8), f(2, 5, 8), i(3), S((6, 5), (4, 1), x.ptr, x))      # rows of the result overlap
    refused(p.rows, S((6, -8), (8, 1), x.ptr, x), f(2, 5, 8), i(3), f(6, 5))
    refused(p.rows, S((1 << 31, 8), (8, 1), x.ptr, x), f(2, 5, 8), i(3), f(6, 5), index=i(6))
    refused(p.outer, f(6, 8), f(7, 5), i(3), f(2, 8, 5))
    refused(p.outer, f(6, 8), f(6, 5), i(3), f(2, 5, 8))
    refused(p.outer, f(6, 8), f(6, 5), i(2), f(2, 8, 5))
    refused(r.route, f(6, 1), i(6, 2), f(6, 2), i(2), i(12), i(6, 2))            # fewer experts than are chosen
    refused(r.route, f(6, 2049), i(6, 2), f(6, 2), i(2050), i(12), i(6, 2))
    refused(r.route, f(6, 8), i(6, 3), f(6, 2), i(9), i(12), i(6, 2))
    refused(r.route, f(6, 8), i(6, 2), f(6, 2), i(8), i(12), i(6, 2))
    refused(r.route, f(6, 8), i(6, 2), f(6, 2), i(9), i(11), i(6, 2))
    same = i(6, 2)
    refused(r.route, f(6, 8), same, f(6, 2), i(9), i(12), same)
    refused(r.gradient, f(6, 8), i(6, 2), f(6, 2), f(6, 1), f(6, 8))
    refused(r.gradient, f(6, 8), i(6, 2), f(6, 2), f(6, 2), f(6, 7))
    refused(c.combine, f(9, 8), i(4, 2), f(4, 3), f(4, 8))
    refused(c.combine, f(9, 8), i(4, 2), f(4, 2), f(4, 7))
    refused(c.gradient, f(4, 8), f(9, 8), i(4, 2), f(4, 2), f(8, 8), f(4, 2))
    refused(c.gradient, f(4, 8), None, i(4, 2), f(4, 2), f(8, 8), f(4, 2))       # y and dweights go together
    refused(m.quantise, f(4, 40), u(4, 32), u(4, 1))
    refused(m.quantise, f(4, 40), u(4, 16), u(4, 1))
    refused(m.values, S((4, 16), (17, 1), u(128).ptr), u(4, 1), f(4, 32))        # rows of codes that are not aligned
    refused(m.rows, u(4, 32), u(4, 2), u(2, 5, 16), u(2, 5, 1), i(3), f(4, 5))
    # one instance does not do another's work
    assert A._drivers.acc_exec_combine(p.handle, None, None, None, None, None) == A.ERR_INVALID
    assert A._drivers.acc_exec_combine(None, None, None, None, None, None) == A.ERR_INVALID
    for args in (("Product", "double"), ("Product", "Int32"), ("Router", "float", 0), ("Router", "float", 65)):
        refused(getattr(A, args[0]), ctx, *args[1:])
    assert np.array_equal(ctx.array(np.ones(3, np.float32)).get(), np.ones(3))


def test_nothing_to_do_is_no_error(A, ctx, ops):
    f, i = (lambda *s: ctx.empty(s, np.float32)), (lambda *s: ctx.empty(s, np.int32))
    ops("Product", "float").rows(f(0, 8), f(2, 5, 8), i(3), f(0, 5))
    ops("Product", "float").rows(f(6, 8), f(2, 0, 8), i(3), f(6, 0))
    offsets, none = ctx.array(np.full(9, -7, np.int32)), i(0)
    ops("Router", "float", 2, True).route(f(0, 8), i(0, 2), f(0, 2), offsets, none, i(0, 2))
    assert np.array_equal(offsets.get(), np.zeros(9))
    ops("Router", "float", 2, True).gradient(f(0, 8), i(0, 2), f(0, 2), f(0, 2), f(0, 8))
    ops("Combiner", "float").combine(f(0, 8), i(0, 2), None, f(0, 8))
    out = ctx.array(np.full((3, 8), 5.0, np.float32))
    ops("Combiner", "float").combine(f(0, 8), ctx.array(np.zeros((3, 2), np.int32)), None, out)
    assert np.array_equal(out.get(), np.zeros((3, 8)))
    ops("Microscale", "float").quantise(f(0, 40), ctx.empty((0, 32), np.uint8), ctx.empty((0, 2), np.uint8))


def test_weights_of_rows_without_columns_have_a_gradient_of_zero(A, ctx, ops):
    say("combine", "no columns")
    op = ops("Combiner", "float")
    place, weights = ctx.array(np.arange(6, dtype=np.int32).reshape(3, 2)), ctx.array(np.ones((3, 2), np.float32))
    dw = ctx.array(np.full((3, 2), np.nan, np.float32))
    empty = lambda rows: ctx.empty((rows, 0), np.float32)
    op.gradient(empty(3), empty(6), place, weights, empty(6), dw)
    assert np.array_equal(dw.get(), np.zeros((3, 2), np.float32))
    op.combine(empty(6), place, weights, empty(3))


@pytest.mark.parametrize("first", [True, False])
def test_columns_of_one_array_are_operand_and_result(A, ctx, ops, first):
    """the result beside the operand in the same rows, on either side; a column in common is refused"""
    rng = np.random.default_rng(2)
    rows, n, k, pitch = 60, 24, 40, 70
    x, w = rng.integers(-3, 4, (rows, k)).astype(np.float32), rng.integers(-3, 4, (2, n, k)).astype(np.float32)
    host = np.full((rows, pitch), 9, np.float32)
    x_at, out_at = (0, 41) if first else (29, 5)
    host[:, x_at:x_at + k] = x
    both, offsets = ctx.array(host), np.array([0, 25, 60], np.int32)
    part = lambda at, width: A.Strided((rows, width), (pitch, 1), both.ptr + 4 * at, both)
    ops("Product", "float").rows(part(x_at, k), ctx.array(w), ctx.array(offsets), part(out_at, n))
    got = both.get()
    assert np.array_equal(got[:, out_at:out_at + n], np.concatenate([x[:25] @ w[0].T, x[25:] @ w[1].T]))
    got[:, out_at:out_at + n] = 9
    assert np.array_equal(got, host)
    for at in (x_at + k - 1, x_at - n + 1):
        if 0 <= at <= pitch - n:
            with pytest.raises(A.AccError):
                ops("Product", "float").rows(part(x_at, k), ctx.array(w), ctx.array(offsets), part(at, n))


def test_a_layer_recorded_into_a_graph_and_replayed_on_changing_inputs(A, ops):
    """router, products with pieces and copies, combination and gradient in one graph; eager calls of the same between the replays"""
    import ctypes as C
    hip = C.CDLL("libamdhip64.so")
    hip.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    hip.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    hip.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    hip.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    hip.hipGraphExecDestroy.argtypes = hip.hipGraphDestroy.argtypes = [C.c_void_p]
    ctx = A.Context(0)
    stream, rng = ctx.stream(), np.random.default_rng(8)
    tokens, experts, choose, width, hidden = 1200, 96, 2, 515, 2051
    slots = tokens * choose
    x, logits = ctx.empty((tokens, width), np.float16), ctx.empty((tokens, experts), np.float16)
    w = ctx.array(rng.integers(-2, 3, (experts, hidden, width)).astype(np.float16))
    router, product, comb = A.Router(ctx, "half", choose, True), A.Product(ctx, "half"), A.Combiner(ctx, "half")

    def arrays():
        return dict(chosen=ctx.empty((tokens, choose), np.int32), weights=ctx.empty((tokens, choose), np.float32), offsets=ctx.empty((experts + 1,), np.int32),
                    order=ctx.empty((slots,), np.int32), place=ctx.empty((tokens, choose), np.int32), h=ctx.empty((slots, hidden), np.float16),
                    out=ctx.empty((tokens, hidden), np.float16), few=ctx.empty((2, 40, 24), np.float16))

    def call(r):
        router.route(logits, r["chosen"], r["weights"], r["offsets"], r["order"], r["place"], stream=stream)
        product.rows(x, w, r["offsets"], r["h"], index=r["order"], per=choose, stream=stream)
        comb.combine(r["h"], r["place"], r["weights"], r["out"], stream=stream)
        column = lambda n: A.Strided((tokens, n), (width, 1), x.ptr, x)
        product.outer(column(40), column(24), halves, r["few"], stream=stream)
    halves = ctx.array(np.array([0, 600, tokens], np.int32))
    recorded, eager = arrays(), arrays()
    fill = lambda: (x.set(rng.integers(-2, 3, (tokens, width)).astype(np.float16)), logits.set(rng.standard_normal((tokens, experts)).astype(np.float16)))
    fill()
    call(eager)
    ctx.sync()
    graph, graph_exec = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    try:
        call(recorded)
    finally:
        rc = hip.hipStreamEndCapture(stream, C.byref(graph))
    assert rc == 0 and graph.value and hip.hipGraphInstantiate(C.byref(graph_exec), graph, None, None, 0) == 0
    for replay in range(4):
        say("replay", replay)
        fill()
        assert hip.hipGraphLaunch(graph_exec, stream) == 0
        ctx.sync()
        call(eager)
        ctx.sync()
        for name in recorded:
            if name != "h":
                assert np.array_equal(recorded[name].get(), eager[name].get()), (replay, name)
    hip.hipGraphExecDestroy(graph_exec)
    hip.hipGraphDestroy(graph)
    for op in (router, product, comb):
        op.destroy()
    ctx.close()


# ------------------------------------------------------------------------------ far apart

class Far(object):
    """rows (or matrices) `apart` bytes from one another in one large allocation"""

    def __init__(self, A, ctx, whole, host, apart, at=0):
        self.A, self.ctx, self.host, self.apart, self.base = A, ctx, host, apart, whole.ptr + at
        assert at + (host.shape[0] - 1) * apart + host[0].nbytes <= whole.nbytes and apart % host.itemsize == 0
        inner, step = [], 1
        for n in reversed(host.shape[1:]):
            inner.insert(0, step)
            step *= n
        self.array = A.Strided(host.shape, [apart // host.itemsize] + inner, self.base, whole)
        self.set(host)

    def part(self, i):
        one = self.host[i]
        return self.A.DeviceArray.view(self.ctx, one.shape, one.dtype, one.size, self.base + i * self.apart)

    def set(self, host):
        for i in range(host.shape[0]):
            self.part(i).set(host[i])

    def get(self):
        return np.stack([self.part(i).get() for i in range(self.host.shape[0])])


@pytest.mark.parametrize("apart", [(700 << 20) + 64, (700 << 20) + 66, (280 << 20) + 16])
def test_arrays_beyond_two_and_four_gigabytes(A, ctx, ops, apart):
    """seven rows, 280 or 700 MB apart: 1.7 GB, where offsets of 32 bits still do, and 4.2; every operand in turn"""
    say("far", apart)
    rng = np.random.default_rng(apart)
    wholes = [ctx.empty((5 << 30,), np.uint8) for _ in range(3)]           # (a result interleaved with an operand is refused)
    rows, n, k = 7, 40, 64
    far = lambda v, at, which=0: Far(A, ctx, wholes[which], v, apart, at)
    small = lambda *s: rng.integers(-3, 4, s).astype(np.float16)
    offsets, index = np.array([0, 3, 7], np.int32), np.array([6, 0, 5, -1, 4, 6, 1], np.int32)
    doff, dindex = ctx.array(offsets), ctx.array(index)
    x, w, g = small(rows, k), small(2, n, k), small(rows, n)
    named = np.where((index >= 0)[:, None], x[index].astype(float), 0.0)
    product, zeros = ops("Product", "half"), np.zeros
    # the rows that are multiplied, the result's rows; by an index, too
    for use in (False, True):
        fx, fo = far(x, 0), far(zeros((rows, n), np.float16), 1 << 20, 1)
        product.rows(fx.array, ctx.array(w), doff, fo.array, index=dindex if use else None)
        taken = named if use else x.astype(float)
        want = np.concatenate([taken[:3] @ w[0].T.astype(float), taken[3:] @ w[1].T.astype(float)])
        assert np.array_equal(fo.get().astype(float), want)
        fg, dw = far(g, 2 << 20), ctx.empty((2, n, k), np.float16)
        product.outer(fg.array, fx.array, doff, dw, index=dindex if use else None)
        want = np.stack([g[:3].T.astype(float) @ taken[:3], g[3:].T.astype(float) @ taken[3:]])
        assert np.array_equal(dw.get().astype(float), want)
    # the matrices, as operand and as result
    many = small(rows, n, k)
    fw, each, out = far(many, 0), ctx.array(np.arange(rows + 1, dtype=np.int32)), ctx.empty((rows, n), np.float16)
    product.rows(ctx.array(x), fw.array, each, out)
    assert np.array_equal(out.get().astype(float), np.einsum("enk,ek->en", many.astype(float), x.astype(float)))
    fd = far(zeros((rows, n, k), np.float16), 1 << 20, 1)
    product.outer(ctx.array(g), ctx.array(x), each, fd.array)
    assert np.array_equal(fd.get().astype(float), g[:, :, None].astype(float) * x[:, None, :])
    # combination
    place = np.array([[6, 0], [5, 4], [1, -1]], np.int32)
    y, dout = small(rows, k), small(3, k)
    fy, fs, fdo = far(y, 0), far(zeros((3, k), np.float16), 1 << 20, 1), far(dout, 2 << 20)
    comb = ops("Combiner", "half")
    comb.combine(fy.array, ctx.array(place), None, fs.array)
    there = place >= 0
    assert np.array_equal(fs.get().astype(float), (y[place].astype(float) * there[:, :, None]).sum(1))
    fdy, dweights = far(zeros((rows, k), np.float16), 3 << 20, 1), ctx.empty((3, 2), np.float32)
    comb.gradient(fdo.array, fy.array, ctx.array(place), None, fdy.array, dweights)
    want = zeros((rows, k))
    for t in range(3):
        for j in range(2):
            if place[t, j] >= 0:
                want[place[t, j]] = dout[t]
    assert np.array_equal(fdy.get().astype(float), want)
    assert np.array_equal(dweights.get(), (dout[:, None, :].astype(float) * y[place]).sum(2) * there)
    # the router
    logits = rng.permutation(rows * 24).reshape(rows, 24).astype(np.float16)
    fl = far(logits, 0)
    ints = [ctx.empty(s, np.int32) for s in ((rows, 2), (25,), (rows * 2,), (rows, 2))]
    weights = ctx.empty((rows, 2), np.float32)
    ops("Router", "half", 2, True).route(fl.array, ints[0], weights, ints[1], ints[2], ints[3])
    assert np.array_equal(ints[0].get(), np.argsort(-logits.astype(float), 1)[:, :2])
    # 4 bits
    micro = ops("Microscale", "half")
    v = rng.choice([-6, -4, -3, -2, -1.5, -1, -0.5, 0, 0.5, 1, 1.5, 2, 3, 4, 6], (rows, k)).astype(np.float16)
    v[:, ::32] = 6                                          # (scales of one, so that codes are the values)
    if apart % 16:
        return                                              # (rows of codes start on 16 bytes)
    fv, fc, fe = far(v, 0), far(zeros((rows, 32), np.uint8), 1 << 20, 1), far(zeros((rows, 2), np.uint8), 2 << 20, 2)
    micro.quantise(fv.array, fc.array, fe.array)
    fb = far(zeros((rows, k), np.float16), 3 << 20, 0)
    micro.values(fc.array, fe.array, fb.array)
    assert np.array_equal(fb.get(), v)
    fo = far(zeros((rows, rows), np.float16), 4 << 20, 0)
    wc, ws = fc.array, fe.array
    turned = lambda a, m: A.Strided((1, rows, m), (0,) + tuple(a.strides), a.ptr, a.owner)
    micro.rows(fc.array, fe.array, turned(wc, 32), turned(ws, 2), ctx.array(np.array([0, rows], np.int32)), fo.array)
    want = v.astype(float) @ v.T.astype(float)
    assert np.array_equal(fo.get(), want.astype(np.float16))


# ------------------------------------------------------------------------------ sums in pieces of an odd number of steps

# A tile of 32 x 64 or 64 x 128, few enough that sums are cut; a step of a sum is 128 bytes, and pieces of nine steps or more are
# wanted of which there are an odd number: steps * tiles / 512, rounded up.  rows, experts, n, k, segments, w's order, index
PIECES = {
    "half": [(128, 1, 1152, 4096, "even", "nk", 0), (128, 1, 1152, 4096, "even", "kn", 2), (256, 1, 2304, 4096, "gaps", "nk", 0), (127, 2, 1086, 4090, "skewed", "kn", 0),
             (12, 3, 1472, 4096, "even", "kn", 0)],
    "bfloat16": [(128, 1, 1152, 4096, "gaps", "nk", 2), (128, 1, 1152, 4096, "even", "kn", 0), (125, 1, 1151, 4093, "even", "nk", 0)],
    "float": [(150, 1, 960, 4096, "even", "nk", 0), (150, 1, 960, 4096, "gaps", "kn", 3), (12, 7, 1472, 1024, "even", "kn", 0), (149, 1, 959, 4095, "even", "nk", 2)],
}


@pytest.mark.parametrize("lead,extra", [(0, 0), (8, 8), (1, 3)])
@pytest.mark.parametrize("elt,case", [(elt, case) for elt in TYPES for case in PIECES[elt]])
def test_every_step_of_a_sum_in_pieces_counts_once(A, ctx, ops, elt, case, lead, extra):
    """whole numbers, whose sums are exact; a step counted twice, or not at all, is another sum"""
    rows, experts, n, k, kind, order, per = case
    say("pieces", elt, case, lead, extra)
    rng = np.random.default_rng(rows + n + k)
    offsets = segments(rng, rows, experts, kind)
    tokens = rows if not per else rows // per + 1
    index = rng.integers(0, tokens * per, rows).astype(np.int32) if per else None
    if per:
        index[[0, rows - 1]] = (-1, tokens * per)
    x, w = rng.integers(-1, 2, (tokens, k)).astype(float), rng.integers(-1, 2, (experts, n, k)).astype(float)
    named = np.arange(rows) if not per else np.where(index < 0, tokens, index // per)
    taken = np.concatenate([x, np.zeros((1, k))])[np.minimum(named, tokens)]
    want = np.zeros((rows, n))
    for e in range(experts):
        want[offsets[e]:offsets[e + 1]] = taken[offsets[e]:offsets[e + 1]] @ w[e].T
    dx, dw = Boxed(A, ctx, store(x, elt), elt, lead, extra, np.nan), Boxed(A, ctx, store(w, elt), elt, lead, extra, np.nan, swap=order == "kn")
    out = Boxed(A, ctx, np.ones((rows, n), STORED[elt]), elt, lead, extra, 7.0)
    ops("Product", elt).rows(dx.array, dw.array, ctx.array(offsets), out.array, index=None if index is None else ctx.array(index), per=per)
    assert np.array_equal(values(out.get(), elt), values(store(want, elt), elt))


@pytest.mark.parametrize("elt,rows,n,k", [("half", 128, 1280, 13824), ("bfloat16", 128, 1280, 13824), ("float", 127, 1277, 13800), ("half", 128, 1280, 13696)])
def test_every_step_of_a_sum_of_four_bit_numbers_in_pieces_counts_once(A, ctx, ops, elt, rows, n, k):
    say("micro pieces", elt, rows, n, k)
    rng = np.random.default_rng(k)
    # ones, halves and their negatives under scales of one: quarters, whose sums are exact
    grid = np.array([0.0, 0.5, 1.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, -0.5, -1.0])
    blocks = (k + 31) // 32
    cx, cw = rng.choice([0, 1, 2, 9, 10], (rows, blocks * 32)), rng.choice([0, 1, 2, 9, 10], (n, blocks * 32))
    ones = lambda m: ctx.array(np.full((m, blocks), 127, np.uint8))
    sw = ones(n)
    out = Boxed(A, ctx, np.ones((rows, n), STORED[elt]), elt, 8, 8, 7.0)
    dw = ctx.array(packed(cw))
    ops("Microscale", elt).rows(ctx.array(packed(cx)), ones(rows), A.Strided((1, n, 16 * blocks), (n * 16 * blocks, 16 * blocks, 1), dw.ptr, dw),
                                A.Strided((1, n, blocks), (n * blocks, blocks, 1), sw.ptr, sw), ctx.array(np.array([0, rows], np.int32)), out.array)
    want = grid[cx] @ grid[cw].T
    assert np.array_equal(values(out.get(), elt), values(store(want, elt), elt))


# ------------------------------------------------------------------------------ starts in any order

@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("rows,experts,ni,nj", [(5000, 2, 70, 90), (5000, 9, 70, 90), (3001, 70, 33, 40), (6000, 8, 264, 256), (400, 131, 60, 72), (64, 6, 24, 40)])
def test_starts_that_go_back_count_as_the_largest_before_them(A, ctx, ops, elt, rows, experts, ni, nj):
    """whole sums and sums in pieces: a row is in one segment, whatever the starts say, and nothing beside the results changes"""
    say("starts", elt, rows, experts, ni, nj)
    rng = np.random.default_rng(rows + experts)
    a, b, w = rng.integers(-1, 2, (rows, ni)).astype(float), rng.integers(-1, 2, (rows, nj)).astype(float), rng.integers(-1, 2, (experts, nj, ni)).astype(float)
    da, db, dw = (Boxed(A, ctx, store(v, elt), elt, 8, 8, np.nan) for v in (a, b, w))
    for offsets in (np.resize([0, rows], experts + 1), np.resize([rows // 2, rows, 0], experts + 1), np.sort(rng.integers(0, rows + 1, experts + 1))[::-1],
                    rng.integers(-rows, 2 * rows, experts + 1)):
        offsets = offsets.astype(np.int32)
        upto = np.maximum.accumulate(np.clip(offsets, 0, rows))
        do = ctx.array(offsets)
        out = Boxed(A, ctx, np.ones((experts, ni, nj), STORED[elt]), elt, 8, 8, 7.0)
        ops("Product", elt).outer(da.array, db.array, do, out.array)
        want, _ = plain_outer(a, b, upto, experts)
        assert np.array_equal(values(out.get(), elt), values(store(want, elt), elt))
        out = Boxed(A, ctx, np.ones((rows, nj), STORED[elt]), elt, 8, 8, 7.0)
        ops("Product", elt).rows(da.array, dw.array, do, out.array)
        want = np.zeros((rows, nj))
        for e in range(experts):
            want[upto[e]:upto[e + 1]] = a[upto[e]:upto[e + 1]] @ w[e].T
        assert np.array_equal(values(out.get(), elt), values(store(want, elt), elt))


# ------------------------------------------------------------------------------ strides of a dimension of one

@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("stride", [0, 1, 8, 40, 1 << 40])
@pytest.mark.parametrize("ni,nj", [(64, 128), (40, 24), (33, 65), (256, 512)])
def test_a_single_row_is_read_whole_whatever_its_stride(A, ctx, ops, elt, stride, ni, nj):
    """the stride of a dimension of one element says nothing: a turned column has one of 1, a broadcast one of 0"""
    rng = np.random.default_rng(ni + nj)
    a, b, w = (rng.integers(-3, 4, s).astype(float) for s in ((1, ni), (1, nj), (1, nj, ni)))
    da, db, dw = (ctx.array(store(v, elt)) for v in (a, b, w))
    row = lambda d, n: A.Strided((1, n), (stride, 1), d.ptr, d)
    offsets, index = ctx.array(np.array([0, 1], np.int32)), ctx.array(np.array([0], np.int32))
    for use in (None, index):
        for order in ("ij", "ji"):
            out = Boxed(A, ctx, np.ones((1, ni, nj), STORED[elt]), elt, 8, 8, 7.0, swap=order == "ji")
            ops("Product", elt).outer(row(da, ni), row(db, nj), offsets, out.array, index=use)
            assert np.array_equal(values(out.get(), elt), a[:, :, None] * b[:, None, :])
        out = Boxed(A, ctx, np.ones((1, nj), STORED[elt]), elt, 8, 8, 7.0)
        ops("Product", elt).rows(row(da, ni), A.Strided((1, nj, ni), (stride, ni, 1), dw.ptr, dw), offsets, out.array, index=use)
        assert np.array_equal(values(out.get(), elt), values(store(a @ w[0].T, elt), elt))


# ------------------------------------------------------------------------------ calls of more than 2^32 threads

def peek(A, ctx, array, first, count):
    """`count` rows of a dense array from row `first` on"""
    n = array.shape[-1]
    return A.DeviceArray.view(ctx, (count, n), array.dtype, count * n, array.ptr + first * n * array.dtype.itemsize).get()


def test_gradient_of_a_combination_of_more_tokens_than_a_launch_has(A, ctx, ops):
    """a workgroup of 64 threads a token, 2^26 tokens and five"""
    say("combine_gradient, many tokens")
    tokens = (1 << 26) + 5
    place = np.full((tokens, 1), -1, np.int32)
    named = np.array([0, 7, (1 << 26) - 1, 1 << 26, tokens - 1])
    place[named, 0] = [3, 0, 4, 1, 2]
    rng = np.random.default_rng(1)
    y, dout = rng.integers(-3, 4, (5, 8)).astype(np.float16), rng.integers(-3, 4, (1, 8)).astype(np.float16)
    one, dy, dweights = ctx.array(dout), ctx.array(np.full((5, 8), 9, np.float16)), ctx.array(np.full((tokens, 1), np.nan, np.float32))
    ops("Combiner", "half").gradient(A.Strided((tokens, 8), (0, 1), one.ptr, one), ctx.array(y), ctx.array(place), None, dy, dweights)
    assert np.array_equal(dy.get(), np.repeat(dout, 5, 0))
    want = np.zeros((tokens, 1), np.float32)
    want[named, 0] = (y[place[named, 0]].astype(float) * dout).sum(1)
    assert np.array_equal(dweights.get(), want)


def test_more_numbers_in_four_bits_than_a_launch_has_threads(A, ctx, ops):
    """four threads a block of 32, 2^30 blocks and some: every row the same one"""
    say("quantise, many blocks")
    rows, k = (1 << 26) + 3, 512
    v = np.resize([6, -4, 3, -2, 1.5, -1, 0.5, 0], (1, k)).astype(np.float16)
    x, codes, scales = ctx.array(v), ctx.empty((rows, k // 2), np.uint8), ctx.empty((rows, k // 32), np.uint8)
    ops("Microscale", "half").quantise(A.Strided((rows, k), (0, 1), x.ptr, x), codes, scales)
    want, one, _ = plain_quantise(v.astype(float))
    for first in (0, (1 << 25) - 2, (1 << 26) - 2, rows - 4):
        assert np.array_equal(peek(A, ctx, codes, first, 4), np.repeat(packed(want), 4, 0))
        assert np.array_equal(peek(A, ctx, scales, first, 4), np.repeat(one, 4, 0))


def test_gradient_of_more_logits_than_a_launch_has_threads(A, ctx, ops):
    """64 lanes a token of 257 experts, 2^26 tokens and three, every one with the same logits"""
    say("route_gradient, many tokens")
    tokens, experts = (1 << 26) + 3, 257
    logits = ctx.array(np.zeros((1, experts), np.float16))
    chosen, weights, dweights = (ctx.empty((tokens, 1), t) for t in (np.int32, np.float32, np.float32))
    e = (np.arange(tokens) % experts).astype(np.int32)
    chosen.set(e[:, None])
    weights.set(np.full((tokens, 1), 1 / 257, np.float32))
    dweights.set(np.full((tokens, 1), 257.0, np.float32))
    out = ctx.empty((tokens, experts), np.float16)
    ops("Router", "half", 1, False).gradient(A.Strided((tokens, experts), (0, 1), logits.ptr, logits), chosen, weights, dweights, out)
    for first in (0, (1 << 26) - 2, tokens - 4):
        want = np.full((4, experts), -1 / 257)                # p ([chosen] dw - w dw), of equal p
        want[np.arange(4), e[first:first + 4]] = 256 / 257
        assert (np.abs(peek(A, ctx, out, first, 4).astype(float) - want) <= 2.0 ** -10 * np.abs(want)).all()


def test_products_of_extents_that_numbers_of_32_bits_would_pass_are_refused(A, ctx, ops):
    """row 2^31 - 1 and a tile's height are beyond 2^31; arrays of one row over and over, so that nothing large is needed to say it"""
    p, m = ops("Product", "half"), ops("Microscale", "half")
    room = ctx.empty((1 << 16,), np.uint8)
    S = lambda shape, strides: A.Strided(shape, strides, room.ptr, room)
    offsets = ctx.array(np.array([0, 0], np.int32))
    for n in (2 ** 31 - 4095, 2 ** 31 - 1):
        for call in (lambda: p.rows(S((n, 8), (0, 1)), S((1, 8, 8), (64, 8, 1)), offsets, A.Strided((n, 8), (8, 1), 1 << 46)),
                     lambda: p.rows(S((8, 8), (8, 1)), S((1, n, 8), (0, 0, 1)), offsets, A.Strided((8, n), (n, 1), 1 << 46)),
                     lambda: p.rows(S((0, n), (0, 1)), S((1, 8, n), (0, 0, 1)), offsets, A.Strided((0, 8), (8, 1), 1 << 46)),
                     lambda: p.rows(S((n, 8), (0, 1)), S((1, 8, 8), (64, 8, 1)), offsets, A.Strided((8, 8), (8, 1), 1 << 46), index=S((8,), (1,))),
                     lambda: p.outer(S((n, 8), (0, 1)), S((n, 8), (0, 1)), offsets, A.Strided((1, 8, 8), (64, 8, 1), 1 << 46)),
                     lambda: p.outer(S((0, n), (0, 1)), S((0, 8), (0, 1)), offsets, A.Strided((1, n, 8), (8 * n, 8, 1), 1 << 46)),
                     lambda: m.rows(S((n, 16), (0, 1)), S((n, 1), (0, 1)), S((1, 8, 16), (0, 16, 1)), S((1, 8, 1), (0, 1, 1)), offsets, A.Strided((n, 8), (8, 1), 1 << 46))):
            with pytest.raises(A.AccError) as e:
                call()
            assert e.value.code == A.ERR_INVALID and "extent" in e.value.message


def test_a_graph_keeps_its_scratch_memory_beside_other_streams_and_behind_a_trim(A):
    """replays of one stream and eager calls of two others at the same time, scratch memory given back in between"""
    import ctypes as C
    hip = C.CDLL("libamdhip64.so")
    hip.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    hip.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    hip.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    hip.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    hip.hipGraphExecDestroy.argtypes = hip.hipGraphDestroy.argtypes = [C.c_void_p]
    ctx = A.Context(0)
    rng = np.random.default_rng(11)
    tokens, experts, choose, width, hidden, rows = 3000, 40, 2, 1500, 96, 40
    router, product = A.Router(ctx, "float", choose, True), A.Product(ctx, "float")

    class Run(object):
        """inputs of its own, what they give, and a stream"""
        def __init__(self):
            self.stream = ctx.stream()
            f = lambda *s: rng.integers(-2, 3, s).astype(np.float32)
            self.x, self.w, self.logits = f(rows, width), f(1, hidden, width), rng.standard_normal((tokens, experts)).astype(np.float32)
            self.dx, self.dw, self.dl, self.a = ctx.array(self.x), ctx.array(self.w), ctx.array(self.logits), f(tokens, 24)
            self.da, self.all, self.few = ctx.array(self.a), ctx.array(np.array([0, rows], np.int32)), ctx.array(np.array([0, tokens // 2, tokens], np.int32))
            whole = lambda *s: ctx.empty(s, np.int32)
            self.out = dict(chosen=whole(tokens, choose), offsets=whole(experts + 1), order=whole(tokens * choose), place=whole(tokens, choose),
                            weights=ctx.empty((tokens, choose), np.float32), long=ctx.empty((rows, hidden), np.float32), outer=ctx.empty((2, 24, 24), np.float32))
            r = plain_route(self.logits.astype(float), choose, True)
            self.want = dict(chosen=r[0], offsets=r[2], order=r[3], place=r[4], long=self.x @ self.w[0].T,
                             outer=np.stack([h.T @ h for h in (self.a[:tokens // 2], self.a[tokens // 2:])]))

        def call(self):
            o = self.out
            router.route(self.dl, o["chosen"], o["weights"], o["offsets"], o["order"], o["place"], stream=self.stream)
            product.rows(self.dx, self.dw, self.all, o["long"], stream=self.stream)
            product.outer(self.da, self.da, self.few, o["outer"], stream=self.stream)

        def right(self):
            for name, v in self.want.items():
                assert np.array_equal(self.out[name].get(), v), name

        def clear(self):
            for v in self.out.values():
                v.set(np.full(v.shape, 77, v.dtype))
    one, others = Run(), [Run(), Run()]
    for r in [one] + others:
        r.call()
    ctx.sync()
    graph, graph_exec = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(one.stream, 2) == 0
    try:
        one.call()
    finally:
        rc = hip.hipStreamEndCapture(one.stream, C.byref(graph))
    assert rc == 0 and graph.value and hip.hipGraphInstantiate(C.byref(graph_exec), graph, None, None, 0) == 0
    freed, held = C.c_size_t(), C.c_size_t()
    for replay in range(4):
        say("replay", replay)
        for r in [one] + others:
            r.clear()
        ctx.sync()
        A.check(A.lib().acc_context_trim(ctx.handle, C.byref(freed)))
        A.check(A.lib().acc_context_scratch_bytes(ctx.handle, C.byref(held)))
        assert held.value > 0                     # (before anything is replayed: the graph's blocks are there)
        for _ in range(5):
            assert hip.hipGraphLaunch(graph_exec, one.stream) == 0
            for r in others:
                r.call()
        ctx.sync()
        for r in [one] + others:
            r.right()
    hip.hipGraphExecDestroy(graph_exec)
    hip.hipGraphDestroy(graph)
    for r in [one] + others:
        A.check(A.lib().acc_stream_destroy(ctx.handle, r.stream))
    A.check(A.lib().acc_context_trim(ctx.handle, C.byref(freed)))
    A.check(A.lib().acc_context_scratch_bytes(ctx.handle, C.byref(held)))
    assert held.value == 0
    for op in (router, product):
        op.destroy()
    ctx.close()


@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("tokens,experts,choose", [(5003, 300, 3), (5120, 512, 8), (5000, 512, 1), (70, 512, 8), (4999, 384, 4), (100, 1024, 4), (90, 769, 2), (66, 2048, 5), (5100, 2048, 5), (80, 1501, 7)])
def test_routes_on_both_sides_of_where_its_forms_change(A, ctx, ops, elt, tokens, experts, choose):
    test_routes(A, ctx, ops, elt, tokens, experts, choose)
