"""Products with matrices of 4-bit whole numbers in groups (include/acc_hip.h, section D) against plain numpy in 64 bits, through the C ABI.

Error bound.  Of every group of a row's k numbers the kernel has t = sum x (16 + q) and the row's sum, in Float32, and s t - s (16 + z)
sum x: of either a sum of up to k products, each exact in Float32 (11 and 5 bits), or, of Float32 rows in three parts, three times as
many.  So the error is at most (3 k + 8) 2^-24 sum |x| s (31 + 16 + z), but the rows here are normal values and their sums' roundings
far from all in one direction: small whole numbers are asked to be exact, and others within that bound's (k + 8) in place of 3 k + 8.
Where many rows share a matrix, it is first rounded to the operator's type, half a unit of every weight.
"""
import sys

import numpy as np
import pytest

from test_gpu_operators import HALF_ULP, TINY, Boxed as Bits, segments, store, values

pytestmark = pytest.mark.gpu
TYPES = ("float", "half", "bfloat16")
UNIT = 2.0 ** -24


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

    def get(elt, group):
        if (elt, group) not in made:
            made[elt, group] = A.Grouped(ctx, elt, group)
        return made[elt, group]
    yield get
    for op in made.values():
        op.destroy()


def packed(q):
    """codes [.., k] as bytes, rows of whole blocks of 32 (what a row has too many: 15, which must not count)"""
    k = q.shape[-1]
    full = np.full(q.shape[:-1] + (-(-k // 32) * 32,), 15, np.uint8)
    full[..., :k] = q
    return full[..., 0::2] | full[..., 1::2] << 4


def unpacked(codes, k):
    return np.stack([codes & 15, codes >> 4], axis=-1).reshape(codes.shape[:-1] + (-1,))[..., :k]


def weights(q, scales, zeros, group):
    """[experts, n, k] in 64 bits"""
    spread = lambda p: np.repeat(np.swapaxes(p, 1, 2).astype(np.float64), group, axis=2)[:, :, :q.shape[2]]
    return (q - (8.0 if zeros is None else spread(zeros))) * spread(scales)


def matrices(rng, experts, n, k, group, elt, with_zeros, whole):
    groups = -(-k // group)
    q = rng.integers(0, 16, (experts, n, k)).astype(np.uint8)
    scales = rng.integers(1, 3, (experts, groups, n)).astype(np.float64) if whole else np.exp(rng.standard_normal((experts, groups, n)) * 0.5) * 0.05
    return q, values(store(scales, elt), elt), rng.integers(0, 16, (experts, groups, n)).astype(np.uint8) if with_zeros else None


def expected(x, w, offsets, rows, index, per):
    out, size = np.zeros((rows, w.shape[1])), np.zeros((rows, w.shape[1]))
    for e in range(w.shape[0]):
        for m in range(max(0, offsets[e]), min(rows, offsets[e + 1])):
            r = m if index is None else index[m] // max(per, 1)
            if index is not None and not 0 <= index[m] or r >= x.shape[0]:
                continue
            out[m] = w[e] @ x[r]
            size[m] = np.abs(w[e]) @ np.abs(x[r])
    return out, size


SHAPES = [(1, 1, 1, 1), (1, 1, 40, 33), (3, 2, 17, 128), (16, 1, 64, 160), (17, 3, 100, 513), (33, 2, 130, 300), (70, 1, 48, 129), (64, 5, 96, 1030), (150, 3, 65, 257), (400, 2, 70, 200)]


@pytest.mark.parametrize("with_zeros", (False, True))
@pytest.mark.parametrize("group", (32, 64, 128, 512))
@pytest.mark.parametrize("elt", TYPES)
def test_products_of_whole_numbers_are_exact(A, ctx, ops, elt, group, with_zeros):
    """sums of whole numbers below 2^24, whatever their order: the exact sum rounded once"""
    rng = np.random.default_rng(group)
    for case, (rows, experts, n, k) in enumerate(SHAPES):
        q, scales, zeros = matrices(rng, experts, n, k, group, elt, with_zeros, True)
        offsets = segments(rng, rows, experts, ("even", "skewed", "gaps")[case % 3])
        per = (0, 1, 3)[case % 3]
        index = None if case % 2 else rng.integers(-2, rows * max(per, 1), rows).astype(np.int32)
        x_rows = rows if index is None else max(1, rows - 1)
        x = rng.integers(-3, 4, (x_rows, k)).astype(np.float64)
        say(elt, group, with_zeros, rows, experts, n, k, per, index is not None)
        loose = case % 3
        want, _ = expected(x, weights(q, scales, zeros, group), offsets, rows, index, per)
        bx, out = Boxed(A, ctx, x, elt, lead=loose, extra=loose), Boxed(A, ctx, np.full((rows, n), 9.0), elt, lead=1, extra=loose, fill=3.0)
        codes, bs = ctx.array(packed(q)), Boxed(A, ctx, scales, elt, lead=loose, extra=loose)
        bz = None if zeros is None else ctx.array(zeros)
        ops(elt, group).rows(bx.array, codes, bs.array, ctx.array(offsets), out.array, zeros=bz, index=None if index is None else ctx.array(index), per=per)
        ctx.sync()
        assert np.array_equal(out.get(), store(want, elt)), (rows, experts, n, k)


@pytest.mark.parametrize("group,with_zeros", ((32, False), (32, True), (64, True), (128, False), (512, True)))
@pytest.mark.parametrize("elt", TYPES)
def test_many_rows_of_many_matrices(A, ctx, ops, elt, group, with_zeros):
    """tiles of 64 rows (Float32: 32) by 256 columns: a last tile of one column, rows and sums that end anywhere, an index, segments of no row"""
    rng = np.random.default_rng(group + 7)
    for case, (rows, experts, n, k) in enumerate(((2000, 25, 900, 300), (1700, 18, 1025, 129), (3000, 40, 700, 1), (1400, 20, 1000, 640), (1500, 19, 784, 95))):
        q, scales, zeros = matrices(rng, experts, n, k, group, elt, with_zeros, True)
        offsets, per = segments(rng, rows, experts, ("even", "skewed", "gaps")[case % 3]), (0, 1, 3)[case % 3]
        index = None if case % 2 else rng.integers(-2, rows * max(per, 1), rows).astype(np.int32)
        x = rng.integers(-3, 4, (rows if index is None else rows - 1, k)).astype(np.float64)
        say(elt, group, with_zeros, rows, experts, n, k, per, index is not None)
        loose = case % 3
        want, _ = expected(x, weights(q, scales, zeros, group), offsets, rows, index, per)
        bx, out = Boxed(A, ctx, x, elt, lead=loose, extra=loose), Boxed(A, ctx, np.full((rows, n), 9.0), elt, lead=1, extra=loose, fill=3.0)
        args = bx.array, ctx.array(packed(q)), Boxed(A, ctx, scales, elt, lead=loose, extra=loose).array, ctx.array(offsets), out.array
        ops(elt, group).rows(*args, zeros=None if zeros is None else ctx.array(zeros), index=None if index is None else ctx.array(index), per=per)
        ctx.sync()
        assert np.array_equal(out.get(), store(want, elt)), (rows, experts, n, k)


@pytest.mark.parametrize("group", (32, 128))
@pytest.mark.parametrize("elt", TYPES)
def test_products_of_any_numbers(A, ctx, ops, elt, group):
    rng = np.random.default_rng(group + 1)
    for rows, experts, n, k in ((1, 1, 300, 1000), (40, 3, 129, 700), (128, 2, 64, 384), (500, 2, 90, 161), (1500, 20, 800, 700)):
        q, scales, zeros = matrices(rng, experts, n, k, group, elt, rows > 1, False)
        x = values(store(rng.standard_normal((rows, k)), elt), elt)
        offsets = segments(rng, rows, experts, "even")
        say(elt, group, rows, experts, n, k)
        w = weights(q, scales, zeros, group)
        want, size = expected(x, w, offsets, rows, None, 0)
        _, most = expected(x, weights(np.full_like(q, 15), np.abs(scales), None, group) * (63.0 / 7.0), offsets, rows, None, 0)
        many = rows / experts > 96
        bound = UNIT * (k + 8) * most + (HALF_ULP[elt] * 1.01 * size if many else 0)
        out = Boxed(A, ctx, np.zeros((rows, n)), elt)
        ops(elt, group).rows(Boxed(A, ctx, x, elt).array, ctx.array(packed(q)), Boxed(A, ctx, scales, elt).array, ctx.array(offsets), out.array, zeros=None if zeros is None else ctx.array(zeros))
        ctx.sync()
        got = values(out.get(), elt)
        off = np.abs(got - want) - (bound + HALF_ULP[elt] * 1.001 * (np.abs(want) + bound) + TINY[elt])
        assert np.all(off <= 0), (off.max(), np.abs(want).max())


@pytest.mark.parametrize("with_zeros", (False, True))
@pytest.mark.parametrize("elt", TYPES)
def test_quantised_and_made_again(A, ctx, ops, elt, with_zeros):
    """codes, scales and zeros as the formulas give them in Float32, division by division; then what they stand for"""
    rng = np.random.default_rng(11)
    for experts, n, k, group in ((1, 1, 1, 32), (2, 3, 31, 32), (1, 5, 200, 64), (3, 7, 128, 128), (1, 4, 1100, 512), (2, 2, 96, 1024)):
        say(elt, with_zeros, experts, n, k, group)
        w = values(store(rng.standard_normal((experts, n, k)) * np.exp(rng.standard_normal((experts, n, 1))), elt), elt).astype(np.float32)
        w[0, 0, : min(k, group)] = 0.0                        # a group of zeros
        groups = -(-k // group)
        full = np.zeros((experts, n, groups * group), np.float32)
        full[:, :, :k] = w
        full = full.reshape(experts, n, groups, group)
        low, high = np.minimum(full.min(3), 0), np.maximum(full.max(3), 0)
        f = np.float32
        scale = values(store((high - low) / f(15) if with_zeros else np.maximum(high, -low) / f(7), elt), elt).astype(np.float32)
        with np.errstate(all="ignore"):
            zero = np.where(scale > 0, np.clip(np.rint(-low / scale), 0, 15), 0).astype(f) if with_zeros else np.full(scale.shape, 8, f)
            q = np.where(scale[..., None] > 0, np.rint(full / scale[..., None]), 0).astype(f)
        q = np.clip(q + zero[..., None], 0, 15).astype(np.uint8).reshape(experts, n, -1)
        blocks = -(-k // 32)
        codes = ctx.array(np.full((experts, n, 16 * blocks), 0xEE, np.uint8))
        scales, zeros = Boxed(A, ctx, np.zeros((experts, groups, n)), elt, lead=1, extra=1, fill=2.0), ctx.array(np.full((experts, groups, n), 99, np.uint8))
        loose = 1 if k % 2 else 0
        ops(elt, group).quantise(Boxed(A, ctx, w, elt, lead=loose, extra=3 * loose).array, codes, scales.array, zeros=zeros if with_zeros else None)
        ctx.sync()
        assert np.array_equal(scales.get(), store(np.swapaxes(scale, 1, 2), elt))
        if with_zeros:
            assert np.array_equal(zeros.get(), np.swapaxes(zero, 1, 2).astype(np.uint8))
        got = unpacked(codes.get(), k)
        assert np.array_equal(got, q[:, :, :k])
        tail = unpacked(codes.get(), 32 * blocks)[:, :, k:]
        assert np.array_equal(tail, np.broadcast_to(zero[:, :, -1:].astype(np.uint8), tail.shape))
        out = Boxed(A, ctx, np.zeros((experts, n, k)), elt, lead=loose, extra=1, fill=1.0)
        ops(elt, group).values(codes, scales.array, out.array, zeros=zeros if with_zeros else None)
        ctx.sync()
        want = weights(got, np.swapaxes(scale, 1, 2).astype(np.float64), np.swapaxes(zero, 1, 2) if with_zeros else None, group)
        assert np.array_equal(out.get(), store(want.astype(np.float32), elt))      # (5 and at most 24 bits: Float32 rounds once, as here)


def test_groups_that_are_not_numbers(A, ctx, ops):
    w = np.ones((1, 4, 96), np.float32)
    w[0, 1, 40], w[0, 2, 95], w[0, 3, 0] = np.nan, np.inf, -np.inf
    op = ops("float", 32)
    for with_zeros in (False, True):
        codes, scales, zeros = ctx.empty((1, 4, 48), np.uint8), ctx.empty((1, 3, 4), np.float32), ctx.empty((1, 3, 4), np.uint8)
        op.quantise(ctx.array(w), codes, scales, zeros=zeros if with_zeros else None)
        out = ctx.empty((1, 4, 96), np.float32)
        op.values(codes, scales, out, zeros=zeros if with_zeros else None)
        ctx.sync()
        nan = np.isnan(out.get().reshape(4, 3, 32))
        want = np.zeros((4, 3), bool)
        want[1, 1] = want[2, 2] = want[3, 0] = True
        assert np.array_equal(nan.all(2), want) and np.array_equal(nan.any(2), want)


def test_rows_do_not_touch_each_other(A, ctx, ops):
    """a row of NaN, or an infinite one, beside others: theirs are what they were; what is no row's is zeros"""
    rng = np.random.default_rng(6)
    for rows in (20, 300):
        q, scales, zeros = matrices(rng, 1, 50, 200, 64, "bfloat16", True, True)
        x = rng.integers(-3, 4, (rows, 200)).astype(np.float64)
        want, _ = expected(x, weights(q, scales, zeros, 64), np.array([2, rows - 3]), rows, None, 0)
        x[5], x[9, 7] = np.nan, np.inf
        out = Boxed(A, ctx, np.full((rows, 50), 4.0), "bfloat16")
        ops("bfloat16", 64).rows(Boxed(A, ctx, x, "bfloat16").array, ctx.array(packed(q)), Boxed(A, ctx, scales, "bfloat16").array, ctx.array(np.array([2, rows - 3], np.int32)), out.array,
                                 zeros=ctx.array(zeros))
        ctx.sync()
        got = values(out.get(), "bfloat16")
        others = np.setdiff1d(np.arange(rows), [5, 9])
        assert np.array_equal(got[others], values(store(want, "bfloat16"), "bfloat16")[others])
        assert np.isnan(got[5]).all() and not np.isfinite(got[9]).any()


def test_products_that_are_refused(A, ctx, ops):
    op = ops("half", 64)
    h, b, i = lambda *s: ctx.empty(s, np.float16), lambda *s: ctx.empty(s, np.uint8), lambda *v: ctx.array(np.array(v, np.int32))
    good = dict(x=h(8, 100), codes=b(2, 30, 64), scales=h(2, 2, 30), offsets=i(0, 4, 8), out=h(8, 30), zeros=b(2, 2, 30), index=None, per=0)
    op.rows(**good)
    codes = good["codes"]
    for w in (dict(x=h(8, 96)), dict(x=h(7, 100)), dict(codes=b(2, 30, 48)), dict(codes=b(3, 30, 64)), dict(scales=h(2, 1, 30)), dict(scales=h(2, 2, 31)), dict(zeros=b(2, 3, 30)),
              dict(offsets=i(0, 8)), dict(out=h(8, 31)), dict(out=h(9, 30)), dict(per=-1), dict(index=i(0, 1)), dict(x=None), dict(codes=None), dict(scales=None), dict(out=None),
              dict(codes=A.Strided((2, 30, 64), (30 * 72, 72, 1), codes.ptr)), dict(codes=A.Strided((2, 30, 64), (1920, 64, 1), codes.ptr + 8)),
              dict(scales=A.Strided((2, 2, 30), (120, 60, 2), good["scales"].ptr)), dict(out=A.Strided((8, 30), (30, 1), good["x"].ptr))):
        with pytest.raises(A.AccError) as e:
            op.rows(**dict(good, **w))
        assert e.value.code == A.ERR_INVALID
    for bad in (0, 16, 48, -32):
        with pytest.raises(A.AccError):
            A.Grouped(ctx, "half", bad)
    q = dict(w=h(2, 30, 100), codes=codes, scales=good["scales"], zeros=good["zeros"])
    op.quantise(**q)
    for w in (dict(w=h(2, 30, 99, ), codes=b(2, 30, 80)), dict(w=h(2, 31, 100)), dict(scales=h(2, 3, 30)), dict(codes=A.Strided((2, 30, 64), (1920, 64, 1), q["w"].ptr))):
        with pytest.raises(A.AccError) as e:
            op.quantise(**dict(q, **w))
        assert e.value.code == A.ERR_INVALID
    with pytest.raises(A.AccError):
        op.values(codes, good["scales"], h(2, 30, 130), zeros=good["zeros"])
    # nothing to do, and sums of nothing
    op.rows(h(0, 100), codes, good["scales"], i(0, 0, 0), h(0, 30))
    out = ctx.array(np.full((8, 30), 7, np.float16))
    op.rows(h(8, 0), b(2, 30, 0), h(2, 0, 30), good["offsets"], out)
    ctx.sync()
    assert np.all(out.get() == 0)
