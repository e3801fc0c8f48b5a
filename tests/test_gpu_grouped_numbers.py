"""Products with matrices of 4-bit whole numbers in groups (include/acc_hip.h, section D): the numbers that they keep, whatever form a call
takes, by results whose rounding is known to the last bit.

A row of one group gives s T, T = sum x (q - z) a whole number.  Here x are whole numbers of at most 3, so T is exact in Float32 (100 times
3 times 15: 13 bits), s T has at most 11 + 13 bits of a 16-bit scale and is exact too, and the result is the exact one rounded once.  Of
Float32 scales the product is rounded, once, and that is the result.

Rows whose numbers share a sign: of every group the kernels add up x (16 + q) and take (16 + z) sum x off, each of them below 31 sum x;
with whole numbers that make this less than 2^24 everything is exact again, and so is the sum over the groups, with scales that are powers
of two.  A form that adds more than 16 to a code loses digits there.

Float32 rows are cut into three parts of 8 bits, each of what the one before has left.  With x of 17 bits, whole numbers of 2^-16 between 1
and 2, four of a group not 0, all that is added up is a whole number of 2^-16 below 31 x 4 x 2 = 2^8: 24 bits, exact, and so are the results of
one group.  With x of 24 bits, one of a group not 0 and s = 1: -(z + 16) x1 + x1 (16 + q) is exact (13 bits), and so is what the second part
adds (within 21); the third part's product rounds once, below 32 |x|, the second parts' beginning once more, to a result below 16 |x|, and
up to two groups of the row add up once: half a unit of 2^-23 times that, (16 + 8 + 16) |x| 2^-23 of the larger |x|, is more than any of it.
"""
import sys

import numpy as np
import pytest

from test_gpu_grouped import Boxed, expected, matrices, packed, weights
from test_gpu_operators import segments, store, values

pytestmark = pytest.mark.gpu
TYPES = ("float", "half", "bfloat16")


def say(*a):
    print("[case]", *a)
    sys.stdout.flush()


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
def rows(A, ctx):
    """rows(elt, group, x, q, scales, zeros, offsets): the products, as they are in memory"""
    made = {}

    def call(elt, group, x, q, scales, zeros, offsets):
        if (elt, group) not in made:
            made[elt, group] = A.Grouped(ctx, elt, group)
        out = Boxed(A, ctx, np.full((x.shape[0], q.shape[1]), 9.0), elt)
        made[elt, group].rows(Boxed(A, ctx, x, elt).array, ctx.array(packed(q)), Boxed(A, ctx, scales, elt).array, ctx.array(np.asarray(offsets, np.int32)), out.array,
                              zeros=None if zeros is None else ctx.array(zeros))
        ctx.sync()
        return out.get()
    yield call
    for op in made.values():
        op.destroy()


# (rows, matrices, n, k): a few rows, a few hundred of one matrix, tiles of 256 columns enough for the device, rows in LDS (the last two)
FORMS = [(3, 1, 70, 100), (129, 1, 70, 100), (300, 1, 70, 31), (700, 2, 4, 100), (5000, 2, 300, 70), (1500, 25, 900, 100), (200, 2, 3100, 100), (40, 2, 3200, 100), (9, 1, 6200, 100)]


@pytest.mark.parametrize("with_zeros", (False, True))
@pytest.mark.parametrize("elt", TYPES)
def test_no_weight_is_rounded(rows, elt, with_zeros):
    """scales with as many bits as their type has, of which (q - z) s has more"""
    rng = np.random.default_rng(21)
    for m, experts, n, k in FORMS:
        q, scales, zeros = matrices(rng, experts, n, k, 128, elt, with_zeros, False)
        x = rng.integers(-3, 4, (m, k)).astype(np.float64)
        offsets = segments(rng, m, experts, "even")
        say(elt, with_zeros, m, experts, n, k)
        want, _ = expected(x, weights(q, scales, zeros, 128), offsets, m, None, 0)
        assert np.array_equal(rows(elt, 128, x, q, scales, zeros, offsets), store(want, elt)), (m, experts, n, k)


def test_half_weights_beyond_the_largest(rows):
    """(q - z) s beyond 65504, as quantising a matrix of 65504 and its negative gives, and results far below it"""
    rng = np.random.default_rng(22)
    for m, experts, n, k in FORMS:
        q, _, _ = matrices(rng, experts, n, k, 128, "half", False, False)
        scales = np.full((experts, 1, n), 8736.0)
        x = rng.integers(-3, 4, (m, k)) * 2.0 ** -12
        offsets = segments(rng, m, experts, "even")
        say(m, experts, n, k)
        want, _ = expected(x, weights(q, scales, None, 128), offsets, m, None, 0)
        got = rows("half", 128, x, q, scales, None, offsets)
        assert np.isfinite(values(got, "half")).all() and np.array_equal(got, store(want, "half")), (m, experts, n, k)


@pytest.mark.parametrize("elt", TYPES)
def test_an_infinity_in_a_row_of_any_form(rows, elt):
    """what the row gives is not a number, however many rows come with it"""
    rng = np.random.default_rng(23)
    for m, experts, n, k in FORMS:
        q, scales, zeros = matrices(rng, experts, n, k, 64, elt, True, True)
        x = rng.integers(-3, 4, (m, k)).astype(np.float64)
        x[1, 5], x[2, k - 1] = np.inf, -np.inf
        offsets = segments(rng, m, experts, "even")
        say(elt, m, experts, n, k)
        got = values(rows(elt, 64, x, q, scales, zeros, offsets), elt)
        assert np.isnan(got[1:3]).all() and np.isfinite(np.delete(got, (1, 2), axis=0)).all(), (m, experts, n, k)


@pytest.mark.parametrize("group", (32, 64, 128, 256))
@pytest.mark.parametrize("elt", ("half", "bfloat16"))
def test_rows_of_one_sign(rows, elt, group):
    """x of all 11 (8) bits and one sign: 31 sum x of a group is below 2^24, and 15 sum x of a row"""
    rng = np.random.default_rng(group)
    for m, experts, n, k in ((3, 1, 70, 270), (129, 1, 70, 260), (40, 2, 3100, 273), (700, 2, 4, 100), (5000, 2, 300, 70), (1500, 25, 900, 257)):
        q, _, zeros = matrices(rng, experts, n, k, group, elt, m % 2 == 1, True)
        scales = 2.0 ** rng.integers(-8, -6, (experts, -(-k // group), n)).astype(np.float64)
        most = 2047 if elt == "half" else 255
        x = rng.integers(most // 2, most + 1, (m, k)).astype(np.float64)
        assert 31 * min(k, group) * most < 2 ** 24 and 2 * 15 * k * most < 2 ** 24
        offsets = segments(rng, m, experts, "even")
        say(elt, group, m, experts, n, k)
        want, _ = expected(x, weights(q, scales, zeros, group), offsets, m, None, 0)
        assert np.array_equal(rows(elt, group, x, q, scales, zeros, offsets), store(want, elt)), (m, experts, n, k)


@pytest.mark.parametrize("elt", ("float", "bfloat16"))
def test_quantising_a_range_beyond_the_largest_number(A, ctx, elt):
    """high - low of a group of numbers is an infinity, its fifteenth is not: the same formula of sixteenths"""
    rng, f, group = np.random.default_rng(31), np.float32, 32
    w = values(store(rng.uniform(-1, 1, (2, 6, 96)), elt), elt).astype(f)
    most = values(store(np.array([3.3e38]), elt), elt).astype(f)[0]
    w[0, 2, :32] *= most
    w[1, 4, 40], w[1, 4, 41] = most, -most
    w[1, 5, 70], w[1, 5, 71] = most, -most / 2
    full = w.reshape(2, 6, 3, group)
    low, high = np.minimum(full.min(3), 0), np.maximum(full.max(3), 0)
    with np.errstate(over="ignore"):
        ranges = high - low
    assert np.isinf(ranges).sum() == 3
    scale = np.where(np.isinf(ranges), (high * f(0.0625) - low * f(0.0625)) / f(15) * f(16), np.where(np.isinf(ranges), 0, ranges) / f(15)).astype(f)
    scale = values(store(scale, elt), elt).astype(f)
    zero = np.clip(np.rint(-low / scale), 0, 15)
    q = np.clip(np.rint(full / scale[..., None]) + zero[..., None], 0, 15).astype(np.uint8).reshape(2, 6, 96)
    codes, scales, zeros = ctx.empty((2, 6, 48), np.uint8), Boxed(A, ctx, np.zeros((2, 3, 6)), elt), ctx.empty((2, 3, 6), np.uint8)
    op = A.Grouped(ctx, elt, group)
    op.quantise(Boxed(A, ctx, w, elt).array, codes, scales.array, zeros=zeros)
    ctx.sync()
    op.destroy()
    assert np.array_equal(scales.get(), store(np.swapaxes(scale, 1, 2), elt)) and np.array_equal(zeros.get(), np.swapaxes(zero, 1, 2).astype(np.uint8))
    assert np.array_equal(codes.get(), packed(q))


def in_parts(x, parts):
    """the first `parts` of the three 8-bit parts of Float32 numbers, added up"""
    left, total = x.astype(np.float32), np.zeros(x.shape, np.float32)
    for _ in range(parts):
        part = (left.view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
        total, left = total + part, left - part
    return total.astype(np.float64)


@pytest.mark.parametrize("with_zeros", (False, True))
@pytest.mark.parametrize("group", (32, 64, 128))
def test_all_three_parts_of_float32_rows(rows, group, with_zeros):
    rng = np.random.default_rng(group + 5)
    for m, experts, n, k in FORMS:
        k = min(k, group)
        q, _, zeros = matrices(rng, experts, n, k, group, "float", with_zeros, True)
        scales = np.full((experts, 1, n), 0.25)
        x = np.zeros((m, k))
        for r in range(m):
            x[r, rng.permutation(k)[:4]] = (2.0 ** 16 + rng.integers(2 ** 7, 2 ** 15, 4) * 2 + 1) * rng.choice([-1, 1], 4) * 2.0 ** -16
        offsets = segments(rng, m, experts, "even")
        say(group, with_zeros, m, experts, n, k)
        w = weights(q, scales, zeros, group)
        want, _ = expected(x, w, offsets, m, None, 0)
        two, _ = expected(in_parts(x, 2), w, offsets, m, None, 0)
        assert np.array_equal(in_parts(x, 3), x) and np.mean(two != want) > 0.2
        assert np.array_equal(rows("float", group, x, q, scales, zeros, offsets), want.astype(np.float32)), (m, experts, n, k)


@pytest.mark.parametrize("with_zeros", (False, True))
@pytest.mark.parametrize("group", (32, 64))
def test_float32_rows_of_all_their_bits(rows, group, with_zeros):
    rng = np.random.default_rng(group + 6)
    for m, experts, n, k in FORMS:
        k = min(k, 2 * group)
        q, _, zeros = matrices(rng, experts, n, k, group, "float", with_zeros, True)
        scales = np.ones((experts, -(-k // group), n))
        x = np.zeros((m, k))
        for first in range(0, k, group):
            x[np.arange(m), rng.integers(first, min(k, first + group), m)] = rng.uniform(1, 2, m).astype(np.float32) * rng.choice([-1, 1], m)
        offsets = segments(rng, m, experts, "even")
        say(group, with_zeros, m, experts, n, k)
        w = weights(q, scales, zeros, group)
        want, _ = expected(x, w, offsets, m, None, 0)
        bound = 40 * 2.0 ** -23 * np.abs(x).max(1, keepdims=True)
        two, _ = expected(in_parts(x, 2), w, offsets, m, None, 0)
        assert np.mean(np.abs(two - want) > bound) > 0.2       # (two parts alone would not do)
        assert np.all(np.abs(rows("float", group, x, q, scales, zeros, offsets) - want) <= bound), (m, experts, n, k)
