"""The router by scores (include/acc_hip.h, section D) against plain numpy in 64 bits, through the C ABI: choices, places and offsets are
asked to be equal, whatever lies next to whatever; weights and gradients within a few units of Float32.

A weight is an exponential, a sum, a quotient, a sum of up to 32 and another quotient, each within a unit or two of 2^-24, so 48 of
them are allowed; a gradient takes the difference of a weight's gradient and the weighted mean of all, whose own error is that of 32
such terms."""
import sys

import numpy as np
import pytest

from test_gpu_operators import HALF_ULP, TINY, Boxed as Bits, store, values

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


def plain(x, bias, choose, groups, keep, normalise, scale):
    """(experts, weights, offsets, order, place)"""
    t, e = x.shape
    with np.errstate(all="ignore"):
        score = 1.0 / (1.0 + np.exp(-x))
        ranked = score + (0.0 if bias is None else bias.astype(np.float64))
        ranked = np.where((x > -np.inf) & (ranked > -np.inf), ranked, -np.inf)
    if keep < groups:
        two = -np.sort(-ranked.reshape(t, groups, -1), axis=2)[:, :, :2]
        of_group = np.where(two[:, :, 0] > -np.inf, np.where(two > -np.inf, two, 0.0).sum(2), -np.inf)
        best = np.argsort(-of_group, axis=1, kind="stable")[:, :keep]
        kept = np.zeros((t, groups), bool)
        np.put_along_axis(kept, best, True, 1)
        ranked = np.where(np.repeat(kept, e // groups, axis=1), ranked, -np.inf)
    experts = np.argsort(-ranked, axis=1, kind="stable")[:, :choose]
    there = np.take_along_axis(ranked, experts, 1) > -np.inf
    s = np.where(there, np.take_along_axis(score, experts, 1), 0.0)
    total = s.sum(1, keepdims=True) if normalise else np.ones((t, 1))
    with np.errstate(all="ignore"):
        weights = np.where(total > 0, scale * s / total, 0.0)
    experts = np.where(there, experts, -1).astype(np.int32)
    flat = experts.reshape(-1)
    order = np.argsort(np.where(flat < 0, e, flat), kind="stable").astype(np.int32)
    some = int((flat >= 0).sum())
    place = np.empty(flat.size, np.int32)
    place[order] = np.arange(flat.size)
    place[flat < 0] = -1
    order[some:] = -1
    return experts, weights, np.concatenate([[0], np.cumsum(np.bincount(flat[flat >= 0], minlength=e))]).astype(np.int32), order, place.reshape(t, choose)


def routed(A, ctx, x, bias, elt, choose, groups, keep, normalise, scale, lead=0, extra=0):
    t, e = x.shape
    op = A.ScoreRouter(ctx, elt, choose, groups, keep, normalise, scale)
    box = Boxed(A, ctx, x, elt, lead=lead, extra=extra, fill=50.0)
    r = [ctx.empty((t, choose), np.int32), ctx.empty((t, choose), np.float32), ctx.empty((e + 1,), np.int32), ctx.empty((t * choose,), np.int32), ctx.empty((t, choose), np.int32)]
    op.route(box.array, *r, bias=None if bias is None else ctx.array(bias.astype(np.float32)))
    ctx.sync()
    op.destroy()
    return [a.get() for a in r]


def same(got, want, scale):
    for k, what in ((0, "experts"), (2, "offsets"), (3, "order"), (4, "place")):
        bad = np.argwhere(got[k] != want[k])
        assert bad.size == 0, (what, bad[:3], got[k][tuple(bad[0])], want[k][tuple(bad[0])])
    assert np.all(np.abs(got[1] - want[1]) <= 48 * UNIT * np.abs(want[1]) + 1e-37 * abs(scale))


SHAPES = [(1, 8, 1, 1, 1), (8, 128, 6, 8, 3), (3, 6, 2, 2, 1), (65, 160, 6, 8, 3), (1000, 256, 8, 8, 4), (300, 64, 1, 1, 1), (70, 2048, 8, 64, 5), (40, 2048, 3, 1, 1), (129, 384, 8, 16, 16),
          (257, 96, 32, 4, 2), (5000, 40, 5, 4, 3), (40000, 16, 2, 1, 1), (17, 1, 1, 1, 1), (33, 1000, 4, 8, 2), (2, 12, 12, 4, 4)]


@pytest.mark.parametrize("elt", TYPES)
@pytest.mark.parametrize("with_bias", (False, True))
def test_choices_are_those_of_64_bits(A, ctx, elt, with_bias):
    rng = np.random.default_rng(3)
    for case, (t, e, choose, groups, keep) in enumerate(SHAPES):
        say(elt, with_bias, t, e, choose, groups, keep)
        x = rng.standard_normal((t, e)) * (1.5, 4.0, 12.0)[case % 3]
        if t > 2:
            x[t // 2] = -np.inf                               # a token that nothing is left for
            x[t // 3, : e - e // 4] = -np.inf
        if t > 8 and e > 4:
            x[5, ::3], x[6] = np.nan, 0.5
            x[7, e // 2], x[4] = np.inf, np.float64(np.finfo(np.float32 if elt == "float" else np.float16).min) / (1 if elt == "float" else 2)
        x = values(store(x, elt), elt)
        bias = (rng.standard_normal(e) * 0.1).astype(np.float32) if with_bias else None
        if with_bias and e > 4:
            bias[e // 3] = -np.inf
        normalise, scale = bool(case % 2), (1.0, 2.5)[case % 2]
        loose = case % 3
        same(routed(A, ctx, x, bias, elt, choose, groups, keep, normalise, scale, lead=loose, extra=loose), plain(x, bias, choose, groups, keep, normalise, scale), scale)


@pytest.mark.parametrize("groups,keep", [(1, 1), (4, 2)])
def test_scores_that_lie_next_to_each_other(A, ctx, groups, keep):
    """biases that bring all experts of a row to within 10^-8 of each other, and of two rows the same; logits where scores are 1 but
    for their last bits; equal logits and biases"""
    rng = np.random.default_rng(4)
    t, e, choose = 200, 64, 6
    x = rng.standard_normal((t, e)).astype(np.float32).astype(np.float64)
    bias = (0.7 - 1.0 / (1.0 + np.exp(-x[0]))).astype(np.float32)           # row 0: 0.7 but for the bias' rounding
    x[1] = x[0]
    for k in range(2, 100):
        x[k] = (x[0] * (1 + rng.integers(-1, 2, e) * 2.0 ** -22)).astype(np.float32)
    same(routed(A, ctx, x, bias, "float", choose, groups, keep, True, 1.0), plain(x, bias, choose, groups, keep, True, 1.0), 1.0)
    x = (rng.integers(14, 40, (t, e)) + rng.integers(0, 3, (t, e)) / 4.0).astype(np.float64)
    for elt in TYPES:
        same(routed(A, ctx, x, None, elt, choose, groups, keep, True, 1.0), plain(x, None, choose, groups, keep, True, 1.0), 1.0)
    x = rng.integers(-2, 3, (t, e)).astype(np.float64)
    bias = (rng.integers(0, 2, e) * 0.25).astype(np.float32)
    for elt in TYPES:
        same(routed(A, ctx, x, bias, elt, choose, groups, keep, False, 3.0), plain(x, bias, choose, groups, keep, False, 3.0), 3.0)


@pytest.mark.parametrize("normalise", (False, True))
@pytest.mark.parametrize("elt", TYPES)
def test_gradient_of_the_logits(A, ctx, elt, normalise):
    rng = np.random.default_rng(6)
    for t, e, choose, groups, keep in ((1, 1, 1, 1, 1), (5, 64, 4, 1, 1), (300, 96, 6, 8, 4), (1000, 256, 8, 8, 4), (33, 130, 32, 2, 2), (9, 2048, 3, 1, 1), (77, 10, 1, 2, 1)):
        say(elt, normalise, t, e, choose)
        x = rng.standard_normal((t, e)) * 2.0
        if t > 4:
            x[2], x[3, 5:] = -np.inf, -np.inf
        x = values(store(x, elt), elt)
        experts = plain(x, None, choose, groups, keep, normalise, 1.0)[0]
        dw = rng.standard_normal((t, choose)).astype(np.float32)
        there, at = experts >= 0, np.maximum(experts, 0)
        with np.errstate(all="ignore"):
            s = np.where(there, 1.0 / (1.0 + np.exp(-np.take_along_axis(x, at, 1))), 0.0)
        d, big = np.where(there, dw, 0.0).astype(np.float64), np.abs(np.where(there, dw, 0.0))
        total = s.sum(1, keepdims=True)
        with np.errstate(all="ignore"):
            share = np.where(total > 0, s / total, 0.0) if normalise else s
        inner, most = ((d * share).sum(1, keepdims=True), (big * share).sum(1, keepdims=True)) if normalise else (0.0, 0.0)
        part, size = 2.5 * share * (d - inner) * (1.0 - s), 2.5 * share * (big + most) * (1.0 - s)
        want, bound = np.zeros((t, e)), np.zeros((t, e))
        for j in range(choose):
            rows = there[:, j]
            want[rows, at[rows, j]], bound[rows, at[rows, j]] = part[rows, j], 64 * UNIT * size[rows, j]
        op = A.ScoreRouter(ctx, elt, choose, groups, keep, normalise, 2.5)
        out = Boxed(A, ctx, np.full((t, e), 9.0), elt, lead=t % 3, extra=t % 2, fill=4.0)
        op.gradient(Boxed(A, ctx, x, elt, extra=t % 3).array, ctx.array(experts), ctx.array(dw), out.array)
        ctx.sync()
        op.destroy()
        off = np.abs(values(out.get(), elt) - want) - (bound + HALF_ULP[elt] * 1.001 * np.abs(want) + TINY[elt])
        assert np.all(off <= 0), off.max()
        # and against differences, of the definition
        if normalise and elt == "float" and t == 300:
            for r, j in ((0, 0), (7, 3), (299, 5)):
                loss = lambda v: float((2.5 * v / v.sum() * dw[r]).sum())
                sig = lambda h: np.array([1.0 / (1.0 + np.exp(-(x[r, at[r, i]] + (h if i == j else 0.0)))) for i in range(choose)])
                assert abs((loss(sig(1e-5)) - loss(sig(-1e-5))) / 2e-5 - want[r, at[r, j]]) < 1e-7


def test_routers_that_are_refused(A, ctx):
    for args in (dict(choose=0), dict(choose=33), dict(choose=2, groups=3), dict(choose=2, groups=4, keep=5), dict(choose=2, groups=4, keep=0), dict(choose=1, groups=128), dict(choose=1, scale=float("nan"))):
        with pytest.raises(A.AccError) as e:
            A.ScoreRouter(ctx, "float", **args)
        assert e.value.code == A.ERR_INVALID
    op = A.ScoreRouter(ctx, "float", 3, 4, 2)
    f, i = lambda *s: ctx.empty(s, np.float32), lambda *s: ctx.empty(s, np.int32)
    good = dict(logits=f(5, 16), experts=i(5, 3), weights=f(5, 3), offsets=i(17), order=i(15), place=i(5, 3), bias=f(16))
    op.route(**good)
    for w in (dict(logits=f(5, 18)), dict(logits=f(5, 4)), dict(experts=i(5, 2)), dict(weights=f(4, 3)), dict(offsets=i(16)), dict(order=i(14)), dict(place=i(3, 5)), dict(bias=f(15)),
              dict(place=good["experts"]), dict(bias=A.Strided((16,), (1,), good["weights"].ptr)), dict(logits=None)):
        with pytest.raises(A.AccError) as e:
            op.route(**dict(good, **w))
        assert e.value.code == A.ERR_INVALID
    many = dict(good, logits=f(5, 2052), offsets=i(2053))
    with pytest.raises(A.AccError):
        op.route(**dict(many, bias=None))
    grad = dict(logits=good["logits"], experts=good["experts"], dweights=f(5, 3), dlogits=f(5, 16))
    op.gradient(**grad)
    for w in (dict(dlogits=f(5, 15)), dict(dlogits=good["logits"]), dict(dweights=f(5, 4)), dict(experts=i(6, 3))):
        with pytest.raises(A.AccError):
            op.gradient(**dict(grad, **w))
    # no tokens
    none = dict(logits=f(0, 16), experts=i(0, 3), weights=f(0, 3), offsets=ctx.array(np.full(17, 9, np.int32)), order=i(0), place=i(0, 3))
    op.route(**none)
    op.gradient(f(0, 16), i(0, 3), f(0, 3), f(0, 16))
    ctx.sync()
    assert np.all(none["offsets"].get() == 0)
    op.destroy()
