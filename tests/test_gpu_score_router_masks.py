"""The router by scores (include/acc_hip.h, section D) where biases and logits are masks: the largest and lowest numbers, infinities, scores that
64 bits no longer hold.  Choices are asked to be those of the definition in 64 bits."""
import sys

import numpy as np
import pytest

from test_gpu_score_router import plain, routed, same

pytestmark = pytest.mark.gpu
LOWEST, LARGEST = np.finfo(np.float32).min, np.finfo(np.float32).max


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


@pytest.mark.parametrize("elt", ("float", "bfloat16"))
@pytest.mark.parametrize("t,size,groups,keep,choose", ((9, 4, 4, 1, 3), (50, 8, 8, 3, 6), (3000, 16, 8, 2, 8), (300, 2, 64, 5, 4)))
def test_biases_that_are_masks(A, ctx, elt, t, size, groups, keep, choose):
    """a group whose biases are all the lowest number has experts to choose, one whose logits are all minus infinity has none"""
    rng, e = np.random.default_rng(size), size * groups
    x = rng.integers(-6, 7, (t, groups, size)) / 2.0
    x[rng.random((t, groups)) < 0.4] = -np.inf                 # (groups without an expert)
    x[t // 2, : groups - 1] = -np.inf
    x = x.reshape(t, e)
    bias = np.zeros((groups, size), np.float32)
    for name, fill in (("lowest", lambda g: LOWEST), ("some lowest", lambda g: LOWEST if g % 2 else 0.0), ("far", lambda g: (LOWEST, LOWEST / 2, -1e38, LARGEST)[g % 4]),
                       ("largest", lambda g: (LARGEST, 3e38, LARGEST / 2)[g % 3]), ("large and small", lambda g: LARGEST if g % 3 else LOWEST)):
        for g in range(groups):
            bias[g] = fill(g)
            bias[g, 1::3] = fill(g + 1) / 2 if name == "far" else fill(g)
        say(elt, t, size, groups, keep, name)
        b = bias.reshape(-1)
        same(routed(A, ctx, x, b, elt, choose, groups, keep, True, 1.0), plain(x, b, choose, groups, keep, True, 1.0), 1.0)


@pytest.mark.parametrize("normalise", (True, False))
def test_scores_that_64_bits_do_not_hold(A, ctx, normalise):
    """from 709.78 below 0 on e^-x is an infinity: a score is 0 there, for the choice and for the weight; one just above is not"""
    rng, t, e, choose = np.random.default_rng(5), 300, 24, 4
    x = (-rng.uniform(705, 714, (t, e))).astype(np.float32).astype(np.float64)
    x[::3] = (-rng.uniform(709.8, 760, x[::3].shape)).astype(np.float32)
    x[1::9, :] = -760.0
    x[1::9, 5], x[1::9, 7] = np.float32(-709.78271484375), np.float32(-709.78265380859375)
    for groups, keep in ((1, 1), (4, 2)):
        say(normalise, groups)
        want = plain(x, None, choose, groups, keep, normalise, 1.0)
        if normalise:
            assert np.any(want[1].sum(1) == 0) and np.any(want[1].sum(1) > 0.9)
        got = routed(A, ctx, x, None, "float", choose, groups, keep, normalise, 1.0)
        same(got, want, 1.0)
        # the gradient: of a token whose scores are all 0 none, and of the others their parts'
        op = A.ScoreRouter(ctx, "float", choose, groups, keep, normalise, 1.0)
        dw, back = rng.standard_normal((t, choose)).astype(np.float32), ctx.empty((t, e), np.float32)
        op.gradient(ctx.array(x.astype(np.float32)), ctx.array(got[0]), ctx.array(dw), back)
        ctx.sync()
        op.destroy()
        share = want[1]
        d = share * (dw - (dw * share).sum(1, keepdims=True)) if normalise else share * dw
        full = np.zeros((t, e))
        np.put_along_axis(full, got[0].astype(np.int64), d, 1)
        assert np.all(np.abs(back.get() - full) <= 200 * 2.0 ** -24 * np.abs(dw).sum(1, keepdims=True) + 1e-37)
