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
