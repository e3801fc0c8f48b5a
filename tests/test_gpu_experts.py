"""The layer of experts (accelerate-cuda_amd/experts.py) against plain numpy in 64 bits, its gradients also against differences.

Bounds.  A sum of n products in Float32 is off by at most (n + 2) 2^-24 of the sum of the products' sizes.  Through a chain of
them, errors are off by at most the sum of these factors times what the chain makes of sizes alone: `sizes` below is the layer with
every matrix, input and answer replaced by its size, h by |Wup| |x| in the activation and its gradient.  The activation doubles a
relative error and adds two roundings; the router's weights are off by twice the logits' error, (width + 2) 2^-24 |Wr| |x|, and a few
roundings.  FACTOR adds all that up for the longest chain, from x by way of y to a matrix' gradient.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -24


def plain(w, x, chosen, dout, sizes=False):
    """(out, weights, dx, gradients) in 64 bits for the experts that were chosen; `sizes`: of sizes alone"""
    mag = np.abs if sizes else (lambda v: v)
    route, up, down, x, dout = (mag(v) for v in (w["route"], w["up"], w["down"], x, dout))
    tokens, choose = chosen.shape
    logits = plain.logits
    picked = np.take_along_axis(logits, chosen, 1)
    p = np.exp(picked - picked.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    out, dx = np.zeros(x.shape), np.zeros(x.shape)
    g = {"route": np.zeros(route.shape), "up": np.zeros(up.shape), "down": np.zeros(down.shape)}
    dp = np.zeros(p.shape)
    for t in range(tokens):
        for j in range(choose):
            e = chosen[t, j]
            h = up[e] @ x[t]
            a = np.maximum(h, 0) ** 2
            y = down[e] @ a
            out[t] += p[t, j] * y
            dp[t, j] = dout[t] @ y
            dy = p[t, j] * dout[t]
            g["down"][e] += np.outer(dy, a)
            dh = 2 * np.maximum(h, 0) * (down[e].T @ dy)
            g["up"][e] += np.outer(dh, x[t])
            dx[t] += up[e].T @ dh
        inner = (p[t] * dp[t]).sum()
        dl = np.zeros(route.shape[1])
        dl[chosen[t]] = p[t] * (dp[t] + inner if sizes else dp[t] - inner)
        g["route"][0] += np.outer(dl, x[t])
        dx[t] += route[0].T @ dl
    return out, p, dx, g


@pytest.fixture(scope="module")
def A():
    import acchip
    return acchip


@pytest.fixture(scope="module")
def ctx(A):
    c = A.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("tokens,width,hidden,experts,choose", [(1, 8, 5, 3, 1), (37, 33, 50, 6, 2), (130, 64, 96, 8, 3)])
def test_a_layer_of_experts_and_its_gradients(ctx, tokens, width, hidden, experts, choose):
    from experts import Experts
    layer = Experts(ctx, width, hidden, experts, choose, seed=tokens)
    rng = np.random.default_rng(tokens)
    x, dout = rng.standard_normal((tokens, width)).astype(np.float32), rng.standard_normal((tokens, width)).astype(np.float32)
    out, kept = layer.forward(ctx.array(x))
    dx, g = layer.backward(kept, ctx.array(dout))
    w = {k: v.get().astype(float) for k, v in layer.w.items()}
    x, dout, chosen = x.astype(float), dout.astype(float), kept[1]["experts"].get()
    plain.logits = x @ w["route"][0].T
    near = (width + 2) * ULP * (np.abs(x) @ np.abs(w["route"][0]).T)
    # what was chosen is largest, but for logits that are too near to tell
    rest = plain.logits.copy()
    np.put_along_axis(rest, chosen, -np.inf, 1)
    assert (np.take_along_axis(plain.logits, chosen, 1).min(1) + 2 * near.max(1) >= rest.max(1)).all()
    factor = 2 * (width + 4) + (hidden + 4) + 2 * (hidden + width + 8) + tokens * choose + choose + 16 + 4 * near.max() / ULP
    want, size = plain(w, x, chosen, dout), plain(w, x, chosen, dout, sizes=True)
    assert (np.abs(out.get() - want[0]) <= factor * ULP * size[0]).all()
    assert (np.abs(kept[1]["weights"].get() - want[1]) <= (4 * near.max() / ULP + 16) * ULP * want[1]).all()
    assert (np.abs(dx.get() - want[2]) <= factor * ULP * size[2]).all()
    for name in g:
        assert (np.abs(g[name].get() - want[3][name]) <= factor * ULP * size[3][name]).all(), name
    # against differences of the formula: the loss <dout, out> along a direction of everything that is learnt, the choice kept
    move = {k: rng.standard_normal(v.shape) for k, v in w.items()}
    step, loss = 1e-5, []
    for s in (step, -step):
        there = {k: w[k] + s * move[k] for k in w}
        plain.logits = x @ there["route"][0].T
        loss.append((dout * plain(there, x, chosen, dout)[0]).sum())
    along = sum((g[k].get() * move[k]).sum() for k in g)
    # (the formula has a third derivative of the size of its second; rounding of the losses, 2^-52 of their sizes over 2 step)
    third = sum((np.abs(move[k]) * size[3][k]).sum() for k in w)
    assert abs((loss[0] - loss[1]) / (2 * step) - along) <= factor * ULP * third + 1e-3 * step * third * 100 + 2.0 ** -50 * np.abs(dout * size[0]).sum() / step
    layer.destroy()


def test_a_step_down_the_gradient_brings_the_answers_nearer(ctx):
    from experts import Experts
    teacher, pupil = Experts(ctx, 40, 24, 4, 2, seed=1), Experts(ctx, 40, 24, 4, 2, seed=2)
    x = ctx.array(np.random.default_rng(5).standard_normal((64, 40)).astype(np.float32))
    want = teacher.forward(x)[0].get()
    losses = []
    for _ in range(4):
        out, kept = pupil.forward(x)
        off = out.get() - want
        losses.append(float((off.astype(float) ** 2).sum()))
        pupil.step(pupil.backward(kept, ctx.array(2 * off / 64))[1], 0.01)
    assert all(b < a for a, b in zip(losses, losses[1:]))
    teacher.destroy()
    pupil.destroy()


@pytest.mark.parametrize("tokens", [1, 50])
def test_answers_in_four_bits_are_those_of_the_operators_one_by_one(A, ctx, tokens):
    from experts import Experts
    layer = Experts(ctx, 64, 160, 6, 2, seed=9)
    layer.quantise()
    x = ctx.array(np.random.default_rng(6).standard_normal((tokens, 64)).astype(np.float32))
    got = layer.serve(x).get()
    r, slots = layer.route(x), tokens * 2
    micro = A.Microscale(ctx, "float")

    def four(a):
        codes, scales = ctx.empty((a.shape[0], 16 * ((a.shape[1] + 31) // 32)), np.uint8), ctx.empty((a.shape[0], (a.shape[1] + 31) // 32), np.uint8)
        micro.quantise(a, codes, scales)
        values = ctx.empty(a.shape, np.float32)
        micro.values(codes, scales, values)
        return codes, scales, values.get().astype(float)

    xc, xs, xv = four(x)
    h = ctx.empty((slots, 160), np.float32)
    micro.rows(xc, xs, *layer.four_bits["up"], r["offsets"], h, index=r["order"], per=2)
    # the products are those of the numbers that the codes stand for
    flat = lambda name: A.DeviceArray.view(ctx, (6 * layer.w[name].shape[1], layer.w[name].shape[2]), np.dtype(np.float32), layer.w[name].size, layer.w[name].ptr)
    up, order, offsets = four(flat("up"))[2].reshape(6, 160, 64), r["order"].get(), r["offsets"].get()
    for e in range(6):
        for m in range(offsets[e], offsets[e + 1]):
            want, size = up[e] @ xv[order[m] // 2], np.abs(up[e]) @ np.abs(xv[order[m] // 2])
            assert (np.abs(h.get()[m] - want) <= (64 + 2) * ULP * size).all()
    a = ctx.array(np.where(h.get() > 0, h.get() * h.get(), np.float32(0)))
    ac, as_, _ = four(a)
    y, out = ctx.empty((slots, 64), np.float32), ctx.empty((tokens, 64), np.float32)
    micro.rows(ac, as_, *layer.four_bits["down"], r["offsets"], y)
    A.Combiner(ctx, "float").combine(y, r["place"], r["weights"], out)
    assert np.array_equal(got, out.get())
    layer.destroy()


def test_the_layer_runs_as_a_command(capsys):
    import experts
    experts.main(64, 3)
    said = capsys.readouterr().out.splitlines()
    assert len(said) == 4 and said[0].startswith("step  0") and said[-1].startswith("in 4 bits")
