"""The decoder's block (accelerate-cuda_amd/decoder.py): its gradients against differences of the block in 64 bits, its steps against
whole sequences, its answers in 4 bits against the same block on the numbers that those stand for."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import acchip as A
    c = A.Context(0)
    yield c
    c.close()


def sigmoid(v):
    return 1.0 / (1.0 + np.exp(-v))


def plain(w, x, offsets, chosen):
    """the block in 64 bits, for the experts that were chosen"""
    z, v = x @ w["z"][0].T, x @ w["v"][0].T
    h = np.zeros(z.shape)
    for b, e in zip(offsets, offsets[1:]):
        state = np.zeros(z.shape[1])
        for t in range(b, e):
            state = sigmoid(z[t]) * state + sigmoid(-z[t]) * v[t]
            h[t] = state
    y = x + h @ w["o"][0].T
    scores = sigmoid(np.take_along_axis(y @ w["route"][0].T, chosen, 1))
    share = scores / scores.sum(1, keepdims=True)
    out = y.copy()
    for t in range(x.shape[0]):
        for j, e in enumerate(chosen[t]):
            out[t] += share[t, j] * (w["down"][e] @ np.maximum(w["up"][e] @ y[t], 0.0) ** 2)
    return out


def matrices(block):
    return {k: v.get().astype(float) for k, v in list(block.w.items()) + list(block.layer.w.items())}


@pytest.mark.parametrize("tokens,width,inner,hidden,experts,choose,groups,keep", [(1, 8, 5, 7, 4, 2, 2, 1), (60, 24, 33, 40, 16, 4, 4, 2)])
def test_a_block_and_its_gradients(ctx, tokens, width, inner, hidden, experts, choose, groups, keep):
    from decoder import Block
    block = Block(ctx, width, inner, hidden, experts, choose, groups, keep, seed=tokens)
    rng = np.random.default_rng(tokens)
    offsets = np.array([0, tokens // 3, tokens // 3, tokens], np.int32)
    x, dout = (rng.standard_normal((tokens, width)).astype(np.float32) for _ in range(2))
    out, kept = block.forward(ctx.array(x), ctx.array(offsets))
    dx, g = block.backward(kept, ctx.array(dout))
    chosen, w = kept[5][1]["experts"].get(), matrices(block)
    x, dout = x.astype(float), dout.astype(float)
    want = plain(w, x, offsets, chosen)
    # (sums of up to `hidden` products in Float32, one behind the other three times; the activation doubles what is off)
    assert np.abs(out.get() - want).max() <= 2.0 ** -24 * 16 * (width + inner + hidden) * (1 + np.abs(want).max())
    g = dict({k: v.get().astype(float) for k, v in g.items()}, x=dx.get().astype(float))
    for name in sorted(g):
        move = rng.standard_normal(g[name].shape)
        loss = []
        for by in (1e-5, -1e-5):
            there = dict(w)
            if name != "x":
                there[name] = w[name] + by * move
            loss.append((dout * plain(there, x + by * move if name == "x" else x, offsets, chosen)).sum())
        along, size = (g[name] * move).sum(), np.linalg.norm(g[name]) * np.linalg.norm(move)
        # (Float32 sums as above, and what a step of 10^-5 leaves of the second derivative's growth)
        assert abs((loss[0] - loss[1]) / 2e-5 - along) <= 2e-5 * size + 1e-6, name
    block.destroy()


def test_a_token_at_a_time_is_the_whole_sequence(ctx):
    """in 4 bits: steps of decoding against whole sequences on the matrices that the 4 bits stand for; states in a table"""
    from decoder import Block
    block = Block(ctx, 40, 50, 64, 8, 2, 4, 3, seed=7)
    rng = np.random.default_rng(7)
    steps, n = 5, 6
    x = rng.standard_normal((n, steps, 40)).astype(np.float32)
    block.quantise()
    for name, (codes, scales, zeros) in block.layer.four_bits.items():
        made = ctx.empty(block.layer.w[name].shape, np.float32)
        block.layer.grouped.values(codes, scales, made, zeros=zeros)
        block.layer.w[name] = made
    offsets = ctx.array((np.arange(n + 1) * steps).astype(np.int32))
    last = block.states(n)
    whole, kept = block.forward(ctx.array(x.reshape(-1, 40)), offsets, last=last)
    whole = whole.get().reshape(n, steps, 40)
    state, rows = block.states(n + 3), np.array([7, 2, 0, 5, 8, 3], np.int32)
    for t in range(steps):
        got = block.serve(ctx.array(np.ascontiguousarray(x[:, t])), state, ctx.array(rows)).get()
        assert np.abs(got - whole[:, t]).max() <= 1e-4 * np.abs(whole).max()
    assert np.abs(state.get()[rows] - last.get()).max() <= 1e-5
    block.destroy()


def test_what_evens_out_the_experts(ctx):
    from decoder import Block
    block = Block(ctx, 24, 16, 24, 8, 2, 2, 2, seed=3)
    x = ctx.array(np.random.default_rng(3).standard_normal((500, 24)).astype(np.float32))
    r = block.layer.route(x)
    counts = np.diff(r["offsets"].get())
    block.layer.balance(r, 0.125)
    assert np.array_equal(block.layer.bias.get(), (0.125 * np.sign(125 - counts)).astype(np.float32))
    block.destroy()


def test_the_example_runs(capsys):
    import decoder
    decoder.main(300, 3)
    assert "in 4 bits" in capsys.readouterr().out
