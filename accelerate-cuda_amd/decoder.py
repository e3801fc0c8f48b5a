"""A decoder's block on the operators of include/acc_hip.h, section D: what was mixes with what is along every sequence, then every token
goes to its experts (experts.py).  It learns from whole sequences and answers a token at a time.

    z, v  = Wz x, Wv x                            products with one matrix
    h     = s(z) h' + (1 - s(z)) v                a gated linear recurrence along the rows of every sequence
    y     = x + Wo h
    out   = y + the layer of experts of y         chosen by scores and a bias

A step of decoding keeps h of every sequence in a table of states, and the experts' matrices in 4 bits.

    python accelerate-cuda_amd/decoder.py [tokens [steps]]
"""
import sys

import numpy as np

import acchip as A
from experts import F1, F2, F3, Experts


class Block(object):
    """rows of `width` in Float32; a state of `inner` channels a sequence; `experts` of which every token takes `choose`"""

    def __init__(self, ctx, width, inner, hidden, experts, choose, groups, keep, seed=0):
        self.ctx, self.width, self.inner = ctx, width, inner
        rng = np.random.default_rng(seed)
        self.w = {}
        for name, shape in (("z", (1, inner, width)), ("v", (1, inner, width)), ("o", (1, width, inner))):
            self.w[name] = ctx.array((rng.standard_normal(shape) / np.sqrt(shape[2])).astype(np.float32))
        self.layer = Experts(ctx, width, hidden, experts, choose, seed + 1, groups, keep)
        self.product, self.recurrence = A.Product(ctx, "float"), A.Recurrence(ctx, "float", "sigmoid")
        self.add = ctx.skeleton(A.SKEL_MAP, "float", env=[F2, F2], out_rank=2, get="arrIn0_0[ix] + arrIn1_0[ix]")
        self.descend = ctx.skeleton(A.SKEL_MAP, "float", env=[F3, F3, F1], out_rank=3, get="arrIn0_0[ix] - arrIn2_0[0] * arrIn1_0[ix]")

    def destroy(self):
        self.layer.destroy()
        for op in (self.product, self.recurrence, self.add, self.descend):
            op.destroy()

    def _floats(self, *shape):
        return self.ctx.empty(shape, np.float32)

    def _sum(self, a, b):
        out = self._floats(*a.shape)
        self.add.map([a, b], out)
        return out

    def _rows(self, x, w, out):
        """all rows with one matrix"""
        self.product.rows(x, w, self.ctx.array(np.array([0, x.shape[0]], np.int32)), out)
        return out

    def states(self, sequences):
        return self.ctx.array(np.zeros((sequences, self.inner), np.float32))

    def _mixed(self, x, recur):
        z, v, h = (self._floats(x.shape[0], self.inner) for _ in range(3))
        self._rows(x, self.w["z"], z)
        self._rows(x, self.w["v"], v)
        recur(z, v, h)
        return z, v, h, self._sum(x, self._rows(h, self.w["o"], self._floats(*x.shape)))

    def forward(self, x, offsets, last=None):
        """the answers to the rows of every sequence, and what `backward` needs; `last`: where the states behind them go"""
        z, v, h, y = self._mixed(x, lambda z, v, h: self.recurrence.scan(z, v, offsets, h, last=last))
        out, kept = self.layer.forward(y)
        return self._sum(y, out), (x, offsets, z, v, h, kept)

    def backward(self, kept, dout):
        """the gradients of x and of all matrices"""
        x, offsets, z, v, h, below = kept
        rows = x.shape[0]
        turned = lambda w: A.Strided.of(w).swap()
        dy, g = self.layer.backward(below, dout)
        dy = self._sum(dout, dy)
        all_rows = self.ctx.array(np.array([0, rows], np.int32))
        g.update({name: self._floats(*w.shape) for name, w in self.w.items()})
        self.product.outer(dy, h, all_rows, g["o"])
        dh, dz, dv = (self._floats(rows, self.inner) for _ in range(3))
        self._rows(dy, turned(self.w["o"]), dh)
        self.recurrence.gradient(z, v, offsets, h, dh, dz, dv)
        self.product.outer(dz, x, all_rows, g["z"])
        self.product.outer(dv, x, all_rows, g["v"])
        dx = self._sum(dy, self._rows(dz, turned(self.w["z"]), self._floats(*x.shape)))
        return self._sum(dx, self._rows(dv, turned(self.w["v"]), self._floats(*x.shape))), g

    def step(self, g, rate):
        """all matrices, a step of `rate` down the gradients"""
        by = self.ctx.array(np.array([rate], np.float32))
        for name, w in self.w.items():
            new = self._floats(*w.shape)
            self.descend.map([w, g[name], by], new)
            self.w[name] = new
        self.layer.step(g, rate)

    def quantise(self):
        self.layer.quantise(grouped=True)

    def serve(self, x, state, index=None):
        """a token of every sequence, whose states are the rows `index` of `state` (replaced in place); experts in 4 bits"""
        _, _, _, y = self._mixed(x, lambda z, v, h: self.recurrence.step(z, v, state, state, h, index=index))
        return self._sum(y, self.layer.serve(y))


def main(tokens=1000, steps=10):
    """a block learns what another one answers; then it answers a token at a time, its experts in 4 bits"""
    ctx = A.Context(0)
    teacher, pupil = (Block(ctx, 96, 128, 160, 16, 4, 4, 2, seed=seed) for seed in (1, 5))
    rng = np.random.default_rng(3)
    offsets = ctx.array(np.concatenate([[0], np.sort(rng.integers(0, tokens, 7)), [tokens]]).astype(np.int32))
    x = ctx.array(rng.standard_normal((tokens, 96)).astype(np.float32))
    want = teacher.forward(x, offsets)[0].get()
    for k in range(steps):
        out, kept = pupil.forward(x, offsets)
        off = out.get() - want
        used = np.diff(kept[5][1]["offsets"].get())
        print("step %2d: %.4f off, experts have %d to %d rows" % (k, np.sqrt(np.mean(off * off)), used.min(), used.max()), flush=True)
        pupil.step(pupil.backward(kept, ctx.array(off * np.float32(2.0 / tokens)))[1], 0.05)
        pupil.layer.balance(kept[5][1], 0.02)
    pupil.quantise()
    starts = offsets.get()
    longest, state, off, size = int(np.diff(starts).max()), pupil.states(8), 0.0, 0.0
    whole = pupil.forward(x, offsets)[0].get()
    for t in range(min(longest, 8)):
        here = np.array([s for s in range(8) if starts[s] + t < starts[s + 1]], np.int32)
        got = pupil.serve(ctx.array(x.get()[starts[here] + t]), state, ctx.array(here)).get()
        off, size = off + np.sum((got - whole[starts[here] + t]) ** 2), size + np.sum(whole[starts[here] + t] ** 2)
    print("a token at a time, in 4 bits: %.3f of the answers' size off" % np.sqrt(off / size))
    teacher.destroy()
    pupil.destroy()
    ctx.close()


if __name__ == "__main__":
    main(*(int(v) for v in sys.argv[1:3]))
