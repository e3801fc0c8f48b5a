"""A layer of experts on the operators of include/acc_hip.h, section D, next to the skeletons: one training step after
the other, then answers from matrices of 4-bit numbers.

    logits[t]  = Wr x[t]                                         a product with one matrix
    experts    = the `choose` largest logits, their weights w    route: slots sorted by expert, in segments; with `groups` by
                                                                 scores and a bias that evens out what the experts have to do
    h          = Wup[e] x[token of the slot]                     a product of rows with their expert's matrix, through the order
    a          = max(h, 0) ^ 2                                   map
    y          = Wdown[e] a                                      a product of rows
    out[t]     = sum_j w[t, j] y[place[t, j]]                    combine

Everything stays on the device; what goes to the host is what `get` is called on.

    python accelerate-cuda_amd/experts.py [tokens [steps]]
"""
import sys

import numpy as np

import acchip as A

F1, F2, F3 = (1, "float"), (2, "float"), (3, "float")


class Experts(object):
    """`experts` pairs of matrices of `width` x `hidden` in Float32, of which every token takes `choose`; with `groups`, those with the
    best scores in the best `keep` groups of experts."""

    def __init__(self, ctx, width, hidden, experts, choose, seed=0, groups=0, keep=1):
        self.ctx, self.width, self.hidden, self.experts, self.choose = ctx, width, hidden, experts, choose
        rng = np.random.default_rng(seed)
        self.w = {}
        for name, shape in (("route", (1, experts, width)), ("up", (experts, hidden, width)), ("down", (experts, width, hidden))):
            self.w[name] = ctx.array((rng.standard_normal(shape) / np.sqrt(shape[2])).astype(np.float32))
        self.product, self.combiner = A.Product(ctx, "float"), A.Combiner(ctx, "float")
        self.router = A.ScoreRouter(ctx, "float", choose, groups, keep) if groups else A.Router(ctx, "float", choose)
        self.bias = ctx.array(np.zeros(experts, np.float32)) if groups else None
        self.micro, self.grouped = A.Microscale(ctx, "float"), A.Grouped(ctx, "float", 32)
        one, other = "arrIn0_0[ix]", "arrIn1_0[ix]"
        self.act = ctx.skeleton(A.SKEL_MAP, "float", env=[F2], out_rank=2, get="%s > 0.0f ? %s * %s : 0.0f" % (one, one, one))
        self.act_gradient = ctx.skeleton(A.SKEL_MAP, "float", env=[F2, F2], out_rank=2, get="%s > 0.0f ? 2.0f * %s * %s : 0.0f" % (one, one, other))
        self.add = ctx.skeleton(A.SKEL_MAP, "float", env=[F2, F2], out_rank=2, get="%s + %s" % (one, other))
        self.descend = ctx.skeleton(A.SKEL_MAP, "float", env=[F3, F3, F1], out_rank=3, get="%s - arrIn2_0[0] * %s" % (one, other))
        share = "(float)arrIn1_0[%d] / %d" % (experts, experts)
        count = "(float)(arrIn1_0[ix + 1] - arrIn1_0[ix])"
        self.even = ctx.skeleton(A.SKEL_MAP, "float", env=[F1, (1, "Int32"), F1], out_rank=1, get="arrIn0_0[ix] + arrIn2_0[0] * (%s < %s ? 1.0f : %s > %s ? -1.0f : 0.0f)" % (count, share, count, share))
        self.four_bits = None

    def destroy(self):
        for op in (self.product, self.router, self.combiner, self.micro, self.grouped, self.act, self.act_gradient, self.add, self.descend, self.even):
            op.destroy()

    def _floats(self, *shape):
        return self.ctx.empty(shape, np.float32)

    def _ints(self, *shape):
        return self.ctx.empty(shape, np.int32)

    def route(self, x):
        """where the tokens go: everything the passes below need to know of it"""
        tokens = x.shape[0]
        r = {"all": self.ctx.array(np.array([0, tokens], np.int32)), "logits": self._floats(tokens, self.experts),
             "experts": self._ints(tokens, self.choose), "weights": self._floats(tokens, self.choose), "offsets": self._ints(self.experts + 1),
             "order": self._ints(tokens * self.choose), "place": self._ints(tokens, self.choose)}
        self.product.rows(x, self.w["route"], r["all"], r["logits"])
        self.router.route(r["logits"], r["experts"], r["weights"], r["offsets"], r["order"], r["place"], **({} if self.bias is None else {"bias": self.bias}))
        return r

    def balance(self, r, rate):
        """the experts' bias, a step of `rate` up for those that had less than their share to do, and down for the others"""
        new = self._floats(self.experts)
        self.even.map([self.bias, r["offsets"], self.ctx.array(np.array([rate], np.float32))], new)
        self.bias = new

    def forward(self, x):
        """the answer to x [tokens, width], and what `backward` needs"""
        r, slots = self.route(x), x.shape[0] * self.choose
        h, a, y, out = self._floats(slots, self.hidden), self._floats(slots, self.hidden), self._floats(slots, self.width), self._floats(x.shape[0], self.width)
        self.product.rows(x, self.w["up"], r["offsets"], h, index=r["order"], per=self.choose)
        self.act.map([h], a)
        self.product.rows(a, self.w["down"], r["offsets"], y)
        self.combiner.combine(y, r["place"], r["weights"], out)
        return out, (x, r, h, a, y)

    def backward(self, kept, dout):
        """the gradients of x and of the matrices"""
        x, r, h, a, y = kept
        slots, tokens = h.shape[0], x.shape[0]
        g = {name: self._floats(*w.shape) for name, w in self.w.items()}
        dy, da, dh, dslots = self._floats(slots, self.width), self._floats(slots, self.hidden), self._floats(slots, self.hidden), self._floats(slots, self.width)
        dweights, dlogits = self._floats(tokens, self.choose), self._floats(tokens, self.experts)
        through, beside, dx = self._floats(tokens, self.width), self._floats(tokens, self.width), self._floats(tokens, self.width)
        turned = lambda w: A.Strided.of(w).swap()
        self.combiner.gradient(dout, y, r["place"], r["weights"], dy, dweights)
        self.product.outer(dy, a, r["offsets"], g["down"])
        self.product.rows(dy, turned(self.w["down"]), r["offsets"], da)
        self.act_gradient.map([h, da], dh)
        self.product.outer(dh, x, r["offsets"], g["up"], index=r["order"], per=self.choose)
        self.product.rows(dh, turned(self.w["up"]), r["offsets"], dslots)
        self.combiner.combine(dslots, r["place"], None, through)
        if self.bias is None:
            self.router.gradient(r["logits"], r["experts"], r["weights"], dweights, dlogits)
        else:
            self.router.gradient(r["logits"], r["experts"], dweights, dlogits)
        self.product.outer(dlogits, x, r["all"], g["route"])
        self.product.rows(dlogits, turned(self.w["route"]), r["all"], beside)
        self.add.map([through, beside], dx)
        return dx, g

    def step(self, g, rate):
        """the matrices, a step of `rate` down the gradients"""
        by = self.ctx.array(np.array([rate], np.float32))
        for name, w in self.w.items():
            new = self._floats(*w.shape)
            self.descend.map([w, g[name], by], new)
            self.w[name] = new

    def _quantised(self, x):
        rows, blocks = x.shape[0], (x.shape[1] + 31) // 32
        codes, scales = self.ctx.empty((rows, 16 * blocks), np.uint8), self.ctx.empty((rows, blocks), np.uint8)
        self.micro.quantise(x, codes, scales)
        return codes, scales

    def quantise(self, grouped=False):
        """the experts' matrices in 4 bits, as `serve` takes them: floating-point numbers, for rows in the same form, or `grouped`, whole
        numbers under a scale and a zero for every 32, for rows as they are"""
        self.four_bits = {}
        if grouped:
            for name in ("up", "down"):
                e, n, k = self.w[name].shape
                b = (k + 31) // 32
                codes, scales, zeros = self.ctx.empty((e, n, 16 * b), np.uint8), self._floats(e, b, n), self.ctx.empty((e, b, n), np.uint8)
                self.grouped.quantise(self.w[name], codes, scales, zeros)
                self.four_bits[name] = (codes, scales, zeros)
            return
        for name in ("up", "down"):
            w = self.w[name]
            e, n, k = w.shape
            codes, scales = self._quantised(A.DeviceArray.view(self.ctx, (e * n, k), w.dtype, w.size, w.ptr))
            self.four_bits[name] = tuple(A.Strided((e, n, p.shape[1]), (n * p.shape[1], p.shape[1], 1), p.ptr, p) for p in (codes, scales))

    def serve(self, x):
        """`forward` with both products in 4 bits"""
        r, slots = self.route(x), x.shape[0] * self.choose
        h, a, y, out = self._floats(slots, self.hidden), self._floats(slots, self.hidden), self._floats(slots, self.width), self._floats(x.shape[0], self.width)
        if len(self.four_bits["up"]) == 3:
            (up, s, z), (down, t, u) = self.four_bits["up"], self.four_bits["down"]
            self.grouped.rows(x, up, s, r["offsets"], h, zeros=z, index=r["order"], per=self.choose)
            self.act.map([h], a)
            self.grouped.rows(a, down, t, r["offsets"], y, zeros=u)
        else:
            self.micro.rows(*self._quantised(x), *self.four_bits["up"], r["offsets"], h, index=r["order"], per=self.choose)
            self.act.map([h], a)
            self.micro.rows(*self._quantised(a), *self.four_bits["down"], r["offsets"], y)
        self.combiner.combine(y, r["place"], r["weights"], out)
        return out


def main(tokens=1000, steps=20):
    """a layer learns what another one answers; then it answers from 4 bits a number"""
    ctx = A.Context(0)
    teacher, pupil = Experts(ctx, 96, 160, 8, 2, seed=1), Experts(ctx, 96, 160, 8, 2, seed=2)
    x = ctx.array(np.random.default_rng(3).standard_normal((tokens, 96)).astype(np.float32))
    want = teacher.forward(x)[0].get()
    for k in range(steps):
        out, kept = pupil.forward(x)
        off = out.get() - want
        print("step %2d: %.4f off" % (k, np.sqrt(np.mean(off * off))), flush=True)
        pupil.step(pupil.backward(kept, ctx.array(off * np.float32(2.0 / tokens)))[1], 0.02)
    whole = pupil.forward(x)[0].get()
    pupil.quantise()
    off = pupil.serve(x).get() - whole
    print("in 4 bits: %.3f of the answers' size off" % (np.linalg.norm(off) / np.linalg.norm(whole)))
    teacher.destroy()
    pupil.destroy()
    ctx.close()


if __name__ == "__main__":
    main(*(int(v) for v in sys.argv[1:3]))
