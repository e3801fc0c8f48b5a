"""The operators of a layer of experts, case by case: products of ragged segments of rows with a matrix each, the router that
makes the segments, the combination that brings the rows back, and the same products on 4-bit operands.

    listed()           the cases, from a few tokens of a decoding step to the rows of a training step
    draw(rng)          another case of the same ranges
    prepare(case, s)   inputs made from the seed `s` and the arrays that results go to
    run(state)         one pass: the framework's operators where `own` is true, elementary operations in 32 bits where it is not
    work(case)         the bytes and operations that a pass cannot do without
    exact(case, s)     what `run` returns, from the definition in 64 bits
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"float": torch.float32, "half": torch.float16, "bfloat16": torch.bfloat16}
SIZE = {"float": 4, "half": 2, "bfloat16": 2}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)          # the magnitudes that the three lower bits of a 4-bit number stand for


def listed():
    return [
        # One decoding step of eight sequences, two experts a token: what counts is the weights that have to be read, and
        # what a call costs.
        {"name": "rows_decode_16", "path": "rows", "type": "bfloat16", "rows": 16, "experts": 8, "n": 1024, "k": 1024, "spread": "even", "order": "nk", "per": 2},
        # A decoding step of a larger batch with many experts: 32 experts' weights pass by once, for a row or two each.
        {"name": "rows_decode_64", "path": "rows", "type": "bfloat16", "rows": 64, "experts": 32, "n": 4096, "k": 2048, "spread": "even", "order": "nk", "per": 2},
        # A prompt's rows on odd sizes, some experts without a row, weights kept the other way round (as the gradient
        # with respect to the rows reads them).
        {"name": "rows_ragged_5003", "path": "rows", "type": "half", "rows": 5003, "experts": 24, "n": 1333, "k": 1001, "spread": "skewed", "order": "kn", "per": 0},
        # The rows of a training step on sixteen experts.
        {"name": "rows_train_32k", "path": "rows", "type": "bfloat16", "rows": 32768, "experts": 16, "n": 4096, "k": 2048, "spread": "skewed", "order": "nk", "per": 2},
        # The array language's own element type, in an ordinary size.
        {"name": "rows_float_8k", "path": "rows", "type": "float", "rows": 8192, "experts": 8, "n": 1024, "k": 1536, "spread": "even", "order": "nk", "per": 0},
        # The gradient of the weights in that training step.
        {"name": "outer_train_32k", "path": "outer", "type": "bfloat16", "rows": 32768, "experts": 16, "n": 4096, "k": 2048, "spread": "skewed", "per": 2},
        # The smallest call: eight tokens of a decoding step are given their experts.
        {"name": "route_8", "path": "route", "type": "float", "tokens": 8, "experts": 64, "choose": 4, "normalise": True, "padding": 0.0},
        # The tokens of a training step, padding among them.
        {"name": "route_64k", "path": "route", "type": "bfloat16", "tokens": 65536, "experts": 128, "choose": 8, "normalise": False, "padding": 0.02},
        # The experts' results of four slots a token summed into the layer's.
        {"name": "combine_16k", "path": "combine", "type": "bfloat16", "tokens": 16384, "choose": 4, "width": 2048},
        # Its gradient, on odd sizes.
        {"name": "combine_gradient_4k", "path": "combine_gradient", "type": "bfloat16", "tokens": 4097, "choose": 6, "width": 1501},
        # 4-bit weights: a decoding step, activations quantised on the way.
        {"name": "micro_decode_32", "path": "micro", "type": "bfloat16", "rows": 32, "experts": 16, "n": 4096, "k": 4096, "spread": "even"},
        # ... and a long prompt.
        {"name": "micro_prompt_16k", "path": "micro", "type": "bfloat16", "rows": 16384, "experts": 8, "n": 4096, "k": 4096, "spread": "even"},
    ]


def _size(rng, low, high):
    """a size between `low` and `high`, even over the logarithm: mostly odd ones, some multiples of 64"""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.4 and n >= 64:
        n = n // 64 * 64
    return max(low, min(high, n))


def draw(rng):
    path = rng.choice(["rows", "rows", "rows", "outer", "outer", "route", "route_gradient", "combine", "combine_gradient", "micro", "micro", "values"])
    if path in ("rows", "outer", "micro"):
        c = {"path": path, "type": rng.choice(["bfloat16", "bfloat16", "half", "float"]) if path != "micro" else rng.choice(["bfloat16", "half"]),
             "rows": _size(rng, 1, 32768), "experts": _size(rng, 1, 64), "n": _size(rng, 32, 4096), "k": _size(rng, 32, 4096), "spread": rng.choice(["even", "skewed"])}
        while c["rows"] * c["n"] * c["k"] * (8 if c["type"] == "float" else 1) > 1 << 38 or c["experts"] * c["n"] * c["k"] > 1 << 28:
            c[rng.choice(["n", "k"])] = _size(rng, 32, 2048)
            c["experts"] = max(1, c["experts"] * 3 // 4)
        if path == "rows":
            c["order"] = rng.choice(["nk", "kn"])
        if path != "micro":
            c["per"] = rng.choice([0, 1, 2, 4])
        return c
    if path in ("route", "route_gradient"):
        experts = _size(rng, 4, 512)
        return {"path": path, "type": rng.choice(["float", "bfloat16", "half"]), "tokens": _size(rng, 1, 65536 if experts <= 128 else 16384), "experts": experts,
                "choose": rng.randint(1, min(8, experts)), "normalise": rng.choice([True, False]), "padding": rng.choice([0.0, 0.02, 0.3])}
    if path == "values":
        return {"path": path, "type": rng.choice(["bfloat16", "half", "float"]), "rows": _size(rng, 1, 16384), "k": _size(rng, 32, 4096)}
    return {"path": path, "type": rng.choice(["bfloat16", "half", "float"]), "tokens": _size(rng, 1, 16384), "choose": rng.randint(1, 4), "width": _size(rng, 64, 2048)}


# ------------------------------------------------------------------------------ inputs

def _shares(c):
    """how likely a row is to go to each expert, before the experts are shuffled"""
    e = c["experts"]
    if c["spread"] == "even":
        return np.full(e, 1.0 / e)
    p = (np.arange(e) + 1.0) ** -0.9
    if e >= 8:
        p[-(e // 8):] = 0.0                                   # experts that no row went to
    return p / p.sum()


def _segments(c, rng):
    """(lengths of the segments on the host, their offsets on the device)"""
    lengths = rng.multinomial(c["rows"], rng.permutation(_shares(c)))
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    return lengths, torch.from_numpy(offsets).cuda()


def _normal(shape, dtype, gen, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(dtype)


def _activations(shape, dtype, gen):
    """normal values, some columns an order of magnitude louder, as the residual stream of a model has them"""
    x = torch.randn(shape, device="cuda", generator=gen)
    loud = torch.rand(shape[-1], device="cuda", generator=gen) < 0.01
    return (x * torch.where(loud, 8.0, 1.0)).to(dtype)


def _weights(c, gen):
    """the experts' matrices, as `experts` x n x k values; where they are kept by columns the view says so"""
    w = _normal((c["experts"], c["k"], c["n"]) if c.get("order") == "kn" else (c["experts"], c["n"], c["k"]), TYPES[c["type"]], gen, c["k"] ** -0.5)
    return w.transpose(1, 2) if c.get("order") == "kn" else w


def _index(c, gen):
    """(which slot each row of the segments is, the rows that the slots' tokens have); no index: the rows lie in order"""
    per = c.get("per", 0)
    if not per:
        return None, c["rows"]
    return torch.randperm(c["rows"], device="cuda", generator=gen).to(torch.int32), (c["rows"] + per - 1) // per


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    rng = np.random.default_rng(int(seed))
    s = _PREPARE[case["path"]](case, gen, rng)
    s["case"] = dict(case)
    return s


def _prepare_rows(c, gen, rng):
    lengths, offsets = _segments(c, rng)
    index, tokens = _index(c, gen)
    dtype = TYPES[c["type"]]
    return {"x": _activations((tokens, c["k"]), dtype, gen), "w": _weights(c, gen), "offsets": offsets, "index": index, "longest": int(lengths.max()),
            "out": torch.empty((c["rows"], c["n"]), dtype=dtype, device="cuda")}


def _prepare_outer(c, gen, rng):
    lengths, offsets = _segments(c, rng)
    index, tokens = _index(c, gen)
    dtype = TYPES[c["type"]]
    return {"a": _normal((c["rows"], c["n"]), dtype, gen, 0.1), "x": _activations((tokens, c["k"]), dtype, gen), "offsets": offsets, "index": index,
            "longest": int(lengths.max()), "out": torch.empty((c["experts"], c["n"], c["k"]), dtype=dtype, device="cuda")}


def _logits(c, gen):
    x = torch.randn((c["tokens"], c["experts"]), device="cuda", generator=gen) * 2.0
    padding = torch.rand((c["tokens"], 1), device="cuda", generator=gen) < c["padding"]
    return torch.where(padding, -math.inf, x).to(TYPES[c["type"]])


def _prepare_route(c, gen, rng):
    t, k = c["tokens"], c["choose"]
    whole = dict(dtype=torch.int32, device="cuda")
    return {"logits": _logits(c, gen), "experts": torch.empty((t, k), **whole), "weights": torch.empty((t, k), device="cuda"),
            "offsets": torch.empty((c["experts"] + 1,), **whole), "order": torch.empty((t * k,), **whole), "place": torch.empty((t, k), **whole)}


def _prepare_route_gradient(c, gen, rng):
    logits = _logits(c, gen)
    experts, weights = _choose(logits, c["choose"], c["normalise"])
    return {"logits": logits, "experts": experts, "weights": weights, "dweights": torch.randn(weights.shape, device="cuda", generator=gen),
            "dlogits": torch.empty_like(logits)}


def _slots(c, gen):
    t, k = c["tokens"], c["choose"]
    place = torch.randperm(t * k, device="cuda", generator=gen).to(torch.int32).reshape(t, k)
    return place, torch.softmax(torch.randn((t, k), device="cuda", generator=gen), dim=1)


def _prepare_combine(c, gen, rng):
    dtype = TYPES[c["type"]]
    place, weights = _slots(c, gen)
    return {"y": _normal((c["tokens"] * c["choose"], c["width"]), dtype, gen), "place": place, "weights": weights,
            "out": torch.empty((c["tokens"], c["width"]), dtype=dtype, device="cuda")}


def _prepare_combine_gradient(c, gen, rng):
    s = _prepare_combine(c, gen, rng)
    s["dout"] = _normal((c["tokens"], c["width"]), TYPES[c["type"]], gen)
    s["dy"], s["dweights"] = torch.empty_like(s["y"]), torch.empty_like(s["weights"])
    return s


def _blocks(k):
    return (k + 31) // 32


def _prepare_micro(c, gen, rng):
    """the weights in 4 bits, as a program that serves a model keeps them; room for the rows' own 4 bits"""
    lengths, offsets = _segments(c, rng)
    dtype, b = TYPES[c["type"]], _blocks(c["k"])
    w = _normal((c["experts"], c["n"], c["k"]), torch.float32, gen, c["k"] ** -0.5)
    codes, scales = _quantised(w.reshape(-1, c["k"]))
    return {"x": _activations((c["rows"], c["k"]), dtype, gen), "codes": codes.reshape(c["experts"], c["n"], b * 16), "scales": scales.reshape(c["experts"], c["n"], b),
            "offsets": offsets, "longest": int(lengths.max()), "xcodes": torch.empty((c["rows"], b * 16), dtype=torch.uint8, device="cuda"),
            "xscales": torch.empty((c["rows"], b), dtype=torch.uint8, device="cuda"), "out": torch.empty((c["rows"], c["n"]), dtype=dtype, device="cuda")}


def _prepare_values(c, gen, rng):
    b = _blocks(c["k"])
    x = _activations((c["rows"], c["k"]), TYPES[c["type"]], gen)
    return {"x": x, "codes": torch.empty((c["rows"], b * 16), dtype=torch.uint8, device="cuda"), "scales": torch.empty((c["rows"], b), dtype=torch.uint8, device="cuda"),
            "out": torch.empty_like(x)}


_PREPARE = {"rows": _prepare_rows, "outer": _prepare_outer, "route": _prepare_route, "route_gradient": _prepare_route_gradient, "combine": _prepare_combine,
            "combine_gradient": _prepare_combine_gradient, "micro": _prepare_micro, "values": _prepare_values}


# ------------------------------------------------------------------------------ the plain forms

def _padded(x, offsets, longest):
    """the rows of the segments as experts x longest x width, zeros behind a segment's end"""
    at = offsets[:-1, None].long() + torch.arange(longest, device=x.device)
    here = at < offsets[1:, None]
    return torch.where(here[:, :, None], x[at.clamp(max=x.shape[0] - 1)], 0.0), at, here


def _gathered(x, index, per):
    return x.float() if index is None else x.float()[(index // per).long()]


def _plain_rows(s, x, w):
    padded, at, here = _padded(x, s["offsets"], s["longest"])
    out = torch.zeros((x.shape[0], w.shape[1]), device=x.device)
    out[at[here]] = torch.bmm(padded, w.transpose(1, 2).contiguous())[here]
    return out.to(s["out"].dtype)


def _plain_outer(s, per):
    x, _, _ = _padded(_gathered(s["x"], s["index"], per), s["offsets"], s["longest"])
    a, _, _ = _padded(s["a"].float(), s["offsets"], s["longest"])
    return torch.bmm(a.transpose(1, 2).contiguous(), x).to(s["out"].dtype)


def _choose(logits, k, normalise):
    x = logits.float()
    best, experts = torch.sort(torch.where(x > -math.inf, x, -math.inf), dim=1, descending=True, stable=True)
    top = best[:, :1]
    powers = torch.where(best > -math.inf, torch.exp(torch.where(best == top, 0.0, best - top)), 0.0)
    total = (powers[:, :k] if normalise else powers).sum(1, keepdim=True)
    chosen = best[:, :k] > -math.inf
    return torch.where(chosen, experts[:, :k], -1).to(torch.int32), torch.where(chosen, powers[:, :k] / total, 0.0)


def _plain_route(s, c):
    experts, weights = _choose(s["logits"], c["choose"], c["normalise"])
    flat = experts.reshape(-1).long()
    keys, order = torch.sort(torch.where(flat < 0, c["experts"], flat), stable=True)
    offsets = torch.searchsorted(keys, torch.arange(c["experts"] + 1, device=keys.device))
    at = torch.arange(flat.numel(), device=keys.device)
    place = torch.empty_like(order)
    place[order] = at
    whole = torch.int32
    return {"experts": experts, "weights": weights, "offsets": offsets.to(whole), "order": torch.where(at < offsets[-1], order, -1).to(whole),
            "place": torch.where(flat < 0, -1, place).to(whole).reshape(experts.shape)}


def _plain_route_gradient(s, c):
    chosen, experts = s["experts"] >= 0, s["experts"].clamp(min=0).long()
    inner = (s["weights"] * s["dweights"]).sum(1, keepdim=True)
    x = s["logits"].float()
    if c["normalise"]:
        d = torch.zeros_like(x).scatter_add_(1, experts, torch.where(chosen, s["weights"] * (s["dweights"] - inner), 0.0))
    else:
        some = x > -math.inf
        top = torch.where(some, x, -math.inf).amax(1, keepdim=True)
        powers = torch.where(some, torch.exp(torch.where(x == top, 0.0, x - top)), 0.0)
        p = torch.where(some, powers / powers.sum(1, keepdim=True), 0.0)
        d = p * (torch.zeros_like(x).scatter_add_(1, experts, torch.where(chosen, s["dweights"], 0.0)) - inner)
    return d.to(s["logits"].dtype)


def _plain_combine(s):
    return (s["y"].float()[s["place"].long()] * s["weights"][:, :, None]).sum(1).to(s["out"].dtype)


def _plain_combine_gradient(s):
    dout, place = s["dout"].float(), s["place"].long()
    dy = torch.zeros(s["y"].shape, device=dout.device)
    dy[place] = dout[:, None, :] * s["weights"][:, :, None]
    return {"dy": dy.to(s["dy"].dtype), "dweights": (s["y"].float()[place] * dout[:, None, :]).sum(2)}


def _quantised(x):
    """(4-bit codes, two a byte, the even place in the low half; a byte of scale for every 32 values) of a matrix's rows"""
    rows, k = x.shape
    b = _blocks(k)
    v = torch.nn.functional.pad(x.float(), (0, 32 * b - k)).reshape(rows, b, 32)
    most = v.abs().amax(2)
    power = torch.where(most > 0, torch.frexp(most)[1].to(torch.int32) - 3, -127).clamp(min=-127)
    a = torch.ldexp(v, -power[:, :, None]).abs()
    code = sum([(a > 0.25), (a >= 0.75), (a > 1.25), (a >= 1.75), (a > 2.5), (a >= 3.5), (a > 5.0)], torch.zeros_like(a, dtype=torch.uint8))
    code = (code + torch.where(torch.signbit(v), 8, 0)).to(torch.uint8).reshape(rows, 16 * b, 2)
    return code[:, :, 0] + code[:, :, 1] * 16, (power + 127).to(torch.uint8)


def _values(codes, scales, k, dtype=torch.float32):
    """what codes and scales stand for"""
    both = torch.stack([codes & 15, codes >> 4], dim=-1).long()
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=dtype, device=codes.device)
    v = grid[both].reshape(*scales.shape, 32)
    return torch.ldexp(v, scales[..., None].to(torch.int32) - 127).reshape(*codes.shape[:-1], -1)[..., :k]


# ------------------------------------------------------------------------------ one pass

_kept = {}


def _operator(name, *arguments):
    """the framework's operator, made once for the program"""
    if not _kept:
        sys.path.insert(0, os.path.join(os.getcwd(), "accelerate-cuda_amd"))
        import acchip
        _kept["module"], _kept["context"] = acchip, acchip.Context(0)
    key = (name,) + arguments
    if key not in _kept:
        _kept[key] = getattr(_kept["module"], name)(_kept["context"], *arguments)
    return _kept[key]


def run(s):
    c, path = s["case"], s["case"]["path"]
    if own:
        return _run_own(s, c, path)
    if path == "rows":
        return _plain_rows(s, _gathered(s["x"], s["index"], c["per"]), s["w"].float())
    if path == "outer":
        return _plain_outer(s, c["per"])
    if path == "route":
        return _plain_route(s, c)
    if path == "route_gradient":
        return _plain_route_gradient(s, c)
    if path == "combine":
        return _plain_combine(s)
    if path == "combine_gradient":
        return _plain_combine_gradient(s)
    codes, scales = _quantised(s["x"])
    x = _values(codes, scales, c["k"])
    if path == "values":
        return x.to(s["x"].dtype)
    return _plain_rows(s, x, _values(s["codes"], s["scales"], c["k"]))


def _run_own(s, c, path):
    if path == "rows":
        _operator("Product", c["type"]).rows(s["x"], s["w"], s["offsets"], s["out"], index=s["index"], per=c["per"])
    elif path == "outer":
        _operator("Product", c["type"]).outer(s["a"], s["x"], s["offsets"], s["out"], index=s["index"], per=c["per"])
    elif path == "route":
        _operator("Router", c["type"], c["choose"], c["normalise"]).route(s["logits"], s["experts"], s["weights"], s["offsets"], s["order"], s["place"])
        return {name: s[name] for name in ("experts", "weights", "offsets", "order", "place")}
    elif path == "route_gradient":
        _operator("Router", c["type"], c["choose"], c["normalise"]).gradient(s["logits"], s["experts"], s["weights"], s["dweights"], s["dlogits"])
        return s["dlogits"]
    elif path == "combine":
        _operator("Combiner", c["type"]).combine(s["y"], s["place"], s["weights"], s["out"])
    elif path == "combine_gradient":
        _operator("Combiner", c["type"]).gradient(s["dout"], s["y"], s["place"], s["weights"], s["dy"], s["dweights"])
        return {"dy": s["dy"], "dweights": s["dweights"]}
    elif path == "values":
        micro = _operator("Microscale", c["type"])
        micro.quantise(s["x"], s["codes"], s["scales"])
        micro.values(s["codes"], s["scales"], s["out"])
    else:
        micro = _operator("Microscale", c["type"])
        micro.quantise(s["x"], s["xcodes"], s["xscales"])
        micro.rows(s["xcodes"], s["xscales"], s["codes"], s["scales"], s["offsets"], s["out"])
    return s["out"]


# ------------------------------------------------------------------------------ what a pass cannot do without

def work(c):
    path = c["path"]
    e = SIZE[c["type"]]
    if path in ("rows", "outer", "micro"):
        m, n, k = c["rows"], c["n"], c["k"]
        met = float(np.sum(1.0 - (1.0 - _shares(c)) ** m))                  # the experts that rows are expected to go to
        tokens = -(-m // c["per"]) if c.get("per") else m
        if path == "micro":
            row = _blocks(k) * 17
            # the rows in their own type once, their 4 bits written and read, the weights' 4 bits once
            return {"bytes": m * (k * e + 2 * row) + met * n * row + m * n * e, "flops": 2.0 * m * n * k}
        if path == "rows":
            return {"bytes": (tokens * k + met * n * k + m * n) * e, "flops": 2.0 * m * n * k}
        return {"bytes": (m * n + tokens * k + c["experts"] * n * k) * e, "flops": 2.0 * m * n * k}
    if path in ("route", "route_gradient"):
        t, x, j = c["tokens"], c["experts"], c["choose"]
        if path == "route":
            return {"bytes": t * x * e + t * j * 16 + 4 * (x + 1), "flops": 3.0 * t * x}
        return {"bytes": (1 if c["normalise"] else 2) * t * x * e + t * j * 12, "flops": 4.0 * t * x}
    if path == "values":
        return {"bytes": 2 * c["rows"] * (c["k"] * e + 17 * _blocks(c["k"])), "flops": 4.0 * c["rows"] * c["k"]}
    t, j, d = c["tokens"], c["choose"], c["width"]
    if path == "combine":
        return {"bytes": t * j * d * e + t * d * e + 8 * t * j, "flops": 2.0 * t * j * d}
    return {"bytes": 2 * t * j * d * e + t * d * e + 12 * t * j, "flops": 3.0 * t * j * d}


# ------------------------------------------------------------------------------ the definitions in 64 bits

def _exact_rows(x, w, offsets):
    """a segment after the other; `w` gives an expert's matrix"""
    ends = offsets.tolist()
    return torch.cat([x[b:e].double() @ w(i).double().t() for i, (b, e) in enumerate(zip(ends, ends[1:]))])


def _exact_micro(x):
    """the nearest of the sixteen numbers, of two as near the one with the even code, under the scale of every 32"""
    rows, k = x.shape
    b = _blocks(k)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    out = torch.zeros((rows, b * 32), dtype=torch.float64, device=x.device)
    out[:, :k] = x.double()
    step = max(1, (1 << 22) // (b * 32))
    for at in range(0, rows, step):
        v = out[at:at + step].reshape(-1, 32)
        most = v.abs().amax(1, keepdim=True)
        scale = torch.exp2(torch.where(most > 0, torch.floor(torch.log2(most)) - 2, -127.0).clamp(min=-127.0))
        a = (v.abs() / scale)[:, :, None]
        off = (a - grid).abs()
        near = off == off.amin(2, keepdim=True)
        even = torch.arange(8, device=x.device) % 2 == 0
        code = torch.where(near, torch.where(even, 2, 1), 0).argmax(2)
        out[at:at + step] = (torch.copysign(grid[code], v) * scale).reshape(-1, b * 32)
    return out[:, :k]


def exact(case, seed):
    s, c, path = prepare(case, seed), case, case["path"]
    if path in ("rows", "outer"):
        x = s["x"] if s["index"] is None else s["x"][torch.div(s["index"], c["per"], rounding_mode="floor").long()]
        if path == "rows":
            return _exact_rows(x, lambda i: s["w"][i], s["offsets"])
        ends = s["offsets"].tolist()
        return torch.stack([s["a"][b:e].double().t() @ x[b:e].double() for b, e in zip(ends, ends[1:])])
    if path in ("micro", "values"):
        x = _exact_micro(s["x"])
        if path == "values":
            return x
        return _exact_rows(x, lambda i: _values(s["codes"][i], s["scales"][i], c["k"], torch.float64), s["offsets"])
    if path == "route":
        x = s["logits"].double()
        weights = torch.softmax(x, 1)
        experts = _choose(s["logits"], c["choose"], c["normalise"])[0]
        weights = torch.where(experts >= 0, weights.gather(1, experts.clamp(min=0).long()), 0.0)
        if c["normalise"]:
            weights = torch.where(experts >= 0, weights / weights.sum(1, keepdim=True), 0.0)
        return {"experts": None, "weights": weights, "offsets": None, "order": None, "place": None}
    if path == "route_gradient":
        x, chosen, experts = s["logits"].double(), s["experts"] >= 0, s["experts"].clamp(min=0).long()
        mask = torch.zeros(x.shape, dtype=torch.bool, device=x.device).scatter_(1, experts, chosen)
        dense = torch.zeros_like(x).scatter_(1, experts, torch.where(chosen, s["dweights"].double(), 0.0))
        p = torch.softmax(torch.where(mask, x, -math.inf) if c["normalise"] else x, 1).nan_to_num(0.0)
        d = p * (dense - (p * dense).sum(1, keepdim=True))
        return torch.where(chosen.any(1, keepdim=True), d, 0.0)
    place, weights = s["place"].long(), s["weights"].double()
    if path == "combine":
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device=place.device)
        for j in range(c["choose"]):
            out += weights[:, j, None] * s["y"][place[:, j]].double()
        return out
    dy, dweights = torch.zeros(s["y"].shape, dtype=torch.float64, device=place.device), torch.zeros_like(weights)
    for j in range(c["choose"]):
        dy[place[:, j]] = weights[:, j, None] * s["dout"].double()
        dweights[:, j] = (s["y"][place[:, j]].double() * s["dout"].double()).sum(1)
    return {"dy": dy, "dweights": dweights}
