"""The recurrence, the router by scores and the grouped 4-bit products at the edges of what they take (include/acc_hip.h, section D): rows and
channels in their billions, by results that are known without a second computation as large."""
import ctypes as C
import sys

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def say(*a):
    print("[case]", *a)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def A():
    import acchip
    return acchip


@pytest.fixture()
def ctx(A):
    c = A.Context(0)
    yield c
    torch.cuda.synchronize()
    c.close()                                                  # (and with it gigabytes of scratch memory)
    torch.cuda.empty_cache()


def edges_of(rng, rows, sequences):
    """offsets of sequences that cover all rows, every third of none"""
    ends = np.sort(rng.integers(1, rows, sequences - 1))
    ends[1::3] = ends[0::3][:len(ends[1::3])]
    return np.concatenate([[0], ends, [rows]]).astype(np.int32)


@pytest.mark.parametrize("rows", (2 ** 30 - 256, 2 ** 30 + 300))
def test_a_narrow_scan_of_a_billion_rows(A, ctx, rows):
    """gates of 0 keep nothing, so h is the values; sequences without a row leave the state that they begin with"""
    rng, sequences = np.random.default_rng(1), 3000
    starts = edges_of(rng, rows, sequences)
    assert starts[-1] == rows and np.all(np.diff(starts) >= 0) and np.sum(np.diff(starts) == 0) > 900
    gates = torch.zeros((rows, 1), dtype=torch.float16, device="cuda")
    values = torch.randint(-9, 10, (rows, 1), dtype=torch.int8, device="cuda").to(torch.float16)
    out = torch.full_like(values, 77.0)
    state = torch.randn((sequences, 1), device="cuda")
    last = torch.full_like(state, 77.0)
    op = A.Recurrence(ctx, "half", "given")
    torch.cuda.synchronize()
    say(rows)
    op.scan(gates, values, torch.from_numpy(starts).cuda(), out, state=state, last=last)
    ctx.sync()
    assert torch.equal(out, values)
    ends = torch.from_numpy(starts[1:].astype(np.int64)).cuda()
    none = torch.from_numpy(np.diff(starts) == 0).cuda()
    assert torch.equal(last[:, 0], torch.where(none, state[:, 0], values[(ends - 1).clamp(min=0), 0].float()))
    op.destroy()


def test_a_narrow_gradient_of_half_a_billion_rows(A, ctx):
    """the same backwards: what a sequence without a row is given behind its end is the gradient of what it begins with"""
    rng, rows, sequences = np.random.default_rng(2), 2 ** 29 + 200, 3000
    starts = edges_of(rng, rows, sequences)
    gates = torch.zeros((rows, 1), dtype=torch.float16, device="cuda")
    dout = torch.randint(-9, 10, (rows, 1), dtype=torch.int8, device="cuda").to(torch.float16)
    h = torch.ones_like(dout)
    dgates, dvalues = torch.full_like(dout, 77.0), torch.full_like(dout, 77.0)
    dlast = torch.randint(-9, 10, (sequences, 1), device="cuda").float()
    dstate = torch.full_like(dlast, 77.0)
    op = A.Recurrence(ctx, "half", "given")
    torch.cuda.synchronize()
    say(rows)
    op.gradient(gates, None, torch.from_numpy(starts).cuda(), h, dout, dgates, dvalues, dlast=dlast, dstate=dstate)
    ctx.sync()
    none = torch.from_numpy(np.diff(starts) == 0).cuda()
    assert torch.equal(dstate, torch.where(none[:, None], dlast, torch.zeros_like(dlast)))
    want, ends = dout.clone(), torch.from_numpy(starts[1:].astype(np.int64)).cuda()
    want[ends[~none] - 1] += dlast[~none].to(torch.float16)
    assert torch.equal(dvalues, want)
    first = torch.from_numpy(starts[:-1].astype(np.int64)).cuda()[~none]
    want[first] = 0.0                                          # (states of zeros: nothing comes before a first row)
    assert torch.equal(dgates, want)
    op.destroy()


@pytest.mark.parametrize("elt,width", (("float", 2 ** 30 + 65), ("half", 2 ** 31 - 4097)))
def test_a_step_of_more_than_a_billion_channels(A, ctx, elt, width):
    """a row of 4 GB and more: every channel is read and written where it is"""
    dtype = {"float": torch.float32, "half": torch.float16}[elt]
    whole = lambda t: torch.randint(-9, 10, (1, width), dtype=torch.int8, device="cuda").to(t)
    gates, values, state = torch.full((1, width), 0.5, dtype=dtype, device="cuda"), whole(dtype), whole(torch.float32)
    out, last = torch.full_like(values, 77.0), torch.full_like(state, 77.0)
    op = A.Recurrence(ctx, elt, "given")
    torch.cuda.synchronize()
    say(elt, width)
    op.step(gates, values, state, last, out)
    ctx.sync()
    state.mul_(0.5).add_(values)                               # (halves of whole numbers: exact)
    assert torch.equal(last, state)
    assert torch.equal(out, state.to(dtype))
    op.destroy()


@pytest.fixture(scope="module")
def hip():
    h = C.CDLL("libamdhip64.so")
    h.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    h.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    h.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    h.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    h.hipGraphExecDestroy.argtypes = h.hipGraphDestroy.argtypes = [C.c_void_p]
    return h


def test_eager_calls_beside_a_capture(A, ctx, hip):
    """a recurrence on one stream while the stream of the last such call is being recorded: it runs at once, and is no part of the graph; a
    large scan, which would have to wait for that stream, is refused, and not recorded either"""
    rng, rows, width, n = np.random.default_rng(4), 6000, 200, 1 << 26
    z, x = (rng.standard_normal((rows, width)).astype(np.float32) for _ in range(2))
    z, x, offsets = ctx.array(z), ctx.array(x), ctx.array(np.array([0, 2500, rows], np.int32))
    outs = [ctx.empty((rows, width), np.float32) for _ in range(2)]
    op = A.Recurrence(ctx, "float", "sigmoid")
    skel = ctx.skeleton(A.SKEL_SCANL1, "Int32", env=[(1, "Int32")], get="arrIn0_0[ix]", combine="x + y")
    ones, sums = ctx.array(np.ones(n, np.int32)), [ctx.empty((n,), np.int32) for _ in range(2)]
    one, two = ctx.stream(), ctx.stream()
    for stream, out, total in zip((one, two, one), (*outs, outs[0]), (*sums, sums[0])):
        skel.scan([ones], n, total, stream=stream)
        op.scan(z, x, offsets, out, stream=stream)
    ctx.sync()
    want = outs[0].get().copy()
    assert np.array_equal(outs[1].get(), want)
    for a in (*outs, sums[1]):
        a.set(np.full(a.shape, 7, a.dtype))
    graph, graph_exec = C.c_void_p(), C.c_void_p()
    assert hip.hipStreamBeginCapture(one, 2) == 0
    try:
        op.scan(z, x, offsets, outs[0], stream=one)
        op.scan(z, x, offsets, outs[1], stream=two)
        with pytest.raises(A.AccError) as refused:
            skel.scan([ones], n, sums[1], stream=two)
        assert refused.value.code == A.ERR_INVALID
    finally:
        rc = hip.hipStreamEndCapture(one, C.byref(graph))
    assert rc == 0 and graph.value and hip.hipGraphInstantiate(C.byref(graph_exec), graph, None, None, 0) == 0
    ctx.sync()
    assert np.array_equal(outs[1].get(), want) and np.all(outs[0].get() == 7.0) and np.all(sums[1].get() == 7)
    skel.scan([ones], n, sums[1], stream=two)
    ctx.sync()
    assert np.array_equal(sums[1].get(), np.arange(1, n + 1, dtype=np.int32))
    for replay in range(4):
        outs[0].set(np.full((rows, width), 9.0, np.float32))
        outs[1].set(np.full((rows, width), 9.0, np.float32))
        ctx.sync()
        assert hip.hipGraphLaunch(graph_exec, one) == 0
        op.scan(z, x, offsets, outs[1], stream=two)
        ctx.sync()
        assert np.array_equal(outs[0].get(), want) and np.array_equal(outs[1].get(), want), replay
    hip.hipGraphExecDestroy(graph_exec)
    hip.hipGraphDestroy(graph)
    op.destroy()


def test_more_numbers_than_a_launch_has_threads_for(A, ctx):
    """33 times the same matrix of 2^30 numbers, quantised and made again: the last is as the first"""
    n, k, experts, group = 2 ** 15, 2 ** 15, 33, 128
    w = torch.empty((n, k), dtype=torch.float16, device="cuda").normal_()
    codes, scales, zeros = (torch.full((experts, *shape), 99, dtype=t, device="cuda") for shape, t in (((n, k // 2), torch.uint8), ((k // group, n), torch.float16), ((k // group, n), torch.uint8)))
    op = A.Grouped(ctx, "half", group)
    torch.cuda.synchronize()
    say("quantise")
    op.quantise(w.expand(experts, n, k), codes, scales, zeros=zeros)
    ctx.sync()
    for a in (codes, scales, zeros):
        assert all(torch.equal(a[0], a[e]) for e in range(1, experts))
    full = w.reshape(n, k // group, group).float()
    low, high = full.amin(2).clamp(max=0.0), full.amax(2).clamp(min=0.0)
    assert torch.equal(scales[-1], ((high - low) / 15.0).half().t())
    del full, low, high
    made = torch.full((experts, n, k), 77.0, dtype=torch.float16, device="cuda")
    say("values")
    op.values(codes, scales, made, zeros=zeros)
    ctx.sync()
    assert all(torch.equal(made[0], made[e]) for e in range(1, experts))
    off = (made[-1].float() - w.float()).abs().reshape(n, k // group, group).amax(2)
    assert torch.all(off <= scales[-1].t().float() * 0.51 + 0.01)          # (half a step; scales and what is made again are rounded, too)
    op.destroy()
