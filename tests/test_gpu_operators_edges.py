"""The recurrence, the router by scores and the grouped 4-bit products at the edges of what they take (include/acc_hip.h, section D): rows and
channels in their billions, by results that are known without a second computation as large."""
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
