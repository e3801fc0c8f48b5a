"""The recurrence, the grouped 4-bit products and the router by scores without a GPU: what they compile, the calls they make on a
stand-in for the HIP runtime, and what they refuse."""
import os
import subprocess

import pytest


@pytest.fixture(scope="module")
def A():
    import acchip
    return acchip


def test_calls_of_every_size_stay_inside_their_memory(A, tmp_path):
    """10 operators, 3000 calls each, eager and as if recorded into a graph"""
    here = os.path.join(os.path.dirname(os.path.abspath(__file__)), "operators_host")
    build = subprocess.run(["make", "-j4", "-C", here, "OUT=%s" % tmp_path, "%s/more" % tmp_path], capture_output=True, text=True)
    assert build.returncode == 0, build.stdout[-3000:] + build.stderr[-3000:]
    A.lib()
    os.symlink(os.path.join(os.path.dirname(os.path.abspath(A.LIB_PATH)), "acc_compile_worker"), tmp_path / "acc_compile_worker")
    (tmp_path / "cache").mkdir()
    run = subprocess.run([str(tmp_path / "more"), str(tmp_path / "cache")], capture_output=True, text=True, timeout=900)
    assert run.returncode == 0 and "wrong 0" in run.stdout, run.stdout[-3000:] + run.stderr[-3000:]
    assert all(int(n) > 100 for n in run.stdout.splitlines()[-2].replace(",", "").split() if n.isdigit())


@pytest.mark.parametrize("elt", ("float", "half", "bfloat16"))
def test_every_unit_compiles(A, tmp_path, elt):
    A.lib().acc_cache_set_dir(str(tmp_path).encode())
    for kind, least, more in ((A.OP_RECUR, 4, dict(gate="sigmoid")), (A.OP_GROUPED, 12, dict(group=64)), (A.OP_SCORE, 12, dict(choose=2, groups=8, keep=3))):
        units, size = A.op_compile_only(kind, elt, **more)
        assert units >= least and size > 3000 * units


def test_arguments_that_there_are_not(A):
    for kind, more in ((A.OP_RECUR, dict(gate="tanh")), (A.OP_GROUPED, dict(group=0)), (A.OP_GROUPED, dict(group=40)), (A.OP_SCORE, dict(choose=0)), (A.OP_SCORE, dict(choose=33)),
                       (A.OP_SCORE, dict(choose=1, groups=6)), (A.OP_SCORE, dict(choose=1, groups=4, keep=0)), (A.OP_SCORE, dict(choose=1, scale=float("inf")))):
        with pytest.raises(A.AccError) as e:
            A.op_compile_only(kind, "float", **more)
        assert e.value.code == A.ERR_INVALID


def test_every_argument_is_asked_for_its_elements(A):
    class There(object):                       # a tensor on the device, as far as a layout asks
        is_cuda, device, shape, itemsize, dtype = True, "cuda:0", (3, 4), 16, "of 16 bytes"

        def data_ptr(self):
            return 4096

        def stride(self):
            return (4, 1)

    class Op(object):
        size, handle = 2, None
    wrong = There()
    for cls, call, n, named in ((A.Recurrence, "scan", 4, ("state", "last", "index")), (A.Recurrence, "gradient", 7, ("state", "dlast", "dstate")), (A.Recurrence, "step", 5, ("index",)),
                                (A.Grouped, "quantise", 3, ("zeros",)), (A.Grouped, "values", 3, ("zeros",)), (A.Grouped, "rows", 5, ("zeros", "index")), (A.ScoreRouter, "route", 6, ("bias",)),
                                (A.ScoreRouter, "gradient", 4, ())):
        for k in range(n):
            with pytest.raises(A.AccError):
                getattr(cls, call)(Op(), *[wrong if k == m else None for m in range(n)])
        for name in named:
            with pytest.raises(A.AccError):
                getattr(cls, call)(Op(), *[None] * n, **{name: wrong})
