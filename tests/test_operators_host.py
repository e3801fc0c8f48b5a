"""The operators' translation units compile for gfx950 without a GPU, and what cannot be served is refused there."""
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def A():
    import acchip
    return acchip


@pytest.mark.parametrize("elt", ("float", "half", "bfloat16"))
def test_every_unit_of_every_operator_compiles_for_gfx950(A, tmp_path, elt):
    A.lib().acc_cache_set_dir(str(tmp_path).encode())
    for kind, least in ((A.OP_PRODUCT, 16), (A.OP_ROUTE, 8), (A.OP_COMBINE, 2), (A.OP_MICRO, 3)):
        units, size = A.op_compile_only(kind, elt, 2)
        assert units >= least and size > 4000 * units


def test_operators_that_there_are_not(A):
    for kind, elt, choose in ((4, "float", 1), (-1, "float", 1), (A.OP_PRODUCT, "double", 1), (A.OP_PRODUCT, "", 1), (A.OP_PRODUCT, None, 1),
                              (A.OP_ROUTE, "float", 0), (A.OP_ROUTE, "float", 65)):
        with pytest.raises(A.AccError) as e:
            A.op_compile_only(kind, elt, choose)
        assert e.value.code == A.ERR_INVALID


def test_layouts_of_arrays_as_the_library_reads_them(A):
    """an acc_strided: rank, four extents, four strides, the address"""
    import struct
    text = A._layout(A.Strided((2, 3, 5), (99, 1, 7), 0x1234))
    assert struct.unpack("@ii4q4qQ", text) == (3, 0, 2, 3, 5, 0, 99, 1, 7, 0, 0x1234)
    assert struct.unpack("@ii4q4qQ", A._layout(A.Strided((2, 3, 5), (99, 1, 7), 16).swap()))[2:10] == (2, 5, 3, 0, 99, 7, 1, 0)
    dense = A.DeviceArray.view(None, (4, 6), __import__("numpy").dtype("f4"), 24, 64)
    assert struct.unpack("@ii4q4qQ", A._layout(dense)) == (2, 0, 4, 6, 0, 0, 6, 1, 0, 0, 64)
    assert A._layout(None) is None


def test_scratch_memory_of_recorded_calls_stays_with_the_graph(tmp_path):
    """on a stand-in for the HIP runtime: what a call recorded into a graph was lent goes to nobody else while the stream lives"""
    import subprocess
    here = os.path.join(os.path.dirname(os.path.abspath(__file__)), "operators_host")
    build = subprocess.run(["make", "-j4", "-C", here, "OUT=%s" % tmp_path, "%s/driver" % tmp_path], capture_output=True, text=True)
    assert build.returncode == 0, build.stdout[-3000:] + build.stderr[-3000:]
    run = subprocess.run([str(tmp_path / "driver")], capture_output=True, text=True, env=dict(os.environ, ACC_HIP_CACHE_DIR=str(tmp_path)), timeout=300)
    assert run.returncode == 0 and "wrong 0" in run.stdout, run.stdout + run.stderr


def test_calls_of_every_size_find_their_units_compiled_and_their_pieces_covered(A, tmp_path):
    """12 operators, 4000 calls each on the stand-in: what op_compile_only has compiled is all they need, and sums that are cut are
    cut into pieces that cover them once"""
    import subprocess
    here = os.path.join(os.path.dirname(os.path.abspath(__file__)), "operators_host")
    build = subprocess.run(["make", "-j4", "-C", here, "OUT=%s" % tmp_path, "%s/walk" % tmp_path], capture_output=True, text=True)
    assert build.returncode == 0, build.stdout[-3000:] + build.stderr[-3000:]
    A.lib()
    os.symlink(os.path.join(os.path.dirname(os.path.abspath(A.LIB_PATH)), "acc_compile_worker"), tmp_path / "acc_compile_worker")
    (tmp_path / "cache").mkdir()
    run = subprocess.run([str(tmp_path / "walk"), str(tmp_path / "cache")], capture_output=True, text=True, timeout=900)
    assert run.returncode == 0 and "wrong 0" in run.stdout, run.stdout[-3000:] + run.stderr[-3000:]
    assert all(int(line.split()[-4]) > 500 for line in run.stdout.splitlines() if line.startswith("bfloat16"))


def test_tensors_that_an_operator_cannot_read_are_refused(A):
    """on the host, or of elements of another size: the kernels would read what is not there"""
    import numpy as np
    import torch
    for t, size in ((torch.zeros(3, 4), 4), (torch.zeros(3, dtype=torch.int64), 4)):
        with pytest.raises(A.AccError) as e:
            A._layout(t, size)
        assert e.value.code == A.ERR_INVALID

    class There(object):                       # a tensor on the device, as far as a layout asks
        is_cuda, device, shape = True, "cuda:0", (3, 4)

        def __init__(self, itemsize):
            self.itemsize, self.dtype = itemsize, "of %d bytes" % itemsize

        def data_ptr(self):
            return 4096

        def stride(self):
            return (4, 1)
    assert A._layout(There(2), 2) == A._layout(A.Strided((3, 4), (4, 1), 4096))
    for itemsize, size in ((4, 2), (2, 4), (8, 4), (4, 1)):
        with pytest.raises(A.AccError):
            A._layout(There(itemsize), size)
        with pytest.raises(A.AccError):
            A._layout(A.DeviceArray.view(None, (4, 6), np.dtype("f%d" % itemsize), 24, 64), size)
    # every argument of every call asks
    class Op(object):
        def __init__(self, cls, size):
            self.cls, self.size, self.handle = cls, size, None
    wrong = There(16)
    for cls, call, n in ((A.Product, "rows", 4), (A.Product, "outer", 4), (A.Router, "route", 6), (A.Router, "gradient", 5), (A.Combiner, "combine", 4),
                         (A.Combiner, "gradient", 6), (A.Microscale, "quantise", 3), (A.Microscale, "values", 3), (A.Microscale, "rows", 6)):
        for k in range(n):
            with pytest.raises(A.AccError) as e:
                getattr(cls, call)(Op(cls, 2), *[wrong if k == m else None for m in range(n)])
            assert "16 bytes" in str(e.value)
    for cls in (A.Product, A.Microscale):
        with pytest.raises(A.AccError):
            cls.rows(Op(cls, 2), *[None] * (4 if cls is A.Product else 6), index=wrong)
