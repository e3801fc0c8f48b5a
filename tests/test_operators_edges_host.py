"""Calls of the operators at the edges of what they take, without a GPU: on a stand-in for the HIP runtime (operators_edges/edges.cpp)."""
import os
import subprocess

import pytest

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "operators_edges")


@pytest.fixture(scope="module")
def edges(tmp_path_factory):
    """run(part): what the program says about it"""
    import acchip
    out = tmp_path_factory.mktemp("edges")
    build = subprocess.run(["make", "-j4", "-C", HERE, "OUT=%s" % out, "%s/edges" % out], capture_output=True, text=True)
    assert build.returncode == 0, build.stdout[-3000:] + build.stderr[-3000:]
    acchip.lib()
    os.symlink(os.path.join(os.path.dirname(os.path.abspath(acchip.LIB_PATH)), "acc_compile_worker"), out / "acc_compile_worker")
    (out / "cache").mkdir()

    def run(part):
        r = subprocess.run([str(out / "edges"), str(out / "cache"), part], capture_output=True, text=True, timeout=300)
        assert r.returncode == 0 and "wrong 0" in r.stdout, r.stdout[-3000:] + r.stderr[-3000:]
    return run


def test_memory_first_lent_under_capture_is_cleared_before_an_eager_call(edges):
    """a recurrence's tagged words: no fill goes into the graph, and none is missing behind it"""
    edges("pool")


def test_eager_calls_do_not_join_the_capture_of_another_stream(edges):
    """recurrences and scans of many tiles are in order across streams; the last one's stream may be under capture by then"""
    edges("order")


def test_eager_calls_do_not_end_the_capture_of_another_stream(edges):
    """asking for an event of that stream would, and so would waiting for the device"""
    edges("beside")


def test_more_numbers_than_a_launch_has_threads_for(edges):
    """matrices of 2^36 numbers and more are quantised, and made again, in several launches"""
    edges("parts")


def test_sequences_without_a_row_are_found_whatever_the_tiles(tmp_path):
    """op_recur.h's own arithmetic of shares, compiled for the host: no offset outside the array is read"""
    csrc = os.path.join(os.path.dirname(HERE), "..", "accelerate-cuda_amd", "csrc", "operators")
    with open(os.path.join(csrc, "op_recur.h")) as f:
        text = f.read()
    at = text.index("ACC_DEV void op_empty_sequences")
    (tmp_path / "function.inc").write_text(text[at:text.index("\n}\n", at) + 3])
    build = subprocess.run(["g++", "-O1", "-fwrapv", "-std=c++17", "-I%s" % tmp_path, "-o", str(tmp_path / "shares"), os.path.join(HERE, "shares.cpp")], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr[-3000:]
    run = subprocess.run([str(tmp_path / "shares")], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "wrong 0" in run.stdout, run.stdout[-3000:]
