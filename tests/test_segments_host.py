"""How the operators' kernels cut rows into segments and segments into tiles (op_common.h), on the CPU: a wave is 64 contexts that
are run in turn and meet wherever lanes exchange something.  The driver sizes grids and the memory for partial sums by a bound that
holds if a row is in one segment, so that is what is asked here, of starts in order and of any others."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OPERATORS = os.path.join(ROOT, "accelerate-cuda_amd", "csrc", "operators")
CLANG = "/opt/rocm/llvm/bin/clang++"

# what op_common.h takes from acc_hip_device.h
STUB = """
#pragma once
#include <ucontext.h>
#include <cstring>
#include <vector>
#define ACC_DEV static inline
#define ACC_XCDS 8
struct wave { ucontext_t back, at[64]; std::vector<char> stack; int lane; bool over[64]; unsigned turn[64]; long long slot[2][64]; };
static wave W;
static int acc_lane() { return W.lane; }
static void (*body)();
static void enter() { body(); W.over[W.lane] = true; }
static void run(void (*f)())
{
  const size_t each = 64 << 10;
  body = f;
  W.stack.resize(64 * each);
  for (int l = 0; l < 64; ++l) {
    getcontext(&W.at[l]);
    W.at[l].uc_stack.ss_sp = W.stack.data() + l * each;
    W.at[l].uc_stack.ss_size = each;
    W.at[l].uc_link = &W.back;
    W.over[l] = false;
    W.turn[l] = 0;
    makecontext(&W.at[l], enter, 0);
  }
  for (bool some = true; some;) {
    some = false;
    for (int l = 0; l < 64; ++l) {
      if (W.over[l]) continue;
      W.lane = l;
      swapcontext(&W.back, &W.at[l]);
      some = some || !W.over[l];
    }
  }
}
/* everybody's v; what the others have put down stays until the meeting after next */
static const long long *meet(const long long v)
{
  const int lane = W.lane;
  long long *all = W.slot[W.turn[lane]++ & 1];
  all[lane] = v;
  swapcontext(&W.at[lane], &W.back);
  return all;
}
template <typename T> ACC_DEV T acc_min(T x, T y) { return x < y ? x : y; }
template <typename T> ACC_DEV T acc_max(T x, T y) { return x > y ? x : y; }
ACC_DEV int acc_readlane(const int v, const int lane) { return (int)meet(v)[lane]; }
ACC_DEV int acc_wave_shift_up1(const int v)
{
  const int lane = W.lane;
  return (int)meet(v)[lane ? lane - 1 : 0];
}
template <typename F> ACC_DEV int acc_wave_scan(const int v, F f, const int lane)
{
  const long long *all = meet(v);
  int x = (int)all[0];
  for (int l = 1; l <= lane; ++l) x = f(x, (int)all[l]);
  return x;
}
template <typename F> ACC_DEV int acc_wave_reduce(const int v, F f) { return acc_wave_scan(v, f, 63 + 0 * W.lane); }
ACC_DEV unsigned long long __ballot(const bool p)
{
  const long long *all = meet(p);
  unsigned long long b = 0;
  for (int l = 0; l < 64; ++l) b |= (unsigned long long)all[l] << l;
  return b;
}
ACC_DEV int __popcll(const unsigned long long x) { return __builtin_popcountll(x); }
"""

SOURCE = """
#include "acc_hip_device.h"
#define OP_ELT 0
#include "op_common.h"
static struct { const int *offsets; int experts, rows, height, n, kind; int *out; } P;
static int lot_of(op_lot *l) { *l = op_segments(P.offsets, P.experts, P.rows, 0, 0); return 0; }
static void count()
{
  op_lot lot;
  int whole, rest;
  lot_of(&lot);
  op_count_tiles(P.offsets, P.experts, P.rows, P.height, lot, &whole, &rest);
  if (acc_lane() == 0) { P.out[0] = whole; P.out[1] = rest; }
}
static void find()
{
  op_lot lot;
  lot_of(&lot);
  const op_tile t = P.kind == OP_ALL ? op_find_tile<OP_ALL>(P.offsets, P.experts, P.rows, P.height, lot, P.n)
                  : P.kind == OP_WHOLE ? op_find_tile<OP_WHOLE>(P.offsets, P.experts, P.rows, P.height, lot, P.n)
                                       : op_find_tile<OP_REST>(P.offsets, P.experts, P.rows, P.height, lot, P.n);
  if (acc_lane() == 0) { P.out[0] = t.expert; P.out[1] = t.begin; P.out[2] = t.end; P.out[3] = t.all; }
}
static void longest()
{
  int b, e;
  const int x = op_nth_longest(P.offsets, P.experts, P.rows, P.n, &b, &e);
  if (acc_lane() == 17) { P.out[0] = x; P.out[1] = b; P.out[2] = e; }
}
static void first()
{
  int runs;
  const int at = op_first_run(P.offsets, P.experts, P.rows, P.height, P.n, &runs);
  if (acc_lane() == 40) { P.out[0] = at; P.out[1] = runs; }
}
extern "C" void go(int what, const int *offsets, int experts, int rows, int height, int kind, int n, int *out)
{
  P = {offsets, experts, rows, height, n, kind, out};
  run(what == 0 ? count : what == 1 ? find : what == 2 ? longest : first);
}
"""
ALL, WHOLE, REST = range(3)


@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    at = tmp_path_factory.mktemp("segments")
    (at / "acc_hip_device.h").write_text(STUB)
    (at / "cut.cpp").write_text(SOURCE)
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O1", "-w", "-fPIC", "-shared", "-I", str(at), "-I", OPERATORS, "-o", str(at / "cut.so"), str(at / "cut.cpp")],
                   check=True, capture_output=True)
    go = C.CDLL(str(at / "cut.so")).go

    def call(what, offsets, rows, height=1, kind=0, n=0):
        out = (C.c_int * 4)()
        go(what, offsets.ctypes.data_as(C.c_void_p), len(offsets) - 1, rows, height, kind, n, out)
        return list(out)
    return call


def starts(rng, rows, experts, kind):
    if kind == "in order":
        return np.sort(rng.integers(0, rows + 1, experts + 1)).astype(np.int32)
    if kind == "to and fro":
        return np.resize([0, rows], experts + 1).astype(np.int32)
    if kind == "anywhere":
        return rng.integers(-rows, 2 * rows + 2, experts + 1).astype(np.int32)
    if kind == "backwards":
        return np.sort(rng.integers(0, rows + 1, experts + 1))[::-1].astype(np.int32)
    return rng.choice([-2 ** 31, 2 ** 31 - 1, 0, rows, rows // 2], experts + 1).astype(np.int32)


def ends(offsets, rows):
    """where the segments end, the one in front of the first expert's first"""
    return np.append(np.maximum.accumulate(np.clip(offsets.astype(np.int64), 0, rows)), rows)


@pytest.mark.parametrize("kind", ["in order", "to and fro", "anywhere", "backwards", "odd"])
@pytest.mark.parametrize("rows,experts,height", [(1, 1, 16), (50, 3, 16), (1000, 5, 32), (700, 61, 64), (900, 63, 32), (2000, 70, 64), (300, 200, 16), (2 ** 31 - 5000, 3, 1 << 28),
                                                 (1 << 30, 130, 1 << 26), (77, 0, 16)])
def test_every_row_is_in_one_tile(cut, kind, rows, experts, height):
    offsets = starts(np.random.default_rng(rows % 1009 + experts), rows, experts, kind)
    upto = ends(offsets, rows)
    from_ = np.append(0, upto[:-1])
    # what grids and partial sums are sized by
    parts = min(rows, experts + 2)
    most = (rows + parts * (height - 1)) // height
    runs = -(-(upto - from_) // height)
    assert runs.sum() <= most
    want = [(s - 1 if s <= experts else -1, b, min(b + height, upto[s]), upto[s] - from_[s])
            for s in range(experts + 2) for b in range(int(from_[s]), int(upto[s]), height)]
    assert [tuple(cut(1, offsets, rows, height, ALL, n)) for n in range(len(want))] == want
    begin, end = cut(1, offsets, rows, height, ALL, len(want))[1:3]
    assert begin >= end
    whole, rest = cut(0, offsets, rows, height)[:2]
    assert [tuple(cut(1, offsets, rows, height, WHOLE, n)) for n in range(whole)] == [t for t in want if t[2] - t[1] == height]
    assert [tuple(cut(1, offsets, rows, height, REST, n)) for n in range(rest)] == [t for t in want if t[2] - t[1] < height]
    assert whole + rest == len(want)
    # a segment's runs among all of them, as their sums are added up
    for s in sorted({0, 1, experts // 2, experts, experts + 1}):
        assert cut(3, offsets, rows, height, n=s)[:2] == [runs[:s].sum(), runs[s]]
    # every expert once, longest first where there are few
    seen = [cut(2, offsets, rows, n=n)[:3] for n in range(experts)]
    assert sorted(e for e, _, _ in seen) == list(range(experts))
    assert all((b, t) == (from_[e + 1], upto[e + 1]) for e, b, t in seen)
    if experts <= 62:
        lengths = [min(t - b, (1 << 26) - 2) for _, b, t in seen]
        assert lengths == sorted(lengths, reverse=True)
