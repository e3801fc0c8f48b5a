// Calls of the recurrence, the grouped 4-bit products and the router by scores of every size and layout on the stand-in for the HIP
// runtime of ../tsan/mock_hip.cpp: launches do nothing, and every launch's shape and arguments are looked at.  What is asked: that no
// call needs a translation unit which acc_op_compile_only has not compiled (argument: the directory of the kernel cache, empty), that
// tiles cover their arrays, that scratch memory and LDS hold what the kernels put there, and that calls which do not fit are refused.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <filesystem>
#include <map>
#include <random>

#include "../../accelerate-cuda_amd/csrc/operators/op_args.h"

// (this program's own versions of four of the stand-in's functions)
#define hipStreamIsCapturing mock_StreamIsCapturing
#define hipModuleLaunchKernel mock_ModuleLaunchKernel
#define hipMalloc mock_Malloc
#define hipFree mock_Free
#include "../tsan/mock_hip.cpp"
#undef hipStreamIsCapturing
#undef hipModuleLaunchKernel
#undef hipMalloc
#undef hipFree

static std::map<uint64_t, size_t> g_blocks;       // device memory: where, and how much
static uint64_t g_next = 1ull << 50;
static int g_wrong = 0;
static long g_calls = 0, g_cleared = 0, g_scans = 0, g_stream = 0, g_tall = 0, g_places = 0;
static bool g_recorded = false;
static int64_t g_element = 2;
static int g_choose = 0;

static void not_so(const char *what, long long a, long long b)
{
  if (++g_wrong <= 20) std::fprintf(stderr, "call %ld: %s (%lld, %lld)\n", g_calls, what, a, b);
}
static int64_t room_behind(const void *p)
{
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  auto it = g_blocks.upper_bound(at);
  if (it == g_blocks.begin()) return 0;
  --it;
  return (int64_t)(it->first + it->second) - (int64_t)at;
}

extern "C" {
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *c)
{
  *c = g_recorded ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
hipError_t hipMalloc(void **p, size_t n)          // (addresses alone: nothing here reads or writes device memory)
{
  g_blocks[g_next] = n;
  *p = reinterpret_cast<void *>(g_next);
  g_next += (n + 4095) / 4096 * 4096 + 4096;
  return hipSuccess;
}
hipError_t hipFree(void *p) { g_blocks.erase(reinterpret_cast<uint64_t>(p)); return hipSuccess; }
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned gx, unsigned gy, unsigned gz, unsigned bx, unsigned, unsigned, unsigned lds, hipStream_t, void **params, void **)
{
  const char *name = reinterpret_cast<const Function *>(f)->name;
  if ((uint64_t)gx * bx > 0xffffffffull || gy != 1 || gz != 1) not_so("more threads than a launch has", gx, bx);
  if (bx > 1024 || lds > 160 * 1024) not_so("a workgroup too large", bx, lds);
  if (!std::strcmp(name, "recur") || !std::strcmp(name, "recur_clear")) {
    const acc_recur_args &a = *static_cast<const acc_recur_args *>(params[0]);
    const int64_t channels = a.strips ? 64 * ((a.width > 64 || g_element == 4) ? 4 / g_element : 1) : 0, words = (int64_t)a.tiles * a.strips * 3 * channels;
    if (a.strips * channels < a.width) not_so("strips do not cover the channels", a.strips, a.width);
    if (room_behind(a.words) < words * 8) not_so("words beyond their memory", room_behind(a.words), words);
    if (a.tag == 0) not_so("no tag", 0, 0);
    if ((a.ticket != nullptr) != g_recorded) not_so("a counter of tiles", a.ticket != nullptr, g_recorded);
    if (a.ticket && room_behind(a.ticket) < 256) not_so("the counter beyond its memory", room_behind(a.ticket), 0);
    if (!std::strcmp(name, "recur")) {
      ++g_scans;
      if ((int64_t)gx != (int64_t)a.tiles * a.strips || bx != 512) not_so("grid of the recurrence", gx, bx);
      bool covered = false;                       // (8, 16 or 32 rows a wave)
      for (int64_t r : {64, 128, 256}) covered = covered || a.tiles == std::max<int64_t>(1, (a.rows + r - 1) / r);
      if (!covered) not_so("tiles do not cover the rows", a.tiles, a.rows);
    } else {
      ++g_cleared;
      if ((int64_t)gx * bx < words) not_so("words that are not cleared", gx, words);
    }
  } else if (!std::strcmp(name, "recur_step")) {
    const acc_recur_args &a = *static_cast<const acc_recur_args *>(params[0]);
    if ((int64_t)gx != a.rows * a.strips || (int64_t)a.strips * 256 * (a.width == 1 ? 1 : 4 / g_element) < a.width) not_so("grid of a step", gx, a.strips);
  } else if (!std::strcmp(name, "grouped")) {
    const acc_grouped_args &a = *static_cast<const acc_grouped_args *>(params[0]);
    const int64_t steps = (a.blocks + 3) / 4;
    if ((int64_t)a.run * a.tiles_j * 16 < a.nj) not_so("tiles do not cover the columns", a.run, a.tiles_j);
    if ((int64_t)gx != (int64_t)a.tiles_i * a.tiles_j) not_so("grid of the products", gx, a.tiles_i);
    const int64_t parts = std::min<int64_t>(a.rows, a.experts + 2), least = (a.rows + parts * (a.height - 1)) / a.height;
    if (a.tiles_i < least) not_so("fewer tiles than segments may have", a.tiles_i, least);
    if (a.run == 16 && bx == 256) {
      ++g_tall;
      const int64_t chunks = a.group >= 128 ? 1 : 128 / a.group, rows = g_element == 4 ? 32 : 64, need = 3 * (16 * rows * (g_element == 4 ? 3 : 1) * 16 + chunks * 272 * 4 * (a.zeros ? 2 : 1)) + 2 * chunks * rows * 4 * (a.zeros || g_element == 4 ? 2 : 1);
      if (a.height != rows || a.nj < 16 || a.codes_stride * 63 + 64 > 0xffffffffll || (int64_t)lds > need || (int64_t)lds < need - 2 * chunks * rows * 4) not_so("LDS of the tall tiles", lds, need);
    } else if (bx >= 512 && lds) {
      ++g_stream;
      const int64_t chunks = a.group >= 128 ? 1 : 128 / a.group, waves = bx / 64, rows = (a.height + 15) / 16;
      const int64_t need = waves * rows * 1024 + steps * a.height * (256 * (g_element == 4 ? 3 : 1) + chunks * 8);
      if ((int64_t)lds < need - steps * a.height * chunks * 4 || (a.height & (a.height - 1)) || a.split < 1 || (a.split & (a.split - 1)) || a.split > waves) not_so("LDS of the products", lds, need);
      if (a.nj < 16 || (a.group >> a.group_shift) != 1) not_so("columns of the form in LDS", a.nj, a.group_shift);
    }
  } else if (!std::strcmp(name, "score")) {
    const acc_route_args &a = *static_cast<const acc_route_args *>(params[0]);
    if ((int64_t)a.block * a.blocks < a.tokens || (int64_t)gx != a.blocks || a.blocks > 256) not_so("blocks of the router", a.block, a.blocks);
    const int64_t needed = a.blocks == 1 && !a.counts ? 6 * (int64_t)a.experts + a.tokens * g_choose : a.experts;
    if ((int64_t)lds < needed * 4 + (int64_t)a.groups * 8) not_so("LDS of the router", lds, needed);
    if (a.counts && room_behind(a.counts) < (int64_t)a.blocks * a.experts * 4) not_so("counts beyond their memory", room_behind(a.counts), a.blocks);
    if (!a.counts && a.blocks != 1) not_so("no memory for counts", a.blocks, 0);
  } else if (!std::strcmp(name, "route_place")) {
    ++g_places;
  }
  return hipSuccess;
}
}

#define OK(call)                                                                        \
  do {                                                                                  \
    int rc__ = (call);                                                                  \
    if (rc__ != ACC_OK) {                                                               \
      std::fprintf(stderr, "%s:%d: %s -> %d: %s\n", __FILE__, __LINE__, #call, rc__, acc_last_error()); \
      std::exit(2);                                                                     \
    }                                                                                   \
  } while (0)
#define REFUSED(call)                                                                   \
  do {                                                                                  \
    if ((call) != ACC_ERR_INVALID) {                                                    \
      std::fprintf(stderr, "%s:%d: not refused: %s\n", __FILE__, __LINE__, #call);      \
      ++g_wrong;                                                                        \
    }                                                                                   \
  } while (0)

static std::mt19937_64 g_random(7);
static int64_t pick(double low, double high)      // even over the logarithm
{
  const double u = std::uniform_real_distribution<double>(0, 1)(g_random);
  const int64_t n = (int64_t)(low * std::pow(high / low, u) + 0.5);
  return g_random() % 2 && n >= 64 ? n / 64 * 64 : n;
}
static bool heads() { return g_random() % 2; }

// an array of its own place, `extra` elements between rows
static acc_strided array(std::initializer_list<int64_t> shape, int64_t lead_bytes = 0, int64_t extra = 0)
{
  static uint64_t place = 0;
  acc_strided a = {};
  a.rank = (int32_t)shape.size();
  int d = 0;
  for (int64_t n : shape) a.shape[d++] = n;
  int64_t step = 1;
  for (int k = a.rank - 1; k >= 0; --k) {
    a.stride[k] = step;
    step *= a.shape[k] + (k == a.rank - 1 ? extra : 0);
  }
  a.ptr = (1ull << 41) + (place++ % 64 << 45) + lead_bytes;      // (far apart)
  return a;
}

static size_t units_in(const char *dir)
{
  size_t n = 0;
  for (const auto &e : std::filesystem::recursive_directory_iterator(dir)) n += e.is_regular_file();
  return n;
}

int main(int, char **argv)
{
  OK(acc_init());
  OK(acc_cache_set_dir(argv[1]));
  acc_context ctx = nullptr;
  OK(acc_context_create(0, &ctx));
  for (const char *type : {"float", "bfloat16"})
    for (int form = 0; form < 5; ++form) {
      acc_op_desc d = {};
      d.kind = form < 2 ? ACC_OP_RECUR : form < 4 ? ACC_OP_GROUPED : ACC_OP_SCORE;
      d.elt_type = type;
      d.gate = form;
      d.group = form == 2 ? 32 : 128;
      d.choose = g_choose = 3;
      d.normalise = 1;
      d.groups = 4;
      d.keep = 2;
      d.scale = 1.0f;
      if (form >= 2) d.gate = 0;
      int32_t units = 0;
      size_t size = 0;
      OK(acc_op_compile_only("gfx950", &d, &units, &size));
      const size_t compiled = units_in(argv[1]);
      acc_op op = nullptr;
      OK(acc_op_create(ctx, &d, &op));
      g_element = *type == 'f' ? 4 : 2;
      for (int call = 0; call < 3000; ++call, ++g_calls) {
        const int64_t lead = heads() ? 0 : g_element * (int64_t)(g_random() % 8), extra = (int64_t)(g_random() % 5);
        const int64_t rows = call % 50 ? pick(1, 1e6) : 0, width = pick(1, 8192), n = pick(1, 300);
        g_recorded = call % 3 == 2;
        if (form < 2) {
          const acc_strided gates = array({rows, width}, lead, extra), values = array({rows, width}, lead, extra), out = array({rows, width}, lead, extra), offsets = array({n + 1}),
                            state = array({n, width}, 0, extra), last = array({n, width}), h = array({rows, width}), dout = array({rows, width}), dx = array({rows, width}),
                            table = array({n + rows, width}), index = array({rows});
          OK(acc_exec_recur(op, &gates, &values, &offsets, nullptr, heads() ? &state : nullptr, heads() ? &last : nullptr, &out, nullptr));
          OK(acc_exec_recur(op, &gates, &values, &offsets, nullptr, &state, &state, &out, nullptr));
          OK(acc_exec_recur_gradient(op, &gates, &values, &offsets, &h, &dout, heads() ? &state : nullptr, nullptr, &out, &dx, heads() ? &last : nullptr, nullptr));
          OK(acc_exec_recur_step(op, &gates, &values, heads() ? &index : nullptr, &table, &table, &out, nullptr));
        } else if (form < 4) {
          const int64_t k = pick(1, 16384), blocks = (k + 31) / 32, groups = (k + d.group - 1) / d.group, m = call % 50 ? pick(1, 20000) : 0, e = pick(1, 64);
          const acc_strided x = array({m, k}, lead, extra), codes = array({e, width, 16 * blocks}, 0, 16 * (extra % 2)), scales = array({e, groups, width}, lead, extra), zeros = array({e, groups, width}),
                            offsets = array({e + 1}), index = array({m}), out = array({m, width}, lead, extra), w = array({e, width, k}, lead, extra);
          OK(acc_exec_grouped_rows(op, &x, &codes, &scales, heads() ? &zeros : nullptr, &offsets, heads() ? &index : nullptr, (int32_t)(g_random() % 3), &out, nullptr));
          if (call % 10) continue;
          OK(acc_exec_grouped_quantise(op, &w, &codes, &scales, heads() ? &zeros : nullptr, nullptr));
          OK(acc_exec_grouped_values(op, &codes, &scales, heads() ? &zeros : nullptr, &w, nullptr));
        } else {
          const int64_t tokens = call % 50 ? pick(1, 3e5) : 0, experts = 4 * pick(2, 512);
          const acc_strided logits = array({tokens, experts}, lead, extra), bias = array({experts}), chosen = array({tokens, 3}), weights = array({tokens, 3}), starts = array({experts + 1}),
                            order = array({tokens * 3}), place = array({tokens, 3}), back = array({tokens, experts}, lead, extra);
          OK(acc_exec_score(op, &logits, heads() ? &bias : nullptr, &chosen, &weights, &starts, &order, &place, nullptr));
          OK(acc_exec_score_gradient(op, &logits, &chosen, &weights, &back, nullptr));
        }
      }
      g_recorded = false;
      OK(acc_op_destroy(op));
      if (units_in(argv[1]) != compiled) not_so("units that calls needed beside those that had been compiled", (long long)(units_in(argv[1]) - compiled), form);
      std::printf("%s %d: %d units\n", type, form, units);
    }

  // refusals, none of which reaches a launch
  acc_op_desc d = {};
  d.kind = ACC_OP_RECUR;
  d.elt_type = "float";
  acc_op op = nullptr;
  OK(acc_op_create(ctx, &d, &op));
  const acc_strided z = array({8, 6}), x = array({8, 6}), out = array({8, 6}), offsets = array({3}), state = array({2, 6}), other = array({8, 5}), none = array({0}), huge = array({0x7fffffff, 1});
  REFUSED(acc_exec_recur(op, nullptr, &x, &offsets, nullptr, nullptr, nullptr, &out, nullptr));
  REFUSED(acc_exec_recur(op, &z, &x, &none, nullptr, nullptr, nullptr, &out, nullptr));
  REFUSED(acc_exec_recur(op, &other, &x, &offsets, nullptr, nullptr, nullptr, &out, nullptr));
  REFUSED(acc_exec_recur(op, &z, &x, &offsets, &offsets, &state, nullptr, &out, nullptr));
  REFUSED(acc_exec_recur(op, &z, &x, &offsets, nullptr, &other, nullptr, &out, nullptr));
  REFUSED(acc_exec_recur(op, &z, &x, &offsets, nullptr, nullptr, nullptr, &x, nullptr));
  REFUSED(acc_exec_recur(op, &huge, &huge, &offsets, nullptr, nullptr, nullptr, &huge, nullptr));
  REFUSED(acc_exec_recur(nullptr, &z, &x, &offsets, nullptr, nullptr, nullptr, &out, nullptr));
  REFUSED(acc_exec_recur_gradient(op, &z, &x, &offsets, nullptr, &x, nullptr, nullptr, &out, &out, nullptr, nullptr));
  REFUSED(acc_exec_recur_step(op, &z, &x, nullptr, nullptr, &state, &out, nullptr));
  REFUSED(acc_exec_score(op, &z, nullptr, &x, &x, &x, &x, &x, nullptr));
  REFUSED(acc_exec_grouped_rows(op, &x, &z, &z, nullptr, &offsets, nullptr, 0, &out, nullptr));
  OK(acc_op_destroy(op));
  d.kind = ACC_OP_GROUPED;
  d.group = 1 << 30;
  OK(acc_op_create(ctx, &d, &op));
  const int64_t most = (1 << 30) + 32;
  const acc_strided pair = array({2}), far = array({1, most}), codes = array({1, 1, most / 2}), scales = array({1, 2, 1}), result = array({1, 1}), matrices = array({1, 1, most});
  REFUSED(acc_exec_grouped_rows(op, &far, &codes, &scales, nullptr, &pair, nullptr, 0, &result, nullptr));
  REFUSED(acc_exec_grouped_quantise(op, &matrices, &codes, &scales, nullptr, nullptr));
  OK(acc_op_destroy(op));
  for (int bad = 0; bad < 6; ++bad) {
    acc_op_desc e = {};
    e.elt_type = "half";
    e.kind = bad < 2 ? ACC_OP_GROUPED : bad < 4 ? ACC_OP_SCORE : bad == 4 ? ACC_OP_RECUR : 4;
    e.group = bad == 0 ? 24 : 0;
    e.choose = 2;
    e.groups = bad == 2 ? 3 : 4;
    e.keep = bad == 3 ? 5 : 1;
    e.gate = bad == 4 ? 2 : 0;
    REFUSED(acc_op_create(ctx, &e, &op));
  }
  OK(acc_context_destroy(ctx));
  std::printf("%ld scans, %ld cleared, %ld products with rows in LDS, %ld of tall tiles, %ld placings\nwrong %d\n", g_scans, g_cleared, g_stream, g_tall, g_places, g_wrong);
  return g_wrong ? 1 : 0;
}
