// Calls of the operators of every size and layout on the stand-in for the HIP runtime of ../tsan/mock_hip.cpp: launches do
// nothing, and every launch's shape and arguments are looked at.  What is asked: that no call needs a translation unit which
// acc_op_compile_only has not compiled (argument: the directory of the kernel cache, empty), and that the pieces of a sum cover
// it once and fit the memory for their results.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <filesystem>
#include <map>
#include <random>

#include "../../accelerate-cuda_amd/csrc/operators/op_args.h"

// (this program's own versions of three of the stand-in's functions)
#define hipModuleLaunchKernel mock_ModuleLaunchKernel
#define hipMalloc mock_Malloc
#define hipFree mock_Free
#include "../tsan/mock_hip.cpp"
#undef hipModuleLaunchKernel
#undef hipMalloc
#undef hipFree

static std::map<uint64_t, size_t> g_blocks;       // device memory: where, and how much
static uint64_t g_next = 1ull << 50;
static int g_wrong = 0;
static bool g_micro = false;
static int64_t g_element = 2;
static long g_calls = 0, g_cut = 0;

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
hipError_t hipMalloc(void **p, size_t n)          // (addresses alone: nothing here reads or writes device memory)
{
  g_blocks[g_next] = n;
  *p = reinterpret_cast<void *>(g_next);
  g_next += (n + 4095) / 4096 * 4096 + 4096;
  return hipSuccess;
}
hipError_t hipFree(void *p) { g_blocks.erase(reinterpret_cast<uint64_t>(p)); return hipSuccess; }
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned gx, unsigned gy, unsigned gz, unsigned bx, unsigned, unsigned, unsigned, hipStream_t, void **params, void **)
{
  if ((uint64_t)gx * bx > 0xffffffffull || gy != 1 || gz != 1) not_so("more threads than a launch has", gx, bx);
  if (std::strcmp(reinterpret_cast<const Function *>(f)->name, "product") != 0) return hipSuccess;
  const acc_product_args &a = *static_cast<const acc_product_args *>(params[0]);
  if (!a.piece) return hipSuccess;
  ++g_cut;
  const int64_t step = 128 / (g_micro ? 1 : g_element);
  if (a.piece % step) not_so("a piece is no whole number of steps", a.piece, step);
  if (a.pieces) {                                 // products of rows
    if ((int64_t)a.pieces * a.piece < a.k || (int64_t)(a.pieces - 1) * a.piece >= a.k) not_so("pieces do not cover the sum", a.pieces, a.piece);
    if ((int64_t)gx != (int64_t)a.tiles_i * a.tiles_j * a.pieces) not_so("grid", gx, a.pieces);
    if (room_behind(a.parts) < (int64_t)a.pieces * a.rows * a.nj * 4) not_so("results of pieces beyond their memory", room_behind(a.parts), a.pieces);
  } else {                                        // of columns: at most so many runs, of segments that are a row's alone
    const int64_t runs = gx / ((int64_t)a.tiles_i * a.tiles_j), parts = std::min<int64_t>(a.rows, a.experts + 2);
    if (runs < (a.rows + parts * (a.piece - 1)) / a.piece) not_so("fewer runs than segments may have", runs, a.piece);
    if (room_behind(a.parts) < runs * a.ni * a.nj * 4) not_so("results of pieces beyond their memory", room_behind(a.parts), runs);
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

static std::mt19937_64 g_random(5);
static int64_t pick(double low, double high)      // even over the logarithm
{
  const double u = std::uniform_real_distribution<double>(0, 1)(g_random);
  const int64_t n = (int64_t)(low * std::pow(high / low, u) + 0.5);
  return g_random() % 2 && n >= 64 ? n / 64 * 64 : n;
}
static bool heads() { return g_random() % 2; }

// an array of its own place, `extra` elements between rows, the last two dimensions exchanged if `turned`
static acc_strided array(std::initializer_list<int64_t> shape, int64_t lead_bytes, int64_t extra, bool turned = false)
{
  static uint64_t place = 0;
  acc_strided a = {};
  a.rank = (int32_t)shape.size();
  int d = 0;
  for (int64_t n : shape) a.shape[d++] = n;
  int order[4] = {0, 1, 2, 3};
  if (turned) std::swap(order[a.rank - 1], order[a.rank - 2]);
  int64_t step = 1;
  for (int k = a.rank - 1; k >= 0; --k) {
    a.stride[order[k]] = step;
    step *= a.shape[order[k]] + (k == a.rank - 1 ? extra : 0);
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
  const char *types[] = {"float", "half", "bfloat16"};
  for (const char *type : types)
    for (int kind : {ACC_OP_PRODUCT, ACC_OP_ROUTE, ACC_OP_COMBINE, ACC_OP_MICRO}) {
      acc_op_desc d = {kind, type, 3, 1};
      int32_t units = 0;
      size_t size = 0;
      OK(acc_op_compile_only("gfx950", &d, &units, &size));
      const size_t compiled = units_in(argv[1]);
      acc_op op = nullptr;
      OK(acc_op_create(ctx, &d, &op));
      g_element = *type == 'f' ? 4 : 2;
      g_micro = kind == ACC_OP_MICRO;
      for (int call = 0; call < 4000; ++call, ++g_calls) {
        const bool plain = heads();               // rows of whole chunks
        const int64_t lead = plain ? 0 : g_element * (int64_t)(g_random() % 8), extra = plain ? 8 * (int64_t)(g_random() % 2) : (int64_t)(g_random() % 5);
        const int64_t rows = pick(1, 1e5), experts = pick(1, 300), n = pick(1, 8192), k = pick(1, 16384), per = (int64_t)(g_random() % 3);
        const acc_strided offsets = array({experts + 1}, 0, 0), index = array({rows}, 0, 0);
        const acc_strided *use = heads() ? &index : nullptr;
        if (kind == ACC_OP_PRODUCT && heads()) {
          const acc_strided x = array({rows, k}, lead, extra), w = array({experts, n, k}, lead, extra, heads()), out = array({rows, n}, lead, extra);
          OK(acc_exec_product_rows(op, &x, &w, &offsets, use, (int32_t)per, &out, nullptr));
        } else if (kind == ACC_OP_PRODUCT) {
          const acc_strided a = array({rows, n}, lead, extra), b = array({rows, k}, lead, extra), out = array({experts, n, k}, lead, extra, heads());
          OK(acc_exec_product_outer(op, &a, &b, &offsets, use, (int32_t)per, &out, nullptr));
        } else if (kind == ACC_OP_ROUTE) {
          const int64_t tokens = pick(1, 2e5), all = std::max<int64_t>(3, pick(3, 2048));
          const acc_strided logits = array({tokens, all}, lead, extra), chosen = array({tokens, 3}, 0, 0), weights = array({tokens, 3}, 0, 0), starts = array({all + 1}, 0, 0),
                            order = array({tokens * 3}, 0, 0), place = array({tokens, 3}, 0, 0), back = array({tokens, all}, lead, extra);
          OK(acc_exec_route(op, &logits, &chosen, &weights, &starts, &order, &place, nullptr));
          OK(acc_exec_route_gradient(op, &logits, &chosen, &weights, &place, &back, nullptr));
        } else if (kind == ACC_OP_COMBINE) {
          const acc_strided y = array({rows, n}, lead, extra), place = array({rows, 3}, 0, 0), weights = array({rows, 3}, 0, 0), out = array({rows, n}, lead, extra),
                            dy = array({rows, n}, lead, extra), dw = array({rows, 3}, 0, 0);
          OK(acc_exec_combine(op, &y, &place, &weights, &out, nullptr));
          OK(acc_exec_combine_gradient(op, &out, &y, &place, &weights, &dy, &dw, nullptr));
        } else {
          const int64_t blocks = heads() ? (k + 31) / 32 : 1 + (int64_t)(g_random() % 6), between = plain ? 0 : (int64_t)(g_random() % 3);
          const acc_strided xc = array({rows, 16 * blocks}, 0, 16 * between), xs = array({rows, blocks}, plain ? 0 : 1, between), wc = array({experts, n, 16 * blocks}, 0, 16 * between),
                            ws = array({experts, n, blocks}, 0, between), out = array({rows, n}, lead, extra), x = array({rows, 32 * blocks}, lead, extra);
          OK(acc_exec_micro_quantise(op, &x, &xc, &xs, nullptr));
          OK(acc_exec_micro_values(op, &xc, &xs, &x, nullptr));
          OK(acc_exec_micro_rows(op, &xc, &xs, &wc, &ws, &offsets, use, (int32_t)per, &out, nullptr));
        }
      }
      OK(acc_op_destroy(op));
      if (units_in(argv[1]) != compiled) not_so("units that calls needed beside those that had been compiled", (long long)(units_in(argv[1]) - compiled), kind);
      std::printf("%s %d: %d units, %ld launches in pieces\n", type, kind, units, g_cut);
    }
  OK(acc_context_destroy(ctx));
  std::printf("wrong %d\n", g_wrong);
  return g_wrong ? 1 : 0;
}
