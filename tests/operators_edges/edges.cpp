// What the operators' drivers ask of the HIP runtime at the edges of what they take, on the stand-in for it of ../tsan/mock_hip.cpp:
// launches do nothing but leave their arguments, fills and events are written down, and a stream is under capture when this program says
// so.  Argument: which part to look at.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>
#include <vector>

#include "../../accelerate-cuda_amd/csrc/operators/op_args.h"

// (this program's own versions of some of the stand-in's functions)
#define hipStreamIsCapturing mock_StreamIsCapturing
#define hipModuleLaunchKernel mock_ModuleLaunchKernel
#define hipMalloc mock_Malloc
#define hipFree mock_Free
#define hipMemsetAsync mock_MemsetAsync
#define hipEventRecord mock_EventRecord
#define hipStreamWaitEvent mock_StreamWaitEvent
#define hipDeviceSynchronize mock_DeviceSynchronize
#include "../tsan/mock_hip.cpp"
#undef hipStreamIsCapturing
#undef hipModuleLaunchKernel
#undef hipMalloc
#undef hipFree
#undef hipMemsetAsync
#undef hipEventRecord
#undef hipStreamWaitEvent
#undef hipDeviceSynchronize

struct Launch {
  std::string name;
  hipStream_t stream;
  unsigned grid, block;
  acc_recur_args recur;                           // of "recur" and "recur_clear"
  acc_grouped_args grouped;                       // of "grouped..."
};
struct Fill { uint64_t from, to; hipStream_t stream; size_t launches; };
static hipStream_t g_capturing = nullptr;
static std::vector<Launch> g_launched;
static std::vector<Fill> g_fills;
static uint64_t g_next = 1ull << 50;
static int g_filled = 0;                          // fills that were asked for on the stream under capture
static int g_joined = 0;                          // events recorded on the stream under capture, and waits of others for what it holds
static int g_synchronised = 0;
static hipError_t g_synchronise = hipSuccess;

extern "C" {
hipError_t hipStreamIsCapturing(hipStream_t s, hipStreamCaptureStatus *c)
{
  *c = s && s == g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned gx, unsigned, unsigned, unsigned bx, unsigned, unsigned, unsigned, hipStream_t s, void **params, void **)
{
  Launch l = {reinterpret_cast<const Function *>(f)->name, s, gx, bx, {}, {}};
  if (l.name.rfind("recur", 0) == 0) l.recur = *static_cast<const acc_recur_args *>(params[0]);
  if (l.name.rfind("grouped", 0) == 0) l.grouped = *static_cast<const acc_grouped_args *>(params[0]);
  g_launched.push_back(l);
  return hipSuccess;
}
hipError_t hipMalloc(void **p, size_t n)          // (addresses alone: nothing here reads or writes device memory)
{
  *p = reinterpret_cast<void *>(g_next);
  g_next += (n + 4095) / 4096 * 4096 + 4096;
  return hipSuccess;
}
hipError_t hipFree(void *) { return hipSuccess; }
hipError_t hipMemsetAsync(void *p, int, size_t n, hipStream_t s)
{
  g_filled += s && s == g_capturing;
  g_fills.push_back({reinterpret_cast<uint64_t>(p), reinterpret_cast<uint64_t>(p) + n, s, g_launched.size()});
  return hipSuccess;
}
hipError_t hipEventRecord(hipEvent_t, hipStream_t s) { g_joined += s && s == g_capturing; return hipSuccess; }
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipSuccess; }
hipError_t hipDeviceSynchronize(void) { ++g_synchronised; return g_synchronise; }
}

#define OK(call)                                                                        \
  do {                                                                                  \
    int rc__ = (call);                                                                  \
    if (rc__ != ACC_OK) {                                                               \
      std::fprintf(stderr, "%s:%d: %s -> %d: %s\n", __FILE__, __LINE__, #call, rc__, acc_last_error()); \
      std::exit(2);                                                                     \
    }                                                                                   \
  } while (0)
static int g_wrong = 0;
#define IS(what)                                                                        \
  do {                                                                                  \
    if (!(what)) {                                                                      \
      std::fprintf(stderr, "%s:%d: not so: %s\n", __FILE__, __LINE__, #what);           \
      ++g_wrong;                                                                        \
    }                                                                                   \
  } while (0)

// a dense array of its own place
static acc_strided array(std::initializer_list<int64_t> shape)
{
  static uint64_t place = 0;
  acc_strided a = {};
  a.rank = (int32_t)shape.size();
  int d = 0;
  for (int64_t n : shape) a.shape[d++] = n;
  int64_t step = 1;
  for (int k = a.rank - 1; k >= 0; --k) {
    a.stride[k] = step;
    step *= a.shape[k];
  }
  a.ptr = (1ull << 41) + (place++ % 64 << 45);    // (far apart)
  return a;
}

static void under_capture(acc_stream s) { g_capturing = static_cast<hipStream_t>(s); }

static acc_op recurrence(acc_context ctx)
{
  acc_op_desc d = {};
  d.kind = ACC_OP_RECUR;
  d.elt_type = "float";
  acc_op op = nullptr;
  OK(acc_op_create(ctx, &d, &op));
  return op;
}
// a scan of several tiles: its launch
static Launch scan(acc_op op, int64_t rows, acc_stream s)
{
  const acc_strided z = array({rows, 64}), x = array({rows, 64}), out = array({rows, 64}), offsets = array({2});
  OK(acc_exec_recur(op, &z, &x, &offsets, nullptr, nullptr, nullptr, &out, s));
  IS(g_launched.back().name == "recur" && g_launched.back().recur.tiles > 1 && g_launched.back().stream == static_cast<hipStream_t>(s));
  return g_launched.back();
}
// whether a fill on a stream not under capture covers the launch's scratch memory, behind launch number `since` and before the last
static bool cleared(const Launch &l, size_t since)
{
  const uint64_t from = reinterpret_cast<uint64_t>(l.recur.words), to = from + (uint64_t)l.recur.tiles * l.recur.strips * 3 * 64 * 8;
  for (const Fill &f : g_fills)
    if (f.launches >= since && f.from <= from - 256 && f.to >= to) return true;
  return false;
}

// memory of tagged words that is first lent to a call under capture: nobody's graph, nobody clears it
static void pool(acc_context ctx)
{
  acc_op op = recurrence(ctx);
  acc_stream one = nullptr, two = nullptr;
  OK(acc_stream_create(ctx, &one));
  OK(acc_stream_create(ctx, &two));
  under_capture(one);
  const Launch recorded = scan(op, 5000, one);
  const size_t fills = g_fills.size();
  IS(g_filled == 0);
  under_capture(nullptr);
  IS(recorded.recur.tag != 0 && recorded.recur.ticket);
  OK(acc_stream_destroy(ctx, one));               // (and with it the graph)
  size_t since = g_launched.size();
  const Launch eager = scan(op, 5000, two);
  IS(eager.recur.words == recorded.recur.words);  // the same block
  IS(g_fills.size() == fills + 1 && cleared(eager, since));
  // once is enough
  const Launch again = scan(op, 5000, two);
  IS(again.recur.words == eager.recur.words && again.recur.tag != eager.recur.tag && g_fills.size() == fills + 1);

  // tags that run out under capture: no fill there, and one before the block's next eager call
  for (acc::ScratchBlock &b : ctx->scratch)
    if (b.protocol == acc::SCRATCH_FLAGS) b.epoch = 0xFFFFFFFFu;
  under_capture(two);
  const Launch last = scan(op, 5000, two);
  IS(last.recur.words == eager.recur.words && last.recur.tag != 0 && g_filled == 0);
  under_capture(nullptr);
  OK(acc_stream_destroy(ctx, two));
  OK(acc_stream_create(ctx, &one));
  since = g_launched.size();
  const Launch behind = scan(op, 5000, one);
  IS(behind.recur.words == eager.recur.words && cleared(behind, since));
  OK(acc_stream_destroy(ctx, one));
  OK(acc_op_destroy(op));
}

int main(int, char **argv)
{
  OK(acc_init());
  OK(acc_cache_set_dir(argv[1]));
  acc_context ctx = nullptr;
  OK(acc_context_create(0, &ctx));
  const std::string part = argv[2];
  if (part == "pool") pool(ctx);
  else IS(!"a part that there is");
  OK(acc_context_destroy(ctx));
  std::printf("wrong %d\n", g_wrong);
  return g_wrong ? 1 : 0;
}
