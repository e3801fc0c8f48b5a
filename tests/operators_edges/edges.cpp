// What the operators' drivers ask of the HIP runtime at the edges of what they take, on the stand-in for it of ../tsan/mock_hip.cpp:
// launches do nothing but leave their arguments, fills and events are written down, and a stream is under capture when this program says
// so.  Argument: which part to look at.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
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
#define hipEventQuery mock_EventQuery
#define hipDeviceSynchronize mock_DeviceSynchronize
#include "../tsan/mock_hip.cpp"
#undef hipStreamIsCapturing
#undef hipModuleLaunchKernel
#undef hipMalloc
#undef hipFree
#undef hipMemsetAsync
#undef hipEventRecord
#undef hipStreamWaitEvent
#undef hipEventQuery
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
static std::map<hipEvent_t, hipStream_t> g_recorded_on;
static int g_ended = 0;                           // captures that a call on another stream has ended
static bool g_done = true;                        // what has been enqueued
static int g_joined = 0;                          // events recorded on the stream under capture, and waits of others for what it holds

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
hipError_t hipEventRecord(hipEvent_t e, hipStream_t s)
{
  g_joined += s && s == g_capturing;
  g_recorded_on[e] = s;
  return hipSuccess;
}
// (either ends the capture, as the HIP runtime has it)
hipError_t hipEventQuery(hipEvent_t e)
{
  const bool captured = g_capturing && g_recorded_on[e] == g_capturing;
  g_ended += captured;
  return captured ? hipErrorCapturedEvent : g_done ? hipSuccess : hipErrorNotReady;
}
hipError_t hipDeviceSynchronize(void)
{
  g_ended += g_capturing != nullptr;
  return g_capturing ? hipErrorStreamCaptureUnsupported : hipSuccess;
}
hipError_t hipStreamWaitEvent(hipStream_t, hipEvent_t, unsigned) { return hipSuccess; }
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

// eager calls of several tiles on other streams while the one that had the last such call is under capture
static void order(acc_context ctx)
{
  acc_op op = recurrence(ctx);
  acc_stream one = nullptr, two = nullptr;
  OK(acc_stream_create(ctx, &one));
  OK(acc_stream_create(ctx, &two));
  scan(op, 5000, one);                            // (the call that is to be recorded, once)
  under_capture(one);
  const Launch recorded = scan(op, 5000, one);
  const Launch eager = scan(op, 5000, two);
  IS(g_joined == 0 && g_filled == 0);             // nothing of `two` waits for the capture, and nothing of it is recorded
  IS(recorded.recur.words != eager.recur.words);
  // it draws its tiles from a counter, which it has cleared: there is no order between it and what runs beside it
  IS(eager.recur.ticket);
  IS(g_launched[g_launched.size() - 2].name == "recur_clear" && g_launched[g_launched.size() - 2].recur.ticket == eager.recur.ticket);
  scan(op, 5000, two);
  IS(g_joined == 0);
  under_capture(nullptr);
  // and when the capture is over, everything is as before
  IS(!scan(op, 5000, two).recur.ticket);
  IS(!scan(op, 5000, one).recur.ticket);

  // a large scan of the array language has no such form: it is refused, outside the capture
  acc_env_sig env[1] = {};
  env[0].rank = env[0].ncomp = 1;
  env[0].type[0] = "Int32";
  acc_skel_desc d = {};
  d.kind = ACC_SKEL_SCANL1;
  d.n_env = 1;
  d.env = env;
  d.elt_type = "Int32";
  d.out_rank = 1;
  d.get = "arrIn0_0[ix]";
  d.combine = "x + y";
  acc_skel skel = nullptr;
  OK(acc_skel_create(ctx, &d, &skel));
  acc_array in = {}, out = {};
  in.rank = in.ncomp = out.rank = out.ncomp = 1;
  in.shape[0] = out.shape[0] = int64_t(1) << 30;
  in.ptr[0] = 1ull << 44;
  out.ptr[0] = 1ull << 45;
  OK(acc_exec_scan(skel, &in, in.shape[0], &out, nullptr, one));
  OK(acc_exec_scan(skel, &in, in.shape[0], &out, nullptr, two));
  OK(acc_exec_scan(skel, &in, in.shape[0], &out, nullptr, one));
  under_capture(one);
  const size_t launched = g_launched.size();
  IS(acc_exec_scan(skel, &in, in.shape[0], &out, nullptr, two) == ACC_ERR_INVALID);
  IS(g_joined == 0 && g_launched.size() == launched);
  in.shape[0] = out.shape[0] = 1000;              // (one that waits for nothing)
  OK(acc_exec_scan(skel, &in, in.shape[0], &out, nullptr, two));
  in.shape[0] = out.shape[0] = int64_t(1) << 30;
  under_capture(nullptr);
  OK(acc_exec_scan(skel, &in, in.shape[0], &out, nullptr, two));
  OK(acc_skel_destroy(skel));
  OK(acc_stream_destroy(ctx, one));
  OK(acc_stream_destroy(ctx, two));
  OK(acc_op_destroy(op));
}

// scratch memory of eager calls while another stream is under capture: what that stream had last is not asked for
static void beside(acc_context ctx)
{
  acc_op op = recurrence(ctx);
  acc_stream one = nullptr, two = nullptr, three = nullptr;
  OK(acc_stream_create(ctx, &one));
  OK(acc_stream_create(ctx, &two));
  OK(acc_stream_create(ctx, &three));
  // one stream alone has had scratch memory, and is under capture when a second one wants some
  const Launch first = scan(op, 5000, one);
  under_capture(one);
  const Launch other = scan(op, 5000, two);
  IS(g_ended == 0 && g_joined == 0 && other.recur.words != first.recur.words);
  const Launch recorded = scan(op, 5000, one);
  IS(recorded.recur.words == first.recur.words);  // (that stream's own)
  under_capture(nullptr);
  // several have had some
  g_done = false;
  const Launch third = scan(op, 5000, three);
  IS(third.recur.words != other.recur.words && third.recur.words != recorded.recur.words);
  under_capture(two);
  g_done = true;
  const Launch fourth = scan(op, 6000, three);
  IS(g_ended == 0 && g_joined == 0 && fourth.recur.words != other.recur.words);
  under_capture(nullptr);
  // and afterwards it is anybody's
  const Launch fifth = scan(op, 4000, one);
  IS(fifth.recur.words == other.recur.words || fifth.recur.words == third.recur.words || fifth.recur.words == fourth.recur.words);
  IS(g_ended == 0);
  OK(acc_stream_destroy(ctx, one));
  OK(acc_stream_destroy(ctx, two));
  OK(acc_stream_destroy(ctx, three));
  OK(acc_op_destroy(op));
}

// matrices of more numbers than a launch has threads for, by a matrix that is there many times
static void parts(acc_context ctx)
{
  acc_op_desc d = {};
  d.kind = ACC_OP_GROUPED;
  d.elt_type = "half";
  d.group = 32;
  acc_op op = nullptr;
  OK(acc_op_create(ctx, &d, &op));
  const int64_t experts = 100, n = 1 << 15, k = (1 << 15) - 7, blocks = (k + 31) / 32;
  acc_strided w = array({experts, n, k}), codes = array({experts, n, 16 * blocks}), scales = array({experts, blocks, n}), zeros = array({experts, blocks, n});
  for (const char *name : {"grouped_quantise", "grouped_values"}) {
    const size_t since = g_launched.size();
    if (!std::strcmp(name, "grouped_quantise")) OK(acc_exec_grouped_quantise(op, &w, &codes, &scales, &zeros, nullptr));
    else OK(acc_exec_grouped_values(op, &codes, &scales, &zeros, &w, nullptr));
    int64_t done = 0;
    for (size_t i = since; i < g_launched.size(); ++i) {
      const Launch &l = g_launched[i];
      IS(l.name == name && (uint64_t)l.grid * l.block <= 0xffffffffull && l.block % 64 == 0);
      IS(l.grouped.first == done);                // (one behind the other, teams of lanes whole)
      done += (int64_t)l.grid * l.block;
    }
    IS(done >= experts * n * blocks * 4 && g_launched.size() - since > 2);
  }
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
  else if (part == "order") order(ctx);
  else if (part == "beside") beside(ctx);
  else if (part == "parts") parts(ctx);
  else IS(!"a part that there is");
  OK(acc_context_destroy(ctx));
  std::printf("wrong %d\n", g_wrong);
  return g_wrong ? 1 : 0;
}
