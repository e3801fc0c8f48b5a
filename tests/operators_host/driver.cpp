// What the operators' drivers do with scratch memory when their calls are recorded into a graph, on the stand-in for the HIP
// runtime of ../tsan/mock_hip.cpp: launches do nothing but say which scratch memory they were given, and a stream is under
// capture when this program says so.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <set>

#include "../../accelerate-cuda_amd/csrc/operators/op_args.h"

// (this program's own versions of five of the stand-in's functions)
#define hipStreamIsCapturing mock_StreamIsCapturing
#define hipModuleLaunchKernel mock_ModuleLaunchKernel
#define hipMalloc mock_Malloc
#define hipFree mock_Free
#define hipMemsetAsync mock_MemsetAsync
#include "../tsan/mock_hip.cpp"
#undef hipStreamIsCapturing
#undef hipModuleLaunchKernel
#undef hipMalloc
#undef hipFree
#undef hipMemsetAsync

static hipStream_t g_capturing = nullptr;
static const void *g_counts = nullptr;          // the scratch memory of the last launch of a router
static std::set<const void *> g_freed;
static long g_filled = 0;                       // fills that were asked for on the stream under capture

extern "C" {
hipError_t hipStreamIsCapturing(hipStream_t s, hipStreamCaptureStatus *c)
{
  *c = s && s == g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
hipError_t hipModuleLaunchKernel(hipFunction_t, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, unsigned, hipStream_t, void **params, void **)
{
  g_counts = static_cast<const acc_route_args *>(params[0])->counts;
  return hipSuccess;
}
hipError_t hipMalloc(void **p, size_t n) { *p = std::malloc(n ? n : 1); return *p ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipFree(void *p) { g_freed.insert(p); return hipSuccess; }      // (kept, so that no later block has its address)
hipError_t hipMemsetAsync(void *, int, size_t, hipStream_t s) { g_filled += s && s == g_capturing; return hipSuccess; }
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

static acc_strided array(acc_devptr p, int64_t rows, int64_t columns)
{
  acc_strided a = {};
  a.rank = columns < 0 ? 1 : 2;
  a.shape[0] = rows;
  a.stride[0] = columns < 0 ? 1 : columns;
  if (columns >= 0) {
    a.shape[1] = columns;
    a.stride[1] = 1;
  }
  a.ptr = p;
  return a;
}

int main()
{
  OK(acc_init());
  acc_context ctx = nullptr;
  OK(acc_context_create(0, &ctx));
  acc_op_desc d = {ACC_OP_ROUTE, "float", 2, 1};
  acc_op router = nullptr;
  OK(acc_op_create(ctx, &d, &router));
  // two sizes, with counts of several workgroups: the second wants a larger block
  const int64_t experts = 32;
  const auto route = [&](int64_t tokens, acc_stream st) -> const void * {
    const acc_devptr at = 1ull << 40;             // (nothing is read or written)
    const acc_strided logits = array(at, tokens, experts), chosen = array(at + (1ull << 32), tokens, 2), weights = array(at + (2ull << 32), tokens, 2),
                      offsets = array(at + (3ull << 32), experts + 1, -1), order = array(at + (4ull << 32), tokens * 2, -1), place = array(at + (5ull << 32), tokens, 2);
    g_counts = nullptr;
    OK(acc_exec_route(router, &logits, &chosen, &weights, &offsets, &order, &place, st));
    return g_counts;
  };
  acc_stream one = nullptr, two = nullptr;
  OK(acc_stream_create(ctx, &one));
  OK(acc_stream_create(ctx, &two));
  const auto under_capture = [&](acc_stream st) { g_capturing = static_cast<hipStream_t>(st); };
  size_t freed = 0, held = 0;

  // a call, the same call recorded, and then others while the graph lives
  const void *eager = route(1000, one);
  IS(eager);
  under_capture(one);
  const void *recorded = route(1000, one);
  IS(recorded == eager);                          // (the pool has what it needs: nothing is allocated under capture)
  const void *again = route(1000, one);
  IS(again == recorded);                          // one behind the other in the same graph
  under_capture(nullptr);
  IS(route(1000, two) != recorded);
  IS(route(900, two) != recorded);
  IS(route(1000, one) != recorded);
  OK(acc_context_trim(ctx, &freed));
  IS(freed > 0 && !g_freed.count(recorded));
  OK(acc_context_scratch_bytes(ctx, &held));
  IS(held > 0);
  // the next graph of that stream is replayed behind the first: it may have the same
  under_capture(one);
  IS(route(1000, one) == recorded);
  // a block that is made under capture: nothing clears it there
  const void *larger = route(6000, one);
  under_capture(nullptr);
  IS(larger != recorded && g_filled == 0);
  IS(route(6000, two) != larger);
  // another stream's graph has its own
  under_capture(two);
  const void *other = route(1000, two);
  under_capture(nullptr);
  IS(other != recorded && other != larger);

  // the stream's graphs go with it, and then its blocks are anybody's
  OK(acc_stream_destroy(ctx, one));
  OK(acc_context_trim(ctx, &freed));
  IS(g_freed.count(recorded) && g_freed.count(larger) && !g_freed.count(other));
  OK(acc_stream_destroy(ctx, two));
  OK(acc_op_destroy(router));
  OK(acc_context_destroy(ctx));
  IS(g_freed.count(other));
  std::printf("wrong %d\n", g_wrong);
  return g_wrong ? 1 : 0;
}
