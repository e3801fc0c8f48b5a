// Which sequences a wave looks at for those without a row: op_empty_sequences of op_recur.h as it stands there (function.inc), on the host,
// a wave of one lane at a time, for tiles in their millions.  What is asked: that no offset outside the array is read, and that all shares
// together look at every sequence once.
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <vector>

#define ACC_DEV static inline
#define OP_WAVES 8

static int64_t g_sequences = 0, g_outside = 0, g_read = 0, g_before = 0;
struct Offsets {
  int operator[](const int64_t i) const
  {
    if (i < 0 || i > g_sequences) ++g_outside;
    if (++g_read - g_before > 1 << 22 || g_outside > 1000) throw 1;      // (a share that never ends)
    return 0;                                     // (every sequence is without a row)
  }
};
struct acc_recur_args {
  float *leave = reinterpret_cast<float *>(16), *enter = nullptr;
  Offsets offsets;
  int64_t enter_stride = 0, leave_stride = 0;
  int32_t sequences = 0, tiles = 0;
};
struct op_pair { float v; };
static std::vector<unsigned char> *g_seen = nullptr;
static int64_t g_kept = 0, g_twice = 0;
static int acc_min(int a, int b) { return std::min(a, b); }
static int acc_max(int a, int b) { return std::max(a, b); }
static unsigned long long g_lane = 0;
static unsigned long long __ballot(bool b) { return b ? 1ull << g_lane : 0; }
static long long op_slot(const acc_recur_args &, const int sequence) { return sequence; }
static op_pair op_state(const float *, long long, long long, int, int) { return {0.0f}; }
static void op_keep(float *, long long, const long long at, int, int, const op_pair &)
{
  ++g_kept;
  if (at < 0 || at >= g_sequences) ++g_outside;
  else if (!g_seen->empty() && (*g_seen)[(size_t)at]++) ++g_twice;
}
#include "function.inc"

int main()
{
  int wrong = 0;
  // (tiles, sequences): as many tiles as 2^30 rows of a scan have, and of a gradient; more sequences than a step of 32 bits covers
  const int64_t cases[][2] = {{1, 5}, {1, 1000}, {40, 70000}, {4194303, 1000}, {4194304, 1000}, {4194305, 1000}, {8388599, 3}, {3000000, 1600000000}, {2, 200000}};
  for (const auto &c : cases) {
    acc_recur_args p;
    p.tiles = (int32_t)c[0];
    p.sequences = (int32_t)(g_sequences = c[1]);
    // every lane of every share where there are few; else a lane at either end, of the shares at both ends
    const int64_t shares = c[0] * OP_WAVES;
    const bool whole = g_sequences <= 200000 && shares <= 4096;
    std::vector<unsigned char> seen(whole ? (size_t)g_sequences : 0);
    g_seen = &seen;
    g_outside = g_read = g_kept = g_twice = 0;
    for (int64_t share = 0; share < shares && g_outside <= 1000; ++share) {
      if (!whole && share > 300 && share < shares - 300) continue;
      for (int lane = 0; lane < 64 && g_outside <= 1000; lane += whole ? 1 : 63) {
        g_lane = (unsigned long long)lane;
        g_before = g_read;
        try {
          op_empty_sequences(p, 1 << 30, (int)share, lane, 0, 1);
        } catch (int) {
          g_outside += 1001;
        }
      }
    }
    const bool missing = whole && g_kept != g_sequences;
    std::printf("%lld tiles, %lld sequences: %lld read, %lld outside, %lld twice%s\n", (long long)c[0], (long long)c[1], (long long)g_read, (long long)g_outside, (long long)g_twice, missing ? ", some missing" : "");
    wrong += g_outside > 0 || g_twice > 0 || missing;
  }
  std::printf("wrong %d\n", wrong);
  return wrong ? 1 : 0;
}
