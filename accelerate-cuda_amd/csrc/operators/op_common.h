/*
 * op_common.h -- what the operators' kernels share: element types and the segments of rows.
 */
#ifndef ACC_OP_COMMON_H
#define ACC_OP_COMMON_H

#include "op_args.h"

typedef unsigned int acc_u4 __attribute__((ext_vector_type(4)));
typedef unsigned int acc_u2 __attribute__((ext_vector_type(2)));
typedef float acc_f4 __attribute__((ext_vector_type(4)));

/* OP_ELT: 0 float, 1 half, 2 bfloat16 */
#if OP_ELT == 0
typedef float op_elt;
#elif OP_ELT == 1
typedef _Float16 op_elt;
#else
typedef __bf16 op_elt;
#endif
#define OP_VALUES (16 / (int)sizeof(op_elt))       /* elements of a chunk of 16 bytes */

/* 16 bytes of memory that start wherever an element may */
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) op_loose { acc_u4 v; };

/* `valid` elements from p on, zeros behind them; p may be anywhere if valid <= 0 */
template <bool ALIGNED> ACC_DEV acc_u4 op_chunk(const op_elt *p, const int valid)
{
  if (ALIGNED) return valid > 0 ? *(const acc_u4 *)p : acc_u4{0, 0, 0, 0};
  if (valid >= OP_VALUES) return ((const op_loose<op_elt> *)p)->v;
  op_elt e[OP_VALUES];
#pragma unroll
  for (int k = 0; k < OP_VALUES; ++k) e[k] = k < valid ? p[k] : (op_elt)0.0f;
  acc_u4 v;
  __builtin_memcpy(&v, e, 16);
  return v;
}

/* v, `bytes` further down: what is shifted in is zeros */
ACC_DEV acc_u4 op_shifted(const acc_u4 v, const int bytes)
{
  const unsigned long long lo = v.x | (unsigned long long)v.y << 32, hi = v.z | (unsigned long long)v.w << 32;
  const int n = 8 * bytes;
  unsigned long long a, b;
  if (bytes >= 8) {
    a = bytes >= 16 ? 0 : hi >> (n - 64);
    b = 0;
  } else {
    a = bytes ? lo >> n | hi << (64 - n) : lo;
    b = hi >> n;
  }
  return acc_u4{(unsigned int)a, (unsigned int)(a >> 32), (unsigned int)b, (unsigned int)(b >> 32)};
}

/* The segments of the rows 0 .. rows-1: number 0 is what lies before the first expert's rows, s the rows of expert s - 1,
 * experts + 1 what lies behind the last one's.  A start that is out of range counts as the nearest row, one that goes back as the
 * largest before it: whatever the starts say, a row is in one segment, so that no row outside the array is ever named, and all
 * segments together have no more tiles than the driver has allowed for. */
ACC_DEV int op_start(const int *offsets, const int experts, const int rows, const int s)
{
  /* (read whether it counts or not: no branch) */
  const int at = offsets[acc_min(s, experts)];
  return s > experts ? rows : acc_min(acc_max(at, 0), rows);
}

/* the lane's of 64 segments from number `base` on, of which the first begins at row `from` (0, or the end of the 64 before
 * them); behind the last one none */
struct op_lot { int begin, end; };
ACC_DEV op_lot op_segments(const int *offsets, const int experts, const int rows, const int base, const int from)
{
  const int lane = acc_lane();
  const int upto = acc_wave_scan(op_start(offsets, experts, rows, base + lane), [](int x, int y) { return acc_max(x, y); }, lane);
  op_lot l;
  l.end = acc_max(from, upto);
  l.begin = acc_wave_shift_up1(l.end);
  if (lane == 0) l.begin = from;
  return l;
}
/* the next 64, from number `base` on */
ACC_DEV op_lot op_segments_behind(const int *offsets, const int experts, const int rows, const int base, const op_lot lot)
{
  return op_segments(offsets, experts, rows, base, acc_readlane(lot.end, 63));
}

/* runs of `height` rows that `n` rows make, the last of them shorter (n + height may pass 2^31) */
ACC_DEV int op_runs(const int n, const int height) { return (int)(((unsigned int)n + (unsigned int)height - 1u) / (unsigned int)height); }

/* Workgroups go to the eight dies in turn: block b of n as a number such that every die has a run of neighbours. */
ACC_DEV long long op_die_run(const long long b, const long long n)
{
  const long long q = n / ACC_XCDS, r = n % ACC_XCDS, die = b % ACC_XCDS;
  return die * q + acc_min<long long>(die, r) + b / ACC_XCDS;
}

/* Tile x of ti x tj as (i, j), x counting down `height` rows of tiles, then on to the next column: the tiles that a die works
 * on at a time are about as many rows as columns, and few of either's operands are wanted. */
ACC_DEV void op_grouped(const int x, const int ti, const int tj, const int height, int *i, int *j)
{
  const int group = x / (height * tj), first = group * height, here = acc_min(height, ti - first), y = x - first * tj;
  *i = first + y % here;
  *j = y / here;
}

/* Whole tiles of `height` rows that the segments have, and segments that end amid another one.  `lot`: the first 64 segments. */
ACC_DEV void op_count_tiles(const int *offsets, const int experts, const int rows, const int height, op_lot lot, int *whole, int *parts)
{
  *whole = *parts = 0;
  for (int base = 0;;) {
    *whole += acc_wave_reduce((lot.end - lot.begin) / height, [](int x, int y) { return x + y; });
    *parts += __popcll(__ballot((lot.end - lot.begin) % height > 0));
    base += 64;
    if (base >= experts + 2) return;
    lot = op_segments_behind(offsets, experts, rows, base, lot);
  }
}

/* The expert with the n-th longest segment, of up to 62 experts (of more: number n), and that: what takes longest is begun
 * first, and the workgroups that are left at the end have little to do. */
ACC_DEV int op_nth_longest(const int *offsets, const int experts, const int rows, const int n, int *begin, int *end)
{
  if (experts > 62) {
    int from = 0;                                  /* the largest start up to the segment's own */
    for (int s = acc_lane(); s <= n; s += 64) from = acc_max(from, op_start(offsets, experts, rows, s));
    *begin = acc_wave_reduce(from, [](int x, int y) { return acc_max(x, y); });
    *end = acc_max(*begin, op_start(offsets, experts, rows, n + 1));
    return n;
  }
  const op_lot lot = op_segments(offsets, experts, rows, 0, 0);
  const int s = acc_lane();
  /* (no two of these are the same; a length beyond 2^26 counts as that) */
  const unsigned int mine = s >= 1 && s <= experts ? (unsigned int)(acc_min(lot.end - lot.begin, (1 << 26) - 2) + 1) << 6 | (63 - s) : 0;
  int longer = 0;
#pragma unroll 4
  for (int k = 1; k <= experts; ++k) longer += (unsigned int)acc_readlane((int)mine, k) > mine;
  const int at = __builtin_ctzll(__ballot((longer == n) & (mine > 0)) | 1ull << 63);
  *begin = acc_readlane(lot.begin, at);
  *end = acc_readlane(lot.end, at);
  return at - 1;
}

/* expert -1: rows of no segment; begin >= end: no such tile; `all`: rows of its segment */
struct op_tile { int expert, begin, end, all; };

/* How segments are cut into runs of `height` rows: all runs, the last of a segment shorter; its whole runs only; or what is
 * left behind those. */
#define OP_ALL 0
#define OP_WHOLE 1
#define OP_REST 2

/* The `tile`-th such run, counted segment after segment: a wave adds up the runs of 64 segments at a time.  Every wave of a
 * workgroup works it out for itself, and the answer is the same in every lane.  `lot`: the first 64 segments. */
template <int KIND> ACC_DEV op_tile op_find_tile(const int *offsets, const int experts, const int rows, const int height, op_lot lot, int tile)
{
  const int lane = acc_lane();
  op_tile t = {-1, 0, 0, 0};
  for (int base = 0;;) {
    int b = lot.begin;
    const int e = lot.end;
    if (KIND == OP_REST) b = e - (e - b) % height;
    const int runs = KIND == OP_WHOLE ? (e - b) / height : op_runs(e - b, height);
    const int upto = acc_wave_scan(runs, [](int x, int y) { return x + y; }, lane);
    const unsigned long long beyond = __ballot(upto > tile);
    if (beyond) {
      const int at = __builtin_ctzll(beyond);
      const int first = acc_readlane(b, at) + (tile - (acc_readlane(upto, at) - acc_readlane(runs, at))) * height;
      t.begin = first;
      t.end = first + acc_min(acc_readlane(e, at) - first, height);
      t.all = acc_readlane(e, at) - acc_readlane(lot.begin, at);
      t.expert = base + at == experts + 1 ? -1 : base + at - 1;
      return t;
    }
    tile -= acc_readlane(upto, 63);
    base += 64;
    if (base >= experts + 2) return t;
    lot = op_segments_behind(offsets, experts, rows, base, lot);
  }
}

/* Of the runs of `height` rows, counted segment after segment: the first of segment number s, and how many that has. */
ACC_DEV int op_first_run(const int *offsets, const int experts, const int rows, const int height, const int s, int *runs)
{
  const int lane = acc_lane();
  int first = 0;
  op_lot lot = op_segments(offsets, experts, rows, 0, 0);
  for (int base = 0;;) {
    const int mine = op_runs(lot.end - lot.begin, height);
    first += acc_wave_reduce(base + lane < s ? mine : 0, [](int x, int y) { return x + y; });
    if (s - base < 64) {
      *runs = acc_readlane(mine, s - base);
      return first;
    }
    base += 64;
    lot = op_segments_behind(offsets, experts, rows, base, lot);
  }
}

#endif
