/*
 * op_recur.h -- a gated linear recurrence along the rows of ragged sequences, its gradient, and one step of it.
 *
 *   h[t] = a[t] h[t-1] + b[t]       per channel; a = gates, b = values (OP_GATE 0), or a = s(gates), b = (1 - a) values with
 *                                   s(z) = 1 / (1 + e^-z) (OP_GATE 1)
 *   u[t] = a[t] (dh[t] + u[t+1])    the gradient that goes on to the row before; g = dh[t] + u[t+1] is that of h[t], then
 *                                   da = g h[t-1], db = g, and for OP_GATE 1  dz = g (h[t-1] - x) a (1 - a), dx = g (1 - a)
 *
 * Both are scans of the maps h -> A h + B, the second from the last row to the first (OP_BACK; rows are counted from the end
 * then).  A row that begins a sequence takes nothing of the row before: it replaces, it does not multiply, so that no infinity
 * and nothing that is not a number passes from one sequence to the next.  A map is no good where A or B is not finite (gates above 1,
 * whose product overflows though the state is small or 0) or the state is infinite (of which an A that has become 0 would make NaN):
 * such a tile waits for the state in front of it, and its waves take their rows one after the other, as the definition has it.  (Half,
 * one sequence of 65536 x 512: 56 us, 12000 where every tile's product overflows.)
 *
 * Bound by memory: every array passes by once.  bfloat16, 32768 rows of 2048 in 8 sequences, sigmoids: 102 us, 3.9 TB/s, the gradient 170,
 * 4.7 (a copy 5.4); what is short of that are the gates, worked out in both passes.  One sequence of 65536 half rows of 512: 56, 3.6, the
 * tiles' waits for those before; Float32, 9001 rows of 1001: 38, 2.9, rows starting amid lines.  A workgroup has a tile of 64 OP_V channels and 8 OP_R rows, a wave OP_R of those, all
 * of them in registers; it goes over them twice, first for the tile's map, and once what comes in from the rows before is known for
 * the results.  That it finds in what the tiles before have left: their maps (A, B), or the state behind them (H), as 64-bit words
 * of a Float32 and the launch's tag, which need no fence.  A tile in which a sequence begins leaves a state at once.  Every tile
 * leaves its map without having waited, so waits end as long as the tiles before are on the device: workgroups start in the order of
 * their numbers, or (in a graph, or beside one that is being recorded: what else runs then nobody knows) draw them from a counter.
 */
#include "op_common.h"

/* OP_V: channels of a lane, a word of a row; OP_THIN: one of 16 bits, for rows of up to 64 */
#if OP_THIN
#define OP_V 1
#else
#define OP_V (4 / (int)sizeof(op_elt))
#endif
#define OP_WAVES 8
#define OP_NEAR 32                                 /* tiles in front that are looked at, at once */

/* a word of memory, which starts wherever an element may */
#if OP_THIN
typedef unsigned short op_word;
#else
typedef unsigned int __attribute__((aligned(sizeof(op_elt)))) op_word;
#endif

struct op_pair { float v[OP_V]; };
ACC_DEV op_pair op_floats(const unsigned int w)
{
  op_elt e[OP_V];
  __builtin_memcpy(e, &w, sizeof(e));
  op_pair f;
#pragma unroll
  for (int k = 0; k < OP_V; ++k) f.v[k] = (float)e[k];
  return f;
}

/* the same, made where it is wanted: what has been made of all rows' words, kept from one pass to the next, takes twice their registers */
ACC_DEV op_pair op_again(unsigned int w)
{
  acc_pin(w);
  return op_floats(w);
}

/* A lane's word of a row (the same for all lanes) from element `at` on.  Where a row ends amid a lane's word, the lane reads one
 * element earlier and shifts (`down` bits): no read goes past the row. */
ACC_DEV unsigned int op_read(const op_elt *row, const unsigned int at)
{
  return __builtin_nontemporal_load((const op_word *)((const char *)row + at * (unsigned int)sizeof(op_elt)));
}
/* `valid` of a lane's channels there are (0 to OP_V); `whole`: in all lanes OP_V */
ACC_DEV void op_write(op_elt *row, const unsigned int at, const bool whole, const int valid, const op_pair &f)
{
  op_elt *const p = (op_elt *)((char *)row + at * (unsigned int)sizeof(op_elt));
  op_elt e[OP_V];
#pragma unroll
  for (int k = 0; k < OP_V; ++k) e[k] = (op_elt)f.v[k];
  unsigned int w = 0;
  __builtin_memcpy(&w, e, sizeof(e));
  if (whole || valid == OP_V) __builtin_nontemporal_store((op_word)w, (op_word *)p);
  else if (valid == 1) *p = e[0];
}

/* what a gate keeps and what it takes in, for a gate of OP_GATE 1: 1 / (1 + e) and e / (1 + e) with e = e^-z, of which neither
 * loses its digits; an exponent beyond 2^126 stays there (the first is below 2^-125 then, and the second 1) */
struct op_gate { float keep, take; };
ACC_DEV op_gate op_gate_of(const float z)
{
  op_gate g;
#if OP_GATE
  const float y = z * -1.44269504f;
  float t = sizeof(op_elt) == 4 ? __builtin_fmaf(z, -1.44269504f, -y) + z * -1.92596303e-8f : 0.0f;
  t = __builtin_fabsf(y) <= 126.0f ? t : 0.0f;     /* (what the product's rounding has lost; Float32 alone can show it) */
  const float most = y > 126.0f ? 126.0f : y;
  const float e = __builtin_amdgcn_exp2f(most) * (1.0f + t * 0.693147181f);
  g.keep = sizeof(op_elt) == 4 ? 1.0f / (1.0f + e) : __builtin_amdgcn_rcpf(1.0f + e);
  g.take = e * g.keep;
#else
  g.keep = z;
  g.take = 1.0f;
#endif
  return g;
}

/* How many of the n offsets, which ascend, are at most a lane's `row`; they count as the nearest row there is.  Lanes' rows ascend
 * by one.  The wave looks at 64 offsets at a time until 64 are left that the first lane's row lies among, and the lanes search
 * those; where the last lane's lies behind them, offsets lie close, and every lane searches memory. */
ACC_DEV int op_upto(const int *offsets, const int n, const int rows, const int row, const int lane)
{
  const auto value = [&](const int i) { return i < n ? acc_min(acc_max(offsets[i], 0), rows) : 0x7fffffff; };
  const int least = acc_readlane(row, 0), most = acc_readlane(row, 63);
  int lo = 0, hi = n;                              /* the count of the first lane's row lies in between */
  while (hi - lo > 63) {
    const int step = (hi - lo) / 64;               /* (one at least) */
    const int c = __popcll(__ballot(value(lo + lane * step) <= least));
    if (c < 64) hi = acc_min(hi, lo + c * step);
    lo += acc_max(c - 1, 0) * step;
  }
  const int mine = value(lo + lane);
  int found = 0;
  if (acc_readlane(mine, 63) > most) {
#pragma unroll
    for (int step = 32; step > 0; step /= 2) found += __builtin_amdgcn_ds_bpermute((found + step - 1) * 4, mine) <= row ? step : 0;
    return lo + found;
  }
  hi = n;
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (value(mid) <= row) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

/* a row of the states, or -1 */
ACC_DEV long long op_slot(const acc_recur_args &p, const int sequence)
{
  const int at = p.index ? p.index[sequence] : sequence;
  return at >= 0 && at < p.states ? at : -1;
}
ACC_DEV op_pair op_state(const float *states, const long long stride, const long long at, const int channel, const int valid)
{
  op_pair f;
#pragma unroll
  for (int k = 0; k < OP_V; ++k) f.v[k] = states && at >= 0 && k < valid ? states[at * stride + channel + k] : 0.0f;
  return f;
}
ACC_DEV void op_keep(float *states, const long long stride, const long long at, const int channel, const int valid, const op_pair &f)
{
  if (!states || at < 0) return;
#pragma unroll
  for (int k = 0; k < OP_V; ++k)
    if (k < valid) states[at * stride + channel + k] = f.v[k];
}

ACC_DEV void op_put(unsigned long long *d, const unsigned int tag, const op_pair &f)
{
#pragma unroll
  for (int k = 0; k < OP_V; ++k) __hip_atomic_store(d + k, (unsigned long long)tag << 32 | __float_as_uint(f.v[k]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
/* whether all of the lane's words carry the tag */
ACC_DEV bool op_get(const unsigned long long *d, const unsigned int tag, op_pair *f)
{
  bool all = true;
#pragma unroll
  for (int k = 0; k < OP_V; ++k) {
    const unsigned long long w = __hip_atomic_load(d + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    all = all && (unsigned int)(w >> 32) == tag;
    f->v[k] = __uint_as_float((unsigned int)w);
  }
  return all;
}

#if OP_STEP
/* one row a sequence: a lane has a word of a row */
extern "C" __global__ void __launch_bounds__(256) recur_step(const acc_recur_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const long long row = blockIdx.x / p.strips, left = p.width - (long long)(blockIdx.x % p.strips) * (256 * OP_V) - (int)threadIdx.x * OP_V;
  if (left <= 0) return;
  const int channel = (int)(p.width - left), valid = acc_min<long long>(left, OP_V);
  /* (asked for before it is known whether the row counts; op_read and op_write count bytes in 32 bits, a row may have more) */
  const long long at = acc_min(channel, p.width - OP_V);
  const int down = (int)(channel - at) * 8 * (int)sizeof(op_elt);
  const op_pair z = op_floats(op_read((const op_elt *)p.gates + row * p.gates_stride + at, 0) >> down);
  const op_pair x = op_floats(op_read((const op_elt *)p.values + row * p.values_stride + at, 0) >> down);
  const long long slot = op_slot(p, (int)row);
  if (slot < 0) return;
  op_pair h = op_state(p.enter, p.enter_stride, slot, channel, valid);
#pragma unroll
  for (int k = 0; k < OP_V; ++k) {
    const op_gate g = op_gate_of(z.v[k]);
    h.v[k] = __builtin_fmaf(g.keep, h.v[k], g.take * x.v[k]);
  }
  op_keep(p.leave, p.leave_stride, slot, channel, valid, h);
  op_write((op_elt *)p.out + row * p.out_stride + channel, 0, false, valid, h);
}
#else

struct op_map { op_pair a, b; };
ACC_DEV float op_largest(const op_pair &f, float most)       /* (what is not a number is not) */
{
#pragma unroll
  for (int k = 0; k < OP_V; ++k) most = __builtin_fmaxf(most, __builtin_fabsf(f.v[k]));
  return most;
}

/* the words of a tile's strip: A, B, H */
ACC_DEV unsigned long long *op_words(const acc_recur_args &p, const long long tile, const int strip, const int plane, const int lane)
{
  return (unsigned long long *)p.words + (((tile * p.strips + strip) * 3 + plane) * 64 + lane) * OP_V;
}

/* sequences without a row leave what they enter with: every tile looks at a share of the sequences (steps in 64 bits: tiles may be millions) */
ACC_DEV void op_empty_sequences(const acc_recur_args &p, const int rows, const int share, const int lane, const int channel, const int valid)
{
  if (!p.leave) return;
  for (long long from = share * 64ll; from < p.sequences; from += p.tiles * (OP_WAVES * 64ll)) {
    const int base = (int)from, s = base + lane, n = acc_min(s, p.sequences - 1);
    const int begin = acc_min(acc_max(p.offsets[n], 0), rows), end = acc_min(acc_max(p.offsets[n + 1], 0), rows);
    unsigned long long none = __ballot(s < p.sequences && end <= begin);
    while (none) {
      const int j = __builtin_ctzll(none);
      none &= none - 1;
      const long long at = op_slot(p, base + j);
      op_keep(p.leave, p.leave_stride, at, channel, valid, op_state(p.enter, p.enter_stride, at, channel, valid));
    }
  }
}

extern "C" __global__ void __launch_bounds__(64 * OP_WAVES) __attribute__((amdgpu_waves_per_eu(4))) recur(const acc_recur_args p)
{
  if (p.guard && *p.guard == 0u) return;
  __shared__ op_map maps[OP_NEAR][64];             /* of the waves' rows; then of the tiles before */
  __shared__ int ends[OP_NEAR];                    /* whether a wave's map forgets what comes in (1), from its first row on (2); then what is there */
  __shared__ unsigned int drawn;
  __shared__ op_pair carried[64];                  /* from wave to wave, where they take turns */
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), rows = (int)p.rows;
  unsigned int number = blockIdx.x;
  if (p.ticket) {
    if (tid == 0) {
      drawn = atomicAdd(p.ticket, 1u);
      if (drawn + 1 == gridDim.x) *p.ticket = 0u;  /* (the last there is: the next launch begins with 0) */
    }
    __syncthreads();
    number = __builtin_amdgcn_readfirstlane(drawn);
  }
  const int tile = (int)(number / (unsigned int)p.strips), strip = (int)(number % (unsigned int)p.strips);
  const int channel = (strip * 64 + lane) * OP_V, valid = acc_max(acc_min(p.width - channel, OP_V), 0);
  if (rows == 0) {
    op_empty_sequences(p, rows, tile * OP_WAVES + wave, lane, channel, valid);
    return;
  }

  /* The wave's rows, in the order of the recurrence: physical row first + r, or (back) first + OP_R - 1 - r.  Rows that there are
   * not are read as the nearest one, lanes without a channel as the last word of the row. */
  const long long from = ((long long)tile * OP_WAVES + wave) * OP_R, first = OP_BACK ? rows - from - OP_R : from;
  const int at = acc_min(channel, p.width - OP_V), down = valid > 0 ? (channel - at) * 8 * (int)sizeof(op_elt) : 0;
  const bool whole = __ballot(valid != OP_V) == 0;
  const auto read_rows = [&](const void *base, const long long stride, const int back, unsigned int (&to)[OP_R]) {
    if (first >= back && first + OP_R <= rows) {
      const op_elt *x = (const op_elt *)base + (first + (OP_BACK ? OP_R - 1 : 0) - back) * stride;
#pragma unroll
      for (int r = 0; r < OP_R; ++r, x += OP_BACK ? -stride : stride) to[r] = op_read(x, at);
    } else {
#pragma unroll
      for (int r = 0; r < OP_R; ++r)
        to[r] = op_read((const op_elt *)base + acc_max<long long>(acc_min<long long>(first + (OP_BACK ? OP_R - 1 - r : r), rows - 1) - back, 0) * stride, at);
    }
  };
  const auto shift_rows = [&](unsigned int (&w)[OP_R]) {
    if (!whole)
#pragma unroll
      for (int r = 0; r < OP_R; ++r) w[r] >>= down;
  };
  unsigned int zw[OP_R], xw[OP_R];
  read_rows(p.gates, p.gates_stride, 0, zw);
  read_rows(OP_BACK ? p.dout : p.values, OP_BACK ? p.dout_stride : p.values_stride, 0, xw);

  /* sequences: lane j counts those that begin up to row first - 1 + j (as 32 bits: rows end well below 2^31) */
  const int row = (int)(first - 1) + lane;
  const int upto = op_upto(p.offsets, p.sequences + 1, rows, row, lane), before = acc_wave_shift_up1(upto);
  const bool inside = row >= 0 && row < rows && upto >= 1 && upto <= p.sequences, change = lane > 0 && upto > before;
  const unsigned long long mask = (1ull << OP_R) - 1;
  const unsigned long long within = __ballot(inside) >> 1 & mask, begins = __ballot(change && inside) >> 1 & mask, stops = __ballot(change) >> 2 & within;
  const auto turned = [](const unsigned long long m) { return OP_BACK ? __brevll(m) >> (64 - OP_R) : m; };
  const unsigned long long here = turned(within), resets = turned(OP_BACK ? stops : begins), leaves = turned(OP_BACK ? begins : stops);
  const auto sequence_of = [&](const int r) { return acc_readlane(upto, (OP_BACK ? OP_R - 1 - r : r) + 1) - 1; };
  const auto entering = [&](const int r) { return op_state(p.enter, p.enter_stride, op_slot(p, sequence_of(r)), channel, valid); };

  /* The wave's map: from the last row on that begins a sequence.  What enters there is kept: where states are replaced in place, it
   * may be gone by the time of the second pass.  (Sequences that begin before end in these rows, too.) */
  const int latest = resets ? 63 - __builtin_clzll(resets) : -1;
  op_map own;
  op_pair entered;
#pragma unroll
  for (int k = 0; k < OP_V; ++k) {
    own.a.v[k] = 1.0f;
    entered.v[k] = 0.0f;
  }
  if (latest >= 0) entered = entering(latest);
  own.b = entered;
  const unsigned long long live = latest >= 0 ? here >> latest << latest : here;
  shift_rows(zw);
  shift_rows(xw);
#pragma unroll
  for (int r = 0; r < OP_R; ++r) {
    if (!(live >> r & 1)) continue;
    const op_pair z = op_floats(zw[r]), x = op_floats(xw[r]);
#pragma unroll
    for (int k = 0; k < OP_V; ++k) {
      const op_gate g = op_gate_of(z.v[k]);
      own.a.v[k] *= g.keep;
      own.b.v[k] = OP_BACK ? g.keep * (x.v[k] + own.b.v[k]) : __builtin_fmaf(g.keep, own.b.v[k], g.take * x.v[k]);
    }
  }
#if OP_BACK
  /* (on their way while the tiles before are looked at) */
  unsigned int hw[OP_R], vw[OP_R];
  read_rows(p.h, p.h_stride, 1, hw);
  if (OP_GATE) read_rows(p.values, p.values_stride, 0, vw);
#endif
  maps[wave][lane] = own;
  if (lane == 0) ends[wave] = resets & 1 ? 2 : resets ? 1 : 0;
  __syncthreads();

  /* the waves' maps put together: up to this wave's, and of all */
  op_map mine, all;
  bool mine_ends = false, all_ends = false;
#pragma unroll
  for (int k = 0; k < OP_V; ++k) {
    all.a.v[k] = 1.0f;
    all.b.v[k] = 0.0f;
  }
  mine = all;
  float off = 0.0f;                                /* is not a number if one of the sums, or the product of all, is not finite */
  const bool fresh = __builtin_amdgcn_readfirstlane(ends[0]) == 2;
#pragma unroll
  for (int w = 0; w < OP_WAVES; ++w) {
    if (w == wave) {
      mine = all;
      mine_ends = all_ends;
    }
    const op_map m = maps[w][lane];
    const bool e = __builtin_amdgcn_readfirstlane(ends[w]) != 0;
#pragma unroll
    for (int k = 0; k < OP_V; ++k) {
      all.b.v[k] = e ? m.b.v[k] : __builtin_fmaf(m.a.v[k], all.b.v[k], m.b.v[k]);
      all.a.v[k] *= m.a.v[k];
    }
    all_ends = all_ends || e;
#pragma unroll
    for (int k = 0; k < OP_V; ++k) off = __builtin_fmaf(all.b.v[k], 0.0f, off);
  }
#pragma unroll
  for (int k = 0; k < OP_V; ++k) off = __builtin_fmaf(all.a.v[k], 0.0f, off);
  const unsigned long long off_lanes = __ballot(off != 0.0f);
  bool odd = off_lanes != 0;                       /* (of any channel: the waves go together) */
  const bool known = all_ends || tile == 0;
  __syncthreads();                                 /* (everybody has read them) */
  if (wave == 0 && !odd) {
    if (known) {
      op_put(op_words(p, tile, strip, 2, lane), p.tag, all.b);
    } else {
      op_put(op_words(p, tile, strip, 0, lane), p.tag, all.a);
      op_put(op_words(p, tile, strip, 1, lane), p.tag, all.b);
    }
  }

  /* What comes in.  Of the tiles in front the nearest OP_NEAR are looked at, a wave takes every eighth, until the nearest state among
   * them is followed by maps alone; those are applied to it one after the other.  (So a state is the same whoever has put it
   * together, to the last bit.)  If it is infinite on the way it is the state of the tile before that counts. */
  op_pair in;
#pragma unroll
  for (int k = 0; k < OP_V; ++k) in.v[k] = 0.0f;
  if (tile > 0 && !fresh) {
    int got[OP_NEAR / OP_WAVES];                   /* 0 nothing, 1 a map, 2 a state */
#pragma unroll
    for (int q = 0; q < OP_NEAR / OP_WAVES; ++q) got[q] = 0;
    int nearest = OP_NEAR;
    for (int polls = 0;;) {
#pragma unroll
      for (int q = 0; q < OP_NEAR / OP_WAVES; ++q) {
        const int n = q * OP_WAVES + wave, t = tile - 1 - n;
        if (t < 0 || (q > 0 && polls == 0)) {      /* (the nearest eight will often do) */
          if (lane == 0) ends[n] = 0;
          continue;
        }
        if (got[q] == 2) continue;
        op_map m;
        if (__ballot(!op_get(op_words(p, t, strip, 2, lane), p.tag, &m.b)) == 0) {
          got[q] = 2;
          maps[n][lane].b = m.b;
        } else if (got[q] == 0) {
          const bool a = op_get(op_words(p, t, strip, 0, lane), p.tag, &m.a), b = op_get(op_words(p, t, strip, 1, lane), p.tag, &m.b);
          if (__ballot(!a || !b) == 0) {
            got[q] = 1;
            maps[n][lane] = m;
          }
        }
        if (lane == 0) ends[n] = got[q];
      }
      __syncthreads();
      const int seen = lane < OP_NEAR && lane < tile ? ends[lane] : 0;
      const unsigned long long states = __ballot(seen == 2), nothing = __ballot(seen == 0);
      __syncthreads();
      nearest = __builtin_ctzll(states | 1ull << 63);
      if (nearest < __builtin_ctzll(nothing)) {    /* (lane 63 has seen nothing) */
        in = maps[nearest][lane].b;
        float most = op_largest(in, 0.0f);
        for (int left = nearest; left > 0; left -= 4) {        /* (four at a time, those that there are not change nothing) */
          op_map m[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) m[n] = maps[acc_max(left - 1 - n, 0)][lane];
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int k = 0; k < OP_V; ++k) {
              in.v[k] = n < left ? __builtin_fmaf(m[n].a.v[k], in.v[k], m[n].b.v[k]) : in.v[k];
              most = __builtin_fmaxf(most, __builtin_fabsf(in.v[k]));
            }
        }
        if (nearest == 0 || __ballot(most == __builtin_inff()) == 0) break;
        __syncthreads();                           /* (everybody has read them, and found the same) */
      }
      if (++polls >= ACC_SPIN_LIMIT) {
        if (tid == 0) acc_report(p.status, ACC_STATUS_SCAN_LOOKBACK);
        break;
      }
    }
    /* (where what comes in is not a number, neither is what goes out, whatever the map) */
    bool none = !all_ends;
#pragma unroll
    for (int k = 0; k < OP_V; ++k) none = none && in.v[k] != in.v[k];
    odd = (off_lanes & ~__ballot(none)) != 0 || __ballot(op_largest(in, 0.0f) == __builtin_inff()) != 0;
    if (wave == 0 && !known && !odd) {
      op_pair h;
#pragma unroll
      for (int k = 0; k < OP_V; ++k) h.v[k] = __builtin_fmaf(all.a.v[k], in.v[k], all.b.v[k]);
      op_put(op_words(p, tile, strip, 2, lane), p.tag, h);
    }
  }

  /* the results, sequence after sequence: what comes in, or what one that begins here enters with */
  op_pair h;
#pragma unroll
  for (int k = 0; k < OP_V; ++k) h.v[k] = odd ? in.v[k] : mine_ends ? mine.b.v[k] : __builtin_fmaf(mine.a.v[k], in.v[k], mine.b.v[k]);
#if OP_BACK
  shift_rows(hw);
  if (OP_GATE) shift_rows(vw);
#endif
  for (int turn = 0; turn < (odd ? OP_WAVES : 1); ++turn) {
    if (odd) {
      __syncthreads();
      if (turn != wave) continue;
      if (wave > 0) h = carried[lane];
    }
    for (int begin = 0; begin < OP_R;) {
      const unsigned long long more = resets & ~0ull << begin << 1;
      const int next = more ? __builtin_ctzll(more) : OP_R;
      const unsigned long long run = here & ~0ull << begin & ((1ull << next) - 1);
      if (resets >> begin & 1) {
        h = entered;
        if (begin != latest) h = entering(begin);
      }
      const int final = run & leaves ? __builtin_ctzll(run & leaves) : -1;
      const long long slot = final >= 0 ? op_slot(p, sequence_of(final)) : -1;
#if OP_BACK
      const op_pair started = op_state(p.state, p.state_stride, slot, channel, valid);
      op_elt *dgates = (op_elt *)p.dgates + (first + OP_R - 1) * p.dgates_stride, *dvalues = (op_elt *)p.dvalues + (first + OP_R - 1) * p.dvalues_stride;
      asm volatile("" : "+s"(dgates), "+s"(dvalues));      /* (or the rows' addresses are kept in registers from sequence to sequence) */
#else
      op_elt *out = (op_elt *)p.out + first * p.out_stride;
      asm volatile("" : "+s"(out));                        /* (or the rows' addresses are kept in registers from sequence to sequence) */
#endif
#pragma unroll
      for (int r = 0; r < OP_R; ++r) {
        if (run >> r & 1) {
          const op_pair z = op_again(zw[r]), x = op_again(xw[r]);
#if OP_BACK
          op_pair b = op_again(hw[r]), dz, dx;
          if (r == final) b = started;
#if OP_GATE
          const op_pair v = op_again(vw[r]);
#endif
#pragma unroll
          for (int k = 0; k < OP_V; ++k) {
            const op_gate g = op_gate_of(z.v[k]);
            const float d = x.v[k] + h.v[k];
            h.v[k] = g.keep * d;
#if OP_GATE
            dx.v[k] = g.take * d;
            dz.v[k] = (b.v[k] - v.v[k]) * (g.keep * dx.v[k]);
#else
            dx.v[k] = d;
            dz.v[k] = b.v[k] * d;
#endif
          }
          op_write(dgates, channel, whole, valid, dz);
          op_write(dvalues, channel, whole, valid, dx);
#else
#pragma unroll
          for (int k = 0; k < OP_V; ++k) {
            const op_gate g = op_gate_of(z.v[k]);
            h.v[k] = __builtin_fmaf(g.keep, h.v[k], g.take * x.v[k]);
          }
          op_write(out, channel, whole, valid, h);
#endif
        }
#if OP_BACK
        dgates -= p.dgates_stride;
        dvalues -= p.dvalues_stride;
#else
        out += p.out_stride;
#endif
      }
      if (final >= 0) op_keep(p.leave, p.leave_stride, slot, channel, valid, h);
      begin = next;
    }
    if (odd) {
      carried[lane] = h;
      if (wave == OP_WAVES - 1) op_put(op_words(p, tile, strip, 2, lane), p.tag, h);
    }
  }
  op_empty_sequences(p, rows, tile * OP_WAVES + wave, lane, channel, valid);
}

/* where tiles are drawn: no tile has left anything yet.  (The launches of a graph carry one tag.) */
extern "C" __global__ void __launch_bounds__(256) recur_clear(const acc_recur_args p)
{
  const long long words = (long long)p.tiles * p.strips * 3 * 64 * OP_V, i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i < words) p.words[i] = 0;
  if (i == 0) *p.ticket = 0u;
}
#endif
