/*
 * op_combine.h -- the experts' rows of a token summed into one, and the gradient of that.
 *
 *   combine    out[t] = sum_j weights[t, j] y[place[t, j]]          (slots j in order, in Float32; place < 0: no row)
 *   gradient   dy[place[t, j]] = weights[t, j] dout[t],   dweights[t, j] = <dout[t], y[place[t, j]]>
 *
 * Bound by memory: every row goes by once.  What keeps it from that bound is waiting, so a lane has the rows of OP_SLOTS slots on
 * their way at once, and no branch turns a load's result into Float32 before the next load is out.  Of 4097 tokens with 6 slots and
 * 1501 bfloat16 columns: combine 21 us (24 with one row at a time), its gradient 40 (44 with a slot's place and weight read in front
 * of its rows; 160 MB, 4.0 TB/s); of 16384 tokens with 8 slots and 2048 columns 120 and 233 us, 5.0 and 4.9 TB/s.
 */
#include "op_common.h"

/* Where a lane's eight columns begin that are the c-th of its row: in rows that end amid eight, the last eight begin earlier, and
 * `skip` of them are the lane's before, too (they are written twice, with the same values, and no access goes past the row).
 * OP_TINY: a row has fewer than eight. */
ACC_DEV int op_eight(const int c, const int width, int *skip)
{
  const int at = OP_ALIGNED || OP_TINY ? c : acc_min(c, width - 8);
  *skip = c - at;
  return at;
}

/* 8 elements, of which `valid` are the row's (all of them, but for OP_TINY) */
struct op_raw8 { acc_u4 v[8 / OP_VALUES]; };
ACC_DEV op_raw8 op_load8(const op_elt *p, const int valid)
{
  op_raw8 r;
#pragma unroll
  for (int h = 0; h < 8 / OP_VALUES; ++h) {
    if (OP_ALIGNED)
      r.v[h] = ((const acc_u4 *)p)[h];
    else
      r.v[h] = op_chunk<false>(p + h * OP_VALUES, OP_TINY ? valid - h * OP_VALUES : OP_VALUES);
  }
  return r;
}
ACC_DEV void op_floats(const op_raw8 &r, float (&f)[8])
{
  op_elt e[8];
  __builtin_memcpy(e, &r, sizeof e);
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = (float)e[k];
}
ACC_DEV void op_store8(op_elt *p, const int valid, const float (&f)[8])
{
  op_elt e[8];
  op_raw8 r;
#pragma unroll
  for (int k = 0; k < 8; ++k) e[k] = (op_elt)f[k];
  __builtin_memcpy(&r, e, sizeof e);
  if (OP_TINY) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < valid) p[k] = e[k];
    return;
  }
#pragma unroll
  for (int h = 0; h < 8 / OP_VALUES; ++h) {
    if (OP_ALIGNED)
      ((acc_u4 *)p)[h] = r.v[h];
    else
      ((op_loose<op_elt> *)(p + h * OP_VALUES))->v = r.v[h];
  }
}

/* a slot's row, or -1 */
ACC_DEV long long op_row(const acc_combine_args &p, const long long slot)
{
  const int at = p.place[slot];
  return at >= 0 && at < p.y_rows ? at : -1;
}

/* a lane has 8 columns of a token */
extern "C" __global__ void __launch_bounds__(256) combine(const acc_combine_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const int pieces = (p.width + 7) / 8;
  const unsigned int n = blockIdx.x * 256 + threadIdx.x, t = p.per_mul ? __umulhi(n, p.per_mul) >> p.per_shift : n;
  if (t >= p.tokens) return;
  int skip;
  const int c = op_eight((int)(n - t * pieces) * 8, p.width, &skip);
  float sum[8] = {};
  for (int first = 0; first < p.choose; first += OP_SLOTS) {         /* OP_SLOTS rows on their way at once */
    long long r[OP_SLOTS];
    float w[OP_SLOTS];
    op_raw8 y[OP_SLOTS];
#pragma unroll
    for (int j = 0; j < OP_SLOTS; ++j) {
      const long long s = (long long)t * p.choose + acc_min(first + j, p.choose - 1);
      r[j] = op_row(p, s);
      w[j] = p.weights ? p.weights[s] : 1.0f;
    }
#pragma unroll
    for (int j = 0; j < OP_SLOTS; ++j) {
      if (first + j >= p.choose) r[j] = -1;
      y[j] = {};
      if (r[j] >= 0) y[j] = op_load8((const op_elt *)p.y + r[j] * p.y_stride + c, p.width - c);
    }
#pragma unroll
    for (int j = 0; j < OP_SLOTS; ++j) {
      float f[8];
      op_floats(y[j], f);
      if (r[j] < 0) w[j] = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] += w[j] * f[k];
    }
  }
  op_store8((op_elt *)p.out + t * p.out_stride + c, p.width - c, sum);
}

/* A workgroup has a token, a wave 512 of its columns at a time (a wave with a whole token: 267 us where this takes 233).  The lanes
 * read 64 slots' places and weights at once; dout goes by once for every OP_SLOTS slots, and a slot without a row asks for dout's
 * again. */
extern "C" __global__ void __launch_bounds__(256) combine_gradient(const acc_combine_args p)
{
  __shared__ float part[4][OP_SLOTS];
  if (p.guard && *p.guard == 0u) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const long long t = blockIdx.x;
  const op_elt *const dout = (const op_elt *)p.dout + t * p.dout_stride;
  int place = -1;                                                    /* of 64 slots, one a lane */
  unsigned int weight = __float_as_uint(1.0f);
  for (int first = 0; first < p.choose; first += OP_SLOTS) {
    if (first % 64 == 0) {
      const bool slot = first + lane < p.choose;
      place = slot ? p.place[t * p.choose + first + lane] : -1;
      if (slot && p.weights) weight = __float_as_uint(p.weights[t * p.choose + first + lane]);
      if (place >= p.y_rows) place = -1;
    }
    int r[OP_SLOTS];
    float w[OP_SLOTS], dot[OP_SLOTS];
#pragma unroll
    for (int j = 0; j < OP_SLOTS; ++j) {
      r[j] = __builtin_amdgcn_readlane(place, (first + j) % 64);
      w[j] = __uint_as_float(__builtin_amdgcn_readlane(weight, (first + j) % 64));
      dot[j] = 0.0f;
    }
    for (int at = threadIdx.x * 8; at < p.width; at += waves * 512) {
      int skip;
      const int c = op_eight(at, p.width, &skip);
      const op_raw8 draw = op_load8(dout + c, p.width - c);
      op_raw8 y[OP_SLOTS];
      if (p.dweights)
#pragma unroll
        for (int j = 0; j < OP_SLOTS; ++j) y[j] = op_load8((r[j] < 0 ? dout : (const op_elt *)p.y + (long long)r[j] * p.y_stride) + c, p.width - c);
      float d[8], own[8];
      op_floats(draw, d);
#pragma unroll
      for (int k = 0; k < 8; ++k) own[k] = k < skip ? 0.0f : d[k];
#pragma unroll
      for (int j = 0; j < OP_SLOTS; ++j) {
        if (r[j] < 0) continue;
        float g[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] = w[j] * d[k];
        op_store8((op_elt *)p.out + (long long)r[j] * p.out_stride + c, p.width - c, g);
      }
      if (p.dweights)
#pragma unroll
        for (int j = 0; j < OP_SLOTS; ++j) {
          float f[8];
          op_floats(y[j], f);
          if (skip > 0)
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = k < skip ? 0.0f : f[k];
#pragma unroll
          for (int k = 0; k < 8; ++k) dot[j] += own[k] * f[k];
        }
    }
    if (!p.dweights) continue;
#pragma unroll
    for (int j = 0; j < OP_SLOTS; ++j) {
      const float all = acc_wave_reduce(dot[j], [](float x, float y) { return x + y; });
      if (lane == 0) part[wave][j] = r[j] < 0 ? 0.0f : all;
    }
    __syncthreads();
    const int j = threadIdx.x;
    if (j < OP_SLOTS && first + j < p.choose) {
      float all = 0.0f;
      for (int i = 0; i < waves; ++i) all += part[i][j];
      p.dweights[t * p.choose + first + j] = all;
    }
    __syncthreads();
  }
}
