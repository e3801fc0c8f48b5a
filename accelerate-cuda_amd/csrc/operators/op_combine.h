/*
 * op_combine.h -- the experts' rows of a token summed into one, and the gradient of that.
 *
 *   combine    out[t] = sum_j weights[t, j] y[place[t, j]]          (slots j in order, in Float32; place < 0: no row)
 *   gradient   dy[place[t, j]] = weights[t, j] dout[t],   dweights[t, j] = <dout[t], y[place[t, j]]>
 *
 * Bound by memory: every row goes by once.
 */
#include "op_common.h"

/* 8 elements as Float32 */
template <bool ALIGNED> ACC_DEV void op_load8(const op_elt *p, const int valid, float (&f)[8])
{
#pragma unroll
  for (int h = 0; h < 8 / OP_VALUES; ++h) {
    const acc_u4 v = op_chunk<ALIGNED>(p + h * OP_VALUES, valid - h * OP_VALUES);
    op_elt e[OP_VALUES];
    __builtin_memcpy(e, &v, 16);
#pragma unroll
    for (int k = 0; k < OP_VALUES; ++k) f[h * OP_VALUES + k] = (float)e[k];
  }
}
template <bool ALIGNED> ACC_DEV void op_store8(op_elt *p, const int valid, const float (&f)[8])
{
#pragma unroll
  for (int h = 0; h < 8 / OP_VALUES; ++h) {
    op_elt e[OP_VALUES];
    acc_u4 v;
#pragma unroll
    for (int k = 0; k < OP_VALUES; ++k) e[k] = (op_elt)f[h * OP_VALUES + k];
    __builtin_memcpy(&v, e, 16);
    const int left = valid - h * OP_VALUES;
    if (ALIGNED) {
      if (left > 0) *(acc_u4 *)(p + h * OP_VALUES) = v;
    } else if (left >= OP_VALUES) {
      ((op_loose<op_elt> *)(p + h * OP_VALUES))->v = v;
    } else {
#pragma unroll
      for (int k = 0; k < OP_VALUES; ++k)
        if (k < left) p[h * OP_VALUES + k] = e[k];
    }
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
  const long long n = (long long)blockIdx.x * 256 + threadIdx.x, t = n / pieces;
  if (t >= p.tokens) return;
  const int c = (int)(n % pieces) * 8;
  float sum[8] = {};
  for (int j = 0; j < p.choose; ++j) {
    const long long r = op_row(p, t * p.choose + j);
    if (r < 0) continue;
    const float w = p.weights ? p.weights[t * p.choose + j] : 1.0f;
    float f[8];
    op_load8<OP_ALIGNED>((const op_elt *)p.y + r * p.y_stride + c, p.width - c, f);
#pragma unroll
    for (int k = 0; k < 8; ++k) sum[k] += w * f[k];
  }
  op_store8<OP_ALIGNED>((op_elt *)p.out + t * p.out_stride + c, p.width - c, sum);
}

/* a wave has a token: dout goes by once for every OP_SLOTS slots */
extern "C" __global__ void __launch_bounds__(256) combine_gradient(const acc_combine_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const int lane = threadIdx.x & 63;
  const long long t = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= p.tokens) return;
  for (int first = 0; first < p.choose; first += OP_SLOTS) {
    long long r[OP_SLOTS];
    float w[OP_SLOTS], dot[OP_SLOTS];
#pragma unroll
    for (int j = 0; j < OP_SLOTS; ++j) {
      const long long s = t * p.choose + first + j;
      r[j] = first + j < p.choose ? op_row(p, s) : -1;
      w[j] = r[j] < 0 ? 0.0f : p.weights ? p.weights[s] : 1.0f;
      dot[j] = 0.0f;
    }
    for (int c = lane * 8; c < p.width; c += 512) {
      float d[8];
      op_load8<OP_ALIGNED>((const op_elt *)p.dout + t * p.dout_stride + c, p.width - c, d);
#pragma unroll
      for (int j = 0; j < OP_SLOTS; ++j) {
        if (r[j] < 0) continue;
        float f[8], g[8];
        if (p.dweights) op_load8<OP_ALIGNED>((const op_elt *)p.y + r[j] * p.y_stride + c, p.width - c, f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (p.dweights) dot[j] += d[k] * f[k];
          g[k] = w[j] * d[k];
        }
        op_store8<OP_ALIGNED>((op_elt *)p.out + r[j] * p.out_stride + c, p.width - c, g);
      }
    }
    if (p.dweights) {
#pragma unroll
      for (int j = 0; j < OP_SLOTS; ++j) {
        const float all = acc_wave_reduce(dot[j], [](float x, float y) { return x + y; });
        if (lane == 0 && first + j < p.choose) p.dweights[t * p.choose + first + j] = r[j] < 0 ? 0.0f : all;
      }
    }
  }
}
