/*
 * op_grouped.h -- matrices of 4-bit whole numbers, neighbours of a row in groups under a scale and a zero:
 *
 *   w[e, n, k] = (q[e, n, k] - z[e, g, n]) s[e, g, n],   g = k / group;   z = 8 where there are no zeros
 *   out[m, n]  = sum_k x[r(m), k] w[e(m), n, k]          for a few rows of each matrix
 *
 * The products are taken of the numbers as they are: a code's four bits are the mantissa's first, of 16 + q (exact in both 16-bit
 * types), the matrix cores add up x (16 + q) and x alone over what a group has of a step, and then
 *
 *   sum += s (sum x (16 + q)) - s (16 + z) (sum x)
 *
 * in Float32: no weight is ever rounded.  What is taken off again is 16 to 31 times a row's sum at most, of whose 24 bits it costs
 * two or three beside the 4-bit numbers' own.  Float32 rows are cut into three bfloat16 each, which hold all 24 bits.  (An infinity
 * in a row makes the row's results NaN.)
 *
 * What counts is that the matrices pass by once.  A lane loads 16 bytes of codes, 32 numbers of a row, straight into registers,
 * OP_AHEAD steps of 128 numbers of k at a time; four lanes then exchange words so that a fragment is 32 neighbours of one
 * group.  The eight waves of a workgroup take every eighth step of the same 16 OP_FN columns and add up what they have by way of
 * LDS, in order.
 */
#include "op_matrix.h"

#define OP_FM (OP_BM / 16)
#define OP_WAVES 8

#if OP_TYPE == 1
#define OP_SIXTEEN 0x4C004C00u
#define OP_FOUR_BITS 0x03C003C0u
#define OP_ONES 0x3C003C00u
#define OP_UP 6                                    /* where a number of the low bits goes */
#else
#define OP_SIXTEEN 0x41804180u
#define OP_FOUR_BITS 0x00780078u
#define OP_ONES 0x3F803F80u
#define OP_UP 3
#endif

/* 8 codes as 16 + q: of neighbours 0 4, 1 5, 2 6, 3 7 */
ACC_DEV acc_u4 op_sixteens(const unsigned int w)
{
  const auto at = [](const unsigned int v) { return (v & OP_FOUR_BITS) | OP_SIXTEEN; };
  return acc_u4{at(w << OP_UP), at(OP_UP >= 4 ? w << (OP_UP - 4) : w >> (4 - OP_UP)), at(w >> (8 - OP_UP)), at(w >> (12 - OP_UP))};
}

/* a row's 8 neighbours in that order, in OP_PARTS parts that add up to them */
#if OP_ELT == 0
#define OP_PARTS 3
#else
#define OP_PARTS 1
#endif
struct op_eight { acc_u4 v[OP_ELT == 0 ? 2 : 1]; };
ACC_DEV void op_parts(const op_eight &x, acc_u4 (&to)[OP_PARTS])
{
#if OP_ELT == 0
  unsigned int f[8];
  __builtin_memcpy(f, &x, 32);
#pragma unroll
  for (int part = 0; part < OP_PARTS; ++part) {
#pragma unroll
    for (int k = 0; k < 4; ++k) to[part][k] = __builtin_amdgcn_perm(f[k + 4], f[k], 0x07060302u);
    if (part + 1 < OP_PARTS)
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = __float_as_uint(__uint_as_float(f[k]) - __uint_as_float(f[k] & 0xffff0000u));
  }
#else
  const acc_u4 v = x.v[0];
  to[0] = acc_u4{__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u), __builtin_amdgcn_perm(v.w, v.y, 0x05040100u),
                 __builtin_amdgcn_perm(v.w, v.y, 0x07060302u)};
#endif
}
ACC_DEV op_frag op_as_frag(const acc_u4 &v)
{
  op_frag f;
  __builtin_memcpy(&f, &v, 16);
  return f;
}

/* `valid` of a row's elements from p on, zeros behind them */
ACC_DEV op_eight op_row8(const op_elt *p, const int valid)
{
  op_eight x;
#pragma unroll
  for (int h = 0; h < 8 / OP_VALUES; ++h) x.v[h] = op_chunk<false>(p + h * OP_VALUES, valid - h * OP_VALUES);
  return x;
}

/* four lanes' words w[f] of numbers 32 g + 8 f on: w[b] becomes those of 32 b + 8 g on */
ACC_DEV void op_turn(acc_u4 &w)
{
  const auto a = __builtin_amdgcn_permlane32_swap(w.x, w.z, false, false), b = __builtin_amdgcn_permlane32_swap(w.y, w.w, false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  w = acc_u4{c[0], c[1], d[0], d[1]};
}

/* four neighbours of a row of scales (or zeros), of which the last ones may not be there */
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) op_e4 { T v[4]; };
template <typename T> ACC_DEV op_e4<T> op_four(const T *p, const int at, const int end)
{
  if (at + 4 <= end) return *(const op_e4<T> *)(p + at);
  op_e4<T> e;
#pragma unroll
  for (int t = 0; t < 4; ++t) e.v[t] = p[acc_min(at + t, end - 1)];
  return e;
}

#if OP_ELEMENTS
/* A team of lanes has a group, a lane eight of its numbers at a time; what a row's last group has too many counts as zeros.  (Once for
 * a matrix: the rows are read twice.) */
extern "C" __global__ void __launch_bounds__(256) grouped_quantise(const acc_grouped_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const int team = acc_min(64, p.group / 8), lane = (int)threadIdx.x % team;
  const long long n = ((long long)blockIdx.x * 256 + threadIdx.x) / team, rows = (long long)p.experts * p.nj;
  const bool here = n < rows * p.groups;
  const long long row = here ? n / p.groups : 0, e = row / p.nj, j = row % p.nj;
  const int g = here ? (int)(n % p.groups) : 0, first = g * p.group, end = acc_min(p.k, first + p.group);
  const op_elt *const w = (const op_elt *)p.w + e * p.w_expert + j * p.w_stride;
  float low = 0.0f, high = 0.0f;
  int bad = 0;
  for (int k = first + lane * 8; k < end; k += team * 8)
    for (int i = k; i < acc_min(k + 8, end); ++i) {
      const float v = (float)w[i];
      low = v < low ? v : low;
      high = v > high ? v : high;
      bad |= !(__builtin_fabsf(v) < __builtin_inff());
    }
  for (int apart = 1; apart < team; apart *= 2) {
    const int other = (acc_lane() ^ apart) * 4;
    const float l = __uint_as_float(__builtin_amdgcn_ds_bpermute(other, __float_as_uint(low))), h = __uint_as_float(__builtin_amdgcn_ds_bpermute(other, __float_as_uint(high)));
    low = l < low ? l : low;
    high = h > high ? h : high;
    bad |= __builtin_amdgcn_ds_bpermute(other, bad);
  }
  if (!here) return;
  /* (divisions as IEEE has them: a number between two codes is rounded the same way wherever this is computed) */
  const op_elt kept = (op_elt)(p.zeros ? (high - low) / 15.0f : (high > -low ? high : -low) / 7.0f);
  const float scale = (float)kept;
  bad |= !(scale < __builtin_inff());
  const float zero = p.zeros ? (scale > 0.0f ? acc_min(acc_max(__builtin_rintf(-low / scale), 0.0f), 15.0f) : 0.0f) : 8.0f;
  unsigned char *const codes = (unsigned char *)p.codes + e * p.codes_expert + j * p.codes_stride;
  for (int k = first + lane * 8; k < acc_min(first + p.group, p.blocks * 32); k += team * 8) {
    unsigned int word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = k + i < end ? (float)w[k + i] : 0.0f, q = scale > 0.0f && !bad ? __builtin_rintf(v / scale) : 0.0f;
      word |= (unsigned int)acc_min(acc_max(q + zero, 0.0f), 15.0f) << 4 * i;
    }
    *(unsigned int *)(codes + k / 2) = word;
  }
  if (lane != 0) return;
  ((op_elt *)p.scales)[e * p.scales_expert + g * p.scales_stride + j] = bad ? (op_elt)__builtin_nanf("") : kept;
  if (p.zeros) ((unsigned char *)p.zeros)[e * p.zeros_expert + g * p.zeros_stride + j] = (unsigned char)zero;
}

/* a lane has eight numbers */
extern "C" __global__ void __launch_bounds__(256) grouped_values(const acc_grouped_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const long long n = (long long)blockIdx.x * 256 + threadIdx.x, row = n / (p.blocks * 4);
  if (row >= (long long)p.experts * p.nj) return;
  const long long e = row / p.nj, j = row % p.nj;
  const int k = (int)(n % (p.blocks * 4)) * 8, g = k / p.group, left = p.k - k;
  const unsigned int word = *(const unsigned int *)((const unsigned char *)p.codes + e * p.codes_expert + j * p.codes_stride + k / 2);
  const float scale = (float)((const op_elt *)p.scales)[e * p.scales_expert + g * p.scales_stride + j];
  const float zero = p.zeros ? (float)((const unsigned char *)p.zeros)[e * p.zeros_expert + g * p.zeros_stride + j] : 8.0f;
  op_elt v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (op_elt)(((float)(word >> 4 * i & 15u) - zero) * scale);
  op_elt *const out = (op_elt *)p.out + e * p.out_expert + j * p.out_stride + k;
  if (left >= 8) {
    acc_u4 u[8 / OP_VALUES];
    __builtin_memcpy(u, v, sizeof(v));
#pragma unroll
    for (int h = 0; h < 8 / OP_VALUES; ++h) ((op_loose<op_elt> *)(out + h * OP_VALUES))->v = u[h];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) out[i] = v[i];
  }
}
#else

#define OP_CHUNKS (OP_GROUP >= 4 ? 1 : 4 / OP_GROUP)        /* groups of a step (OP_GROUP: blocks of 32 of a group, 4: or more) */
struct op_step {
  acc_u4 w[OP_FN];
  op_eight x[OP_FM][4];
  op_e4<op_elt> s[OP_CHUNKS][OP_FN];
  op_e4<unsigned char> z[OP_CHUNKS][OP_FN];
};

extern "C" __global__ void __launch_bounds__(64 * OP_WAVES) grouped(const acc_grouped_args p)
{
  if (p.guard && *p.guard == 0u) return;
  __shared__ acc_f4 parts[OP_WAVES - 1][OP_FM * OP_FN][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l = lane & 15, g = lane >> 4;
  const op_tile tile = op_find_tile<OP_ALL>(p.offsets, p.experts, (int)p.rows, OP_BM, op_segments(p.offsets, p.experts, (int)p.rows, 0, 0), (int)(blockIdx.x / p.tiles_j));
  if (tile.begin >= tile.end) return;
  const int j0 = (int)(blockIdx.x % p.tiles_j) * 16 * OP_FN;

  acc_f4 c[OP_FM][OP_FN];
#pragma unroll
  for (int i = 0; i < OP_FM; ++i)
#pragma unroll
    for (int j = 0; j < OP_FN; ++j) c[i][j] = acc_f4{0.0f, 0.0f, 0.0f, 0.0f};
  int arow[OP_FM];
#pragma unroll
  for (int i = 0; i < OP_FM; ++i) {
    const int m = tile.begin + i * 16 + l;
    arow[i] = p.index ? op_listed(p.index, m, tile.begin, tile.end, p.x_rows, p.per_mul, p.per_shift) : m < tile.end ? m : -1;
  }
  if (tile.expert >= 0 && p.x_rows > 0) {
    /* (rows that there are not are read as the first one, and columns as the last: what comes of them is not written) */
    const unsigned char *w[OP_FN];
    const op_elt *x[OP_FM], *const scales = (const op_elt *)p.scales + tile.expert * p.scales_expert;
    const unsigned char *const zeros = (const unsigned char *)p.zeros + tile.expert * p.zeros_expert;
#pragma unroll
    for (int j = 0; j < OP_FN; ++j) w[j] = (const unsigned char *)p.codes + tile.expert * p.codes_expert + (long long)acc_min(j0 + j * 16 + l, p.nj - 1) * p.codes_stride;
#pragma unroll
    for (int i = 0; i < OP_FM; ++i) x[i] = (const op_elt *)p.x + (long long)acc_max(arow[i], 0) * p.x_stride;
    const int steps = (p.blocks + 3) / 4;
    const auto load = [&](const int n, op_step &s) {
      const int k = n * 128;
#pragma unroll
      for (int j = 0; j < OP_FN; ++j) s.w[j] = __builtin_nontemporal_load((const acc_u4 *)(w[j] + acc_min(n * 4 + g, p.blocks - 1) * 16));
#pragma unroll
      for (int q = 0; q < OP_CHUNKS; ++q) {
        const int at = acc_min((k + q * (128 / OP_CHUNKS)) >> p.group_shift, p.groups - 1);
#pragma unroll
        for (int j = 0; j < OP_FN; ++j) {
          s.s[q][j] = op_four(scales + at * p.scales_stride, j0 + j * 16 + g * 4, p.nj);
          if (p.zeros) s.z[q][j] = op_four(zeros + at * p.zeros_stride, j0 + j * 16 + g * 4, p.nj);
        }
      }
      if (k + 128 <= p.k) {
#pragma unroll
        for (int i = 0; i < OP_FM; ++i)
#pragma unroll
          for (int b = 0; b < 4; ++b) s.x[i][b] = op_row8(x[i] + k + b * 32 + g * 8, 8);
      } else {
#pragma unroll
        for (int i = 0; i < OP_FM; ++i)
#pragma unroll
          for (int b = 0; b < 4; ++b) s.x[i][b] = op_row8(x[i] + k + b * 32 + g * 8, p.k - k - b * 32 - g * 8);
      }
    };
    const auto add = [&](op_step &s) {
      const acc_f4 none = {0.0f, 0.0f, 0.0f, 0.0f};
      const op_frag ones = op_as_frag(acc_u4{OP_ONES, OP_ONES, OP_ONES, OP_ONES});
#pragma unroll
      for (int j = 0; j < OP_FN; ++j) op_turn(s.w[j]);
#pragma unroll
      for (int q = 0; q < OP_CHUNKS; ++q) {
        acc_f4 t[OP_FM][OP_FN], sum[OP_FM];
#pragma unroll
        for (int i = 0; i < OP_FM; ++i) {
          sum[i] = none;
#pragma unroll
          for (int j = 0; j < OP_FN; ++j) t[i][j] = none;
        }
#pragma unroll
        for (int b = q * 4 / OP_CHUNKS; b < (q + 1) * 4 / OP_CHUNKS; ++b) {
          op_frag v[OP_FN];
#pragma unroll
          for (int j = 0; j < OP_FN; ++j) v[j] = op_as_frag(op_sixteens(s.w[j][b]));
#pragma unroll
          for (int i = 0; i < OP_FM; ++i) {
            acc_u4 part[OP_PARTS];
            op_parts(s.x[i][b], part);
#pragma unroll
            for (int n = OP_PARTS - 1; n >= 0; --n) {
              const op_frag y = op_as_frag(part[n]);
              sum[i] = op_mfma(ones, y, sum[i]);
#pragma unroll
              for (int j = 0; j < OP_FN; ++j) t[i][j] = op_mfma(v[j], y, t[i][j]);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < OP_FN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float scale = (float)s.s[q][j].v[r], off = scale * (16.0f + (p.zeros ? (float)s.z[q][j].v[r] : 8.0f));
#pragma unroll
            for (int i = 0; i < OP_FM; ++i) c[i][j][r] += __builtin_fmaf(scale, t[i][j][r], -off * sum[i][r]);
          }
      }
    };
    for (int n = wave; n < steps; n += OP_WAVES * OP_AHEAD) {
      op_step s[OP_AHEAD];
#pragma unroll
      for (int u = 0; u < OP_AHEAD; ++u)
        if (n + u * OP_WAVES < steps) load(n + u * OP_WAVES, s[u]);
      __builtin_amdgcn_sched_barrier(0);           /* (all loads first) */
#pragma unroll
      for (int u = 0; u < OP_AHEAD; ++u)
        if (n + u * OP_WAVES < steps) add(s[u]);
    }
  }

  if (wave > 0)
#pragma unroll
    for (int i = 0; i < OP_FM; ++i)
#pragma unroll
      for (int j = 0; j < OP_FN; ++j) parts[wave - 1][i * OP_FN + j][lane] = c[i][j];
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int i = 0; i < OP_FM; ++i) {
    const int m = tile.begin + i * 16 + l;
#pragma unroll
    for (int j = 0; j < OP_FN; ++j)
#pragma unroll
      for (int w = 0; w < OP_WAVES - 1; ++w) c[i][j] += parts[w][i * OP_FN + j][lane];
    if (m >= tile.end) continue;
    op_elt *out = (op_elt *)p.out + (long long)m * p.out_stride;
#pragma unroll
    for (int j = 0; j < OP_FN; ++j) op_write4(out, j0 + j * 16 + 4 * g, p.nj, c[i][j], arow[i] < 0 || tile.expert < 0);
  }
}
#endif
