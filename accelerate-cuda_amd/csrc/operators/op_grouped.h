/*
 * op_grouped.h -- matrices of 4-bit whole numbers, neighbours of a row in groups under a scale and a zero:
 *
 *   w[e, n, k] = (q[e, n, k] - z[e, g, n]) s[e, g, n],   g = k / group;   z = 8 where there are no zeros
 *   out[m, n]  = sum_k x[r(m), k] w[e(m), n, k]          for a few rows of each matrix
 *
 * The products are taken of the numbers as they are: a code's four bits become the highest of the mantissa of 16 + q, exact in either
 * 16-bit type; the matrix cores add up x (16 + q) over what a group has of a step, beginning with -(z + 16) sum x, and that times s is
 * added up in Float32: no weight is ever rounded.  What is taken off again costs two or three of the 24 bits of a sum, more where a
 * row's numbers share a sign and the sums of x (q - z) are small beside sum x: half rows of one sign, 4096 numbers in groups of 128, are
 * 5.3e-6 off before the result is rounded.  (With the codes at the end of the mantissa, 1024 + q and 64 + q, such rows were 1.4e-4
 * off, and calls no faster for want of three shifts: 64 rows, 16 of 4096 x 2048: 23.4 us and 23.3 as here; 2048, 8 of 4096 x 4096: 131 and 119.) Float32 rows are cut into three bfloat16 each, which hold all 24 bits;
 * the first parts, 8 bits each, are added up and what is too much of them taken off before the others come, which is exact or nearly so
 * (150 rows of 12 matrices of 1333 x 1001 in groups of 32, 21 us: 1.2e-7 off; all at once 6e-7, and up to 1.4e-6 at other sizes).  (An infinity in a row makes the row's results NaN.)
 *
 * What counts is that the matrices pass by once, and that their codes are nearly all that is read.  A lane loads 16 bytes of them, 32
 * numbers of a row.  Where a matrix has many columns for a compute unit, the rows lie in LDS and waves go over the columns (OP_STREAM);
 * where it has few, what counts is how soon all of it is on its way, and the waves of a workgroup take every so many steps of the same
 * 16 OP_FN columns and add up what they have by way of LDS, in order.  64 half rows, 16 matrices of 4096 x 2048 in groups of 64 with
 * zeros: 22 us, of which the codes' loads alone take 13 (5.8 TB/s), what is in front of them 8 with the launch; bfloat16 in groups of 128,
 * 16 rows, 8 of 4096 x 4096: 21 us; 1 row, 1 of 4096 x 4096: 6.4.  Many rows are matter for the matrix cores (OP_WIDE).
 */
#include "op_matrix.h"

#define OP_FM (OP_BM / 16)

/* a constant in a register of the lanes' (an instruction takes one of two constants only from elsewhere, and "and, or" is one then) */
ACC_DEV unsigned int op_lane_word(unsigned int v)
{
  asm("" : "+v"(v));
  return v;
}
/* 8 codes as OP_D + q, in 16 bits each: of neighbours 0 4, 1 5, 2 6, 3 7 */
#define OP_D 16.0f
#if OP_ELT == 1
#define OP_ONES 0x3C003C00u
ACC_DEV acc_u4 op_numbers(const unsigned int w)
{
  const unsigned int d = op_lane_word(0x4C004C00u);
  const auto at = [d](const unsigned int v) { return (v & 0x03C003C0u) | d; };
  return acc_u4{at(w << 6), at(w << 2), at(w >> 2), at(w >> 6)};
}
#else
#define OP_ONES 0x3F803F80u
ACC_DEV acc_u4 op_numbers(const unsigned int w)
{
  const unsigned int d = op_lane_word(0x41804180u);
  const auto at = [d](const unsigned int v) { return (v & 0x00780078u) | d; };
  return acc_u4{at(w << 3), at(w >> 1), at(w >> 5), at(w >> 9)};
}
#endif

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

/* Four lanes have words w[f] of numbers 32 g + 8 f on.  Where a step has one group that is as good an order as any; where it has
 * several, w[b] becomes those of 32 b + 8 g on.  OP_FIRST: the first number of a lane's b-th word. */
#define OP_CHUNKS (OP_GROUP >= 4 ? 1 : 4 / OP_GROUP)        /* groups of a step (OP_GROUP: blocks of 32 of a group, 4: or more) */
#define OP_BLOCKS (4 / OP_CHUNKS)                  /* words of a group in a step */
#define OP_FIRST(b, g) (OP_CHUNKS > 1 ? 32 * (b) + 8 * (g) : 32 * (g) + 8 * (b))
ACC_DEV void op_turn(acc_u4 &w)
{
  if (OP_CHUNKS == 1) return;
  const auto a = __builtin_amdgcn_permlane32_swap(w.x, w.z, false, false), b = __builtin_amdgcn_permlane32_swap(w.y, w.w, false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false), d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  w = acc_u4{c[0], c[1], d[0], d[1]};
}

/* four neighbours of a row of scales (or zeros); `whole`: they are all there, in every lane */
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) op_e4 { T v[4]; };
template <typename T> ACC_DEV op_e4<T> op_four(const T *p, const bool whole, const int at, const int end)
{
  if (whole) return *(const op_e4<T> *)(p + at);
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
  const long long n = (p.first + (long long)blockIdx.x * 256 + threadIdx.x) / team, rows = (long long)p.experts * p.nj;
  const bool here = n < rows * p.groups;
  const long long row = here ? n / p.groups : 0, e = row / p.nj, j = row % p.nj;
  const int g = here ? (int)(n % p.groups) : 0, first = g * p.group, end = acc_min(p.k, first + p.group);
  const op_elt *const w = (const op_elt *)p.w + e * p.w_expert + j * p.w_stride;
  float low = 0.0f, high = 0.0f;
  int bad = 0;
  for (int k = first + lane * 8; k < end; k += team * 8) {
    const op_eight x = op_row8(w + k, end - k);
    op_elt e[8];
    __builtin_memcpy(e, &x, sizeof(e));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = (float)e[i];
      low = v < low ? v : low;
      high = v > high ? v : high;
      bad |= !(__builtin_fabsf(v) < __builtin_inff());
    }
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
  const float range = high - low < __builtin_inff() ? (high - low) / 15.0f : (high * 0.0625f - low * 0.0625f) / 15.0f * 16.0f;
  const op_elt kept = (op_elt)(p.zeros ? range : (high > -low ? high : -low) / 7.0f);
  const float scale = (float)kept;
  bad |= !(scale < __builtin_inff());
  const float zero = p.zeros ? (scale > 0.0f ? acc_min(acc_max(__builtin_rintf(-low / scale), 0.0f), 15.0f) : 0.0f) : 8.0f;
  unsigned char *const codes = (unsigned char *)p.codes + e * p.codes_expert + j * p.codes_stride;
  for (int k = first + lane * 8; k < acc_min(first + p.group, p.blocks * 32); k += team * 8) {
    const op_eight x = op_row8(w + k, end - k);
    op_elt e[8];
    __builtin_memcpy(e, &x, sizeof(e));
    unsigned int word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float v = (float)e[i], q = scale > 0.0f && !bad ? __builtin_rintf(v / scale) : 0.0f;
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
  const long long n = p.first + (long long)blockIdx.x * 256 + threadIdx.x, row = n / (p.blocks * 4);
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

/* what products of a group begin with */
ACC_DEV float op_begin(const float sum, const float zero) { return -(zero + OP_D) * sum; }

/* the sums behind that, of 16 rows: sum x, of Float32 ones that of the first part, and of the other parts in `second` */
template <typename F> ACC_DEV void op_sums(const int q, F fragment, acc_f4 &sum, acc_f4 &second)
{
  const op_frag ones = op_as_frag(acc_u4{OP_ONES, OP_ONES, OP_ONES, OP_ONES});
  sum = second = acc_f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int b = q * OP_BLOCKS; b < (q + 1) * OP_BLOCKS; ++b) {
    sum = op_mfma(ones, fragment(b, 0), sum);
#pragma unroll
    for (int part = OP_PARTS - 1; part > 0; --part) second = op_mfma(ones, fragment(b, part), second);
  }
}
/* of Float32 rows: the other parts' beginning, behind their products */
ACC_DEV float op_rest(const float t, const float second, const float zero) { return OP_ELT == 0 ? __builtin_fmaf(-(zero + OP_D), second, t) : t; }

#if OP_STREAM
/* The form whose rows lie in LDS, cut and in the order of fragments, with their sums by groups: p.height rows of a tile (a power of
 * two up to 16, or 16 OP_FM).  A wave goes over columns, 16 at a time, or over a part of k of the same columns as its neighbours where
 * there are few (p.split of them, whose sums then meet in LDS).  It takes OP_AHEAD steps at a time while the codes of the next ones
 * are on their way; their scales and zeros, of 16 columns, are a load of 16 bytes in as many lanes as it takes, and go round by way of
 * LDS (asked for by every lane that wants them they cost more of the cache's time than the codes).  No load is behind a branch, so that
 * what is on its way can be counted: steps and columns that there are not are read as the last ones. */
#define OP_NOTED (OP_AHEAD * OP_CHUNKS)            /* groups of so many steps */
#define OP_SIZE ((int)sizeof(op_elt))              /* lanes of a group's 16 scales; one has its zeros */

extern "C" __global__ void __launch_bounds__(64 * OP_WAVES) grouped(const acc_grouped_args p)
{
  if (p.guard && *p.guard == 0u) return;
  extern __shared__ acc_u4 shared[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l = lane & 15, g = lane >> 4;
  const op_tile tile = op_find_tile<OP_ALL>(p.offsets, p.experts, (int)p.rows, p.height, op_segments(p.offsets, p.experts, (int)p.rows, 0, 0), (int)(blockIdx.x / p.tiles_j));
  if (tile.begin >= tile.end) return;
  const int steps = (p.blocks + 3) / 4, rows = tile.end - tile.begin, tiles = (p.nj + 15) / 16, height = OP_HEIGHT ? OP_HEIGHT : p.height;
  const int j0 = (int)(blockIdx.x % p.tiles_j) * p.run, here = acc_min(p.run, tiles - j0);       /* tiles of columns */
  const bool sums = tile.expert >= 0 && p.x_rows > 0 && steps > 0;
  acc_u4 *const notes = shared;                    /* [waves][OP_FM][64]: a wave's scales and zeros; its sums, where they meet */
  acc_u4 *const x = notes + OP_WAVES * OP_FM * 64; /* [steps][4][parts][4][height] */
  float *const sum = (float *)(x + steps * 16 * OP_PARTS * height);       /* [steps][chunks][height], and Float32's second ones */
  float *const offset = OP_ELT == 0 ? sum + steps * OP_CHUNKS * height : sum;
  const auto row_of = [&](const int i) { return p.index ? op_listed(p.index, tile.begin + i, tile.begin, tile.end, p.x_rows, p.per_mul, p.per_shift) : tile.begin + i; };
  const auto write = [&](const int jt, const acc_f4 (&c)[OP_FM]) {
#pragma unroll
    for (int i = 0; i < OP_FM; ++i) {
      const int m = i * 16 + l;
      if (m < rows) op_write4((op_elt *)p.out + (long long)(tile.begin + m) * p.out_stride, jt * 16 + 4 * g, p.nj, c[i], !sums || row_of(m) < 0);
    }
  };
  if (!sums) {
    const acc_f4 none[OP_FM] = {};
    for (int t = wave; t < here; t += OP_WAVES) write(j0 + t, none);
    return;
  }

  const unsigned char *const codes = (const unsigned char *)p.codes + tile.expert * p.codes_expert, *const zeros = (const unsigned char *)p.zeros + tile.expert * p.zeros_expert;
  const op_elt *const scales = (const op_elt *)p.scales + tile.expert * p.scales_expert;
  const int split = p.split, each = (steps + split - 1) / split, n0 = wave % split * each, n1 = acc_min(steps, n0 + each), stride = OP_WAVES / split;
  const int mine = wave / split, turns = (here + stride - 1) / stride, own = n1 > n0 && mine < here ? (here - mine + stride - 1) / stride : 0;
  const int last_tile = p.nj % 16 ? tiles - 1 : -1, last_step = p.blocks % 4 ? steps - 1 : -1;      /* that are not whole */
  const unsigned int pitch = (unsigned int)p.codes_stride, row = l * pitch + g * 16, last_row = acc_min(l, p.nj - 1 - last_tile * 16) * pitch + g * 16;
  const unsigned int early = (unsigned int)acc_max(0, g - (p.blocks - 1 - last_step * 4)) * 16;
  /* codes of columns jt, step n: an address that is the same in all lanes, and 32 bits of the lane's */
  const auto load = [&](const int jt, const int n, acc_u4 &w) {
    const unsigned int at = (jt != last_tile ? row : last_row) - (n != last_step ? 0u : early);
    w = __builtin_nontemporal_load((const acc_u4 *)(codes + ((long long)jt * 16 * p.codes_stride + n * 64) + at));
  };
  /* the lane's part of the scales and zeros of 16 columns from step n on (of the last columns: the last 16 there are) */
  const bool scale_lane = lane < OP_NOTED * OP_SIZE;
  const int noted = scale_lane ? lane / OP_SIZE : acc_min(lane - OP_NOTED * OP_SIZE, OP_NOTED - 1);
  const char *const note_base = scale_lane || !OP_ZEROS ? (const char *)scales + lane % OP_SIZE * 16 : (const char *)zeros;
  const long long note_stride = scale_lane || !OP_ZEROS ? p.scales_stride * OP_SIZE : p.zeros_stride;
  const auto load_note = [&](const int jt, const int n, acc_u4 &note) {
    const int column = jt != last_tile ? jt * 16 : p.nj - 16, group = acc_min(((n * 128) >> p.group_shift) + noted, p.groups - 1);
    note = ((const op_loose<unsigned char> *)(note_base + (group * note_stride + column * (scale_lane || !OP_ZEROS ? OP_SIZE : 1))))->v;
  };
  acc_f4 c[OP_FM];
  const char *const my_notes = (const char *)(notes + wave * OP_FM * 64);
  /* step n's products, the first of its groups being the at-th that is noted; `down`: the columns' places among the noted 16 */
  const auto add = [&](const int n, const int at, const int down, acc_u4 w) {
    op_turn(w);
    /* (of Float32's many fragments in groups of 32 no addresses are kept from step to step: there are not the registers, and a wait for
     * one that has been put into memory is a wait for all codes on their way: 27 us in place of 23 for 150 rows of 12 matrices of
     * 1333 x 1001.  Elsewhere, where there are registers, it costs 3 in 100) */
    int row = l, quarter = g;
    if (OP_PARTS > 1 && OP_CHUNKS > 2) {
      acc_pin(row);
      acc_pin(quarter);
    }
#pragma unroll
    for (int q = 0; q < OP_CHUNKS; ++q) {
      const int noted_at = at + q;
      op_e4<op_elt> s;
      op_e4<unsigned char> z;
      if (down == 0) {
        __builtin_memcpy(&s, __builtin_assume_aligned(my_notes + (noted_at * 16 + quarter * 4) * OP_SIZE, 4 * OP_SIZE), sizeof(s));
        if (OP_ZEROS) __builtin_memcpy(&z, __builtin_assume_aligned(my_notes + OP_NOTED * OP_SIZE * 16 + noted_at * 16 + quarter * 4, 4), sizeof(z));
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int k = acc_min(quarter * 4 + r + down, 15);
          s.v[r] = *(const op_elt *)(my_notes + (noted_at * 16 + k) * OP_SIZE);
          if (OP_ZEROS) z.v[r] = *(const unsigned char *)(my_notes + OP_NOTED * OP_SIZE * 16 + noted_at * 16 + k);
        }
      }
      acc_f4 t[OP_FM];
      float second[OP_FM];
#pragma unroll
      for (int i = 0; i < OP_FM; ++i) {
        const int place = (n * OP_CHUNKS + q) * height + ((i * 16 + row) & (height - 1));
        const float f = sum[place];
        second[i] = OP_ELT == 0 ? offset[place] : 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r) t[i][r] = op_begin(f, OP_ZEROS ? (float)z.v[r] : 8.0f);
      }
#pragma unroll
      for (int part = 0; part < OP_PARTS; ++part)
#pragma unroll
        for (int b = q * OP_BLOCKS; b < (q + 1) * OP_BLOCKS; ++b) {
          const op_frag v = op_as_frag(op_numbers(w[b]));
#pragma unroll
          for (int i = 0; i < OP_FM; ++i) t[i] = op_mfma(v, op_as_frag(x[(((n * 4 + b) * OP_PARTS + part) * 4 + quarter) * height + ((i * 16 + row) & (height - 1))]), t[i]);
        }
#pragma unroll
      for (int i = 0; i < OP_FM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) t[i][r] = op_rest(t[i][r], second[i], OP_ZEROS ? (float)z.v[r] : 8.0f);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < OP_FM; ++i) c[i][r] = __builtin_fmaf((float)s.v[r], t[i][r], c[i][r]);
    }
  };
  const auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < OP_FM; ++i) c[i] = acc_f4{0.0f, 0.0f, 0.0f, 0.0f};
  };
  const int lots = n1 > n0 ? (n1 - n0 + OP_AHEAD - 1) / OP_AHEAD : 0, all = own * lots;
  acc_u4 ring[OP_AHEAD], note;
  if (all > 0) {
    load_note(j0 + mine, n0, note);
#pragma unroll
    for (int u = 0; u < OP_AHEAD; ++u) load(j0 + mine, acc_min(n0 + u, n1 - 1), ring[u]);
  }

  /* the rows: a lane has eight neighbours of one; rows that there are not stay as LDS is, and nobody's */
  for (int at = tid; at < steps * 16 * rows; at += 64 * OP_WAVES) {
    const int i = at / (steps * 16), k = (at - i * steps * 16) * 8, n = k / 128, kk = k % 128, r = row_of(i);
    const int b = OP_CHUNKS > 1 ? kk / 32 : kk / 8 % 4, quarter = OP_CHUNKS > 1 ? kk / 8 % 4 : kk / 32;
    acc_u4 v[OP_PARTS];
    op_parts(op_row8((const op_elt *)p.x + (long long)acc_max(r, 0) * p.x_stride + k, p.k - k), v);
#pragma unroll
    for (int part = 0; part < OP_PARTS; ++part) x[(((n * 4 + b) * OP_PARTS + part) * 4 + quarter) * height + i] = v[part];
  }
  __syncthreads();
  for (int n = wave; n < steps; n += OP_WAVES)
#pragma unroll
    for (int q = 0; q < OP_CHUNKS; ++q)
#pragma unroll
      for (int i = 0; i < OP_FM; ++i) {
        acc_f4 t, d;
        op_sums(q, [&](const int b, const int part) { return op_as_frag(x[(((n * 4 + b) * OP_PARTS + part) * 4 + g) * height + ((i * 16 + l) & (height - 1))]); }, t, d);
        const int at = (n * OP_CHUNKS + q) * height + i * 16 + l;
        if (g == 0 && i * 16 + l < height) {
          sum[at] = t[0];
          if (OP_ELT == 0) offset[at] = d[0];
        }
      }
  __syncthreads();

  int jt = j0 + mine, n = n0;
  clear();
  for (int at = 0; at < all; ++at) {
    notes[wave * OP_FM * 64 + lane] = note;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const bool end = n + OP_AHEAD >= n1, more = at + 1 < all;
    const int next_jt = end & more ? jt + stride : jt, next_n = !more ? n : end ? n0 : n + OP_AHEAD;
    load_note(next_jt, next_n, note);
    const int down = jt == last_tile ? 16 - p.nj % 16 : 0, group = (n * 128) >> p.group_shift;
#pragma unroll
    for (int u = 0; u < OP_AHEAD; u += 2) {        /* (two at a time: a line of memory has two steps of a row) */
      if (n + u < n1) add(n + u, OP_CHUNKS > 1 ? u * OP_CHUNKS : (((n + u) * 128) >> p.group_shift) - group, down, ring[u]);
      __builtin_amdgcn_sched_barrier(0);           /* (a step's rows out of LDS when it is their turn: registers) */
      if (n + u + 1 < n1) add(n + u + 1, OP_CHUNKS > 1 ? (u + 1) * OP_CHUNKS : (((n + u + 1) * 128) >> p.group_shift) - group, down, ring[u + 1]);
      __builtin_amdgcn_sched_barrier(0);
      load(next_jt, acc_min(next_n + u, n1 - 1), ring[u]);
      load(next_jt, acc_min(next_n + u + 1, n1 - 1), ring[u + 1]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (end) {
      /* (waves of the same columns meet twice for each of their tiles) */
      if (split > 1) {
#pragma unroll
        for (int i = 0; i < OP_FM; ++i) ((acc_f4 *)notes)[(wave * OP_FM + i) * 64 + lane] = c[i];
        __syncthreads();
        if (wave % split == 0)
#pragma unroll
          for (int i = 0; i < OP_FM; ++i)
            for (int w = 1; w * each < steps; ++w) c[i] += ((const acc_f4 *)notes)[((wave + w) * OP_FM + i) * 64 + lane];
        __syncthreads();
      }
      if (wave % split == 0) write(jt, c);
      clear();
    }
    jt = next_jt;
    n = next_n;
  }
  if (split > 1)
    for (int t = own; t < turns; ++t) {
      __syncthreads();
      __syncthreads();
    }
}
#elif OP_WIDE
/* The form for many rows of a matrix: tiles of 64 rows (of Float32: 32, in three parts) by 256 columns, four waves of 64 of them, two
 * workgroups a compute unit.  The rows of a step of 128 lie in LDS, three steps at a time: the one whose products are taken, the next
 * one, whose sums by groups are taken meanwhile (of 16 rows by a wave), and the one after that, on its way there.  A wave makes its 64
 * columns' codes into numbers itself, in registers: 16 columns' are used for all rows.  bfloat16, 2048 rows of 8 matrices of 4096 x 4096 in
 * groups of 128: 110 us, 624 TFLOP/s.  Loads are not what it waits for (without those of
 * the codes 1 us less, of the rows 7): a step's 64 instructions of the matrix cores take as long as the 200 others beside them, of which
 * a half makes numbers, and of two waves a SIMD one covers the other only in part.  (128 rows and eight waves a workgroup: 154, a
 * segment's short last tile being as long as a whole one; the numbers of the next 32 made ready between the products: 132 and more,
 * for want of registers.) */
#define OP_PER (OP_ELT == 0 ? 2 : 4)               /* rows of a tile, in sixteens */
#define OP_ROWS (16 * OP_PER)
#define OP_SIZE ((int)sizeof(op_elt))
#define OP_COLUMNS 256
#define OP_LINE (OP_COLUMNS + 16)                  /* scales (zeros) of a group: 16 places in front, for a tile with fewer columns */

/* What the 16 rows' places of a step's word b, quarter g are turned by: other numbers for all 16, so that a row's eighths go to other banks;
 * and for the quarters 0 and 1, 2 and 3, of whose lanes 16 are served at a time (four, four more twelve on, and eight of the other quarter
 * between those), such that these still lie beside each other. */
ACC_DEV int op_turn_of(const int b, const int g) { return OP_CHUNKS > 1 ? 4 * b + g : b | (g & 1) << 3 | ((g ^ g >> 1) & 1) << 2; }

template <int N> struct op_count { static constexpr int value = N; };

extern "C" __global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) grouped(const acc_grouped_args p)
{
  if (p.guard && *p.guard == 0u) return;
  extern __shared__ acc_u4 shared[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l = lane & 15, g = lane >> 4;
  const op_tile tile = op_find_tile<OP_ALL>(p.offsets, p.experts, (int)p.rows, OP_ROWS, op_segments(p.offsets, p.experts, (int)p.rows, 0, 0), (int)(blockIdx.x / p.tiles_j));
  if (tile.begin >= tile.end) return;
  const int steps = (p.blocks + 3) / 4, rows = tile.end - tile.begin, j0 = (int)(blockIdx.x % p.tiles_j) * OP_COLUMNS;
  acc_u4 *const x = shared;                        /* [3][16][parts][OP_ROWS]: eight neighbours of a row, a row's places turned by their number */
  float *const scale = (float *)(x + 3 * 16 * OP_PARTS * OP_ROWS);         /* [3][chunks][OP_LINE], and the zeros' */
  float *const zero = scale + 3 * OP_CHUNKS * OP_LINE;
  float *const sum = OP_ZEROS ? zero + 3 * OP_CHUNKS * OP_LINE : zero;     /* [2][chunks][OP_ROWS]; what products begin with, where zeros are 8 */
  float *const offset = sum + 2 * OP_CHUNKS * OP_ROWS;                     /* Float32: the second ones */
  acc_f4 c[OP_PER][4];
#pragma unroll
  for (int i = 0; i < OP_PER; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) c[i][j] = acc_f4{0.0f, 0.0f, 0.0f, 0.0f};
  const auto row_of = [&](const int m) { return p.index ? op_listed(p.index, tile.begin + m, tile.begin, tile.end, p.x_rows, p.per_mul, p.per_shift) : tile.begin + acc_min(m, rows - 1); };

  if (tile.expert >= 0 && p.x_rows > 0 && steps > 0) {
    /* a lane's places among the rows: eight neighbours, of rows 16 apart */
    const int chunk = tid & 15, first = tid >> 4, place = ((OP_CHUNKS > 1 ? chunk : chunk % 4 * 4 + chunk / 4) * OP_PARTS * OP_ROWS) + (first ^ (OP_CHUNKS > 1 ? op_turn_of(chunk / 4, chunk % 4) : op_turn_of(chunk % 4, chunk / 4)));
    const op_elt *from[OP_PER];
#pragma unroll
    for (int u = 0; u < OP_PER; ++u) from[u] = (const op_elt *)p.x + (long long)acc_max(row_of(first + 16 * u), 0) * p.x_stride + chunk * 8;
    /* ... and among the scales and zeros: 16 bytes of a group's (of the last columns: as many as there are) */
    constexpr int wide = 16 / OP_SIZE, lanes = OP_COLUMNS / wide;
    const int scale_at = acc_min(j0 + (tid < OP_CHUNKS * lanes ? tid % lanes * wide : 0), p.nj - wide), zero_at = acc_min(j0 + tid % 16 * 16, p.nj - 16);
    const op_elt *const scales = (const op_elt *)p.scales + tile.expert * p.scales_expert + scale_at;
    const unsigned char *const zeros = (const unsigned char *)p.zeros + tile.expert * p.zeros_expert + zero_at;
    op_eight v[OP_PER];
    acc_u4 scale_note, zero_note;
    const auto load = [&](const int n) {
      const int group = (n * 128) >> p.group_shift;
      scale_note = ((const op_loose<op_elt> *)(scales + acc_min(group + tid / lanes % OP_CHUNKS, p.groups - 1) * p.scales_stride))->v;
      if (OP_ZEROS) zero_note = ((const op_loose<unsigned char> *)(zeros + acc_min(group + tid / 16 % OP_CHUNKS, p.groups - 1) * p.zeros_stride))->v;
      if (n * 128 + 128 <= p.k) {
#pragma unroll
        for (int u = 0; u < OP_PER; ++u)
#pragma unroll
          for (int h = 0; h < 8 / OP_VALUES; ++h) v[u].v[h] = ((const op_loose<op_elt> *)(from[u] + n * 128 + h * OP_VALUES))->v;
      } else {
#pragma unroll
        for (int u = 0; u < OP_PER; ++u) v[u] = op_row8(from[u] + n * 128, p.k - n * 128 - chunk * 8);
      }
    };
    const auto put = [&](const int to) {
#pragma unroll
      for (int u = 0; u < OP_PER; ++u) {
        acc_u4 parts[OP_PARTS];
        op_parts(v[u], parts);
#pragma unroll
        for (int part = 0; part < OP_PARTS; ++part) x[(to * 16 * OP_PARTS + part) * OP_ROWS + place + 16 * u] = parts[part];
      }
      if (tid < OP_CHUNKS * lanes) {
        op_elt e[wide];
        __builtin_memcpy(e, &scale_note, 16);
        float *const line = scale + (to * OP_CHUNKS + tid / lanes) * OP_LINE + 16 + (scale_at - j0);
#pragma unroll
        for (int t = 0; t < wide; ++t) line[t] = (float)e[t];
      }
      if (OP_ZEROS && tid < OP_CHUNKS * 16) {
        float *const line = zero + (to * OP_CHUNKS + tid / 16) * OP_LINE + 16 + (zero_at - j0);
#pragma unroll
        for (int t = 0; t < 16; ++t) line[t] = (float)(zero_note[t / 4] >> t % 4 * 8 & 255u);
      }
    };
    /* the lane's fragment of rows 16 i on of a wave's */
    const auto row16 = [&](const int buffer, const int b, const int i, const int part) {
      return op_as_frag(x[((buffer * 16 + b * 4 + g) * OP_PARTS + part) * OP_ROWS + i * 16 + (l ^ op_turn_of(b, g))]);
    };
    const auto add_up = [&](const int buffer, const int slot) {
      if (OP_PER < 4 && wave >= OP_PER) return;
#pragma unroll
      for (int q = 0; q < OP_CHUNKS; ++q) {
        acc_f4 t, d;
        op_sums(q, [&](const int b, const int part) { return row16(buffer, b, wave, part); }, t, d);
        const int at = (slot * OP_CHUNKS + q) * OP_ROWS + wave * 16 + l;
        if (g == 0) {
          sum[at] = OP_ZEROS ? t[0] : op_begin(t[0], 8.0f);
          if (OP_ELT == 0) offset[at] = d[0];
        }
      }
    };

    /* codes: 16 columns are 16 rows of bytes; columns and blocks that there are not are read as the last ones */
    const int column = acc_min(j0 + wave * 64, p.nj - 1), left = p.nj - 1 - column, last_step = p.blocks % 4 ? steps - 1 : -1;
    const unsigned char *const codes = (const unsigned char *)p.codes + tile.expert * p.codes_expert + column * p.codes_stride;
    const unsigned int early = (unsigned int)acc_max(0, g - (p.blocks - 1 - (steps - 1) * 4)) * 16;
    unsigned int at_code[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) at_code[j] = (unsigned int)acc_min(16 * j + l, left) * (unsigned int)p.codes_stride + g * 16;
    acc_u4 w[4];
    const auto load_codes = [&](const int n, const int j) {
      w[j] = *(const acc_u4 *)(codes + (long long)n * 64 + (at_code[j] - (n != last_step ? 0u : early)));
    };

    load(0);
    put(0);
    load(acc_min(1, steps - 1));
    put(1);
    load(acc_min(2, steps - 1));
#pragma unroll
    for (int j = 0; j < 4; ++j) load_codes(0, j);
    __syncthreads();
    add_up(0, 0);
    /* the products of 16 M rows (a segment's last tile may have few) */
    const auto products = [&](const auto fragments) {
      constexpr int M = decltype(fragments)::value;
      int now = 0, next = 1, then = 2;
      for (int n = 0; n < steps; ++n) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) op_turn(w[j]);
#pragma unroll
        for (int q = 0; q < OP_CHUNKS; ++q) {
          op_frag y[OP_BLOCKS][M][OP_PARTS];
          float f[M], o[M];
#pragma unroll
          for (int i = 0; i < M; ++i) {
#pragma unroll
            for (int b = 0; b < OP_BLOCKS; ++b)
#pragma unroll
              for (int part = 0; part < OP_PARTS; ++part) y[b][i][part] = row16(now, q * OP_BLOCKS + b, i, part);
            const int at = ((n & 1) * OP_CHUNKS + q) * OP_ROWS + i * 16 + l;
            f[i] = sum[at];
            o[i] = OP_ELT == 0 ? offset[at] : 0.0f;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = (now * OP_CHUNKS + q) * OP_LINE + 16 + wave * 64 + j * 16 + g * 4;
            const acc_f4 s = *(const acc_f4 *)(scale + at), z = OP_ZEROS ? *(const acc_f4 *)(zero + at) : s;
            op_frag numbers[OP_BLOCKS];
#pragma unroll
            for (int b = 0; b < OP_BLOCKS; ++b) numbers[b] = op_as_frag(op_numbers(w[j][q * OP_BLOCKS + b]));
            if (q == OP_CHUNKS - 1) load_codes(acc_min(n + 1, steps - 1), j);
            acc_f4 t[M];
#pragma unroll
            for (int i = 0; i < M; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) t[i][r] = OP_ZEROS ? op_begin(f[i], z[r]) : f[i];
#pragma unroll
            for (int part = 0; part < OP_PARTS; ++part)
#pragma unroll
              for (int b = 0; b < OP_BLOCKS; ++b)
#pragma unroll
                for (int i = 0; i < M; ++i) t[i] = op_mfma(numbers[b], y[b][i][part], t[i]);
#pragma unroll
            for (int i = 0; i < M; ++i)
#pragma unroll
              for (int r = 0; r < 4; ++r) c[i][j][r] = __builtin_fmaf(s[r], op_rest(t[i][r], o[i], OP_ZEROS ? z[r] : 8.0f), c[i][j][r]);
            /* (the next steps' rows and sums amid the products: every wave has some to go on with) */
            if (q == 0 && j == 0) {
              put(then);
              load(acc_min(n + 3, steps - 1));
            }
            if (q == 0 && j == 1) add_up(next, (n + 1) & 1);
          }
        }
        const int was = now;
        now = next;
        next = then;
        then = was;
      }
    };
    if (OP_PER > 2 && rows > 32) products(op_count<OP_PER>{});
    else if (rows > 16) products(op_count<2>{});
    else products(op_count<1>{});
  }
#pragma unroll
  for (int i = 0; i < OP_PER; ++i) {
    const int m = i * 16 + l;
    if (m >= rows) continue;
    const bool none = tile.expert < 0 || row_of(m) < 0;
    op_elt *const out = (op_elt *)p.out + (long long)(tile.begin + m) * p.out_stride;
#pragma unroll
    for (int j = 0; j < 4; ++j) op_write4(out, j0 + wave * 64 + j * 16 + 4 * g, p.nj, c[i][j], none);
  }
}
#else
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
    const auto load_as = [&](const bool whole, const int n, op_step &s) {
      const int k = n * 128;
#pragma unroll
      for (int j = 0; j < OP_FN; ++j) s.w[j] = __builtin_nontemporal_load((const acc_u4 *)(w[j] + acc_min(n * 4 + g, p.blocks - 1) * 16));
#pragma unroll
      for (int q = 0; q < OP_CHUNKS; ++q) {
        const int at = acc_min((k + q * (128 / OP_CHUNKS)) >> p.group_shift, p.groups - 1);
#pragma unroll
        for (int j = 0; j < OP_FN; ++j) {
          s.s[q][j] = op_four(scales + at * p.scales_stride, whole, j0 + j * 16 + g * 4, p.nj);
          if (OP_ZEROS) s.z[q][j] = op_four(zeros + at * p.zeros_stride, whole, j0 + j * 16 + g * 4, p.nj);
        }
      }
#pragma unroll
      for (int i = 0; i < OP_FM; ++i)
#pragma unroll
        for (int b = 0; b < 4; ++b) s.x[i][b] = op_row8(x[i] + k + OP_FIRST(b, g), whole ? 8 : p.k - k - OP_FIRST(b, g));
    };
    const auto load = [&](const int n, op_step &s) {
      if (n * 128 + 128 <= p.k && j0 + 16 * OP_FN <= p.nj) load_as(true, n, s);
      else load_as(false, n, s);
    };
    const auto add = [&](op_step &s) {
      const acc_f4 none = {0.0f, 0.0f, 0.0f, 0.0f};
      const op_frag ones = op_as_frag(acc_u4{OP_ONES, OP_ONES, OP_ONES, OP_ONES});
#pragma unroll
      for (int j = 0; j < OP_FN; ++j) op_turn(s.w[j]);
#pragma unroll
      for (int q = 0; q < OP_CHUNKS; ++q) {
        acc_f4 t[OP_FM][OP_FN], rest[OP_FM][OP_FN], sum[OP_FM], second[OP_FM];      /* rest: of Float32's other parts */
#pragma unroll
        for (int i = 0; i < OP_FM; ++i) {
          sum[i] = second[i] = none;
#pragma unroll
          for (int j = 0; j < OP_FN; ++j) t[i][j] = rest[i][j] = none;
        }
#pragma unroll
        for (int b = q * OP_BLOCKS; b < (q + 1) * OP_BLOCKS; ++b) {
          op_frag v[OP_FN];
#pragma unroll
          for (int j = 0; j < OP_FN; ++j) v[j] = op_as_frag(op_numbers(s.w[j][b]));
#pragma unroll
          for (int i = 0; i < OP_FM; ++i) {
            acc_u4 part[OP_PARTS];
            op_parts(s.x[i][b], part);
#pragma unroll
            for (int n = OP_PARTS - 1; n >= 0; --n) {
              const op_frag y = op_as_frag(part[n]);
              acc_f4 &sums = n == 0 ? sum[i] : second[i];
              sums = op_mfma(ones, y, sums);
#pragma unroll
              for (int j = 0; j < OP_FN; ++j) {
                acc_f4 &to = n == 0 ? t[i][j] : rest[i][j];
                to = op_mfma(v[j], y, to);
              }
            }
          }
        }
#pragma unroll
        for (int j = 0; j < OP_FN; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float scale = (float)s.s[q][j].v[r], zero = OP_ZEROS ? (float)s.z[q][j].v[r] : 8.0f;
#pragma unroll
            for (int i = 0; i < OP_FM; ++i) {
              const float first = t[i][j][r] + op_begin(sum[i][r], zero);
              c[i][j][r] = __builtin_fmaf(scale, OP_ELT == 0 ? first + op_rest(rest[i][j][r], second[i][r], zero) : first, c[i][j][r]);
            }
          }
      }
    };
    for (int n = wave * OP_AHEAD; n < steps; n += OP_WAVES * OP_AHEAD) {
      op_step s[OP_AHEAD];
#pragma unroll
      for (int u = 0; u < OP_AHEAD; ++u)
        if (n + u < steps) load(n + u, s[u]);
      __builtin_amdgcn_sched_barrier(0);           /* (all loads first) */
#pragma unroll
      for (int u = 0; u < OP_AHEAD; ++u)
        if (n + u < steps) add(s[u]);
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
#endif
