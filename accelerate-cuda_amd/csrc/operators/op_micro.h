/*
 * op_micro.h -- 4-bit floating-point numbers under shared scales, after the published microscaling formats (MXFP4): 32
 * neighbours share a power of two, a byte of exponent (127 for 1; 255: not a number); an element has a sign, two bits of
 * exponent and one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6.  Two elements a byte, the even place in the low half.
 *
 * The scale of a block is the power of two of its largest magnitude, less the two of the largest element's; elements are
 * rounded to the nearest, of two as near to the one with the even code, and to 6 above it.
 *
 * Bound by memory: 16384 x 4096 bfloat16 numbers, 134 MB read and 36 written, take 32 us to quantise, 5.3 TB/s (55 with comparisons in
 * place of the target's conversions, and a division by the blocks of a row), and 35 us to make again, 4.9 TB/s; Float32 52 and 75.
 */
#include "op_common.h"

/* two elements' codes in byte `n` of `to`: the target's own conversion rounds as said above, and takes the scale as the
 * exponent of a Float32 */
template <int N> ACC_DEV unsigned int op_codes(const unsigned int to, const float x, const float y, const float scale)
{
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(to, x, y, scale, N);
}
template <int N> ACC_DEV void op_values(const unsigned int codes, const float scale, float *to)
{
  const auto v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, N);
  to[0] = v[0];
  to[1] = v[1];
}

/* A lane's place: eight elements of a block, four lanes a block, blocks row after row.  (Rows by multiplication, the driver's
 * divisor; a launch has fewer than 2^30 blocks.) */
struct op_eight { long long row; int block, first; bool here; };
ACC_DEV op_eight op_mine(const acc_micro_args &p)
{
  const long long n = (long long)blockIdx.x * 256 + threadIdx.x;
  const unsigned int block = (unsigned int)(n >> 2);
  const unsigned int row = p.per_mul ? __umulhi(block, p.per_mul) >> p.per_shift : block;
  op_eight e;
  e.row = row;
  e.block = (int)(block - row * (unsigned int)p.blocks);
  e.first = e.block * 32 + (int)(n & 3) * 8;
  e.here = row < p.rows;
  return e;
}

/* four lanes have a block of 32, 8 elements each; a lane's elements are 4 bytes of codes */
extern "C" __global__ void __launch_bounds__(256) micro_quantise(const acc_micro_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const op_eight at = op_mine(p);
  const int quarter = (int)threadIdx.x & 3;
  float f[8];
#pragma unroll
  for (int h = 0; h < 8 / OP_VALUES; ++h) {
    const acc_u4 v = op_chunk<OP_ALIGNED>((const op_elt *)p.x + at.row * p.x_stride + at.first + h * OP_VALUES, at.here ? p.k - at.first - h * OP_VALUES : 0);
    op_elt e[OP_VALUES];
    __builtin_memcpy(e, &v, 16);
#pragma unroll
    for (int k = 0; k < OP_VALUES; ++k) f[h * OP_VALUES + k] = (float)e[k];
  }
  /* the largest magnitude by its bits: what is no number, or infinite, is larger than any other */
  unsigned int most = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) most = acc_max(most, __float_as_uint(f[k]) & 0x7fffffffu);
  most = acc_max(most, acc_dpp<0xB1, 0xf>(most, most));          /* the neighbour's, then the other pair's */
  most = acc_max(most, acc_dpp<0x4E, 0xf>(most, most));
  /* a subnormal Float32 is below 2^-126: its scale is the smallest one anyway */
  const int exponent = (int)(most >> 23);
  const int byte = exponent == 255 ? 255 : acc_max(exponent - 2, 0);
  const float scale = __uint_as_float((unsigned int)byte << 23);
  unsigned int codes = 0;
  codes = op_codes<0>(codes, f[0], f[1], scale);
  codes = op_codes<1>(codes, f[2], f[3], scale);
  codes = op_codes<2>(codes, f[4], f[5], scale);
  codes = op_codes<3>(codes, f[6], f[7], scale);
  if (byte == 255) codes = 0;
  if (!at.here) return;
  *(unsigned int *)(p.codes + at.row * p.codes_stride + at.block * 16 + quarter * 4) = codes;
  if (quarter == 0) p.scales[at.row * p.scales_stride + at.block] = (unsigned char)byte;
}

/* a lane has 8 elements */
extern "C" __global__ void __launch_bounds__(256) micro_values(const acc_micro_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const op_eight at = op_mine(p);
  if (!at.here) return;
  const unsigned int codes = *(const unsigned int *)(p.codes + at.row * p.codes_stride + at.block * 16 + ((int)threadIdx.x & 3) * 4);
  const int byte = p.scales[at.row * p.scales_stride + at.block];
  const float scale = __uint_as_float((unsigned int)byte << 23);
  op_elt *out = (op_elt *)p.out + at.row * p.x_stride + at.first;
  float f[8];
  op_values<0>(codes, scale, f);
  op_values<1>(codes, scale, f + 2);
  op_values<2>(codes, scale, f + 4);
  op_values<3>(codes, scale, f + 6);
  op_elt e[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) e[k] = (op_elt)(byte == 255 ? __builtin_nanf("") : f[k]);
#pragma unroll
  for (int h = 0; h < 8 / OP_VALUES; ++h) {
    const int left = p.k - at.first - h * OP_VALUES;
    acc_u4 v;
    __builtin_memcpy(&v, e + h * OP_VALUES, 16);
    if (OP_ALIGNED) {
      if (left > 0) *(acc_u4 *)(out + h * OP_VALUES) = v;
    } else if (left >= OP_VALUES) {
      ((op_loose<op_elt> *)(out + h * OP_VALUES))->v = v;
    } else {
#pragma unroll
      for (int k = 0; k < OP_VALUES; ++k)
        if (k < left) out[h * OP_VALUES + k] = e[h * OP_VALUES + k];
    }
  }
}
