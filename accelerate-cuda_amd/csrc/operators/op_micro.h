/*
 * op_micro.h -- 4-bit floating-point numbers under shared scales, after the published microscaling formats (MXFP4): 32
 * neighbours share a power of two, a byte of exponent (127 for 1; 255: not a number); an element has a sign, two bits of
 * exponent and one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6.  Two elements a byte, the even place in the low half.
 *
 * The scale of a block is the power of two of its largest magnitude, less the two of the largest element's; elements are
 * rounded to the nearest, of two as near to the one with the even code, and to 6 above it.
 */
#include "op_common.h"

/* the code of x * scale */
ACC_DEV unsigned int op_code(const float x, const float scale)
{
  const float v = x * scale, a = __builtin_fabsf(v);
  const unsigned int m = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.0f);
  return m | (__float_as_uint(x) >> 31 << 3);
}

/* four lanes have a block of 32, 8 elements each; a lane's elements are 4 bytes of codes */
extern "C" __global__ void __launch_bounds__(256) micro_quantise(const acc_micro_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const long long n = (long long)blockIdx.x * 256 + threadIdx.x, block = n >> 2, row = block / p.blocks;
  const int b = (int)(block % p.blocks), c = b * 32 + (int)(n & 3) * 8;
  const bool here = row < p.rows;
  float f[8];
#pragma unroll
  for (int h = 0; h < 8 / OP_VALUES; ++h) {
    const acc_u4 v = op_chunk<OP_ALIGNED>((const op_elt *)p.x + row * p.x_stride + c + h * OP_VALUES, here ? p.k - c - h * OP_VALUES : 0);
    op_elt e[OP_VALUES];
    __builtin_memcpy(e, &v, 16);
#pragma unroll
    for (int k = 0; k < OP_VALUES; ++k) f[h * OP_VALUES + k] = (float)e[k];
  }
  /* the largest magnitude by its bits: what is no number, or infinite, is larger than any other */
  unsigned int most = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) most = acc_max(most, __float_as_uint(f[k]) & 0x7fffffffu);
  most = acc_max(most, (unsigned int)__shfl_xor((int)most, 1));
  most = acc_max(most, (unsigned int)__shfl_xor((int)most, 2));
  /* a subnormal Float32 is below 2^-126: its scale is the smallest one anyway */
  const int exponent = (int)(most >> 23);
  const int byte = exponent == 255 ? 255 : acc_max(exponent - 2, 0);
  const float scale = __builtin_ldexpf(1.0f, 127 - acc_min(byte, 254));
  unsigned int codes = 0;
  if (byte < 255)
#pragma unroll
    for (int k = 0; k < 8; ++k) codes |= op_code(f[k], scale) << (4 * k);
  if (!here) return;
  *(unsigned int *)(p.codes + row * p.codes_stride + b * 16 + (n & 3) * 4) = codes;
  if ((n & 3) == 0) p.scales[row * p.scales_stride + b] = (unsigned char)byte;
}

/* a lane has 8 elements */
extern "C" __global__ void __launch_bounds__(256) micro_values(const acc_micro_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const long long n = (long long)blockIdx.x * 256 + threadIdx.x, block = n >> 2, row = block / p.blocks;
  if (row >= p.rows) return;
  const int b = (int)(block % p.blocks), c = b * 32 + (int)(n & 3) * 8;
  const unsigned int codes = *(const unsigned int *)(p.codes + row * p.codes_stride + b * 16 + (n & 3) * 4);
  const int byte = p.scales[row * p.scales_stride + b];
  op_elt *out = (op_elt *)p.out + row * p.x_stride + c;
  op_elt e[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const unsigned int code = codes >> (4 * k);
    /* 0, 1/2, then 2^(e - 1) (1 + m / 2) */
    const unsigned int m = code & 7u;
    const float a = m < 2 ? 0.5f * (float)m : __uint_as_float(((m >> 1) + 126u) << 23 | (m & 1u) << 22);
    const float v = byte == 255 ? __builtin_nanf("") : __builtin_ldexpf(code & 8u ? -a : a, byte - 127);
    e[k] = (op_elt)v;
  }
#pragma unroll
  for (int h = 0; h < 8 / OP_VALUES; ++h) {
    const int left = p.k - c - h * OP_VALUES;
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
