/*
 * op_matrix.h -- what the products' kernels share: elements in memory, fragments, the matrix instructions.
 */
#ifndef ACC_OP_MATRIX_H
#define ACC_OP_MATRIX_H

#include "op_common.h"

#if OP_TYPE == 3
typedef unsigned char op_mem;
#else
typedef op_elt op_mem;
#endif
#define OP_EPC (16 / (int)sizeof(op_mem))          /* elements of a chunk of 16 bytes */
#define OP_STEP (8 * OP_EPC)                       /* the step of the sum, in elements */

#if OP_TYPE == 0
typedef acc_f4 op_frag;                            /* four values of r for one i */
ACC_DEV acc_f4 op_mfma(const op_frag x, const op_frag y, acc_f4 c)
{
#pragma unroll
  for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[t], y[t], c, 0, 0, 0);
  return c;
}
#elif OP_TYPE == 1
typedef _Float16 op_frag __attribute__((ext_vector_type(8)));
ACC_DEV acc_f4 op_mfma(const op_frag x, const op_frag y, const acc_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0); }
#elif OP_TYPE == 2
typedef __bf16 op_frag __attribute__((ext_vector_type(8)));
ACC_DEV acc_f4 op_mfma(const op_frag x, const op_frag y, const acc_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0); }
#else
typedef int op_i8 __attribute__((ext_vector_type(8)));
typedef acc_u4 op_frag;                            /* a block of 32 */
/* `sx` holds the scales of four fragments, x's the nx-th */
ACC_DEV acc_f4 op_mfma_scaled(const op_frag &x, const op_frag &y, const acc_f4 c, const int sx, const int nx, const int sy, const int ny)
{
  const op_i8 a = {(int)x.x, (int)x.y, (int)x.z, (int)x.w, 0, 0, 0, 0}, b = {(int)y.x, (int)y.y, (int)y.z, (int)y.w, 0, 0, 0, 0};
  /* (the byte to take is part of the instruction; which it is, is known once the loops are unrolled) */
#define OP_CASE(i, j) case 4 * i + j: return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 4, 4, i, sx, j, sy);
#define OP_CASES(i) OP_CASE(i, 0) OP_CASE(i, 1) OP_CASE(i, 2) OP_CASE(i, 3)
  switch (4 * nx + ny) { OP_CASES(0) OP_CASES(1) OP_CASES(2) OP_CASES(3) }
  return c;
}
#endif

#define OP_NOWHERE 0x80000000u                     /* an offset beyond the end of every buffer: reads as zeros */
#define OP_FARTHEST 0x7fffffffll                   /* the longest buffer */

/* what an index of rows lo .. hi - 1 says of row m (of one beside them: something), and which row that is, divided as the arguments
 * say; -1: none */
ACC_DEV int op_entry(const int *index, const int m, const int lo, const int hi) { return index[(unsigned int)acc_max(lo, acc_min(m, hi - 1))]; }
ACC_DEV int op_named(const int at, const int m, const int lo, const int hi, const int limit, const unsigned int per_mul, const unsigned int per_shift)
{
  /* (by nothing: per_mul is 0) */
  const int r = (int)(__umulhi((unsigned int)at, per_mul) >> per_shift) + (at & (per_mul ? 0 : -1));
  return (m >= lo) & (m < hi) & ((unsigned int)at < 0x80000000u) & (r < limit) ? r : -1;
}
ACC_DEV int op_listed(const int *index, const int m, const int lo, const int hi, const int limit, const unsigned int per_mul, const unsigned int per_shift)
{
  return op_named(op_entry(index, m, lo, hi), m, lo, hi, limit, per_mul, per_shift);
}

/* four neighbours of a row of the result, from column j on, wherever it starts; `none`: of no row, whatever the sums say (a
 * matrix may hold infinities: no row times that is zeros all the same) */
template <typename T> ACC_DEV void op_write4(T *out, const int j, const int end, const acc_f4 c, const bool none)
{
  struct __attribute__((packed, aligned(sizeof(T)))) op_e4 { T v[4]; };
  op_e4 e;
#pragma unroll
  for (int t = 0; t < 4; ++t) e.v[t] = (T)(none ? 0.0f : c[t]);
  if (j + 4 <= end) {
    *(op_e4 *)(out + j) = e;
  } else {
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (j + t < end) out[j + t] = e.v[t];
  }
}

/* Two neighbouring fragments of the result, columns j .. j + 31, of which a lane has four of either (g: its quarter of the wave).  Of
 * 16 bits, quarters exchange halves first, so that a lane has eight neighbours, and four lanes half a cache line: with 8 bytes a
 * lane, 230 MB of gradients took 97 us. */
ACC_DEV void op_write_pair(op_elt *out, const int j, const int end, const int g, const acc_f4 c, const acc_f4 d, const bool none)
{
#if OP_ELT == 0
  op_write4(out, j + 4 * g, end, c, none);
  op_write4(out, j + 16 + 4 * g, end, d, none);
#else
  op_elt x[4], y[4];
  unsigned int u[2], v[2];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    x[t] = (op_elt)(none ? 0.0f : c[t]);
    y[t] = (op_elt)(none ? 0.0f : d[t]);
  }
  __builtin_memcpy(u, x, 8);
  __builtin_memcpy(v, y, 8);
  const auto lo = __builtin_amdgcn_permlane16_swap(u[0], v[0], false, false), hi = __builtin_amdgcn_permlane16_swap(u[1], v[1], false, false);
  const acc_u4 all = {lo[0], hi[0], lo[1], hi[1]};
  const int at = j + (g & 1) * 16 + (g >> 1) * 8;
  if (at + 8 <= end) {
    ((op_loose<op_elt> *)(out + at))->v = all;
  } else {
    op_elt e[8];
    __builtin_memcpy(e, &all, 16);
#pragma unroll
    for (int t = 0; t < 8; ++t)
      if (at + t < end) out[at + t] = e[t];
  }
#endif
}

#endif
