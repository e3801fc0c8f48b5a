/*
 * op_micro_product.h -- products of segments of rows with a matrix each, both operands 4-bit numbers under shared scales
 * (op_micro.h), on the scaled matrix instructions: out[m, n] = sum_k a[r(m), k] b[e(m), n, k].
 *
 * A lane's operand of the 16 x 16 x 128 instruction is one block of 32 of one row, 16 bytes of codes and its scale.
 */
#include "op_common.h"

typedef int op_i8 __attribute__((ext_vector_type(8)));

#define OP_NJ 4                                    /* fragments of 16 columns that a wave has */

/* block `block` of a row: its codes and scale; zeros where there is none */
ACC_DEV void op_block(const unsigned char *codes, const unsigned char *scales, const int block, const int blocks, op_i8 *v, int *scale)
{
  acc_u4 c = {0, 0, 0, 0};
  int s = 127;
  if (codes && block < blocks) {
    c = *(const acc_u4 *)(codes + (long long)block * 16);
    s = scales[block];
  }
  *v = op_i8{(int)c.x, (int)c.y, (int)c.z, (int)c.w, 0, 0, 0, 0};
  *scale = s;
}

extern "C" __global__ void __launch_bounds__(256) micro_product(const acc_micro_product_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
  const op_tile tile = op_find_tile(p.offsets, p.experts, (int)p.rows, 16, blockIdx.x / p.tiles_j);
  if (tile.begin >= tile.end) return;
  const int j0 = ((int)(blockIdx.x % p.tiles_j) * 4 + wave) * 16 * OP_NJ;
  const int m = tile.begin + (lane & 15);

  long long r = m;
  bool row = m < tile.end && tile.expert >= 0;
  if (row && p.index) {
    const int at = p.index[m];
    r = p.per > 1 ? at / p.per : at;
    row = at >= 0 && r < p.a_rows;
  }
  const bool none = !row;          /* (a block of the matrix may be no number: no row times that is zeros all the same) */
  const unsigned char *a = row ? p.a + r * p.a_stride : (const unsigned char *)0, *sa = p.sa + (row ? r * p.sa_stride : 0);
  const unsigned char *b[OP_NJ], *sb[OP_NJ];
  acc_f4 c[OP_NJ];
#pragma unroll
  for (int j = 0; j < OP_NJ; ++j) {
    const int n = j0 + j * 16 + (lane & 15);
    const bool column = n < p.n && tile.expert >= 0;
    b[j] = column ? p.b + tile.expert * p.b_expert + n * p.b_stride : (const unsigned char *)0;
    sb[j] = p.sb + (column ? tile.expert * p.sb_expert + n * p.sb_stride : 0);
    c[j] = acc_f4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  for (int k = 0; k < p.blocks; k += 4) {
    op_i8 va, vb;
    int xa, xb;
    op_block(a, sa, k + g, p.blocks, &va, &xa);
#pragma unroll
    for (int j = 0; j < OP_NJ; ++j) {
      op_block(b[j], sb[j], k + g, p.blocks, &vb, &xb);
      c[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(vb, va, c[j], 4, 4, 0, xb, 0, xa);
    }
  }
  if (m >= tile.end) return;
  op_elt *out = (op_elt *)p.out + (long long)m * p.out_stride;
#pragma unroll
  for (int j = 0; j < OP_NJ; ++j)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int n = j0 + j * 16 + 4 * g + t;
      if (n < p.n) out[n] = (op_elt)(none ? 0.0f : c[j][t]);
    }
}
