/*
 * op_skinny.h -- products of segments of a few rows: out[m, n] = sum_k a[r(m), k] b[e(m), n, k] where an expert has no more
 * than a tile of OP_BM rows or two, both operands' rows along k, in whole chunks.
 *
 * What counts is that the experts' matrices pass by once, as fast as memory gives them.  Nothing of them is used twice, so
 * nothing goes by way of LDS: a lane loads its part of a fragment, 16 bytes of a column of the result, straight into
 * registers, OP_AHEAD steps of 128 bytes of k at a time.  The four waves of a workgroup take every fourth step of the same
 * 16 OP_FN columns -- a small call's matrices are spread over four times the waves that way -- and add up what they have
 * by way of LDS, in order.  Bound by memory: 64 rows, two of each of 32 matrices of 4096 x 2048 bfloat16 numbers, 537 MB: 85 us, 6.3
 * TB/s (partly out of the memory-side cache); 16 rows, 8 of 1024 x 1024, 17 MB: 6 us, which is about a launch.
 */
#include "op_matrix.h"

#define OP_FM (OP_BM / 16)
#define OP_WAVES 4
#define OP_AHEAD 3                                  /* (2, 3 and 4 take the same time within 2 %) */

extern "C" __global__ void __launch_bounds__(64 * OP_WAVES) product(const acc_product_args p)
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

  const int size = (int)sizeof(op_mem), row_bytes = p.k * size;
  const int astride = (int)p.a_stride * size, bstride = (int)p.b_stride * size;
  int arow[OP_FM];
#pragma unroll
  for (int i = 0; i < OP_FM; ++i) {
    const int m = tile.begin + i * 16 + l;
    arow[i] = p.index_a ? op_listed(p.index_a, m, tile.begin, tile.end, p.a_rows, p.per_mul, p.per_shift) : m < tile.end ? m : -1;
  }
  if (tile.expert >= 0) {
    /* buffers: of a from the tile's first row (with an index, from its first), of b from the tile's first column on */
    const int first = p.index_a ? 0 : tile.begin, columns = acc_min(16 * OP_FN, p.nj - j0);
    const __amdgpu_buffer_rsrc_t a = __builtin_amdgcn_make_buffer_rsrc((void *)((const op_mem *)p.a + first * p.a_stride), 0, (int)OP_FARTHEST, 0x00020000);
    const __amdgpu_buffer_rsrc_t b = __builtin_amdgcn_make_buffer_rsrc((void *)((const op_mem *)p.b + tile.expert * p.b_expert + j0 * p.b_stride), 0,
                                                                       (columns - 1) * bstride + row_bytes, 0x00020000);
    unsigned int aat[OP_FM], bat[OP_FN];
#pragma unroll
    for (int i = 0; i < OP_FM; ++i) aat[i] = arow[i] < 0 ? OP_NOWHERE : (unsigned int)((arow[i] - first) * astride) + 16 * g;
#pragma unroll
    for (int j = 0; j < OP_FN; ++j) bat[j] = (unsigned int)((j * 16 + l) * bstride) + 16 * g;
#if OP_TYPE == 3
    const __amdgpu_buffer_rsrc_t as = __builtin_amdgcn_make_buffer_rsrc((void *)(p.a_scales + first * p.a_scales_stride), 0, (int)OP_FARTHEST, 0x00020000);
    const __amdgpu_buffer_rsrc_t bs = __builtin_amdgcn_make_buffer_rsrc((void *)(p.b_scales + tile.expert * p.b_scales_expert + j0 * p.b_scales_stride), 0,
                                                                        (int)((columns - 1) * p.b_scales_stride) + p.k / 16, 0x00020000);
    unsigned int asat[OP_FM], bsat[OP_FN];
#pragma unroll
    for (int i = 0; i < OP_FM; ++i) asat[i] = arow[i] < 0 ? OP_NOWHERE : (unsigned int)((arow[i] - first) * (int)p.a_scales_stride);
#pragma unroll
    for (int j = 0; j < OP_FN; ++j) bsat[j] = (unsigned int)((j * 16 + l) * (int)p.b_scales_stride);
#endif
    for (int at = wave * 128; at < row_bytes; at += OP_WAVES * OP_AHEAD * 128) {
      acc_u4 va[OP_AHEAD][OP_FM][2], vb[OP_AHEAD][OP_FN][2];
#if OP_TYPE == 3
      unsigned int sa[OP_AHEAD][OP_FM][2], sb[OP_AHEAD][OP_FN][2];
#endif
#pragma unroll
      for (int u = 0; u < OP_AHEAD; ++u) {
        const int k = at + u * OP_WAVES * 128;         /* the same in all lanes */
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool in = k + 64 * h + 16 * g < row_bytes;
#pragma unroll
          for (int j = 0; j < OP_FN; ++j) vb[u][j][h] = __builtin_amdgcn_raw_buffer_load_b128(b, in ? bat[j] : OP_NOWHERE, k + 64 * h, 0);
#pragma unroll
          for (int i = 0; i < OP_FM; ++i) va[u][i][h] = __builtin_amdgcn_raw_buffer_load_b128(a, in ? aat[i] : OP_NOWHERE, k + 64 * h, 0);
#if OP_TYPE == 3
          /* (four blocks' scales; the lane's own is the g-th.  Rows are whole fours of blocks) */
          const bool some = k + 64 * h < row_bytes;
#pragma unroll
          for (int j = 0; j < OP_FN; ++j) sb[u][j][h] = __builtin_amdgcn_raw_buffer_load_b32(bs, some ? bsat[j] : OP_NOWHERE, k / 16 + 4 * h, 0);
#pragma unroll
          for (int i = 0; i < OP_FM; ++i) sa[u][i][h] = __builtin_amdgcn_raw_buffer_load_b32(as, some ? asat[i] : OP_NOWHERE, k / 16 + 4 * h, 0);
#endif
        }
      }
      __builtin_amdgcn_sched_barrier(0);               /* (all loads first: left to itself the compiler takes turns, to save registers) */
#pragma unroll
      for (int u = 0; u < OP_AHEAD; ++u)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < OP_FM; ++i)
#pragma unroll
            for (int j = 0; j < OP_FN; ++j) {
              op_frag x, y;
              __builtin_memcpy(&x, &vb[u][j][h], 16);
              __builtin_memcpy(&y, &va[u][i][h], 16);
#if OP_TYPE == 3
              c[i][j] = op_mfma_scaled(x, y, c[i][j], (int)(sb[u][j][h] >> (8 * g)), 0, (int)(sa[u][i][h] >> (8 * g)), 0);
#else
              c[i][j] = op_mfma(x, y, c[i][j]);
#endif
            }
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
    for (int j = 0; j < OP_FN; j += 2) op_write_pair(out, j0 + j * 16, p.nj, g, c[i][j], c[i][j + 1], arow[i] < 0);
  }
}
