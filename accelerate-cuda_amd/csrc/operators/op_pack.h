/*
 * op_pack.h -- an operand whose rows start anywhere, as the products' aligned form wants it: rows of whole chunks of 16 bytes,
 * one behind the other, with zeros behind the last column and the last row (which add nothing to a sum).
 *
 * A lane has a chunk.  Bound by memory: 4690 rows of 3367 bfloat16 and 5 matrices of 2021 x 3367, 31 and 68 MB, take 17.8 us on
 * average, 5.6 TB/s read and written.
 */
#include "op_common.h"

extern "C" __global__ void __launch_bounds__(256) pack(const acc_pack_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const unsigned int n = blockIdx.x * 256 + threadIdx.x, r = p.per_mul ? __umulhi(n, p.per_mul) >> p.per_shift : n;
  if (r >= p.rows_out * p.batches) return;
  const unsigned int batch = r / p.rows_out, row = r - batch * p.rows_out;
  const int c = (int)(n - r * p.chunks) * OP_VALUES;
  const op_elt *from = (const op_elt *)p.in + (long long)batch * p.batch_stride + (long long)row * p.row_stride + c;
  ((acc_u4 *)p.out)[n] = op_chunk<false>(from, row < p.rows ? p.cols - c : 0);
}
