/*
 * op_product.h -- products of segments of rows with a matrix each, on the matrix cores.
 *
 *   rows   out[m, n] = sum_k a[r(m), k] b[e(m), n, k]       for every row m of expert e(m)'s segment
 *   outer  out[e, i, j] = sum_{m in e} a[r(m), i] b[r(m), j]
 *
 * Both are C[i, j] = sum_r A(i, r) B(j, r) over tiles of OP_BM x OP_BN results; what differs is whether an operand's rows in
 * memory run along r (OP_A_FAST, OP_B_FAST) or across it.  A step of the sum covers 128 bytes along r of an operand
 * (64 elements of 16 bits, 32 of Float32).
 */
#include "op_common.h"

#define OP_BR (128 / OP_SIZE)                      /* the step of the sum, in elements */
#define OP_THREADS (64 * OP_WM * OP_WN)
#define OP_FM (OP_BM / OP_WM / 16)                 /* fragments of 16 x 16 that a wave has of the result */
#define OP_FN (OP_BN / OP_WN / 16)

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
#else
typedef __bf16 op_frag __attribute__((ext_vector_type(8)));
ACC_DEV acc_f4 op_mfma(const op_frag x, const op_frag y, const acc_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0); }
#endif

/* One operand's tile of a step in LDS, in chunks of 16 bytes.
 *   rows along r: TILE rows of 8 chunks; row i's chunk c lies at c ^ (i & 7), so that the 16 rows of a fragment are read
 *   from all banks.
 *   rows across r: OP_BR rows of TILE elements.
 * A lane's fragment holds, for its i (lane % 16), the r of its quarter of the wave (lane / 16): 8 of 32 in a row for 16 bits,
 * 4 of 16 for Float32 -- any order of r will do that both operands keep. */
template <bool FAST, int TILE> struct op_operand {
  static constexpr int CHUNKS = TILE * 8;                         /* of a step */
  static constexpr int MINE = (CHUNKS + OP_THREADS - 1) / OP_THREADS;
  static constexpr int PITCH = FAST ? 8 : TILE / OP_EPC;          /* chunks of a row */

  const op_elt *base;
  long long stride;
  const int *index;              /* which row of memory row m of the segments is; 0: its own number */
  const int *gate;               /* outer, the operand without an index: the other one's; a row that has no partner counts as none */
  int per;
  long long limit;               /* rows an index may name */
  int lo, hi;                    /* the rows of memory that count: along r the i's, across it the r's */
  int minor, extent;             /* across r: the tile's first element of a row, and the row's length; along r: -, the sum's length */
  const op_elt *row[FAST ? MINE : 1];

  ACC_DEV const op_elt *address(const int m) const
  {
    if (m < lo || m >= hi) return (const op_elt *)0;
    const int *named = index ? index : gate;
    if (named) {
      const int at = named[m], r = per > 1 ? at / per : at;
      if (at < 0 || r >= limit) return (const op_elt *)0;
      if (index) return base + (long long)r * stride;
    }
    return base + (long long)m * stride;
  }

  ACC_DEV void start(const int tid, const int first)              /* first: along r the tile's first i */
  {
    if (FAST) {
#pragma unroll
      for (int q = 0; q < MINE; ++q) {
        const int s = tid + q * OP_THREADS, i = s / 8;
        row[q] = s < CHUNKS ? address(first + i) : (const op_elt *)0;
        if (row[q]) row[q] += (((s % 8) ^ (i & 7))) * OP_EPC;
      }
    }
  }

  ACC_DEV void load(acc_u4 (&v)[MINE], const int tid, const int r0) const
  {
#pragma unroll
    for (int q = 0; q < MINE; ++q) {
      const int s = tid + q * OP_THREADS;
      if (FAST) {
        const int c = ((s % 8) ^ ((s / 8) & 7)) * OP_EPC;
        v[q] = op_chunk<OP_ALIGNED>(row[q] + r0, row[q] ? extent - (r0 + c) : 0);
      } else {
        const op_elt *p = s < CHUNKS ? address(r0 + s / PITCH) : (const op_elt *)0;
        const int c = minor + (s % PITCH) * OP_EPC;
        v[q] = op_chunk<OP_ALIGNED>(p + c, p ? extent - c : 0);
      }
    }
  }

  ACC_DEV static void store(acc_u4 *lds, const acc_u4 (&v)[MINE], const int tid)
  {
#pragma unroll
    for (int q = 0; q < MINE; ++q) {
      const int s = tid + q * OP_THREADS;
      if (CHUNKS % OP_THREADS == 0 || s < CHUNKS) lds[s] = v[q];
    }
  }

  /* the fragment of rows i0 .. i0 + 15 and the step's half `h` */
  ACC_DEV static op_frag fragment(const acc_u4 *lds, const int i0, const int h, const int lane)
  {
    const int i = i0 + (lane & 15), g = lane >> 4;
    op_frag f;
    if (FAST) {
      const acc_u4 v = lds[i * 8 + ((h * 4 + g) ^ (i & 7))];
      __builtin_memcpy(&f, &v, 16);
    } else {
      const op_elt *e = (const op_elt *)lds;
#pragma unroll
      for (int t = 0; t < OP_EPC; ++t) f[t] = e[(h * (OP_BR / 2) + g * OP_EPC + t) * TILE + i];
    }
    return f;
  }
};

typedef op_operand<OP_A_FAST, OP_BM> op_a;
typedef op_operand<OP_B_FAST, OP_BN> op_b;

extern "C" __global__ void __launch_bounds__(OP_THREADS) product(const acc_product_args p)
{
  if (p.guard && *p.guard == 0u) return;
  __shared__ acc_u4 lds_a[2][op_a::CHUNKS], lds_b[2][op_b::CHUNKS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wi = (wave / OP_WN) * (OP_BM / OP_WM), wj = (wave % OP_WN) * (OP_BN / OP_WN);

  /* the tile, and the sum's range */
  int expert, i0, j0, iend, jend, r0, r1;
#if OP_OUTER
  {
    const long long b = blockIdx.x;
    expert = (int)(b / ((long long)p.tiles_i * p.tiles_j));
    const int t = (int)(b % ((long long)p.tiles_i * p.tiles_j));
    i0 = (t / p.tiles_j) * OP_BM;
    j0 = (t % p.tiles_j) * OP_BN;
    iend = p.ni;
    jend = p.nj;
    op_segment(p.offsets, p.experts, (int)p.rows, expert + 1, &r0, &r1);
  }
#else
  {
    const int t = blockIdx.x / p.tiles_j;
    j0 = (int)(blockIdx.x % p.tiles_j) * OP_BN;
    const op_tile tile = op_find_tile(p.offsets, p.experts, (int)p.rows, OP_BM, t);
    if (tile.begin >= tile.end) return;
    expert = tile.expert;
    i0 = tile.begin;
    iend = tile.end;
    jend = p.nj;
    r0 = 0;
    r1 = expert < 0 ? 0 : p.k;
  }
#endif

  op_a a;
  op_b b;
  a.base = (const op_elt *)p.a;
  a.stride = p.a_stride;
  a.index = p.index_a;
  a.limit = p.a_rows;
  a.gate = b.gate = (const int *)0;
  a.per = b.per = p.per;
  b.base = (const op_elt *)p.b;
  b.stride = p.b_stride;
#if OP_OUTER
  b.index = p.index_b;
  b.limit = p.b_rows;
  if (!p.index_a && p.index_b) { a.gate = p.index_b; a.limit = p.b_rows; }
  if (!p.index_b && p.index_a) { b.gate = p.index_a; b.limit = p.a_rows; }
  a.lo = b.lo = r0;
  a.hi = b.hi = r1;
  a.minor = i0;
  a.extent = p.ni;
  b.minor = j0;
  b.extent = p.nj;
#else
  b.base += (long long)acc_max(expert, 0) * p.b_expert;
  b.index = (const int *)0;
  b.limit = 0;
  a.lo = i0;
  a.hi = iend;
  a.minor = 0;
  a.extent = p.k;
  b.lo = 0;
  b.hi = OP_B_FAST ? jend : p.k;
  b.minor = j0;
  b.extent = OP_B_FAST ? p.k : jend;
#endif
  a.start(tid, i0);
  b.start(tid, j0);

  acc_f4 c[OP_FM][OP_FN];
#pragma unroll
  for (int i = 0; i < OP_FM; ++i)
#pragma unroll
    for (int j = 0; j < OP_FN; ++j) c[i][j] = acc_f4{0.0f, 0.0f, 0.0f, 0.0f};

  acc_u4 va[op_a::MINE], vb[op_b::MINE];
  if (r0 < r1) {
    a.load(va, tid, r0);
    b.load(vb, tid, r0);
  }
  int buf = 0;
  for (int r = r0; r < r1; r += OP_BR, buf ^= 1) {
    /* two buffers, one barrier a step: whoever writes into a buffer has passed the barrier that every wave reached after
     * it last read it */
    op_a::store(lds_a[buf], va, tid);
    op_b::store(lds_b[buf], vb, tid);
    __syncthreads();
    if (r + OP_BR < r1) {
      a.load(va, tid, r + OP_BR);
      b.load(vb, tid, r + OP_BR);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      op_frag fa[OP_FM], fb[OP_FN];
#pragma unroll
      for (int i = 0; i < OP_FM; ++i) fa[i] = op_a::fragment(lds_a[buf], wi + i * 16, h, lane);
#pragma unroll
      for (int j = 0; j < OP_FN; ++j) fb[j] = op_b::fragment(lds_b[buf], wj + j * 16, h, lane);
#pragma unroll
      for (int i = 0; i < OP_FM; ++i)
#pragma unroll
        for (int j = 0; j < OP_FN; ++j) c[i][j] = op_mfma(fb[j], fa[i], c[i][j]);
    }
  }

  /* b's fragment is the instruction's first operand: a lane has four neighbouring j of one i */
#pragma unroll
  for (int i = 0; i < OP_FM; ++i) {
    const int ri = i0 + wi + i * 16 + (lane & 15);
    if (ri >= iend) continue;
    op_elt *out = (op_elt *)p.out + (long long)ri * p.out_stride;
    bool none = false;           /* (a matrix may hold infinities: no row times that is zeros all the same) */
#if OP_OUTER
    out += (long long)expert * p.out_expert;
#else
    none = p.index_a && !a.address(ri);
#endif
#pragma unroll
    for (int j = 0; j < OP_FN; ++j) {
      const int cj = j0 + wj + j * 16 + 4 * (lane >> 4);
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (cj + t < jend) out[cj + t] = (op_elt)(none ? 0.0f : c[i][j][t]);
    }
  }
}
