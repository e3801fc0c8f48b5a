/*
 * op_product.h -- products of segments of rows with a matrix each, on the matrix cores.
 *
 *   rows   out[m, n] = sum_k a[r(m), k] b[e(m), n, k]       for every row m of expert e(m)'s segment
 *   outer  out[e, i, j] = sum_{m in e} a[r(m), i] b[r(m), j]
 *
 * Both are C[i, j] = sum_r A(i, r) B(j, r) over tiles of OP_BM x OP_BN results; what differs is whether an operand's rows in
 * memory run along r (OP_A_FAST, OP_B_FAST) or across it.  A step of the sum covers 128 bytes of an operand along r, a cache
 * line: 64 elements of 16 bits, 32 of Float32, 256 of 4 bits (OP_TYPE 3: both operands as op_micro.h makes them, each with
 * its scales).  Two steps lie in LDS.  The matrix cores work on half a step, whose fragments are in registers, while the next
 * half's are read; one barrier a step, in its middle, says that everybody's share of the next step has arrived and that
 * nobody reads this one any more, so that the next but one may take its place.
 *
 * A wave of the largest tile has 128 x 64 results in 128 registers, and reads 12 fragments of LDS for 32 products of a half step.
 * Of the cycles in which a compute unit has work, the matrix cores are busy in 78 % (8192^3 bfloat16; outer 72, 4 bits 45) and LDS
 * in 29 (27, 22), without a bank conflict; what is left are waits for one another at the barrier, two waves a SIMD covering them
 * only in part, then, where sums are short, the 10 us a tile has in front of its first product and behind its last (32768 rows, 16
 * of 4096 x 2048: 60 %).  Measured: bfloat16 8192^3 along the sum 768 us, 1431 TFLOP/s; the matrix
 * turned 782, both turned (outer) 819, with an index 868; 4 bits 295, 3730; Float32 4096^3 962, 143.  A sum may be in pieces (few
 * tiles, long sums): each is a workgroup's, goes out in Float32, and product_join adds them up in order.
 */
#include "op_matrix.h"

#define OP_THREADS (64 * OP_WM * OP_WN)
#define OP_GROUP (OP_BM >= 256 ? 4 : OP_BM >= 128 ? 8 : 16)   /* rows of tiles that are gone through together: 8192^3 takes a tenth less than column by column */
#define OP_FM (OP_BM / OP_WM / 16)                 /* fragments of 16 x 16 that a wave has of the result */
#define OP_FN (OP_BN / OP_WN / 16)

/* OP_INDEX, outer: 0: no index, 1: of b's rows, 2: of a's */
#define OP_PLAIN 0
#define OP_LISTED 1
#define OP_GATED 2

typedef __attribute__((address_space(3))) void *op_lds_ptr;

/* Where row r of an operand lies, in bytes, as a load takes it whose buffer ends before 2 GB: the top bit set, and none (r < 0)
 * is 0 -- as a load of such a number beyond the end of a buffer of them is.  With that bit turned, it is an offset, and none
 * is beyond the end of every buffer. */
ACC_DEV unsigned int op_place_of(const int r, const int stride) { return r < 0 ? 0u : (unsigned int)(r * stride) | OP_NOWHERE; }

/* One operand's share of a step in LDS, in chunks of 16 bytes.
 *   rows along r: TILE rows of 8 chunks; row i's chunk c lies at c ^ (i % 8): the eight lanes that are served together read
 *     neighbouring rows' chunks from all banks.
 *   rows across r: OP_STEP rows of TILE elements; a row's units of 16 elements lie at u ^ f(r), so that the rows that are
 *     read together (four neighbours, for 16 bits, and those eight further on; every fourth, for Float32) lie in other banks.
 * A lane's fragment holds, for its i (lane % 16), the r of its quarter of the wave (lane / 16): 8 of 32 in a row for 16 bits,
 * 4 of 16 for Float32, a block of 32 for 4 bits.
 *
 * OP_ALIGNED: rows are whole chunks and start on one.  A lane's chunks go from memory straight to LDS, by way of a buffer
 * that starts at the tile (or the step) and ends where the rows that count do: what lies beyond reads as zeros, and
 * addresses are one offset of 32 bits a chunk (the driver sees to it that they suffice).
 * Otherwise rows start anywhere; chunks go by way of registers, with addresses of 64 bits.  A chunk that would reach
 * beyond its row's end is read that much earlier and shifted into place, or, across r, where it ends within the next row
 * and that is there, read as it lies (see `whole`): no read leaves the operand.  128 x 128 tiles, half, 5003 rows of 24 segments
 * by 1333 x 1001: 46 us, 41 in the aligned form by 1336 x 1000; 5000 x 5001 x 5001: 475, so that large ones are copied first. */
template <bool FAST, int TILE, int WAVES, int LIST> struct op_operand {
  static constexpr int CHUNKS = TILE * 8;                         /* of a step */
  static constexpr int MINE = (CHUNKS + OP_THREADS - 1) / OP_THREADS;
  static constexpr int PITCH = FAST ? 8 : TILE / OP_EPC;          /* chunks of a row */
  static constexpr int UNITS = TILE / 16;                         /* across r: of a row */
  static constexpr int SIZE = (int)sizeof(op_mem);
  /* 4 bits: the scales of a step's rows lie behind them, those of the first half, then of the second; in each, words that hold
   * the same block of up to four rows 16 apart, as the fragments of a wave's up to 64 rows want them */
  static constexpr int SHARE = TILE / WAVES < 64 ? TILE / WAVES : 64;
  static constexpr int SCALE_WORDS = TILE / SHARE * 64;           /* of a half */
  static constexpr int SCALES = OP_TYPE == 3 ? 2 * SCALE_WORDS / 4 : 0;
  static_assert(CHUNKS % 64 == 0 && (CHUNKS % OP_THREADS == 0 || OP_THREADS % CHUNKS == 0), "whole waves, the same number each");

  const unsigned char *base;     /* along r: of the operand; across it: of the tile's first column */
  long long stride;              /* of a row, in bytes */
  const int *index;              /* which row of memory row m of the segments is; 0: its own number.  LIST: OP_PLAIN: there is none;
                                  * OP_LISTED: along r perhaps one, across r one; OP_GATED: the other operand's (a row without
                                  * a partner counts as none) */
  unsigned int per_mul, per_shift;
  int limit;                     /* rows of the operand that an index may name; across r: rows that there are */
  int lo, hi;                    /* the rows that count: along r the i's, across it the r's */
  int extent;                    /* elements of a row that count, from `base` on */
  int column;                    /* along r: the lane's chunks' first element (the same of all of them) */
  /* whether a lane's chunks lie equally far apart in memory: the rows between them are as many, and swizzled alike (for
   * Float32 across r they are not) */
  static constexpr bool EVEN = FAST ? LIST == OP_PLAIN : OP_TYPE != 0;
  static constexpr int APART = CHUNKS < OP_THREADS ? 0 : OP_THREADS / PITCH;
#if OP_ALIGNED
  unsigned int offset[EVEN ? 1 : MINE];   /* of the lane's chunks, in bytes: along r from the tile's first row, across it from the step's */
  __amdgpu_buffer_rsrc_t buffer; /* along r */
#else
  long long offset[!FAST && EVEN ? 1 : MINE];   /* of the lane's chunks, in bytes: along r from `base`, across it from the step's first row (with an index:
                                  * from the row's beginning) */
#endif
  /* a lane's q-th chunk of a step: where there are fewer chunks than lanes, several waves bring the same ones */
  ACC_DEV static int slot(const int tid, const int q) { return CHUNKS < OP_THREADS ? tid % CHUNKS : tid + q * OP_THREADS; }
  ACC_DEV static int swizzle(const int r)
  {
    return (OP_TYPE == 0 ? r >> 2 & 3 : (r & 3) | (r >> 1 & 4)) & (UNITS - 1);
  }
  /* of a slot: its row, and its first element there */
  ACC_DEV static int major(const int s) { return s / PITCH; }
  ACC_DEV static int element(const int s)
  {
    const int i = s / PITCH, c = s % PITCH;
    if (FAST) return (c ^ (i & 7)) * OP_EPC;
    constexpr int U = 16 / OP_EPC;                                /* chunks of a unit: 2 of 16 bits, 4 of Float32 */
    return ((c / U ^ swizzle(i)) * U + c % U) * OP_EPC;
  }

  /* which row of memory row m is, along r; -1: none */
  ACC_DEV int number(const int m) const
  {
    if (LIST == OP_PLAIN || !index) return m < hi ? m : -1;
    return op_listed(index, m, lo, hi, limit, per_mul, per_shift);
  }

  /* along r: where the lane's rows are, from row `first` on; across r: where its columns are */
  ACC_DEV void start(const int tid, const int first)
  {
    column = FAST ? element(slot(tid, 0)) : 0;
#if OP_ALIGNED
    if (FAST) {
      /* (rows behind the last that counts may be read if there are any: what comes of them is not written) */
      const unsigned char *from = index ? base : base + first * stride;
      const long long rows = index ? limit : hi - first;
      buffer = __builtin_amdgcn_make_buffer_rsrc((void *)from, 0, (int)acc_min<long long>(OP_FARTHEST, rows > 0 ? (rows - 1) * stride + (long long)extent * SIZE : 0), 0x00020000);
    }
#endif
    /* (an index is read of all rows at once: one after the other, four times its latency stood in front of a tile) */
    int rows_of[MINE];
    if (FAST && LIST != OP_PLAIN) {
      if (index) {
#pragma unroll
        for (int q = 0; q < MINE; ++q) rows_of[q] = op_entry(index, first + major(slot(tid, q)), lo, hi);
#pragma unroll
        for (int q = 0; q < MINE; ++q) rows_of[q] = op_named(rows_of[q], first + major(slot(tid, q)), lo, hi, limit, per_mul, per_shift);
      } else {
#pragma unroll
        for (int q = 0; q < MINE; ++q) rows_of[q] = first + major(slot(tid, q)) < hi ? first + major(slot(tid, q)) : -1;
      }
    }
#pragma unroll
    for (int q = 0; q < MINE; ++q) {
      const int s = slot(tid, q), m = first + major(s), number = FAST && LIST != OP_PLAIN ? rows_of[q] : m < hi ? m : -1;
#if OP_ALIGNED
      if (EVEN && q > 0) continue;
      if (FAST) {
        /* (without an index, the rows that do not count lie behind the buffer's end) */
        const int r = LIST == OP_PLAIN ? m : number;
        offset[q] = r < 0 ? OP_NOWHERE : (unsigned int)((LIST == OP_LISTED && index ? r : r - first) * (int)stride + element(s) * SIZE);
      } else {
        /* (columns beyond the result's: any will do) */
        offset[q] = (unsigned int)(element(s) < extent ? element(s) : 0) * SIZE + (LIST == OP_LISTED ? 0 : (unsigned int)(major(s) * (int)stride));
      }
#else
      if (!FAST && EVEN && q > 0) continue;
      /* (a row that does not count: the operand's first, which there is where there are steps at all; what comes of it is not written) */
      offset[q] = FAST ? acc_max(number, 0) * stride + column * SIZE : (element(s) < extent ? element(s) : 0) * SIZE + (LIST == OP_PLAIN ? major(s) * stride : 0);
#endif
    }
  }

#if OP_ALIGNED
  /* ask for the lane's q-th chunk of the step at r, straight to LDS; `wave` is the same in all lanes, and known to be.
   * `named`, across r with an index: where the chunk's row lies (see op_place_of) */
  ACC_DEV void bring(acc_u4 *lds, const int wave, const int q, const int r, const int named) const
  {
    const op_lds_ptr to = (op_lds_ptr)(lds + (CHUNKS < OP_THREADS ? wave * 64 % CHUNKS : wave * 64 + q * OP_THREADS));
    const unsigned int at = offset[EVEN ? 0 : q];
    const int further = EVEN ? q * APART * (int)stride : 0;       /* (the same in all lanes) */
    if (FAST) {
      const unsigned int from = r + column < extent ? at : OP_NOWHERE;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, to, 16, from, r * SIZE + further, 0, 0);
    } else if (LIST == OP_LISTED) {
      const __amdgpu_buffer_rsrc_t all = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)OP_FARTHEST, 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(all, to, 16, ((unsigned int)named ^ OP_NOWHERE) + at, 0, 0, 0);
    } else {
      const __amdgpu_buffer_rsrc_t rest =
          __builtin_amdgcn_make_buffer_rsrc((void *)(base + r * stride), 0, (int)acc_min<long long>(OP_FARTHEST, acc_max(0, hi - r) * stride), 0x00020000);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rest, to, 16, LIST == OP_GATED ? (((unsigned int)named ^ OP_NOWHERE) & OP_NOWHERE) | at : at, further, 0, 0);
    }
  }
#else
  /* the same by way of registers: `load` asks, whoever has asked puts what has come into LDS a step later.  `whole`: every
   * chunk of the step is read where it lies.  Along r, all of them end within their rows.  Across r, without an index every row
   * counts; and a chunk that reaches beyond its row's end ends within the next one (what it holds of that makes results that
   * are not written), so that none of the step's rows may be the operand's last.  OP_TINY: a row is shorter than a chunk. */
  template <int N> ACC_DEV bool whole(const int r, const int (&named)[N]) const
  {
    if (OP_TINY) return false;
    if (FAST) return r + OP_STEP <= extent;
    bool inside = extent >= TILE;
    if (!inside && stride >= 16) {
      if (LIST == OP_LISTED) {
        bool last = limit < 2;
#pragma unroll
        for (int q = 0; q < MINE; ++q) last |= named[q] == limit - 1;
        inside = __ballot(last) == 0;
      } else {
        inside = r + OP_STEP < limit;
      }
    }
    return inside & ((LIST != OP_PLAIN) | (r + OP_STEP <= hi));
  }
  ACC_DEV void load(acc_u4 &v, const int tid, const int q, const int r, const int named, const bool whole) const
  {
    const int s = slot(tid, q);
    if (whole) {
      const unsigned char *p;
      if (FAST) p = base + (long long)r * SIZE + offset[q];
      else if (LIST == OP_PLAIN) p = base + (r + (EVEN ? q * APART : 0)) * stride + offset[EVEN ? 0 : q];
      else p = base + (named < 0 ? 0 : LIST == OP_GATED ? r + major(s) : named) * stride + offset[EVEN ? 0 : q];
      v = ((const op_loose<op_mem> *)p)->v;
      if (!FAST && LIST != OP_PLAIN && named < 0) v = acc_u4{0, 0, 0, 0};
      return;
    }
    /* elements of the row that are wanted first, and how many there are */
    const int m = r + major(s), n = FAST ? 0 : LIST == OP_PLAIN ? (m < hi ? m : -1) : LIST == OP_GATED && named >= 0 ? m : named, c = FAST ? r + column : element(s);
    const unsigned char *row = FAST ? base + offset[q] - column * SIZE : base + (long long)acc_max(n, 0) * stride;
#if OP_TINY
    op_mem e[OP_EPC];
#pragma unroll
    for (int k = 0; k < OP_EPC; ++k) e[k] = c + k < extent ? ((const op_mem *)row)[c + k] : (op_mem)0;
    __builtin_memcpy(&v, e, 16);
#else
    const int at = acc_min(c, extent - OP_EPC);
    v = op_shifted(((const op_loose<op_mem> *)(row + (long long)at * SIZE))->v, (c - at) * SIZE);
#endif
    if (n < 0) v = acc_u4{0, 0, 0, 0};
  }
#endif

  /* Where a lane's part of the fragments of a wave lies whose first row is `first`, a multiple of 64 or all that the waves
   * have: worked out once, so that a fragment is a constant further on (along r), or an exclusive or (across it). */
  struct reader {
    int at[2];                   /* along r: chunks, of either half; across r: elements */
    int unit, flip;              /* across r: the wave's first unit, and what the lane's rows have theirs flipped by */
    int scale;                   /* 4 bits: words, behind the chunks */
  };
  ACC_DEV static reader reads(const int first, const int lane)
  {
    const int l = lane & 15, g = lane >> 4;
    reader w = {};
    if (FAST) {
      w.at[0] = (first + l) * 8 + (g ^ (l & 7));
      w.at[1] = (first + l) * 8 + ((4 + g) ^ (l & 7));
      w.scale = first / SHARE * 64 + g * 16 + l;
    } else {
      const int r = OP_TYPE == 0 ? 4 * g : 8 * g + (l >> 2);
      w.at[0] = r * TILE + (OP_TYPE == 0 ? l : (l & 3) * 4);
      w.at[1] = w.at[0] + OP_STEP / 2 * TILE;
      w.unit = first / 16;
      w.flip = swizzle(r);
    }
    return w;
  }
  /* the n-th fragment of the step's half h */
  ACC_DEV static op_frag fragment(const acc_u4 *lds, const reader &w, const int n, const int h)
  {
    op_frag f;
    if (FAST) {
      const acc_u4 v = lds[w.at[h] + n * 128];
      __builtin_memcpy(&f, &v, 16);
    } else {
      const int at = w.at[h] + (((w.unit + n) ^ w.flip) << 4);
#if OP_TYPE == 0
      const float *e = (const float *)lds + at;
#pragma unroll
      for (int t = 0; t < 4; ++t) f[t] = e[t * TILE];
#else
      /* 4 x 16 elements at a time, turned on the way: lane l of a quarter names the four of row l / 4 from 4 (l % 4) on, and
       * gets the four rows' l-th */
      typedef short op_s4 __attribute__((ext_vector_type(4)));
      const short *e = (const short *)lds + at;
      const op_s4 one = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) op_s4 *)e);
      const op_s4 two = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) op_s4 *)(e + 4 * TILE));
      __builtin_memcpy(&f, &one, 8);
      __builtin_memcpy((char *)&f + 8, &two, 8);
#endif
    }
    return f;
  }
  /* 4 bits: the scales of fragments 4 n to 4 n + 3 */
  ACC_DEV static int scale(const acc_u4 *lds, const reader &w, const int n, const int h) { return ((const int *)(lds + CHUNKS))[w.scale + h * SCALE_WORDS + n * 64]; }
};

typedef op_operand<OP_A_FAST, OP_BM, OP_WM, OP_A_FAST ? OP_LISTED : OP_INDEX == 0 ? OP_PLAIN : OP_INDEX == 1 ? OP_GATED : OP_LISTED> op_a;
typedef op_operand<OP_B_FAST, OP_BN, OP_WN, OP_INDEX == 0 ? OP_PLAIN : OP_INDEX == 1 ? OP_LISTED : OP_GATED> op_b;

/* a step of both operands */
#define OP_STAGE (op_a::CHUNKS + op_a::SCALES + op_b::CHUNKS + op_b::SCALES)
#define OP_B_AT (op_a::CHUNKS + op_a::SCALES)

/* Half a step: the products of fa and fb; meanwhile half h of the step in `lds` is read into na and nb, a few fragments for
 * every row of products, and `also(i)`, i from 0 to OP_FM - 1, goes on.  The order is kept as it stands here: left to itself
 * the compiler puts all reads in front of all products.  b's fragment is the instruction's first operand: a lane then has
 * four neighbouring j of one i.
 * OP_ROLL: na is fa, a fragment of which is read anew as soon as its products are under way.  That is for the forms whose
 * addresses and scales leave no registers for a second set. */
#define OP_SM ((OP_FM + 3) / 4)
#define OP_SN ((OP_FN + 3) / 4)
#define OP_ROLL (OP_TYPE == 3 || OP_OUTER || (OP_TYPE == 0 && !OP_B_FAST))
template <typename F>
ACC_DEV void op_half(acc_f4 (&c)[OP_FM][OP_FN], op_frag (&fa)[OP_FM], op_frag (&fb)[OP_FN], op_frag (&na)[OP_FM], op_frag (&nb)[OP_FN],
#if OP_TYPE == 3
                     const int (&sa)[OP_SM], const int (&sb)[OP_SN], int (&nsa)[OP_SM], int (&nsb)[OP_SN],
#endif
                     const acc_u4 *lds, op_a::reader wa, op_b::reader wb, const int h, F also)
{
  /* (not to be worked out for every fragment ahead of the loop: there are not the registers for that) */
  if (!OP_A_FAST) asm volatile("" : "+v"(wa.flip));
  if (!OP_B_FAST) asm volatile("" : "+v"(wb.flip));
  constexpr int READS = OP_ROLL ? (OP_FN + OP_FM - 1) / OP_FM : (OP_FM + OP_FN + OP_FM - 1) / OP_FM;
#pragma unroll
  for (int i = 0; i < OP_FM; ++i) {
#pragma unroll
    for (int n = i * READS; n < (i + 1) * READS; ++n) {
#if OP_TYPE == 3
      if (n % 4 == 0 && n < OP_FN) nsb[n / 4] = op_b::scale(lds + OP_B_AT, wb, n / 4, h);
#endif
      if (n < OP_FN) nb[n] = op_b::fragment(lds + OP_B_AT, wb, n, h);
      else if (!OP_ROLL && n < OP_FN + OP_FM) na[n - OP_FN] = op_a::fragment(lds, wa, n - OP_FN, h);
    }
    also(i);
#pragma unroll
#if OP_TYPE == 3
    for (int j = 0; j < OP_FN; ++j) c[i][j] = op_mfma_scaled(fb[j], fa[i], c[i][j], sb[j / 4], j % 4, sa[i / 4], i % 4);
    if (i % 4 == 0) nsa[i / 4] = op_a::scale(lds, wa, i / 4, h);
#else
    for (int j = 0; j < OP_FN; ++j) c[i][j] = op_mfma(fb[j], fa[i], c[i][j]);
#endif
    if (OP_ROLL) fa[i] = op_a::fragment(lds, wa, i, h);
    __builtin_amdgcn_sched_barrier(0);
  }
}

/* everything that this wave has asked for has come (what it asked for LDS, too), then everybody's */
ACC_DEV void op_meet(const bool loads)
{
  if (loads) __builtin_amdgcn_s_waitcnt(0 | 7 << 4);              /* vmcnt and lgkmcnt 0, in this target's encoding */
  else __builtin_amdgcn_s_waitcnt(15 | 7 << 4 | 3 << 14);         /* lgkmcnt 0 */
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

/* outer, OP_PLACES: where the rows lie that an index names, worked out once for all tiles (not OP_ALIGNED: their numbers, and one
 * more; 0, as beyond the end, is none) */
#if OP_PLACES
extern "C" __global__ void __launch_bounds__(256) product_places(const acc_product_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const int m = (int)(blockIdx.x * 256 + threadIdx.x);
  if (m >= p.rows) return;
  const int r = op_listed(OP_INDEX == 1 ? p.index_b : p.index_a, m, 0, (int)p.rows, OP_INDEX == 1 ? p.b_rows : p.a_rows, p.per_mul, p.per_shift);
  p.places[m] = OP_ALIGNED ? op_place_of(r, (int)(OP_INDEX == 1 ? p.b_stride : p.a_stride) * (int)sizeof(op_mem)) : (unsigned int)(r + 1);
}
#endif

/* (at least two waves a SIMD: more than 256 registers would leave a compute unit to a workgroup of four waves) */
extern "C" __global__ void __launch_bounds__(OP_THREADS) __attribute__((amdgpu_waves_per_eu(2))) product(const acc_product_args p)
{
  if (p.guard && *p.guard == 0u) return;
  /* (two variables, not one of two parts: loads to one are then known to leave the other alone) */
  __shared__ acc_u4 lds0[OP_STAGE], lds1[OP_STAGE];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = (wave / OP_WN) * (OP_BM / OP_WM), wj = (wave % OP_WN) * (OP_BN / OP_WN);

  /* the tile, and the sum's range; every die has a run of tiles of its own, neighbours of which share operands */
  int expert, i0, j0, iend, jend, r0, r1;
  float *part = (float *)0;     /* where a piece of a sum goes */
#if OP_OUTER
  {
    /* (segments are of any length: the longest first, each on all dies) */
    const int tiles = p.tiles_i * p.tiles_j, n = (int)(blockIdx.x / tiles);
    int i, j;
    if (p.piece == 0) {
      expert = op_nth_longest(p.offsets, p.experts, (int)p.rows, n, &r0, &r1);
    } else {
      const op_tile run = op_find_tile<OP_ALL>(p.offsets, p.experts, (int)p.rows, p.piece, op_segments(p.offsets, p.experts, (int)p.rows, 0, 0), n);
      if (run.expert < 0) return;
      expert = run.expert;
      if (run.all > p.piece) part = p.parts + (long long)n * p.ni * p.nj;
      r0 = run.begin;
      r1 = run.end;
    }
    op_grouped((int)op_die_run(blockIdx.x % tiles, tiles), p.tiles_i, p.tiles_j, OP_GROUP, &i, &j);
    i0 = i * OP_BM;
    j0 = j * OP_BN;
    iend = p.ni;
    jend = p.nj;
  }
#else
  {
    /* Whole tiles first, then those that end a segment, which take less long.  (The grid is for the worst lengths; the tiles
     * that there are, are shared out evenly.) */
    int whole, rest, i, j;
    const op_lot lot = op_segments(p.offsets, p.experts, (int)p.rows, 0, 0);
    op_count_tiles(p.offsets, p.experts, (int)p.rows, OP_BM, lot, &whole, &rest);
    const unsigned int grid = (unsigned int)(p.tiles_i * p.tiles_j), n = p.piece ? blockIdx.x / grid : 0u, at = blockIdx.x - n * grid;
    const long long first = (long long)whole * p.tiles_j, all = first + (long long)rest * p.tiles_j;
    if (at >= all) return;
    op_tile tile;
    if (at < first) {
      op_grouped((int)op_die_run(at, first), whole, p.tiles_j, OP_GROUP, &i, &j);
      tile = op_find_tile<OP_WHOLE>(p.offsets, p.experts, (int)p.rows, OP_BM, lot, i);
    } else {
      op_grouped((int)op_die_run(at - first, all - first), rest, p.tiles_j, OP_GROUP, &i, &j);
      tile = op_find_tile<OP_REST>(p.offsets, p.experts, (int)p.rows, OP_BM, lot, i);
    }
    j0 = j * OP_BN;
    if (tile.begin >= tile.end) return;
    expert = tile.expert;
    i0 = tile.begin;
    iend = tile.end;
    jend = p.nj;
    r0 = 0;
    r1 = expert < 0 ? 0 : p.k;
    if (p.piece) {
      part = p.parts + n * p.rows * p.nj;
      r0 = acc_min(r1, (int)n * p.piece);
      r1 = acc_min(r1, r0 + p.piece);
    }
  }
#endif

#if !OP_ALIGNED
  /* (a last column of tiles that would reach beyond the result's edge across r starts earlier: some results are worked out
   * twice, to the same value, and no chunk reaches beyond its row) */
  if (OP_OUTER) i0 = acc_max(0, acc_min(i0, p.ni - OP_BM));
  if (!OP_B_FAST) j0 = acc_max(0, acc_min(j0, p.nj - OP_BN));
  /* (rows of an operand that has none: there is nothing to add up, and no first row to read in their place) */
  if ((OP_INDEX == 1 ? p.b_rows : p.a_rows) < 1) r1 = r0;
#endif
  op_a a;
  op_b b;
  a.base = (const unsigned char *)p.a;
  b.base = (const unsigned char *)p.b;
  a.stride = p.a_stride * op_a::SIZE;
  b.stride = p.b_stride * op_b::SIZE;
  a.index = p.index_a;
  a.limit = p.a_rows;
  a.per_mul = b.per_mul = p.per_mul;
  a.per_shift = b.per_shift = p.per_shift;
#if OP_OUTER
  b.index = (const int *)0;
  b.limit = p.b_rows;
  a.lo = b.lo = r0;
  a.hi = b.hi = r1;
  a.base += (long long)i0 * op_a::SIZE;
  b.base += (long long)j0 * op_b::SIZE;
  a.extent = p.ni - i0;
  b.extent = p.nj - j0;
  a.start(tid, r0);
  b.start(tid, r0);
#else
  b.base += acc_max(expert, 0) * p.b_expert * op_b::SIZE;
  b.index = (const int *)0;
  b.limit = p.k;
  /* (both end where the sum does, which in pieces is not where the rows do: the step behind it has to be zeros, see the loop) */
  a.lo = i0;
  a.hi = iend;
  a.extent = r1;
  b.lo = 0;
  if (OP_B_FAST) {
    b.hi = jend;
    b.extent = r1;
  } else {
    b.hi = r1;
    b.base += (long long)j0 * op_b::SIZE;
    b.extent = jend - j0;
  }
  a.start(tid, i0);
  b.start(tid, OP_B_FAST ? j0 : 0);
#endif

  acc_f4 c[OP_FM][OP_FN];
#pragma unroll
  for (int i = 0; i < OP_FM; ++i)
#pragma unroll
    for (int j = 0; j < OP_FN; ++j) c[i][j] = acc_f4{0.0f, 0.0f, 0.0f, 0.0f};

  if (r0 < r1) {
    op_frag fa[OP_FM], fb[OP_FN], ga[OP_FM], gb[OP_FN];
    const auto nothing = [](int) {};
    /* outer, with an index: which rows of memory the rows of the lane's chunks are, of the step that is to be asked for next
     * -- in the aligned form, where they lie.  (The tile is square: the same rows for both operands.)  With OP_PLACES another
     * kernel has worked that out: the tile of 256 x 256 leaves no registers for it, and its spilled registers' loads would
     * wait for the chunks' (8192^3: 825 TFLOP/s). */
    int named[op_a::MINE > op_b::MINE ? op_a::MINE : op_b::MINE] = {};
#if OP_PLACES
    const __amdgpu_buffer_rsrc_t places = __builtin_amdgcn_make_buffer_rsrc((void *)p.places, 0, r1 * 4, 0x00020000);
    const int mine_at = op_a::major(op_a::slot(tid, 0)) * 4;
#endif
    const auto look_at = [&](const int q, const int r) {
#if OP_PLACES
      if (q < op_a::MINE) named[q] = (int)__builtin_amdgcn_raw_buffer_load_b32(places, mine_at, (r + q * op_a::APART) * 4, 0) - (OP_ALIGNED ? 0 : 1);
#elif OP_INDEX != 0
      static_assert(OP_BM == OP_BN, "a row for both");
      if (q < op_a::MINE) {
        named[q] = op_listed(OP_INDEX == 1 ? p.index_b : p.index_a, r + op_a::major(op_a::slot(tid, q)), r0, r1, OP_INDEX == 1 ? p.b_rows : p.a_rows, p.per_mul, p.per_shift);
#if OP_ALIGNED
        named[q] = (int)op_place_of(named[q], (int)(OP_INDEX == 1 ? b.stride : a.stride));
#endif
      }
#endif
    };
    const auto look = [&](const int r) {
#pragma unroll
      for (int q = 0; q < op_a::MINE; ++q) look_at(q, r);
    };
#if OP_TYPE == 3
    /* The scales go by way of registers, a lane a row of either operand: asked for two steps ahead of their use, put into LDS
     * one step ahead. */
    int fsa[OP_SM], fsb[OP_SN], gsa[OP_SM], gsb[OP_SN];
    static_assert(OP_BM + OP_BN <= OP_THREADS, "a lane a row");
    const int at = tid % (OP_BM + OP_BN), blocks = r1 / 16;
    const bool of_a = at < OP_BM;
    const int si = of_a ? at : at - OP_BM, share = of_a ? op_a::SHARE : op_b::SHARE;
    const int scale_row = of_a ? a.number(i0 + si) : b.number(j0 + si);
    /* (a row that there is not reads the matrix's first scales: what comes of it is not written) */
    const unsigned char *scales = of_a && scale_row >= 0 ? p.a_scales + scale_row * p.a_scales_stride
                                                         : p.b_scales + expert * p.b_scales_expert + acc_max(scale_row, 0) * p.b_scales_stride;
    const int scale_byte = (of_a ? op_a::CHUNKS * 16 : (OP_B_AT + op_b::CHUNKS) * 16) + (si / share * 64 + si % 16) * 4 + si % share / 16;
    const int scale_half = (of_a ? op_a::SCALE_WORDS : op_b::SCALE_WORDS) * 4;
    struct __attribute__((packed)) op_word { unsigned int v; };
    unsigned int scale[2];
    const auto ask_scales = [&](const int r) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = r / 16 + 4 * h;
#if OP_TINY
        /* (a row has fewer than four) */
        scale[h] = 0;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const unsigned int one = scales[acc_min(k + n, blocks - 1)];
          scale[h] |= (k + n < blocks ? one : 0u) << (8 * n);
        }
#else
        /* four, wherever they start; beyond the row's end its last four, which are shifted into place when they have come */
        scale[h] = ((const op_word *)(scales + acc_min(k, blocks - 4)))->v;
#endif
      }
    };
    const auto put_scales = [&](acc_u4 *lds, const int r) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int beyond = OP_TINY ? 0 : acc_max(0, r / 16 + 4 * h - (blocks - 4));
        const unsigned int four = beyond < 4 ? scale[h] >> (8 * beyond) : 0u;
#pragma unroll
        for (int n = 0; n < 4; ++n) ((unsigned char *)lds)[scale_byte + h * scale_half + n * 64] = (unsigned char)(four >> (8 * n));
      }
    };
#define OP_SCALES_F fsa, fsb, gsa, gsb,
#define OP_SCALES_G gsa, gsb, fsa, fsb,
#else
#define OP_SCALES_F
#define OP_SCALES_G
    const auto ask_scales = [](int) {};
    const auto put_scales = [](acc_u4 *, int) {};
#endif
    const op_a::reader wa = op_a::reads(wi, lane);
    const op_b::reader wb = op_b::reads(wj, lane);
    const auto first = [&]() {
#pragma unroll
      for (int j = 0; j < OP_FN; ++j) fb[j] = op_b::fragment(lds0 + OP_B_AT, wb, j, 0);
#pragma unroll
      for (int i = 0; i < OP_FM; ++i) fa[i] = op_a::fragment(lds0, wa, i, 0);
#if OP_TYPE == 3
#pragma unroll
      for (int j = 0; j < OP_SN; ++j) fsb[j] = op_b::scale(lds0 + OP_B_AT, wb, j, 0);
#pragma unroll
      for (int i = 0; i < OP_SM; ++i) fsa[i] = op_a::scale(lds0, wa, i, 0);
#endif
    };
    /* a lane's chunks of a step, shared out over the half's fragments */
    constexpr int ALL = op_a::MINE + op_b::MINE, EACH = (ALL + OP_FM - 1) / OP_FM;
#if OP_ALIGNED
    const auto bring = [&](acc_u4 *lds, const int n, const int r) {
      if (n < op_a::MINE) a.bring(lds, wave, n, r, named[n]);
      else if (n < ALL) b.bring(lds + OP_B_AT, wave, n - op_a::MINE, r, named[n - op_a::MINE]);
    };
    look(r0);
    ask_scales(r0);
#pragma unroll
    for (int n = 0; n < ALL; ++n) bring(lds0, n, r0);
    put_scales(lds0, r0);
    ask_scales(r0 + OP_STEP);
    look(r0 + OP_STEP);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < ALL; ++n) bring(lds1, n, r0 + OP_STEP);
    __builtin_amdgcn_sched_barrier(0);
    /* the first step has come when no more than the second one's loads, which were asked for behind it, are under way */
    __builtin_amdgcn_s_waitcnt((ALL & 15) | 7 << 4 | (ALL >> 4) << 14);
    op_meet(false);
    put_scales(lds1, r0 + OP_STEP);
    ask_scales(r0 + 2 * OP_STEP);
    first();
    /* the step at r lies in `here`, the fragments of its first half in fa, fb */
    const auto round = [&](acc_u4 *here, acc_u4 *there, const int r) {
      op_half(c, fa, fb, ga, gb, OP_SCALES_F here, wa, wb, 1, [&](const int i) {
        look_at(i, r + 2 * OP_STEP);
      });
      op_meet(true);
      put_scales(here, r + 2 * OP_STEP);
      ask_scales(r + 3 * OP_STEP);
      op_half(c, OP_ROLL ? fa : ga, gb, fa, fb, OP_SCALES_G there, wa, wb, 0, [&](const int i) {
#pragma unroll
        for (int n = 0; n < EACH; ++n) bring(here, i * EACH + n, r + 2 * OP_STEP);
      });
    };
#else
    acc_u4 va[op_a::MINE], vb[op_b::MINE];
#define OP_LOAD(r)                                                                          \
    do {                                                                                    \
      if (a.whole(r, named) & b.whole(r, named)) {                                                        \
        _Pragma("unroll") for (int n = 0; n < op_a::MINE; ++n) a.load(va[n], tid, n, r, named[n], true);  \
        _Pragma("unroll") for (int n = 0; n < op_b::MINE; ++n) b.load(vb[n], tid, n, r, named[n], true);  \
      } else if ((r) < r1) {                                                                \
        _Pragma("unroll") for (int n = 0; n < op_a::MINE; ++n) a.load(va[n], tid, n, r, named[n], false); \
        _Pragma("unroll") for (int n = 0; n < op_b::MINE; ++n) b.load(vb[n], tid, n, r, named[n], false); \
      } else {                                                                              \
        _Pragma("unroll") for (int n = 0; n < op_a::MINE; ++n) va[n] = acc_u4{0, 0, 0, 0};  \
        _Pragma("unroll") for (int n = 0; n < op_b::MINE; ++n) vb[n] = acc_u4{0, 0, 0, 0};  \
      }                                                                                     \
      look((r) + OP_STEP);                                                                  \
      ask_scales(r);                                                                        \
    } while (0)
#define OP_STORE(lds, r)                                                                     \
    do {                                                                                    \
      _Pragma("unroll") for (int n = 0; n < op_a::MINE; ++n) lds[op_a::slot(tid, n)] = va[n];           \
      _Pragma("unroll") for (int n = 0; n < op_b::MINE; ++n) lds[OP_B_AT + op_b::slot(tid, n)] = vb[n]; \
      put_scales(lds, r);                                                                   \
    } while (0)
    look(r0);
    OP_LOAD(r0);
    OP_STORE(lds0, r0);
    OP_LOAD(r0 + OP_STEP);
    op_meet(false);
    first();
    const auto round = [&](acc_u4 *here, acc_u4 *there, const int r) {
      OP_STORE(there, r + OP_STEP);
      OP_LOAD(r + 2 * OP_STEP);
      op_half(c, fa, fb, ga, gb, OP_SCALES_F here, wa, wb, 1, nothing);
      op_meet(false);
      op_half(c, OP_ROLL ? fa : ga, gb, fa, fb, OP_SCALES_G there, wa, wb, 0, nothing);
    };
#endif
    /* (An odd number of steps has one of zeros behind it: with a way out between the two, the sums would change registers.  What
     * makes it zeros is that operands end at r1 -- extent along r, hi across it -- and not where their rows do.) */
    int r = r0;
#if OP_ALIGNED
    if (i0 + wi >= iend) {
      /* a wave whose rows lie behind the segment's end only brings its share */
      const auto idle = [&](acc_u4 *here, const int r) {
#pragma unroll
        for (int q = 0; q < op_a::MINE; ++q) look_at(q, r + 2 * OP_STEP);
        op_meet(true);
        put_scales(here, r + 2 * OP_STEP);
        ask_scales(r + 3 * OP_STEP);
#pragma unroll
        for (int n = 0; n < ALL; ++n) bring(here, n, r + 2 * OP_STEP);
      };
      do {
        idle(lds0, r);
        idle(lds1, r + OP_STEP);
        r += 2 * OP_STEP;
      } while (r < r1);
    } else
#endif
    do {
      round(lds0, lds1, r);
      round(lds1, lds0, r + OP_STEP);
      r += 2 * OP_STEP;
    } while (r < r1);
    /* what is still on its way to LDS arrives before the workgroup gives it up */
    __builtin_amdgcn_s_waitcnt(0 | 7 << 4);
  }

#pragma unroll
  for (int i = 0; i < OP_FM; ++i) {
    const int ri = i0 + wi + i * 16 + (lane & 15);
    if (ri >= iend) continue;
    op_elt *out = (op_elt *)p.out + (long long)ri * p.out_stride;
    bool none = false;
#if OP_OUTER
    out += (long long)expert * p.out_expert;
#else
    none = p.index_a && a.number(ri) < 0;
#endif
    if (part) {
#pragma unroll
      for (int j = 0; j < OP_FN; ++j) op_write4(part + (long long)ri * p.nj, j0 + wj + j * 16 + 4 * (lane >> 4), jend, c[i][j], none);
    } else {
#pragma unroll
      for (int j = 0; j < OP_FN; j += 2) op_write_pair(out, j0 + wj + j * 16, jend, lane >> 4, c[i][j], c[i][j + 1], none);
    }
  }
}

/* The pieces of a sum added up, in order; a lane has four neighbours of a row.  Outer: of the experts with more pieces than one, and
 * zeros for those without rows. */
extern "C" __global__ void __launch_bounds__(256) product_join(const acc_product_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const int quads = (p.nj + 3) / 4;
  op_elt *out = (op_elt *)p.out;
  const float *from = p.parts;
#if OP_OUTER
  const int blocks = (int)(((long long)p.ni * quads + 255) / 256), expert = (int)(blockIdx.x / blocks), rows = p.ni;
  const long long u = (long long)(blockIdx.x % blocks) * 256 + threadIdx.x, apart = (long long)p.ni * p.nj;
  int pieces;
  const int first = op_first_run(p.offsets, p.experts, (int)p.rows, p.piece, expert + 1, &pieces);
  if (pieces == 1) return;
  from += first * apart;
  out += (long long)expert * p.out_expert;
#else
  const long long u = (long long)blockIdx.x * 256 + threadIdx.x, apart = p.rows * p.nj, rows = p.rows;
  const int pieces = p.pieces;
#endif
  const long long i = u / quads;
  const int j = (int)(u - i * quads) * 4, left = acc_min(4, p.nj - j);
  if (i >= rows) return;
  from += i * p.nj + j;
  acc_f4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int n = 0; n < pieces; n += 4) {
    struct __attribute__((packed, aligned(4))) op_f4 { float v[4]; } v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float *q = from + acc_min(n + k, pieces - 1) * apart;
      if (left == 4) {
        v[k] = *(const op_f4 *)q;
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t) v[k].v[t] = t < left ? q[t] : 0.0f;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (n + k < pieces)
#pragma unroll
        for (int t = 0; t < 4; ++t) sum[t] += v[k].v[t];
  }
  op_write4(out + i * p.out_stride, j, p.nj, sum, false);
}
