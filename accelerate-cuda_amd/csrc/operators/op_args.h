/*
 * op_args.h -- what the drivers of the operators (operators.cpp) hand to their kernels: one structure a kernel, included
 * by both sides.  Strides are in elements, pointers are device addresses; `guard` is the word of an array-level loop that
 * says whether it still runs (0: no loop), as ACC_GUARDED instances of the skeletons take it.
 */
#ifndef ACC_OP_ARGS_H
#define ACC_OP_ARGS_H

#ifndef __HIPCC_RTC__
#include <cstdint>
#endif

/* products of segments of rows: see op_product.h */
struct acc_product_args {
  const void *a, *b;            /* the operands */
  void *out;
  const int32_t *offsets;       /* experts + 1 segment starts */
  const int32_t *index_a;       /* which row of `a` (outer: or of `b`) each row of the segments is; 0: its own number */
  const int32_t *index_b;
  const uint8_t *a_scales, *b_scales;   /* 4 bits: a byte for every 32 elements */
  int64_t a_stride, b_stride;   /* from one row of the array in memory to the next (4 bits: in bytes, as every length along r) */
  int64_t b_expert;             /* rows: from one expert's matrix to the next */
  int64_t a_scales_stride, b_scales_stride, b_scales_expert;
  int64_t out_stride, out_expert;
  int64_t rows;                 /* rows of the segments, all told */
  int32_t a_rows, b_rows;       /* rows that an index may name */
  int32_t ni, nj;               /* the result's extents: rows: -, n; outer: i, j */
  int32_t k;                    /* rows: the summed dimension */
  int32_t experts;
  uint32_t per_mul, per_shift;  /* an index at is divided: (at * per_mul) >> (32 + per_shift); per_mul 0: it is not */
  int32_t tiles_i, tiles_j;     /* the grid's tiles */
  int32_t piece, pieces;        /* a sum in pieces (0: in one): outer: of up to `piece` rows; rows: `pieces` of `piece` elements of k */
  float *parts;                 /* their results */
  uint32_t *places;             /* outer, with an index, in large tiles: where the rows lie that it names, a number a row */
  const uint32_t *guard;
};

/* an operand copied into rows of whole chunks: see op_pack.h */
struct acc_pack_args {
  const void *in;
  void *out;                    /* batches x rows_out rows of `chunks` chunks */
  int64_t batch_stride, row_stride;
  uint32_t batches, rows, rows_out, chunks;
  int32_t cols, pad;
  uint32_t per_mul, per_shift;  /* a division by `chunks` */
  const uint32_t *guard;
};

/* the router: see op_route.h */
struct acc_route_args {
  const void *logits;
  int32_t *chosen;              /* tokens x choose experts */
  float *weights;
  int32_t *offsets, *order, *place;
  const float *dweights;        /* gradient only */
  void *dlogits;
  uint32_t *counts;             /* scratch: a row of `experts` counts for every workgroup */
  int64_t tokens, logits_stride, dlogits_stride;
  int32_t experts, choose;
  int32_t normalise, blocks;
  int32_t block, pad;           /* tokens of a workgroup */
  const uint32_t *guard;
};

/* the combination: see op_combine.h */
struct acc_combine_args {
  const void *y, *dout;
  void *out;                    /* combine: the sums; gradient: the rows' gradient */
  const int32_t *place;
  const float *weights;
  float *dweights;
  int64_t tokens, y_rows, y_stride, out_stride, dout_stride;
  int32_t choose, width;
  uint32_t per_mul, per_shift;  /* combine: division by a row's pieces of eight */
  const uint32_t *guard;
};

/* 4-bit numbers under shared scales: see op_micro.h */
struct acc_micro_args {
  const void *x;                /* quantise: the values; values: - */
  void *out;                    /* values: the values */
  uint8_t *codes, *scales;
  int64_t rows, x_stride, codes_stride, scales_stride;
  int32_t k, blocks;
  uint32_t per_mul, per_shift;  /* division by `blocks`, as for the products' indices */
  const uint32_t *guard;
};

#endif
