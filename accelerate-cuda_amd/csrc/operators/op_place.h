/*
 * op_place.h -- what comes behind a router's choices: the slots sorted by expert, stably, a histogram, a scan and a permutation.  Whoever
 * includes this says how many tokens a wave has at a time (OP_TOKENS), and how many waves place slots (OP_THREADS, OP_WAVES).
 */
#ifndef ACC_OP_PLACE_H
#define ACC_OP_PLACE_H

/* the slots first .. last - 1 of a workgroup that wave w takes: whole tokens, in order */
ACC_DEV long long op_share(const acc_route_args &p) { return (long long)((p.block + OP_WAVES * OP_TOKENS - 1) / (OP_WAVES * OP_TOKENS)) * OP_TOKENS; }

/* Place of every slot from first on, below last, of one wave: `start[e]` is the place of its first slot of expert e.  64 at a
 * time, in order; lanes of the same expert find one another bit by bit. */
ACC_DEV void op_place(const acc_route_args &p, const int *chosen, const long long first, const long long last, int *start, const int bits, const int lane)
{
  for (long long s = first; s < last; s += 64) {
    const long long mine = s + lane;
    const int e = mine < last ? chosen[mine] : -1;
    unsigned long long same = __ballot(e >= 0);
    for (int b = 0; b < bits; ++b) {
      const unsigned long long has = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? has : ~has;
    }
    if (e >= 0) {
      const int before = __popcll(same & ((1ull << lane) - 1));
      const int at = start[e] + before;
      if (before == 0) start[e] = at + __popcll(same);
      p.order[at] = (int)mine;
      p.place[mine] = at;
    } else if (mine < last) {
      p.place[mine] = -1;
    }
  }
}

ACC_DEV int op_index_bits(const int experts) { return experts > 1 ? 32 - __builtin_clz(experts - 1) : 0; }

/* counts[w][e] -> the place of wave w's first slot of expert e, where the workgroup's first one is at base[e] */
ACC_DEV void op_starts(const acc_route_args &p, int *counts, const int *base, const int tid)
{
  for (int e = tid; e < p.experts; e += OP_THREADS) {
    int at = base[e], n[OP_WAVES];
#pragma unroll
    for (int w = 0; w < OP_WAVES; ++w) n[w] = counts[w * p.experts + e];
#pragma unroll
    for (int w = 0; w < OP_WAVES; ++w) {
      counts[w * p.experts + e] = at;
      at += n[w];
    }
  }
  __syncthreads();
}

/* base[e] += the sum of total[0 .. e-1], by the first wave; *all is the sum of all; the offsets go out if asked for */
ACC_DEV void op_bases(const acc_route_args &p, int *base, const int *total, const bool write, const int tid, int *all)
{
  if (tid < 64) {
    int carry = 0;
    for (int b = 0; b < p.experts; b += 64) {
      const int e = b + tid, n = e < p.experts ? total[e] : 0;
      const int upto = acc_wave_scan(n, [](int x, int y) { return x + y; }, tid);
      if (e < p.experts) {
        base[e] += carry + upto - n;
        if (write) p.offsets[e + 1] = carry + upto;
      }
      carry += acc_readlane(upto, 63);
    }
    if (tid == 0) {
      *all = carry;
      if (write) p.offsets[0] = 0;
    }
  }
  __syncthreads();
}

/* behind it, where there are several workgroups (256 at most): everybody adds up the counts, those before it and all */
extern "C" __global__ void __launch_bounds__(OP_THREADS) route_place(const acc_route_args p)
{
  if (p.guard && *p.guard == 0u) return;
  extern __shared__ int shared[];
  __shared__ int all;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long first = (long long)blockIdx.x * p.block, last = acc_min<long long>(p.tokens, first + p.block), share = op_share(p);
  const long long mine = (first + wave * share) * p.choose, end = acc_min(last, first + (wave + 1) * share) * p.choose;
  int *counts = shared, *base = shared + OP_WAVES * p.experts, *sums = base + p.experts;
  for (int i = tid; i < (OP_WAVES + 2) * p.experts; i += OP_THREADS) counts[i] = 0;
  __syncthreads();
  /* the wave's own slots, once more */
  for (long long s = mine + lane; s < end; s += 64) {
    const int e = p.chosen[s];
    if (e >= 0) atomicAdd(&counts[wave * p.experts + e], 1);
  }
  /* a wave adds up the counts of 64 experts, of every workgroup or of every few, 16 of them on their way at once */
  const int lots = (p.experts + 63) / 64, shares = lots < OP_WAVES ? OP_WAVES / lots : 1;
  for (int lot = wave % acc_min(lots, OP_WAVES); lot < lots; lot += OP_WAVES) {
    const int e = lot * 64 + lane, mine_from = lots < OP_WAVES ? wave / lots : 0;
    if (mine_from >= shares) break;
    int before = 0, total = 0;
    /* (256 workgroups' counts of 2048 experts: offsets of 32 bits do) */
    unsigned int at = (unsigned int)(mine_from * p.experts + acc_min(e, p.experts - 1));
    const unsigned int apart = (unsigned int)(shares * p.experts);
    int b = mine_from;
    for (; b + 15 * shares < p.blocks; b += 16 * shares) {
      int n[16];
#pragma unroll
      for (int k = 0; k < 16; ++k, at += apart) n[k] = (int)p.counts[at];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        total += n[k];
        before += b + k * shares < (int)blockIdx.x ? n[k] : 0;
      }
    }
#pragma unroll 4
    for (; b < p.blocks; b += shares, at += apart) {
      const int n = (int)p.counts[at];
      total += n;
      before += b < (int)blockIdx.x ? n : 0;
    }
    if (e < p.experts) {
      atomicAdd(&base[e], before);
      atomicAdd(&sums[e], total);
    }
  }
  __syncthreads();
  op_bases(p, base, sums, blockIdx.x == 0, tid, &all);
  op_starts(p, counts, base, tid);
  op_place(p, p.chosen, mine, end, counts + wave * p.experts, op_index_bits(p.experts), lane);
  /* what lies behind the last expert's slots, each workgroup its part */
  for (long long s = acc_max<long long>(all, first * p.choose) + tid; s < last * p.choose; s += OP_THREADS) p.order[s] = -1;
}

#endif
