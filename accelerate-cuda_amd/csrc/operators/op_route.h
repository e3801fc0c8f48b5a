/*
 * op_route.h -- the router of a layer of experts: the largest logits of every token, their weights, and the tokens' slots
 * sorted by expert, stably: a row-wise selection, a histogram, a scan and a permutation in one or two launches.
 *
 * A token has OP_LANES neighbouring lanes with OP_PER neighbouring logits each.  The lanes agree on the largest value left; of
 * equal ones the lowest lane has the lowest index.
 */
#include "op_common.h"

#define OP_TOKENS (64 / OP_LANES)                  /* tokens a wave has at a time */
#define OP_WAVES (OP_THREADS / 64)
#define OP_NONE (-__builtin_inff())

/* the largest of a token's lanes, in all of them */
ACC_DEV float op_group_max(float v)
{
#pragma unroll
  for (int d = 1; d < OP_LANES; d *= 2) v = __builtin_fmaxf(v, __shfl_xor(v, d));
  return v;
}
ACC_DEV float op_group_sum(float v)
{
#pragma unroll
  for (int d = 1; d < OP_LANES; d *= 2) v += __shfl_xor(v, d);
  return v;
}

/* a lane's logits: what is not a number counts as minus infinity, as what lies behind the row's end does */
ACC_DEV void op_logits(const acc_route_args &p, const long long t, const int sub, float (&v)[OP_PER])
{
  const op_elt *x = (const op_elt *)p.logits + t * p.logits_stride;
#pragma unroll
  for (int c = 0; c < OP_PER; c += OP_VEC) {
    const int e = sub * OP_PER + c;
    op_elt w[OP_VEC];
    if (OP_VEC > 1) {
      /* (rows of a multiple of OP_VEC elements, aligned to as many) */
      typedef op_elt vec __attribute__((ext_vector_type(OP_VEC)));
      if (t < p.tokens && e < p.experts) {
        const vec u = *(const vec *)(x + e);
        __builtin_memcpy(w, &u, sizeof(w));
      }
    } else if (t < p.tokens && e < p.experts) {
      w[0] = x[e];
    }
#pragma unroll
    for (int k = 0; k < OP_VEC; ++k) {
      const float f = t < p.tokens && e + k < p.experts ? (float)w[k] : OP_NONE;
      v[c + k] = f > OP_NONE ? f : OP_NONE;
    }
  }
}

/* exp(x - most), where an infinite `most` leaves the values that reach it */
ACC_DEV float op_power(const float x, const float most) { return x == OP_NONE ? 0.0f : x == most ? 1.0f : __expf(x - most); }

/* place of every slot of a workgroup's tokens: `start[w * experts + e]` is the place of the first slot that wave w has of
 * expert e; a wave takes its slots 64 at a time, in order.  Lanes of the same expert find one another bit by bit. */
ACC_DEV void op_place(const acc_route_args &p, const long long first, const long long last, int *start, const int bits, const int wave, const int lane)
{
  const long long slots = last - first, share = (slots + OP_WAVES * 64 - 1) / (OP_WAVES * 64) * 64;
  for (long long s = first + wave * share; s < acc_min(last, first + (wave + 1) * share); s += 64) {
    const long long mine = s + lane;
    const int e = mine < acc_min(last, first + (wave + 1) * share) ? p.chosen[mine] : -1;
    unsigned long long same = __ballot(e >= 0);
    for (int b = 0; b < bits; ++b) {
      const unsigned long long has = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? has : ~has;
    }
    if (e >= 0) {
      const int before = __popcll(same & ((1ull << lane) - 1));
      const int at = start[wave * p.experts + e] + before;
      if (before == 0) start[wave * p.experts + e] = at + __popcll(same);
      p.order[at] = (int)mine;
      p.place[mine] = at;
    } else if (mine < last && mine < first + (wave + 1) * share) {
      p.place[mine] = -1;
    }
  }
}

/* how many slots each wave has of each expert, of the workgroup's slots first .. last-1 */
ACC_DEV void op_count(const acc_route_args &p, const long long first, const long long last, int *counts, const int tid)
{
  for (int i = tid; i < OP_WAVES * p.experts; i += OP_THREADS) counts[i] = 0;
  __syncthreads();
  const long long slots = last - first, share = (slots + OP_WAVES * 64 - 1) / (OP_WAVES * 64) * 64;
  for (long long s = first + tid; s < last; s += OP_THREADS) {
    const int e = p.chosen[s];
    if (e >= 0) atomicAdd(&counts[(int)((s - first) / share) * p.experts + e], 1);
  }
  __syncthreads();
}

ACC_DEV int op_bits(const int experts) { return experts > 1 ? 32 - __builtin_clz(experts - 1) : 0; }

/* counts[w][e] -> the place of wave w's first slot of expert e, where the workgroup's first one is at base[e] */
ACC_DEV void op_starts(const acc_route_args &p, int *counts, const int *base, const int tid)
{
  for (int e = tid; e < p.experts; e += OP_THREADS) {
    int at = base[e];
    for (int w = 0; w < OP_WAVES; ++w) {
      const int n = counts[w * p.experts + e];
      counts[w * p.experts + e] = at;
      at += n;
    }
  }
  __syncthreads();
}

/* base[e] += the sum of total[0 .. e-1], by the first wave; the offsets go out if asked for; returns nothing but the sum of all */
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

/* workgroup b has the tokens b * OP_BLOCK .. ; with one workgroup the slots are placed at once, otherwise the counts go out */
extern "C" __global__ void __launch_bounds__(OP_THREADS) route(const acc_route_args p)
{
  if (p.guard && *p.guard == 0u) return;
  extern __shared__ int shared[];                  /* OP_WAVES * experts counts, experts bases, experts totals */
  __shared__ int all;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int sub = lane % OP_LANES;
  const long long first = (long long)blockIdx.x * OP_BLOCK, last = acc_min<long long>(p.tokens, first + OP_BLOCK);

  for (long long base = first + wave * OP_TOKENS; base < last; base += OP_WAVES * OP_TOKENS) {
    const long long t = base + lane / OP_LANES;
    float v[OP_PER];
    op_logits(p, t, sub, v);
    float total = 0.0f, most = OP_NONE;
    if (!p.normalise) {
      float m = OP_NONE;
#pragma unroll
      for (int k = 0; k < OP_PER; ++k) m = __builtin_fmaxf(m, v[k]);
      most = op_group_max(m);
#pragma unroll
      for (int k = 0; k < OP_PER; ++k) total += op_power(v[k], most);
      total = op_group_sum(total);
    }
    for (int j = 0; j < p.choose; ++j) {
      float m = OP_NONE;
#pragma unroll
      for (int k = 0; k < OP_PER; ++k) m = __builtin_fmaxf(m, v[k]);
      const float best = op_group_max(m);
      if (j == 0) most = best;
      /* the lowest lane of the token that has it, and there the lowest index */
      unsigned long long have = __ballot(m == best && best > OP_NONE);
      if (OP_LANES < 64) have &= ((1ull << OP_LANES) - 1) << (lane / OP_LANES * OP_LANES);
      const bool owner = have != 0 && __builtin_ctzll(have) == lane;
      int at = -1;
      bool taken = !owner;
#pragma unroll
      for (int k = 0; k < OP_PER; ++k) {
        const bool it = !taken && v[k] == best;
        if (it) {
          at = sub * OP_PER + k;
          v[k] = OP_NONE;
          taken = true;
        }
      }
      const float power = op_power(best, most);
      if (p.normalise) total += power;
      if (t < last && (owner || (have == 0 && sub == 0))) {
        p.chosen[t * p.choose + j] = at;
        p.weights[t * p.choose + j] = power;
      }
    }
    /* the powers become weights: the lanes that wrote them have made them visible to their wave */
    __threadfence_block();
    if (t < last)
      for (int j = sub; j < p.choose; j += OP_LANES) {
        const float w = p.weights[t * p.choose + j];
        p.weights[t * p.choose + j] = w > 0.0f ? w / total : 0.0f;
      }
  }
  __threadfence_block();
  __syncthreads();

  int *counts = shared, *base = shared + OP_WAVES * p.experts, *sums = base + p.experts;
  op_count(p, first * p.choose, last * p.choose, counts, tid);
  for (int e = tid; e < p.experts; e += OP_THREADS) {
    int n = 0;
    for (int w = 0; w < OP_WAVES; ++w) n += counts[w * p.experts + e];
    if (p.blocks > 1) p.counts[(long long)blockIdx.x * p.experts + e] = n;
    base[e] = 0;
    sums[e] = n;
  }
  if (p.blocks > 1) return;
  __syncthreads();
  op_bases(p, base, sums, true, tid, &all);
  op_starts(p, counts, base, tid);
  op_place(p, 0, p.tokens * p.choose, counts, op_bits(p.experts), wave, lane);
  for (long long s = all + tid; s < p.tokens * p.choose; s += OP_THREADS) p.order[s] = -1;
}

/* behind it, where there are several workgroups: everybody adds up the counts, those before it and all */
extern "C" __global__ void __launch_bounds__(OP_THREADS) route_place(const acc_route_args p)
{
  if (p.guard && *p.guard == 0u) return;
  extern __shared__ int shared[];
  __shared__ int all;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long first = (long long)blockIdx.x * OP_BLOCK, last = acc_min<long long>(p.tokens, first + OP_BLOCK);
  int *counts = shared, *base = shared + OP_WAVES * p.experts, *sums = base + p.experts;
  for (int e = tid; e < p.experts; e += OP_THREADS) {
    int before = 0, total = 0;
    for (int b = 0; b < p.blocks; ++b) {
      const int n = (int)p.counts[(long long)b * p.experts + e];
      total += n;
      before += b < (int)blockIdx.x ? n : 0;
    }
    base[e] = before;
    sums[e] = total;
  }
  __syncthreads();
  op_bases(p, base, sums, blockIdx.x == 0, tid, &all);
  op_count(p, first * p.choose, last * p.choose, counts, tid);
  op_starts(p, counts, base, tid);
  op_place(p, first * p.choose, last * p.choose, counts, op_bits(p.experts), wave, lane);
  /* what lies behind the last expert's slots, each workgroup its part */
  const long long slots = p.tokens * p.choose, mine = first * p.choose, end = last * p.choose;
  for (long long s = acc_max<long long>(all, mine) + tid; s < acc_min(end, slots); s += OP_THREADS) p.order[s] = -1;
}

/* d logit_i = w_i (dw_i - sum_j w_j dw_j) of the chosen ones; where the weights are not normalised over them, of all:
 * p_i ([i chosen] dw_i - sum) */
extern "C" __global__ void __launch_bounds__(OP_THREADS) route_gradient(const acc_route_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const int tid = threadIdx.x, lane = tid & 63, sub = lane % OP_LANES;
  const long long t = ((long long)blockIdx.x * OP_WAVES + (tid >> 6)) * OP_TOKENS + lane / OP_LANES;
  const bool here = t < p.tokens;
  float v[OP_PER], d[OP_PER], inner = 0.0f;
  if (!p.normalise) {
    op_logits(p, t, sub, v);
    float m = OP_NONE, total = 0.0f;
#pragma unroll
    for (int k = 0; k < OP_PER; ++k) m = __builtin_fmaxf(m, v[k]);
    m = op_group_max(m);
#pragma unroll
    for (int k = 0; k < OP_PER; ++k) total += v[k] = op_power(v[k], m);
    total = op_group_sum(total);
#pragma unroll
    for (int k = 0; k < OP_PER; ++k) v[k] = v[k] > 0.0f ? v[k] / total : 0.0f;
  }
  for (int j = sub; j < p.choose; j += OP_LANES)
    if (here && p.chosen[t * p.choose + j] >= 0) inner += p.weights[t * p.choose + j] * p.dweights[t * p.choose + j];
  inner = op_group_sum(inner);
#pragma unroll
  for (int k = 0; k < OP_PER; ++k) d[k] = p.normalise ? 0.0f : -v[k] * inner;
  for (int j = 0; j < p.choose; ++j) {
    const int e = here ? p.chosen[t * p.choose + j] : -1;
    if (e < 0 || e / OP_PER != sub) continue;
    const float w = p.weights[t * p.choose + j], dw = p.dweights[t * p.choose + j];
#pragma unroll
    for (int k = 0; k < OP_PER; ++k)
      if (e % OP_PER == k) d[k] = p.normalise ? w * (dw - inner) : v[k] * (dw - inner);
  }
  if (!here) return;
  op_elt *out = (op_elt *)p.dlogits + t * p.dlogits_stride;
#pragma unroll
  for (int c = 0; c < OP_PER; c += OP_VEC) {
    const int e = sub * OP_PER + c;
    if (e >= p.experts) break;
    typedef op_elt vec __attribute__((ext_vector_type(OP_VEC)));
    op_elt w[OP_VEC];
#pragma unroll
    for (int k = 0; k < OP_VEC; ++k) w[k] = (op_elt)d[c + k];
    if (OP_VEC > 1) {
      vec u;
      __builtin_memcpy(&u, w, sizeof(w));
      *(vec *)(out + e) = u;
    } else {
      out[e] = w[0];
    }
  }
}
