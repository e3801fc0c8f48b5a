/*
 * op_route.h -- the router of a layer of experts: the largest logits of every token, their weights, and the tokens' slots
 * sorted by expert, stably: a row-wise selection, a histogram, a scan and a permutation in one or two launches.
 *
 * A token has OP_LANES neighbouring lanes with OP_PER logits each.  A logit is a key: its bits, made to compare as whole
 * numbers do, above the index turned round, so that of equal ones the lowest index is the largest -- 32 bits for logits of
 * 16, 64 for Float32; 0 is no logit.  A lane sorts its keys once; then the token's lanes agree on the largest of their first
 * ones, `choose` times, and whoever had it moves up.  Bound by that agreement: 16384 tokens of 64 Float32 logits, four chosen, take
 * 12 us in all where memory is 1.
 */
#include "op_common.h"

#define OP_TOKENS (64 / OP_LANES)                  /* tokens a wave has at a time */
#define OP_WAVES (OP_THREADS / 64)
#define OP_NONE (-__builtin_inff())

#if OP_ELT == 0
typedef unsigned long long op_key;
typedef unsigned int op_bits_t;
#define OP_SHIFT 32
#else
typedef unsigned int op_key;
typedef unsigned short op_bits_t;
#define OP_SHIFT 16
#endif
#define OP_SIGN ((op_bits_t)1 << (OP_SHIFT - 1))

/* minus infinity and what is not a number: 0; minus zero counts as zero */
ACC_DEV op_key op_key_of(const op_elt x, const int index)
{
  const float f = (float)x;
  op_bits_t b;
  __builtin_memcpy(&b, &x, sizeof(b));
  b = f == 0.0f ? (op_bits_t)0 : b;
  b = b & OP_SIGN ? (op_bits_t)~b : (op_bits_t)(b | OP_SIGN);
  return f > OP_NONE ? (op_key)b << OP_SHIFT | (op_key)(0xffffu - (unsigned int)index) : (op_key)0;
}
ACC_DEV float op_value_of(const op_key k)
{
  op_bits_t b = (op_bits_t)(k >> OP_SHIFT);
  b = b & OP_SIGN ? (op_bits_t)(b ^ OP_SIGN) : (op_bits_t)~b;
  op_elt x;
  __builtin_memcpy(&x, &b, sizeof(x));
  return k ? (float)x : OP_NONE;
}
ACC_DEV int op_index_of(const op_key k) { return k ? (int)(0xffffu - ((unsigned int)k & 0xffffu)) : -1; }

/* f over a token's lanes, in all of them (f in any order): within 16 lanes by neighbours, pairs, mirrored halves; beyond by
 * exchanges of rows */
template <typename T, typename F> ACC_DEV T op_group(T v, F f)
{
  if (OP_LANES > 1) v = f(v, acc_dpp<0xB1, 0xf>(v, v));
  if (OP_LANES > 2) v = f(v, acc_dpp<0x4E, 0xf>(v, v));
  if (OP_LANES > 4) v = f(v, acc_dpp<0x141, 0xf>(v, v));
  if (OP_LANES > 8) v = f(v, acc_dpp<0x140, 0xf>(v, v));
  if (OP_LANES > 16) {
    unsigned int w[sizeof(T) / 4], a[sizeof(T) / 4], b[sizeof(T) / 4];
    T x, y;
    __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
    for (int k = 0; k < (int)(sizeof(T) / 4); ++k) {
      const auto r = __builtin_amdgcn_permlane16_swap(w[k], w[k], false, false);
      a[k] = r[0];
      b[k] = r[1];
    }
    __builtin_memcpy(&x, a, sizeof(T));
    __builtin_memcpy(&y, b, sizeof(T));
    v = f(x, y);
  }
  if (OP_LANES > 32) {
    unsigned int w[sizeof(T) / 4], a[sizeof(T) / 4], b[sizeof(T) / 4];
    T x, y;
    __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
    for (int k = 0; k < (int)(sizeof(T) / 4); ++k) {
      const auto r = __builtin_amdgcn_permlane32_swap(w[k], w[k], false, false);
      a[k] = r[0];
      b[k] = r[1];
    }
    __builtin_memcpy(&x, a, sizeof(T));
    __builtin_memcpy(&y, b, sizeof(T));
    v = f(x, y);
  }
  return v;
}
ACC_DEV float op_group_max(const float v) { return op_group(v, [](float x, float y) { return __builtin_fmaxf(x, y); }); }
ACC_DEV float op_group_sum(const float v) { return op_group(v, [](float x, float y) { return x + y; }); }

/* a lane's logits as they lie in memory; beyond the row's end (or for no token) minus infinity */
ACC_DEV void op_logits(const acc_route_args &p, const long long t, const bool here, const int sub, op_elt (&v)[OP_PER])
{
  const op_elt *x = (const op_elt *)p.logits + (here ? t : 0) * p.logits_stride;
#pragma unroll
  for (int c = 0; c < OP_PER; c += OP_VEC) {
    const int e = sub * OP_PER + c;
    const bool some = here && e < p.experts;
    if (OP_VEC > 1) {
      /* (rows of a multiple of OP_VEC elements, aligned to as many) */
      typedef op_elt vec __attribute__((ext_vector_type(OP_VEC)));
      vec u;
#pragma unroll
      for (int k = 0; k < OP_VEC; ++k) u[k] = (op_elt)OP_NONE;
      if (some) u = *(const vec *)(x + e);
#pragma unroll
      for (int k = 0; k < OP_VEC; ++k) v[c + k] = u[k];
    } else {
      v[c] = some ? x[e] : (op_elt)OP_NONE;
    }
  }
}

/* exp(x - most) for an x up to `most`, by the power of two; an infinite `most` leaves the values that reach it.  (Without a
 * branch; where `most` is minus infinity there is nothing to choose, and no use for what comes of it.) */
ACC_DEV float op_power(const float x, const float most)
{
  const float d = x == most ? 0.0f : x - most;
  return __builtin_amdgcn_exp2f(d * 1.44269504f);
}

/* largest first: bitonic over a power of two of keys, every comparison known */
ACC_DEV void op_sort(op_key (&k)[OP_PER])
{
#pragma unroll
  for (int size = 2; size <= OP_PER; size *= 2)
#pragma unroll
    for (int step = size / 2; step > 0; step /= 2)
#pragma unroll
      for (int i = 0; i < OP_PER; ++i) {
        const int j = i ^ step;
        if (j > i) {
          const op_key x = k[i], y = k[j];
          const bool down = (i & size) == 0;
          const op_key most = x > y ? x : y, least = x > y ? y : x;
          k[i] = down ? most : least;
          k[j] = down ? least : most;
        }
      }
}

#include "op_place.h"

#if OP_TALL
/* The selection for many tokens or experts: a lane has a token (OP_HALVES lanes, which share its logits) and OP_CHOOSE keys in
 * order, and puts every logit where it belongs among them: the new j-th key is the middle one of the j-th, the one in front of
 * it and the logit's, an instruction for keys of 32 bits.  That is 15 instructions a logit for 64 lanes at once, a third of what
 * the lanes of a token need to agree on as many.  Rows come by way of LDS, 128 bytes of them a lane at a time, so that lines are
 * read whole; a row's share lies 16 bytes further than as many lines, which spreads the lanes' reads over the banks.  65536 tokens
 * of 128 bfloat16 logits, eight chosen, with a lane a token: 15.7 us of a bound of 4 by memory (17 MB read, 4 written) and of about
 * 5 by instructions; a SIMD has one wave then, whose waits nothing covers. */
#define OP_COLUMNS (128 / (int)sizeof(op_elt))
#define OP_TALL_TOKENS (64 / OP_HALVES)            /* of a wave; a token has OP_HALVES lanes, as many apart */
#define OP_TALL_THREADS (256 * OP_HALVES)
#define OP_APART (128 * OP_HALVES + 16)
typedef op_elt op_vec __attribute__((ext_vector_type(OP_VALUES)));

ACC_DEV op_key op_middle(const op_key a, const op_key b, const op_key c)
{
  /* (spelt in full, as the compiler knows the instruction) */
  const op_key low = a < b ? a : b, high = a < b ? b : a, most = high < c ? high : c;
  return low > most ? low : most;
}

/* what the first and the second of two lanes hold that are 16 or 32 apart, in both */
template <typename T> ACC_DEV void op_both(const T v, const int apart, T *first, T *second)
{
  unsigned int w[sizeof(T) / 4], a[sizeof(T) / 4], b[sizeof(T) / 4];
  __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
  for (int k = 0; k < (int)(sizeof(T) / 4); ++k) {
    const auto r = apart == 16 ? __builtin_amdgcn_permlane16_swap(w[k], w[k], false, false) : __builtin_amdgcn_permlane32_swap(w[k], w[k], false, false);
    a[k] = r[0];
    b[k] = r[1];
  }
  __builtin_memcpy(first, a, sizeof(T));
  __builtin_memcpy(second, b, sizeof(T));
}

/* what a shifted chunk has behind the row's end is no logit (whole chunks have none there) */
ACC_DEV op_elt op_there(const acc_route_args &p, const op_elt v, const int index) { return OP_VEC > 1 || index < p.experts ? v : (op_elt)OP_NONE; }

ACC_DEV void op_insert(op_key (&k)[OP_CHOOSE], const op_key y)
{
#pragma unroll
  for (int j = OP_CHOOSE - 1; j > 0; --j) k[j] = op_middle(k[j - 1], k[j], y);
  k[0] = k[0] > y ? k[0] : y;
}

extern "C" __global__ void __launch_bounds__(OP_TALL_THREADS) route(const acc_route_args p)
{
  if (p.guard && *p.guard == 0u) return;
  extern __shared__ int shared[];
  __shared__ __align__(16) unsigned char tiles[OP_TALL_THREADS / 64][OP_TALL_TOKENS * OP_APART];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, token = lane % OP_TALL_TOKENS, share = lane / OP_TALL_TOKENS;
  const long long first = (long long)blockIdx.x * p.block, last = acc_min<long long>(p.tokens, first + p.block);
  unsigned char *tile = tiles[wave];
  for (int e = tid; e < p.experts; e += OP_TALL_THREADS) shared[e] = 0;
  __syncthreads();
  for (long long at = first + wave * OP_TALL_TOKENS; at < last; at += 256) {
    const int rows = (int)acc_min<long long>(OP_TALL_TOKENS, last - at);
    const op_elt *x = (const op_elt *)p.logits + at * p.logits_stride;
    op_key k[OP_CHOOSE];
    float total = 0.0f, most = OP_NONE;
#pragma unroll
    for (int j = 0; j < OP_CHOOSE; ++j) k[j] = 0;
    op_vec next[8];
    const auto ask = [&](const int c0) {           /* (rows that there are not: the last one; columns: minus infinity) */
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int n8 = i * 64 + lane, r = acc_min(n8 / (8 * OP_HALVES), rows - 1), c = c0 + n8 % (8 * OP_HALVES) * OP_VALUES;
#pragma unroll
        for (int n = 0; n < OP_VALUES; ++n) next[i][n] = (op_elt)OP_NONE;
        if (c < p.experts) {
          const op_elt *row = x + r * p.logits_stride;
          if (OP_VEC > 1) {
            next[i] = *(const op_vec *)(row + c);
          } else {
            /* (rows start anywhere; what would reach beyond the row's end is read earlier and shifted into place) */
            const int from = acc_min(c, p.experts - OP_VALUES);
            acc_u4 u = ((const op_loose<op_elt> *)(row + from))->v;
            if (from < c) u = op_shifted(u, (c - from) * (int)sizeof(op_elt));
            __builtin_memcpy(&next[i], &u, 16);
          }
        }
      }
    };
    ask(0);
    for (int c0 = 0; c0 < p.experts; c0 += OP_HALVES * OP_COLUMNS) {
#pragma unroll
      for (int i = 0; i < 8; ++i) *(op_vec *)(tile + (i * 64 + lane) / (8 * OP_HALVES) * OP_APART + lane % (8 * OP_HALVES) * 16) = next[i];
      if (c0 + OP_HALVES * OP_COLUMNS < p.experts) ask(c0 + OP_HALVES * OP_COLUMNS);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      const unsigned char *mine = tile + token * OP_APART + share * 128;
      for (int i = 0; i < 8; ++i) {
        const op_vec v = *(const op_vec *)(mine + i * 16);
#pragma unroll
        for (int n = 0; n < OP_VALUES; ++n) op_insert(k, op_key_of(op_there(p, v[n], c0 + share * OP_COLUMNS + i * OP_VALUES + n), c0 + share * OP_COLUMNS + i * OP_VALUES + n));
      }
      if (!p.normalise) {
        const float now = op_value_of(k[0]);
        total *= op_power(most, now);
        most = now;
        for (int i = 0; i < 8; ++i) {
          const op_vec v = *(const op_vec *)(mine + i * 16);
#pragma unroll
          for (int n = 0; n < OP_VALUES; ++n) {
            const float f = (float)op_there(p, v[n], c0 + share * OP_COLUMNS + i * OP_VALUES + n);
            total += op_power(f > OP_NONE ? f : OP_NONE, most);
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    /* a token's lanes put together what they have */
#pragma unroll
    for (int apart = OP_TALL_TOKENS; apart < 64; apart *= 2) {
      op_key other[OP_CHOOSE];
      float here, there, here_most, there_most;
      op_both(total, apart, &here, &there);
#pragma unroll
      for (int j = 0; j < OP_CHOOSE; ++j) {
        op_key one;
        op_both(k[j], apart, &one, &other[j]);
        k[j] = one;
      }
      here_most = op_value_of(k[0]);
      there_most = op_value_of(other[0]);
#pragma unroll
      for (int j = 0; j < OP_CHOOSE; ++j) op_insert(k, other[j]);
      most = op_value_of(k[0]);
      total = here * op_power(here_most, most) + there * op_power(there_most, most);
    }
    if (token >= rows) continue;
    most = op_value_of(k[0]);
    float power[OP_CHOOSE];
    int expert[OP_CHOOSE];
#pragma unroll
    for (int j = 0; j < OP_CHOOSE; ++j) {
      power[j] = op_power(op_value_of(k[j]), most);
      if (p.normalise) total += power[j];
    }
#pragma unroll
    for (int j = 0; j < OP_CHOOSE; ++j) {
      expert[j] = op_index_of(k[j]);
      power[j] = expert[j] < 0 ? 0.0f : power[j] / total;
    }
    if (share == 0) {
      __builtin_memcpy(p.chosen + (at + token) * OP_CHOOSE, expert, sizeof expert);
#pragma unroll
      for (int j = 0; j < OP_CHOOSE; ++j)
        if (expert[j] >= 0) atomicAdd(&shared[expert[j]], 1);
    }
    if (share == OP_HALVES - 1) __builtin_memcpy(p.weights + (at + token) * OP_CHOOSE, power, sizeof power);
  }
  __syncthreads();
  for (int e = tid; e < p.experts; e += OP_TALL_THREADS) p.counts[(long long)blockIdx.x * p.experts + e] = shared[e];
}
#else
/* workgroup b has the tokens b * block .. ; with one workgroup the slots are placed at once, otherwise the counts go out */
extern "C" __global__ void __launch_bounds__(OP_THREADS) route(const acc_route_args p)
{
  if (p.guard && *p.guard == 0u) return;
  extern __shared__ int shared[];                  /* OP_WAVES * experts counts, experts bases, experts totals, a single workgroup's slots */
  __shared__ int all;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, sub = lane % OP_LANES;
  const long long first = (long long)blockIdx.x * p.block, last = acc_min<long long>(p.tokens, first + p.block), share = op_share(p);
  const long long mine = first + wave * share, end = acc_min(last, mine + share);
  int *counts = shared, *base = shared + OP_WAVES * p.experts, *sums = base + p.experts, *slots = sums + p.experts;
  for (int i = tid; i < OP_WAVES * p.experts; i += OP_THREADS) counts[i] = 0;
  __syncthreads();

  op_elt next[OP_PER];
  op_logits(p, mine + lane / OP_LANES, mine + lane / OP_LANES < end, sub, next);
  for (long long at = mine; at < end; at += OP_TOKENS) {
    const long long t = at + lane / OP_LANES;
    const bool here = t < end;
    op_elt x[OP_PER];
    op_key k[OP_PER];
#pragma unroll
    for (int i = 0; i < OP_PER; ++i) x[i] = next[i];
    op_logits(p, t + OP_TOKENS, t + OP_TOKENS < end, sub, next);     /* (on its way while these are sorted) */
#pragma unroll
    for (int i = 0; i < OP_PER; ++i) k[i] = op_key_of(x[i], sub * OP_PER + i);
    op_sort(k);
    /* the j-th choice stays with lane j of the token, OP_SELS of them a lane */
    op_key chosen[OP_SELS];
    float total = 0.0f, most = OP_NONE;
#pragma unroll
    for (int s = 0; s < OP_SELS; ++s) {
      chosen[s] = 0;
      const int n = acc_min(OP_LANES, p.choose - s * OP_LANES);
      for (int j = 0; j < n; ++j) {
        const op_key best = op_group(k[0], [](op_key a, op_key b) { return a > b ? a : b; });
        const bool owner = k[0] == best;           /* (no two keys are the same, but for 0) */
        chosen[s] = sub == j ? best : chosen[s];
#pragma unroll
        for (int i = 0; i + 1 < OP_PER; ++i) k[i] = owner ? k[i + 1] : k[i];
        k[OP_PER - 1] = owner ? (op_key)0 : k[OP_PER - 1];
      }
      if (s == 0) most = op_value_of(op_group(chosen[0], [](op_key a, op_key b) { return a > b ? a : b; }));
    }
    float power[OP_SELS];
#pragma unroll
    for (int s = 0; s < OP_SELS; ++s) {
      power[s] = op_power(op_value_of(chosen[s]), most);
      if (p.normalise) total += power[s];
    }
    if (!p.normalise)
#pragma unroll
      for (int i = 0; i < OP_PER; ++i) {
        const float f = (float)x[i];
        total += op_power(f > OP_NONE ? f : OP_NONE, most);
      }
    total = op_group_sum(total);
#pragma unroll
    for (int s = 0; s < OP_SELS; ++s) {
      const int j = s * OP_LANES + sub;
      if (here && j < p.choose) {
        const int e = op_index_of(chosen[s]);
        p.chosen[t * p.choose + j] = e;
        if (p.blocks == 1) slots[t * p.choose + j] = e;
        p.weights[t * p.choose + j] = e < 0 ? 0.0f : power[s] / total;
        if (e >= 0) atomicAdd(&counts[wave * p.experts + e], 1);
      }
    }
  }
  __threadfence_block();
  __syncthreads();

  for (int e = tid; e < p.experts; e += OP_THREADS) {
    int n = 0;
#pragma unroll
    for (int w = 0; w < OP_WAVES; ++w) n += counts[w * p.experts + e];
    if (p.blocks > 1) p.counts[(long long)blockIdx.x * p.experts + e] = n;
    base[e] = 0;
    sums[e] = n;
  }
  if (p.blocks > 1) return;
  __syncthreads();
  op_bases(p, base, sums, true, tid, &all);
  op_starts(p, counts, base, tid);
  op_place(p, slots, mine * p.choose, end * p.choose, counts + wave * p.experts, op_index_bits(p.experts), lane);
  for (long long s = all + tid; s < p.tokens * p.choose; s += OP_THREADS) p.order[s] = -1;
}

#endif

/* d logit_i = w_i (dw_i - sum_j w_j dw_j) of the chosen ones; where the weights are not normalised over them, of all:
 * p_i ([i chosen] dw_i - sum).  Bound by waiting: a choice is read, then its weights, and those once more for the lane that has it.
 * 65536 tokens of 128 bfloat16 logits, eight chosen: 13.8 us normalised (a floor of 4.8 by memory), 19.5 not (8.3); Float32 16.5
 * (8.3) and 22.7 (15.3); 8 tokens of 64 a launch. */
extern "C" __global__ void __launch_bounds__(OP_THREADS) route_gradient(const acc_route_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const int tid = threadIdx.x, lane = tid & 63, sub = lane % OP_LANES;
  const long long t = ((long long)blockIdx.x * OP_WAVES + (tid >> 6)) * OP_TOKENS + lane / OP_LANES;
  const bool here = t < p.tokens;
  float v[OP_PER], d[OP_PER], inner = 0.0f;
  if (!p.normalise) {
    op_elt x[OP_PER];
    op_logits(p, t, here, sub, x);
    float m = OP_NONE, total = 0.0f;
#pragma unroll
    for (int k = 0; k < OP_PER; ++k) {
      const float f = (float)x[k];
      v[k] = f > OP_NONE ? f : OP_NONE;
      m = __builtin_fmaxf(m, v[k]);
    }
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
    if (OP_VEC > 1) {
      typedef op_elt vec __attribute__((ext_vector_type(OP_VEC)));
      vec u;
#pragma unroll
      for (int k = 0; k < OP_VEC; ++k) u[k] = (op_elt)d[c + k];
      *(vec *)(out + e) = u;
    } else {
      out[e] = (op_elt)d[c];
    }
  }
}
