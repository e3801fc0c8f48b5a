/*
 * op_score.h -- a router that scores experts one by one, s = 1 / (1 + e^-x), and chooses by s + bias: the best `keep` groups of
 * neighbouring experts, by the sum of their two best, then the best OP_CHOOSE experts of those; weights are the chosen scores alone.
 *
 * A token has OP_LANES neighbouring lanes, each with up to OP_PER neighbouring logits in registers, a group or an even part of one.  What
 * is ranked is Float32 in the high bits of a 64-bit number that compares as one, with the index turned round in the low bits, so that of
 * equal ones the lowest index is the largest.  A lane puts its numbers where they belong among its best, two instructions a place, and
 * the token's lanes then exchange what they have.
 *
 * Scores of 64 bits decide.  Float32 ones are off by 2.3 10^-7 at most, and what lies closer than several times that (and is not the
 * same logit and bias, which is a tie wherever it is computed) is decided again in 64 bits, a wave for a token, when the others are
 * done: of normal logits, 256 experts and eight groups one token in some thousands.  All of them are where logits are all equal, as
 * of a router that begins with zeros, and groups have to be chosen (32768 tokens: 198 us), or all far below 0 (-20: 201, without groups 140).
 *
 * Bound by no one thing of the card's: 32768 tokens of 256 bfloat16 logits, eight chosen of four of eight groups, take 42 us, of which
 * the placing is 10 and the instructions of the choice some 12; memory is 4.  A wave's steps wait for one another (with four waves a
 * workgroup 55, with sixteen, which have 128 registers each, 59).
 */
#include "op_common.h"

#define OP_TOKENS (64 / OP_LANES)                  /* tokens a wave has at a time */
#define OP_WAVES (OP_THREADS / 64)
#include "op_place.h"

#define OP_NONE (-__builtin_inff())
#define OP_SELECT_WAVES (OP_FEW ? 4 : 8)           /* (sixteen have too few registers each) */
#define OP_KEYS (OP_CHOOSE + 1)                    /* one more, to see how near it is */

/* (without the instructions that make quiet what is not a number: there is nothing of the kind among these) */
ACC_DEV double op_most(const double a, const double b)
{
  double r;
  asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
ACC_DEV double op_least(const double a, const double b)
{
  double r;
  asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

/* what the neighbour `apart` lanes away has; up to 16 lanes, one that has the same where as many neighbours already have the same */
template <typename T> ACC_DEV T op_other(const T v, const int apart)
{
  if (apart == 1) return acc_dpp<0xB1, 0xf>(v, v);
  if (apart == 2) return acc_dpp<0x4E, 0xf>(v, v);
  if (apart == 4) return acc_dpp<0x141, 0xf>(v, v);
  if (apart == 8) return acc_dpp<0x140, 0xf>(v, v);
  unsigned int w[sizeof(T) / 4];
  __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
  for (int k = 0; k < (int)(sizeof(T) / 4); ++k) w[k] = __builtin_amdgcn_ds_bpermute((acc_lane() ^ apart) * 4, w[k]);
  T r;
  __builtin_memcpy(&r, w, sizeof(T));
  return r;
}

/* what an expert is ranked by, and nothing (minus infinity) for one that cannot be chosen */
ACC_DEV float op_score_of(const float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f)); }
ACC_DEV float op_ranked(const float x, const float bias)
{
  const float r = op_score_of(x) + bias;
  return x > OP_NONE && r > OP_NONE ? acc_min(r, 3.40282347e38f) + 0.0f : OP_NONE;
}
ACC_DEV double op_ranked64(const float x, const float bias)
{
  const double r = 1.0 / (1.0 + exp(-(double)x)) + (double)bias;
  return x > OP_NONE && r > (double)OP_NONE ? r : (double)OP_NONE;
}
ACC_DEV double op_key_of(const float ranked, const int index)
{
  const double d = (double)ranked;
  unsigned long long b;
  __builtin_memcpy(&b, &d, 8);
  if (ranked > OP_NONE) b |= (unsigned int)(ranked < 0.0f ? index : 2047 - index);
  double k;
  __builtin_memcpy(&k, &b, 8);
  return k;
}
ACC_DEV float op_value_of(const double key)
{
  unsigned long long b;
  __builtin_memcpy(&b, &key, 8);
  b &= ~2047ull;
  double d;
  __builtin_memcpy(&d, &b, 8);
  return (float)d;
}
ACC_DEV int op_index_of(const double key)
{
  unsigned long long b;
  __builtin_memcpy(&b, &key, 8);
  const int low = (int)(b & 2047ull);
  return key > (double)OP_NONE ? (key < 0.0 ? low : 2047 - low) : -1;
}
/* How near two ranked numbers may be to be told apart.  A score is off by a unit of the reciprocal, half a one of its sum, a quarter of
 * one of the exponential and a part of the product's in front of it, 2.3 10^-7 together, and what is ranked by half a unit more: two
 * by twice that.  And what a group's sum may be off itself. */
ACC_DEV float op_near(const float v) { return 6e-7f + 1.6e-7f * __builtin_fabsf(v); }
ACC_DEV float op_off(const float best, const float next) { return 6e-7f + 1.6e-7f * __builtin_fabsf(best) + (next > OP_NONE ? 1.6e-7f * __builtin_fabsf(next) : 0.0f); }

ACC_DEV void op_insert(double (&k)[OP_KEYS], const double y)
{
#pragma unroll
  for (int j = OP_KEYS - 1; j > 0; --j) k[j] = op_least(k[j - 1], op_most(k[j], y));
  k[0] = op_most(k[0], y);
}

/* the two best of a group and of some more of it */
struct op_two { float best, next; };
ACC_DEV void op_put(op_two &t, const float v)
{
  t.next = __builtin_amdgcn_fmed3f(t.best, t.next, v);       /* (the middle one: next <= best) */
  t.best = v > t.best ? v : t.best;
}
template <typename T> ACC_DEV T op_sum_of(const T best, const T next) { return next > (T)OP_NONE ? best + next : best; }
/* (of biases of the type's lowest value, too, the sum of a group that has something to choose is no infinity: near others, not none) */
ACC_DEV float op_group_sum(const op_two &t) { return t.best > OP_NONE ? acc_max(-3.40282347e38f, acc_min(3.40282347e38f, op_sum_of(t.best, t.next))) : OP_NONE; }

ACC_DEV float op_logit(const acc_route_args &p, const long long t, const int e) { return (float)((const op_elt *)p.logits)[t * p.logits_stride + e]; }
ACC_DEV float op_bias(const acc_route_args &p, const int e) { return p.bias ? p.bias[e] : 0.0f; }

/* the weight of a chosen logit from those of all: `shift` is taken off the exponents where all are negative, so that small scores keep
 * their proportions; scores that are zero in 64 bits, where e^-x is beyond the largest number, are zero */
ACC_DEV float op_part(const float x, const float shift) { return x < -709.78268f ? 0.0f : x < 0.0f ? expf(x - shift) / (1.0f + expf(x)) : 1.0f / (1.0f + expf(-x)); }

/* Token t again, in 64 bits: lane j has the j-th choice.  A lane has every 64th expert. */
#define OP_AGAIN (OP_LANES * OP_PER > 64 ? OP_LANES * OP_PER / 64 : 1)
ACC_DEV int op_again(const acc_route_args &p, const long long t, const int lane)
{
  const int size = p.experts / p.groups;
  const auto largest = [](double a, double b) { return op_most(a, b); };
  double v[OP_AGAIN];
#pragma unroll
  for (int i = 0; i < OP_AGAIN; ++i) {
    const int e = acc_min(i * 64 + lane, p.experts - 1);
    v[i] = op_ranked64(op_logit(p, t, e), op_bias(p, e));
    if (i * 64 + lane >= p.experts) v[i] = (double)OP_NONE;
  }
  if (p.keep < p.groups) {
    double mine = (double)OP_NONE;                 /* lane g: group g's */
    for (int g = 0; g < p.groups; ++g) {
      double best = (double)OP_NONE, next = best;
#pragma unroll
      for (int i = 0; i < OP_AGAIN; ++i) {
        const int in = i * 64 + lane - g * size;
        const double w = in >= 0 && in < size ? v[i] : (double)OP_NONE;
        next = op_most(next, op_least(best, w));
        best = op_most(best, w);
      }
      const double all = acc_wave_reduce(best, largest);
      /* (the first lane that has it gives its next) */
      const unsigned long long has = __ballot(best == all);
      const double second = acc_wave_reduce(lane == __builtin_ctzll(has) ? next : best, largest);
      if (lane == g) mine = all > (double)OP_NONE ? op_sum_of(all, second) : all;
    }
    int before = 0;
    for (int g = 0; g < p.groups; ++g) {
      const double other = acc_readlane(mine, g);
      before += other > mine || (other == mine && g < lane);
    }
    const unsigned long long kept = __ballot(lane < p.groups && before < p.keep);
#pragma unroll
    for (int i = 0; i < OP_AGAIN; ++i)
      if (i * 64 + lane < p.experts && !(kept >> ((i * 64 + lane) / size) & 1)) v[i] = (double)OP_NONE;
  }
  int chosen = -1;
  for (int j = 0; j < OP_CHOOSE; ++j) {
    double best = (double)OP_NONE;
    int index = 0x7fffffff;
#pragma unroll
    for (int i = OP_AGAIN - 1; i >= 0; --i) {
      if (v[i] >= best && v[i] > (double)OP_NONE) index = i * 64 + lane;
      best = op_most(best, v[i]);
    }
    const double all = acc_wave_reduce(best, largest);
    if (!(all > (double)OP_NONE)) break;
    const int first = acc_wave_reduce(best == all ? index : 0x7fffffff, [](int a, int b) { return a < b ? a : b; });
    if (lane == j) chosen = first;
#pragma unroll
    for (int i = 0; i < OP_AGAIN; ++i)
      if (i * 64 + lane == first) v[i] = (double)OP_NONE;
  }
  return chosen;
}

/* workgroup b has the tokens b * block .. ; with one workgroup the slots are placed at once, otherwise the counts go out */
extern "C" __global__ void __launch_bounds__(64 * OP_SELECT_WAVES) score(const acc_route_args p)
{
  if (p.guard && *p.guard == 0u) return;
  extern __shared__ int shared[];                  /* OP_FEW: 4 * experts counts, experts bases, experts totals, slots; else experts counts; groups */
  __shared__ int all;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), sub = lane % OP_LANES, token = lane / OP_LANES;
  const long long first = (long long)blockIdx.x * p.block, last = acc_min<long long>(p.tokens, first + p.block);
  const long long share = (long long)((p.block + OP_SELECT_WAVES * OP_TOKENS - 1) / (OP_SELECT_WAVES * OP_TOKENS)) * OP_TOKENS;
  const long long mine = first + wave * share, end = acc_min(last, mine + share);
  const int lots = OP_FEW ? OP_SELECT_WAVES : 1, size = p.experts / p.groups;
  int *const counts = shared + (OP_FEW ? wave * p.experts : 0), *const base = shared + lots * p.experts, *const sums = base + p.experts, *const slots = sums + p.experts;
  float *const groups = (float *)(OP_FEW ? slots + (last - first) * OP_CHOOSE : base) + (wave * OP_TOKENS + token) * 2 * p.groups;      /* sums, and what they may be off */
  for (int i = tid; i < lots * p.experts; i += 64 * OP_SELECT_WAVES) shared[i] = 0;
  __syncthreads();

  /* the lane's logits: a part of a group that it shares with others, or all of it */
  const int lanes = OP_LANES / p.groups, part = (size + lanes - 1) / lanes, own = sub / lanes;
  const int from = own * size + sub % lanes * part, count = acc_max(0, acc_min(part, size - sub % lanes * part));
  bool later = false;
  for (long long at = mine; at < end; at += OP_TOKENS) {
    const long long t = at + token;
    const bool here = t < end;
    const op_elt *const x = (const op_elt *)p.logits + (here ? t : mine) * p.logits_stride + from;
    acc_u4 raw[OP_PER / OP_VALUES];
#pragma unroll
    for (int c = 0; c < OP_PER / OP_VALUES; ++c) raw[c] = op_chunk<false>(x + c * OP_VALUES, count - c * OP_VALUES);
    float r[OP_PER];
#pragma unroll
    for (int c = 0; c < OP_PER / OP_VALUES; ++c) {
      op_elt e[OP_VALUES];
      __builtin_memcpy(e, &raw[c], 16);
      float bias[OP_VALUES];
#pragma unroll
      for (int i = 0; i < OP_VALUES; ++i) bias[i] = 0.0f;
      if (p.bias) {
        if (c * OP_VALUES + OP_VALUES <= count) {
#pragma unroll
          for (int h = 0; h < OP_VALUES / 4; ++h) {
            const acc_u4 u = ((const op_loose<float> *)(p.bias + from + c * OP_VALUES + h * 4))->v;
            __builtin_memcpy(bias + h * 4, &u, 16);
          }
        } else {
#pragma unroll
          for (int i = 0; i < OP_VALUES; ++i)
            if (c * OP_VALUES + i < count) bias[i] = p.bias[from + c * OP_VALUES + i];
        }
      }
#pragma unroll
      for (int i = 0; i < OP_VALUES; ++i) r[c * OP_VALUES + i] = c * OP_VALUES + i < count ? op_ranked((float)e[i], bias[i]) : OP_NONE;
    }
    bool unsure = false;
    if (p.keep < p.groups) {
      op_two two = {OP_NONE, OP_NONE};
#pragma unroll
      for (int k = 0; k < OP_PER; ++k) op_put(two, r[k]);
#pragma unroll
      for (int apart = 1; apart < OP_LANES; apart *= 2) {
        const float best = op_other(two.best, apart), next = op_other(two.next, apart);
        if (apart < lanes) {
          op_put(two, best);
          op_put(two, next);
        }
      }
      const float s = op_group_sum(two), off = op_off(two.best, two.next);
      groups[2 * own] = s;
      groups[2 * own + 1] = off;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      /* a group stays if fewer than `keep` are larger for certain, and is in doubt if as many may be */
      int before = 0, above = 0, beside = 0;
#pragma unroll 4
      for (int o = 0; o < p.groups; ++o) {
        const float v = groups[2 * o], near = off + groups[2 * o + 1];
        before += v > s || (v == s && o < own);
        above += v > s + near;
        beside += v >= s - near && o != own;
      }
      unsure = s > OP_NONE && above < p.keep && beside >= p.keep;
      if (before >= p.keep)
#pragma unroll
        for (int k = 0; k < OP_PER; ++k) r[k] = OP_NONE;
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    double key[OP_KEYS];
#pragma unroll
    for (int j = 0; j < OP_KEYS; ++j) key[j] = (double)OP_NONE;
#pragma unroll
    for (int k = 0; k < OP_PER; ++k) {
      op_insert(key, op_key_of(r[k], from + k));
      __builtin_amdgcn_sched_barrier(0);           /* (or all are made first: registers) */
    }
#pragma unroll
    for (int apart = 1; apart < OP_LANES; apart *= 2) {
      double other[OP_KEYS];
#pragma unroll
      for (int j = 0; j < OP_KEYS; ++j) other[j] = op_other(key[j], apart);
#pragma unroll
      for (int j = 0; j < OP_KEYS; ++j) op_insert(key, other[j]);
      __builtin_amdgcn_sched_barrier(0);
    }
    /* the j-th choice is the affair of lane j % OP_LANES: whether the one behind it is too near, its weight */
    int expert[(OP_CHOOSE + OP_LANES - 1) / OP_LANES];
#pragma unroll
    for (int j = 0; j < OP_CHOOSE; ++j) {
      if (j % OP_LANES == sub) expert[j / OP_LANES] = op_index_of(key[j]);
      const float v = op_value_of(key[j]), w = op_value_of(key[j + 1]);
      if (j % OP_LANES == sub && here && w > OP_NONE && v - w <= op_near(v)) {
        const int a = op_index_of(key[j]), b = op_index_of(key[j + 1]);
        unsure = unsure || op_logit(p, t, a) != op_logit(p, t, b) || op_bias(p, a) != op_bias(p, b);
      }
    }
    /* ... and, where the first that is not chosen may be as good as the last that is, whether there are more such, of other logits */
    const float end_value = op_value_of(key[OP_CHOOSE]), end_near = end_value - op_near(end_value);
    const bool edge = here && end_value > OP_NONE && op_value_of(key[OP_CHOOSE - 1]) - end_value <= op_near(end_value);
    if (__ballot(edge) != 0) {
      const int a = acc_max(op_index_of(key[OP_CHOOSE]), 0);
      const float end_logit = op_logit(p, here ? t : mine, a), end_bias = op_bias(p, a);
#pragma unroll
      for (int k = 0; k < OP_PER; ++k)
        if (edge && r[k] >= end_near && op_key_of(r[k], from + k) < key[OP_CHOOSE])
          unsure = unsure || op_logit(p, t, from + k) != end_logit || op_bias(p, from + k) != end_bias;
    }
    /* (a token that is to be decided again is marked, and left for when the registers are free) */
    const unsigned long long doubt = __ballot(unsure && here);
    later = later || doubt != 0;
    const bool sure = here && (doubt >> (OP_LANES < 64 ? token * OP_LANES : 0) & (OP_LANES < 64 ? (1ull << (OP_LANES & 63)) - 1 : ~0ull)) == 0;
    if (here && !sure && sub == 0) __hip_atomic_store(p.chosen + t * OP_CHOOSE, -2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    float w[(OP_CHOOSE + OP_LANES - 1) / OP_LANES], most = OP_NONE, total = 0.0f;
#pragma unroll
    for (int s = 0; s < (OP_CHOOSE + OP_LANES - 1) / OP_LANES; ++s) {
      const bool some = here && s * OP_LANES + sub < OP_CHOOSE && expert[s] >= 0;
      w[s] = some ? op_logit(p, t, expert[s]) : OP_NONE;
      most = w[s] > most ? w[s] : most;
    }
#pragma unroll
    for (int apart = 1; apart < OP_LANES; apart *= 2) {
      const float other = op_other(most, apart);
      most = other > most ? other : most;
    }
    const float shift = p.normalise ? acc_min(most, 0.0f) : 0.0f;
#pragma unroll
    for (int s = 0; s < (OP_CHOOSE + OP_LANES - 1) / OP_LANES; ++s) {
      w[s] = op_part(w[s], shift);
      total += w[s];
    }
#pragma unroll
    for (int apart = 1; apart < OP_LANES; apart *= 2) total += op_other(total, apart);
#pragma unroll
    for (int s = 0; s < (OP_CHOOSE + OP_LANES - 1) / OP_LANES; ++s) {
      const int j = s * OP_LANES + sub;
      if (!sure || j >= OP_CHOOSE) continue;
      const int e = expert[s];
      p.chosen[t * OP_CHOOSE + j] = e;
      if (OP_FEW) slots[t * OP_CHOOSE + j] = e;
      p.weights[t * OP_CHOOSE + j] = e < 0 ? 0.0f : !p.normalise ? p.scale * w[s] : total > 0.0f ? p.scale * (w[s] / total) : 0.0f;
      if (e >= 0) atomicAdd(&counts[e], 1);
    }
  }
  if (later) {
    __threadfence();
    for (long long at = mine; at < end; at += 64) {
      const bool here = at + lane < end;
      unsigned long long marked = __ballot(here && __hip_atomic_load(p.chosen + (at + (here ? lane : 0)) * OP_CHOOSE, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == -2);
      while (marked) {
        const long long t = at + __builtin_ctzll(marked);
        marked &= marked - 1;
        const int e = op_again(p, t, lane);
        const float x = e >= 0 ? op_logit(p, t, e) : OP_NONE;
        const float most = acc_wave_reduce(x, [](float a, float b) { return a > b ? a : b; }), w = op_part(x, p.normalise ? acc_min(most, 0.0f) : 0.0f);
        const float total = acc_wave_reduce(w, [](float a, float b) { return a + b; });
        if (lane >= OP_CHOOSE) continue;
        p.chosen[t * OP_CHOOSE + lane] = e;
        if (OP_FEW) slots[t * OP_CHOOSE + lane] = e;
        p.weights[t * OP_CHOOSE + lane] = e < 0 ? 0.0f : !p.normalise ? p.scale * w : total > 0.0f ? p.scale * (w / total) : 0.0f;
        if (e >= 0) atomicAdd(&counts[e], 1);
      }
    }
  }
  __threadfence_block();
  __syncthreads();
  if (!OP_FEW) {
    for (int e = tid; e < p.experts; e += 64 * OP_SELECT_WAVES) p.counts[(long long)blockIdx.x * p.experts + e] = (unsigned int)shared[e];
    return;
  }
#if OP_FEW
  for (int e = tid; e < p.experts; e += OP_THREADS) {
    int n = 0;
#pragma unroll
    for (int w = 0; w < OP_WAVES; ++w) n += shared[w * p.experts + e];
    base[e] = 0;
    sums[e] = n;
  }
  __syncthreads();
  op_bases(p, base, sums, true, tid, &all);
  op_starts(p, shared, base, tid);
  op_place(p, slots, mine * OP_CHOOSE, end * OP_CHOOSE, counts, op_index_bits(p.experts), lane);
  for (long long s = all + tid; s < p.tokens * OP_CHOOSE; s += OP_THREADS) p.order[s] = -1;
#endif
}

/* d logit_j = d score_j s_j (1 - s_j) of the chosen ones, zero elsewhere; d score = scale dw, or, where weights are normalised,
 * scale (dw_j - sum_i dw_i share_i) / sum s.  A token has OP_ROW lanes, one a choice, which then write 16 bytes of its row each: 32768
 * tokens of 256 in bfloat16 11.4 us, 3.1 TB/s of the 36 MB.  Bound by vector instructions, which take 96 in 100 of the SIMDs' cycles:
 * every lane compares every choice with each of its columns, to write what are nearly all zeros.  (share_j (1 - s_j) is what a score's part in the sum comes to: nothing is divided by a sum of small scores.) */
extern "C" __global__ void __launch_bounds__(256) score_gradient(const acc_route_args p)
{
  if (p.guard && *p.guard == 0u) return;
  const int lane = acc_lane(), j = lane % OP_ROW;
  const long long t = ((long long)blockIdx.x * 256 + threadIdx.x) / OP_ROW;
  const bool here = t < p.tokens;
  const int e = here && j < OP_CHOOSE ? p.chosen[t * OP_CHOOSE + j] : -1;
  const bool some = e >= 0 && e < p.experts;
  const float x = some ? op_logit(p, t, e) : OP_NONE, dw = some ? p.dweights[t * OP_CHOOSE + j] : 0.0f;
  float most = x;
#pragma unroll
  for (int apart = 1; apart < OP_ROW; apart *= 2) {
    const float other = op_other(most, apart);
    most = other > most ? other : most;
  }
  const float s = op_part(x, p.normalise ? acc_min(most, 0.0f) : 0.0f), rest = x >= 0.0f ? expf(-x) / (1.0f + expf(-x)) : 1.0f / (1.0f + expf(x));
  float total = s;
#pragma unroll
  for (int apart = 1; apart < OP_ROW; apart *= 2) total += op_other(total, apart);
  const float share = p.normalise ? (total > 0.0f ? s / total : 0.0f) : s;
  float inner = p.normalise ? dw * share : 0.0f;
#pragma unroll
  for (int apart = 1; apart < OP_ROW; apart *= 2) inner += op_other(inner, apart);
  const float d = some ? p.scale * share * (dw - inner) * rest : 0.0f;

  op_elt *const out = (op_elt *)p.dlogits + (here ? t : 0) * p.dlogits_stride;
  for (int c = j * OP_VALUES; c - j * OP_VALUES < p.experts; c += OP_ROW * OP_VALUES) {
    op_elt v[OP_VALUES];
#pragma unroll
    for (int k = 0; k < OP_VALUES; ++k) v[k] = (op_elt)0.0f;
#pragma unroll
    for (int n = 0; n < OP_CHOOSE; ++n) {
      const int from = (lane - j + n) * 4, at = __builtin_amdgcn_ds_bpermute(from, e) - c;
      const op_elt value = (op_elt)__uint_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_uint(d)));
#pragma unroll
      for (int k = 0; k < OP_VALUES; ++k) v[k] = at == k ? value : v[k];
    }
    if (!here || c >= p.experts) continue;
    if (c + OP_VALUES <= p.experts) {
      acc_u4 u;
      __builtin_memcpy(&u, v, 16);
      ((op_loose<op_elt> *)(out + c))->v = u;
    } else {
#pragma unroll
      for (int k = 0; k < OP_VALUES; ++k)
        if (c + k < p.experts) out[c + k] = v[k];
    }
  }
}
