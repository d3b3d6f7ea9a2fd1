// Routing with a balance bias and groups of experts (b200dnn_moe_gate).
//
//   s = softmax(x) or 1 / (1 + exp(-x));   c = s + bias;   group score: the largest c of the group, or the sum of its two largest;
//   the topk_groups best groups; the topk largest c in them, ties to the lower index;   w = s (/ their sum) * scale
//
// The order is that of scores held in 64 bits: with 16384 tokens over 256 experts some pair of neighbours in some token lies closer than 32 bits tell.
#pragma once
#include "common.cuh"

namespace b200 {

constexpr int kGateMaxTopk = 16;

struct GateArgs {
  const void *logits; int64_t ld; int logits_bf16;
  const float *bias;
  int T, E, k, sigmoid, groups, top_groups, per_group, top2, renorm;
  float scale;
  int32_t *ids; float *weights;
  int chunk; int32_t *counts;             // tokens of one CTA; [CTA][E] slots per expert, null when not wanted
};

// Values as unsigned numbers of the same order; 0 is left for experts that are out, 1 for a NaN.
__device__ __forceinline__ unsigned long long gate_key(double c) {
  if (c != c) return 1ull;
  const unsigned long long b = (unsigned long long)__double_as_longlong(c);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

// The largest key of the warp and the lowest of the ids that lanes name for it (the key as two words: each a reduction in hardware).
__device__ __forceinline__ void gate_best(unsigned long long &key, int &id) {
  const unsigned all = 0xffffffffu, hi = (unsigned)(key >> 32), lo = (unsigned)key;
  const unsigned top_hi = __reduce_max_sync(all, hi), top_lo = __reduce_max_sync(all, hi == top_hi ? lo : 0u);
  id = (int)__reduce_min_sync(all, hi == top_hi && lo == top_lo ? (unsigned)id : 0x7fffffffu);
  key = (unsigned long long)top_hi << 32 | top_lo;
}

__device__ __forceinline__ float gate_logit(const GateArgs &a, int64_t at) {
  return a.logits_bf16 ? bf16_bits_to_f32(__ldg(reinterpret_cast<const uint16_t *>(a.logits) + at)) : __ldg(reinterpret_cast<const float *>(a.logits) + at);
}

// A token in 64 bits, in three parts.  Scores s and keys lie in memory, expert after expert.
// The softmax's largest logit (a warp's reduction)
__device__ __forceinline__ float gate_largest(const GateArgs &a, int64_t t, int lane) {
  float mx = __int_as_float(0xff800000);
  for (int e = lane; e < a.E; e += 32) mx = fmaxf(mx, gate_logit(a, t * a.ld + e));
#pragma unroll
  for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  return mx;
}
// An expert's exponential, and its score and key from it
__device__ __forceinline__ double gate_exp(const GateArgs &a, int64_t t, int e, float mx) {
  const double x = (double)gate_logit(a, t * a.ld + e);
  return exp(a.sigmoid ? -x : x - (double)mx);
}
__device__ __forceinline__ unsigned long long gate_score(const GateArgs &a, int e, double sum, double &s) {
  s = (a.sigmoid ? 1.0 : s) / (a.sigmoid ? 1.0 + s : sum);
  return gate_key(a.bias ? s + (double)a.bias[e] : s);
}
// The choice, by one warp (the keys are used up).  Lane i < k returns the i-th and its score.
__device__ __noinline__ void gate_choose(const GateArgs &a, const double *s, unsigned long long *key, int lane, int &id, double &score) {
  // the largest key of experts [from, to) but `without`, and its id
  auto best = [&](int from, int to, int without, unsigned long long &top, int &id_of) {
    top = 0ull; id_of = 0x7fffffff;
    for (int e = from + lane; e < to; e += 32) {
      const unsigned long long k = key[e];
      if (e != without && k > top) { top = k; id_of = e; }
    }
    gate_best(top, id_of);
  };
  unsigned long long top;
  int id_of;
  if (a.groups > 1) {
    // lane g: the score of group g
    unsigned long long mine = 0ull;
#pragma unroll 1
    for (int g = 0; g < a.groups; ++g) {
      double total = 0.0;
      int first = -1;
#pragma unroll 1
      for (int r = 0; r <= a.top2; ++r) {
        best(g * a.per_group, (g + 1) * a.per_group, first, top, id_of);
        if (top == 0ull) break;              // a group of one expert
        first = id_of;
        const double c = top == 1ull ? __longlong_as_double(0x7ff8000000000000ll) : __longlong_as_double((long long)(top >> 63 ? top & 0x7fffffffffffffffull : ~top));
        total = r == 0 ? c : total + c;
      }
      if (lane == g) mine = gate_key(total);
    }
    int rank = 0;
#pragma unroll 1
    for (int g = 0; g < a.groups; ++g) {
      const unsigned long long other = __shfl_sync(0xffffffffu, mine, g);
      rank += other > mine || (other == mine && g < lane);
    }
    const unsigned chosen = __ballot_sync(0xffffffffu, lane < a.groups && rank < a.top_groups);
    for (int g = 0; g < a.groups; ++g)
      if (!((chosen >> g) & 1u)) for (int e = g * a.per_group + lane; e < (g + 1) * a.per_group; e += 32) key[e] = 0ull;
    __syncwarp();
  }
  id = 0; score = 0.0;
#pragma unroll 1
  for (int r = 0; r < a.k; ++r) {
    best(0, a.E, -1, top, id_of);
    if (lane == r) { id = id_of; score = s[id_of]; }
    if (lane == 0) key[id_of] = 0ull;
    __syncwarp();
  }
}

// The same in 32 bits, where these are enough.  f32 scores carry errors of a few steps, and the choice is taken for the one that 64 bits would make when every comparison that decides it is clear
// by more than these: between neighbours among the chosen, between the last of them and all that is left (of which the best stands for the others; their errors are bounded with it), between the last chosen group and the next.
// (Experts with one logit and one bias have one score in either width, and go by their index; where the last choice is one of several such, it is all of these that the next has to be behind.)  Choices that are not clear, one token in two thousand over 256 experts with continuous
// logits, are put in order by the 64-bit scores of these alone.  False: the token needs all its scores in 64 bits.  Returns the weights' scores in f32; the sum of the chosen is left to the caller.
__device__ __forceinline__ uint32_t gate_key(float c) {      // (no NaN)
  const int b = __float_as_int(c);
  return (uint32_t)(b ^ (b >> 31 | (int)0x80000000));
}
__device__ __forceinline__ float gate_value(uint32_t key) {
  return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}
template <int N> __device__ __forceinline__ float gate_sum(const float (&v)[N]) {
  if constexpr (N == 1) return v[0];
  else {
    float h[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) h[i] = v[2 * i] + v[2 * i + 1];
    return gate_sum<N / 2>(h);
  }
}
// 1 / x to 2^-23 for x >= 1 (0 for infinity)
__device__ __forceinline__ float gate_rcp(float x) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

// Sorts PER keys of a lane, largest first (Batcher's odd-even merge sort, 1968; PER a power of two).
template <int PER> __device__ __forceinline__ void gate_sort(uint32_t (&v)[PER]) {
#pragma unroll
  for (int p = 1; p < PER; p *= 2)
#pragma unroll
    for (int k = p; k >= 1; k /= 2)
#pragma unroll
      for (int j = k % p; j + k < PER; j += 2 * k)
#pragma unroll
        for (int i = 0; i < k; ++i)
          if (i + j + k < PER && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const uint32_t lo = min(v[i + j], v[i + j + k]);
            v[i + j] = max(v[i + j], v[i + j + k]);
            v[i + j + k] = lo;
          }
}

// x, bias: minus infinity behind the last expert.  group_of: groups of the lane's experts, a byte each.
template <int PER>
__device__ __forceinline__ bool gate_token_f32(const GateArgs &a, int t, const float (&x)[PER], const float (&bias)[PER], const uint32_t (&group_of)[(PER + 3) / 4], int lane, int &id,
                                               float &score) {
  const unsigned all = 0xffffffffu;
  float mx = 0.f, sum = 1.f, most = 1.f;       // of the softmax: largest logit, denominator; bound of the scores
  uint32_t key[PER];
  {
    float s[PER];
    if (a.sigmoid) {
#pragma unroll
      for (int j = 0; j < PER; ++j) s[j] = gate_rcp(1.0f + __expf(-x[j]));
    } else {
      mx = __int_as_float(0xff800000);
#pragma unroll
      for (int j = 0; j < PER; ++j) mx = fmaxf(mx, x[j]);
#pragma unroll
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(all, mx, o));
#pragma unroll
      for (int j = 0; j < PER; ++j) s[j] = __expf(x[j] - mx);
      sum = gate_sum<PER>(s);
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(all, sum, o);
      most = __fdividef(1.0f, sum);
#pragma unroll
      for (int j = 0; j < PER; ++j) s[j] *= most;
      // (a NaN, an infinity, or minus infinity throughout: there is no softmax)
      if (!(sum >= 0.99f && sum < 3e38f)) return false;
    }
    bool nan = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const float c = s[j] + bias[j];
      nan |= c != c;
      key[j] = gate_key(c);
    }
    if (__any_sync(all, nan)) return false;
    if (a.E != PER * 32) {
#pragma unroll
      for (int j = 0; j < PER; ++j) if (j * 32 + lane >= a.E) key[j] = 0u;
    }
  }
  // Errors, relative: the exponential (ex2.approx, 2^-22) with the rounding of its argument, 6e-8 for every unit of it, twice for a softmax (its difference is rounded too); a sum and a quotient: 7e-7 together;
  // a softmax's denominator up to 4e-6.  A group's two scores, each at most `most`: 1.2e-7 |d| exp(-|d|) of it, which 1e-7 covers (and the rounding of its sum, see sum_err).
  const float off = a.sigmoid ? 8e-7f : 5e-6f;
  bool clear = true;
  if (a.groups > 1) {
    uint32_t first = 0u, second = 0u;          // lane g: the two largest keys of group g
    const unsigned per = (unsigned)a.per_group;
    if (per % 32 == 0) {
      // Groups of whole elements: the two largest of every element over the lanes, by halves -- a lane hands half of the elements that it still has to the lane across and takes in the
      // other half's; lane l is left with element l / (32 / PER).  (Reductions element by element: 17 of 34 us for 16384 tokens, 256 experts in eight groups.)
      uint32_t t1[PER], t2[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) { t1[j] = key[j]; t2[j] = 0u; }
      auto merge = [&](int i, uint32_t o1, uint32_t o2) {
        t2[i] = max(min(t1[i], o1), max(t2[i], o2));
        t1[i] = max(t1[i], o1);
      };
#pragma unroll
      for (int half = PER / 2, bit = 16; bit >= 1; half /= 2, bit /= 2) {
        const bool upper = lane & bit;
        if (half == 0) merge(0, __shfl_xor_sync(all, t1[0], bit), __shfl_xor_sync(all, t2[0], bit));
#pragma unroll
        for (int i = 0; i < half; ++i) {
          const uint32_t s1 = upper ? t1[i] : t1[i + half], s2 = upper ? t2[i] : t2[i + half];
          t1[i] = upper ? t1[i + half] : t1[i];
          t2[i] = upper ? t2[i + half] : t2[i];
          merge(i, __shfl_xor_sync(all, s1, bit), __shfl_xor_sync(all, s2, bit));
        }
      }
      const int elements = (int)per / 32;
      for (int i = 0; i < elements; ++i) {     // of group `lane`
        const int from = min(lane * elements + i, PER - 1) * (32 / PER);
        const uint32_t o1 = __shfl_sync(all, t1[0], from), o2 = __shfl_sync(all, t2[0], from);
        second = max(min(first, o1), max(second, o2));
        first = max(first, o1);
      }
    } else {
      auto best_two = [&](uint32_t t1, uint32_t t2, int g) {      // of a lane's members
        const uint32_t m1 = __reduce_max_sync(all, t1);
        if (lane == g) first = m1;
        if (a.top2) {
          const bool mine = lane == __ffs(__ballot_sync(all, t1 == m1)) - 1;
          const uint32_t m2 = __reduce_max_sync(all, mine ? t2 : t1);
          if (lane == g) second = m2;
        }
      };
      for (int g = 0; g < a.groups; ++g) {
        uint32_t t1 = 0u, t2 = 0u;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const uint32_t k = (unsigned)(j * 32 + lane) - (unsigned)g * per < per ? key[j] : 0u;
          t2 = max(t2, min(t1, k));
          t1 = max(t1, k);
        }
        best_two(t1, t2, g);
      }
    }
    if (!a.top2) second = 0u;
    // (a group of one expert has no second)
    const uint32_t mine = lane >= a.groups ? 0u : second ? gate_key(gate_value(first) + gate_value(second)) : first;
    // A bias can make the two of a sum large and their sum small, of any group: its roundings go by the largest pair (an infinite one has no error, a sum that overflows is clear of nothing).
    float sum_err = 0.f;
    if (a.top2 && a.bias) {
      const float v1 = fabsf(gate_value(first)), v2 = fabsf(gate_value(second));
      const bool pair = lane < a.groups && second != 0u && finite_f32(v1) && finite_f32(v2);
      sum_err = 3e-7f * __uint_as_float(__reduce_max_sync(all, pair ? __float_as_uint(v1 + v2) : 0u));
    }
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint32_t other = __shfl_sync(all, mine, g);
      rank += other > mine || (other == mine && g < lane);
    }
    unsigned chosen = __ballot_sync(all, lane < a.groups && rank < a.top_groups);
    if (a.top_groups < a.groups) {
      auto group_at = [&](int r) { return __ffs(__ballot_sync(all, lane < a.groups && rank == r)) - 1; };
      auto value_of = [&](int g) { return gate_value(__shfl_sync(all, mine, g)); };
      auto behind = [&](float u, float v, float more) { return u - v > 4.f * (off + 1e-7f) * most + 3e-7f * (fabsf(u) + fabsf(v)) + more + 1e-36f; };
      const int last = group_at(a.top_groups - 1), next = group_at(a.top_groups);
      const float u = value_of(last), v = value_of(next);
      clear = behind(u, v, sum_err);
      if (!clear && (a.sigmoid || !a.bias)) {
        // The last group that is in and the first that is out are too close (in 16384 tokens of 256 experts two or three times): their scores in 64 bits, from their members', where these two are
        // clear of the others and the members that count are clear of those that do not.
        clear = (a.top_groups < 2 || behind(value_of(group_at(a.top_groups - 2)), u, sum_err)) && (a.top_groups + 1 >= a.groups || behind(v, value_of(group_at(a.top_groups + 1)), sum_err));
        double total[2];
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          const int g = i ? next : last;
          int members[2] = {-1, -1};
          uint32_t top = 0u, before = 0u;
#pragma unroll 1
          for (int r = 0; r <= a.top2 + 1; ++r) {
            uint32_t best = 0u; int at = 0;
#pragma unroll
            for (int j = 0; j < PER; ++j) {
              const int e = j * 32 + lane;
              if ((unsigned)(e - g * (int)per) < per && e != members[0] && e != members[1] && key[j] > best) { best = key[j]; at = e; }
            }
            before = top;
            top = __reduce_max_sync(all, best);
            const int e = (int)__reduce_min_sync(all, best == top ? (unsigned)at : 0x7fffffffu);
            if (r <= a.top2 && top != 0u) members[r] = e;
            // the first that does not count: clearly behind, or there is none
            if (r == a.top2 + 1 && top != 0u && !behind(gate_value(before), gate_value(top), 0.f)) clear = false;
          }
          double c = 0.0;
          if (lane < 2 && members[lane] >= 0) {
            const double x64 = (double)gate_logit(a, t * a.ld + members[lane]), e64 = exp(a.sigmoid ? -x64 : x64 - (double)mx);
            c = a.sigmoid ? 1.0 / (1.0 + e64) + (a.bias ? (double)a.bias[members[lane]] : 0.0) : e64;
          }
          total[i] = __shfl_sync(all, c, 0) + __shfl_sync(all, c, 1);
        }
        if (clear && (total[1] > total[0] || (total[1] == total[0] && next < last))) chosen ^= 1u << last | 1u << next;
      }
#pragma unroll
      for (int j = 0; j < PER; ++j) if (!((chosen >> ((group_of[j / 4] >> (j % 4 * 8)) & 31u)) & 1u)) key[j] = 0u;
    }
  }
  // The choice, and the best that is left behind it: every lane's keys in order, the largest head of all lanes taken again and again.
  const int rounds = a.k + (a.k < a.top_groups * a.per_group);
  uint32_t head[PER], my_key = 0u;
  int my_id = 0, my_lane = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) head[j] = key[j];
  gate_sort<PER>(head);
  for (int r = 0; r < rounds; ++r) {
    const uint32_t top = __reduce_max_sync(all, head[0]);
    const int from = __ffs(__ballot_sync(all, head[0] == top)) - 1;
    if (lane == from) {
#pragma unroll
      for (int j = 0; j + 1 < PER; ++j) head[j] = head[j + 1];
      head[PER - 1] = 0u;
    }
    if (lane == r) { my_key = top; my_lane = from; }
  }
  const uint32_t key_behind = __shfl_down_sync(all, my_key, 1);
  // the lowest index of the largest key, again and again, from the r0-th choice on (keys of a lane that are chosen become 0)
  auto choose = [&](int r0, int r1) {
#pragma unroll 1
    for (int r = r0; r < r1; ++r) {
      uint32_t best = key[0]; int at = 0;
#pragma unroll
      for (int j = 1; j < PER; ++j) if (key[j] > best) { best = key[j]; at = j; }
      const uint32_t top = __reduce_max_sync(all, best);
      const int e = __reduce_min_sync(all, best == top ? (unsigned)(at * 32 + lane) : 0x7fffffffu);
#pragma unroll
      for (int j = 0; j < PER; ++j) if (e == j * 32 + lane) key[j] = 0u;
      if (lane == r) { my_id = e; my_key = top; }
    }
  };
  const bool equal = __any_sync(all, lane + 1 < rounds && my_key == key_behind);
  if (!equal) {
    // which of its lane's experts a choice is
#pragma unroll
    for (int j = 0; j < PER; ++j) if (__shfl_sync(all, key[j], my_lane) == my_key) my_id = j * 32 + my_lane;
  } else choose(0, rounds);
  float my_x = 0.f, my_b = 0.f;
  auto look = [&](int r1) {
    if (lane < r1) {
      my_x = gate_logit(a, t * a.ld + my_id);
      my_b = a.bias ? a.bias[my_id] : 0.f;
    }
    if (a.sigmoid) score = __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-my_x)));
    else {
      // the difference, and what its rounding left out (of minus infinity: nothing)
      const float d = __fsub_rn(my_x, mx), back = __fsub_rn(d, my_x), rest = __fsub_rn(__fsub_rn(my_x, __fsub_rn(d, back)), __fadd_rn(mx, back));
      score = d < -1e30f ? 0.f : __fdiv_rn(expf(d) * (1.0f + rest), sum);
    }
  };
  // Is this lane's choice before the next lane's in 64 bits too?  By the errors of these two; where the choices end, those that are not in front of the next one have to lie behind as well (all_behind).
  // Without a bias these have smaller scores, and smaller errors; with one, any expert's score may lie behind a tiny one, and it is the error of the largest that counts.
  const float most_err = 2.f * (off + 1.2e-7f) * most;      // (an exponential's argument adds |x| exp(-|x|) < 0.4 of its rounding)
  bool same = false, all_behind = false;       // same: one logit and one bias
  auto before_next = [&]() {
    const float c = gate_value(my_key), c2 = __shfl_down_sync(all, c, 1), x2 = __shfl_down_sync(all, my_x, 1), b2 = __shfl_down_sync(all, my_b, 1), s2 = __shfl_down_sync(all, score, 1);
    const float err = off + (a.sigmoid ? 6e-8f * fmaxf(fabsf(my_x), fabsf(x2)) : 1.2e-7f * fmaxf(mx - my_x, mx - x2));
    same = my_x == x2 && my_b == b2;
    const float clear_by = c - c2 - (3e-7f * (fabsf(c) + fabsf(c2)) + 1e-36f), own = 2.f * err * fmaxf(score, s2);
    all_behind = clear_by > (a.bias ? most_err : own);
    return clear_by > own;
  };
  look(rounds);
  bool apart = before_next();
  id = my_id;
  bool past = true;
  if (rounds > a.k && a.bias) {
    // The cut: the largest error that can lie behind it, or, where that is too much, every expert's own (one token in some thousands: the keys below the last choice's are those that are left).
    if (__shfl_sync(all, (int)(apart && !all_behind), a.k - 1)) {
      const uint32_t key1 = __shfl_sync(all, my_key, a.k - 1);
      const float x1 = __shfl_sync(all, my_x, a.k - 1), c1 = gate_value(key1), err1 = (off + (a.sigmoid ? 6e-8f * fabsf(x1) : 1.2e-7f * (mx - x1))) * __shfl_sync(all, score, a.k - 1);
      const float ninf = __int_as_float(0xff800000);
      bool behind = true;
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (key[j] != 0u && key[j] < key1) {
          const float x2 = gate_logit(a, t * a.ld + j * 32 + lane), c2 = gate_value(key[j]);
          const float s2 = a.sigmoid ? gate_rcp(1.0f + __expf(-x2)) : __expf(x2 - mx) * most, err2 = (off + (a.sigmoid ? 6e-8f * fabsf(x2) : 1.2e-7f * (mx - x2))) * s2;
          behind &= c2 == ninf || c1 - c2 > err1 + err2 + 3e-7f * (fabsf(c1) + fabsf(c2)) + 1e-36f;      // (a bias of minus infinity: no error)
        }
      behind = __all_sync(all, behind);
      if (lane == a.k - 1) apart = behind;
    }
  }
  if (rounds > a.k && __shfl_sync(all, (int)(same && !apart), a.k - 1)) {
    // The last choice and the best that is left are one in logit and bias: what has to lie clearly behind is the best expert that is not.
    const float x1 = __shfl_sync(all, my_x, a.k - 1), b1 = __shfl_sync(all, my_b, a.k - 1), c1 = gate_value(__shfl_sync(all, my_key, a.k - 1)), s1 = __shfl_sync(all, score, a.k - 1);
    uint32_t best = 0u;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = j * 32 + lane;
      if (key[j] > best && (gate_logit(a, t * a.ld + e) != x1 || (a.bias && a.bias[e] != b1))) best = key[j];
    }
    best = __reduce_max_sync(all, best);
    const float c2 = gate_value(best), err = off + (a.sigmoid ? 6e-8f * fmaxf(fabsf(x1), 16.f) : 1.2e-7f * fmaxf(mx - x1, 1.f));
    past = best == 0u || c1 - c2 > (a.bias ? most_err : 2.f * err * s1) + 3e-7f * (fabsf(c1) + fabsf(c2)) + 1e-36f;
  }
  if (__all_sync(all, clear && past && (lane + 1 >= rounds || apart || same))) return true;
  // Some neighbours are too close.  Choices up to one that is clearly behind its predecessor, at the k-th or later, hold the right ones: these are put in order by 64-bit scores.
  if (!__all_sync(all, clear) || (!a.sigmoid && a.bias)) return false;
  const int candidates = a.top_groups * a.per_group, more = min(min(32, candidates), a.k + 8);
  choose(equal ? rounds : 0, more);
  look(more);
  before_next();
  const unsigned ends = __ballot_sync(all, all_behind && lane + 1 >= a.k && lane + 1 < more) | (more == candidates ? 1u << (more - 1) : 0u);
  if (ends == 0u) return false;
  const int p = __ffs(ends);                   // so many of them
  const double e64 = exp(a.sigmoid ? -(double)my_x : (double)my_x - (double)mx), c64 = a.sigmoid ? 1.0 / (1.0 + e64) + (double)my_b : e64;
  int rank = 0, from = 0;
#pragma unroll 1
  for (int q = 0; q < p; ++q) {
    const double c2 = __shfl_sync(all, c64, q);
    const int id2 = __shfl_sync(all, my_id, q);
    rank += c2 > c64 || (c2 == c64 && id2 < my_id);
  }
#pragma unroll 1
  for (int q = 0; q < p; ++q) if (__shfl_sync(all, rank, q) == lane) from = q;
  id = __shfl_sync(all, my_id, from);
  score = __shfl_sync(all, score, from);
  return true;
}

// Slots' places: rank of each of a chunk's slots inside its expert, behind next[e] rows.  All threads of a CTA; cnt: 32 bytes an expert, the slots that each warp has for it.
__device__ __forceinline__ void gate_places(const int32_t *ids, int64_t s0, int64_t s_end, int E, int *next, uint4 *cnt, int32_t *slot_to_row) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t front[8];                           // ones for the warps in front of this one
#pragma unroll
  for (int i = 0; i < 8; ++i) { const int n = warp - 4 * i; front[i] = n <= 0 ? 0u : n >= 4 ? 0x01010101u : 0x01010101u >> (32 - 8 * n); }
  for (; s0 < s_end; s0 += blockDim.x) {
    for (int i = tid; i < 2 * E; i += blockDim.x) cnt[i] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    const int64_t s = s0 + tid;
    const int e = s < s_end ? ids[s] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int before = __popc(same & ((1u << lane) - 1u));
    if (e >= 0 && before == 0) reinterpret_cast<uint8_t *>(cnt)[e * 32 + warp] = (uint8_t)__popc(same);
    __syncthreads();
    if (e >= 0) {
      const uint4 u = cnt[2 * e], v = cnt[2 * e + 1];
      unsigned row = (unsigned)(next[e] + before);
      row = __dp4a(u.x, front[0], row); row = __dp4a(u.y, front[1], row); row = __dp4a(u.z, front[2], row); row = __dp4a(u.w, front[3], row);
      row = __dp4a(v.x, front[4], row); row = __dp4a(v.y, front[5], row); row = __dp4a(v.z, front[6], row); row = __dp4a(v.w, front[7], row);
      slot_to_row[s] = (int32_t)row;
    }
    if (s0 + blockDim.x >= s_end) break;
    __syncthreads();
    for (int i = tid; i < E; i += blockDim.x) {
      const uint4 u = cnt[2 * i], v = cnt[2 * i + 1];
      unsigned n = (unsigned)next[i];
      const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) n = __dp4a(w[j], 0x01010101u, n);
      next[i] = (int)n;
    }
    __syncthreads();
  }
}
// next[e] += rows of the experts in front of e (one warp)
__device__ __forceinline__ void gate_offsets(const int *total, int *next, int E) {
  const int lane = threadIdx.x & 31;
  int carry = 0;
  for (int base = 0; base < E; base += 32) {
    const int e = base + lane, n = e < E ? total[e] : 0;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += v; }
    if (e < E) next[e] += carry + sum - n;
    carry += __shfl_sync(0xffffffffu, sum, 31);
  }
}

__host__ __device__ __forceinline__ int gate_pad(int E) { return (E + 3) & ~3; }      // counts of a chunk: whole vectors of four

// A CTA per chunk of tokens, a warp per token.  With a single chunk the places follow at once.  Bound by instruction issue, about 1200 a token: 16384 tokens over 256 experts in eight groups
// 25 us (0.70 of the issue slots), and 10 for the launch behind it.  Every token that goes to 64 bits costs its CTA microseconds: 16384 tokens whose scores a bias tells apart by 1e-9 alone 400 to 500 us.
struct GateRowsArgs { const int32_t *ids, *counts; int T, E, k, chunk; int32_t *expert_counts, *slot_to_row; };
constexpr int kGateThreads = 1024;
template <int PER> constexpr int kGateTokenThreads = PER <= 8 ? 1024 : 512;      // (registers for PER experts a lane)
template <int PER>
__global__ void __launch_bounds__(kGateTokenThreads<PER>) gate_kernel(const GateArgs a, const GateRowsArgs rows) {
  extern __shared__ int sm[];
  __shared__ int n_slow;
  int *hist = sm, *next = sm + gate_pad(a.E), *slow = sm + 2 * gate_pad(a.E) + 8 * a.E;      // (between them 32 bytes an expert)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t0 = blockIdx.x * a.chunk, t1 = min(a.T, t0 + a.chunk);
  const bool count = a.counts || rows.expert_counts || rows.slot_to_row;
  for (int i = threadIdx.x; i < a.E; i += blockDim.x) hist[i] = next[i] = 0;
  if (threadIdx.x == 0) n_slow = 0;
  __syncthreads();
  float bias[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) bias[j] = j * 32 + lane >= a.E ? __int_as_float(0xff800000) : a.bias ? a.bias[j * 32 + lane] : 0.f;
  uint32_t group_of[(PER + 3) / 4] = {};
#pragma unroll
  for (int j = 0; j < PER; ++j) group_of[j / 4] |= (uint32_t)(min(j * 32 + lane, a.E - 1) / a.per_group) << (j % 4 * 8);
  for (int t = t0 + warp; t < t1; t += (int)(blockDim.x >> 5)) {
    float x[PER];
    if (a.logits_bf16) {
      const uint16_t *p = reinterpret_cast<const uint16_t *>(a.logits) + t * a.ld + lane;
#pragma unroll
      for (int j = 0; j < PER; ++j) x[j] = j * 32 + lane < a.E ? bf16_bits_to_f32(__ldg(p + j * 32)) : __int_as_float(0xff800000);
    } else {
      const float *p = reinterpret_cast<const float *>(a.logits) + t * a.ld + lane;
#pragma unroll
      for (int j = 0; j < PER; ++j) x[j] = j * 32 + lane < a.E ? __ldg(p + j * 32) : __int_as_float(0xff800000);
    }
    int id; float w;
    bool done = gate_token_f32<PER>(a, t, x, bias, group_of, lane, id, w);
    if (a.renorm && done) {
      float sum = lane < a.k ? w : 0.f;
#pragma unroll
      for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      w = __fdiv_rn(w, sum);
      done = __shfl_sync(0xffffffffu, sum, 0) >= 1e-30f;      // (else the scores of the chosen are zero in 32 bits, or not whole)
    }
    if (!done) {
      if (lane == 0) slow[atomicAdd(&n_slow, 1)] = t;
      continue;
    }
    if (lane < a.k) {
      a.ids[(int64_t)t * a.k + lane] = id;
      if (a.weights) a.weights[(int64_t)t * a.k + lane] = w * a.scale;
      if (count) atomicAdd(&hist[id], 1);
    }
  }
  __syncthreads();
  // Tokens that 32 bits do not decide, by all threads: a thread per expert for the scores (an exponential and a quotient in 64 bits are thousands of clocks one after the other: a warp by itself took
  // 15 us for a token of 256 experts, and everyone waited), a warp for the choice.
  for (int i = 0; i < n_slow; ++i) {
    const int t = slow[i];
    double *s = reinterpret_cast<double *>(sm + 2 * gate_pad(a.E));
    unsigned long long *key = reinterpret_cast<unsigned long long *>(s + a.E);
    const float mx = a.sigmoid ? 0.f : gate_largest(a, t, lane);
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) s[e] = gate_exp(a, t, e, mx);
    __syncthreads();
    double sum = 1.0;
    if (!a.sigmoid) {
      sum = 0.0;
      for (int e = lane; e < a.E; e += 32) sum += s[e];
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      __syncthreads();
    }
    for (int e = threadIdx.x; e < a.E; e += blockDim.x) {
      double v = s[e];
      key[e] = gate_score(a, e, sum, v);
      s[e] = v;
    }
    __syncthreads();
    if (warp == 0) {
      int id; double score, all = 0.0;
      gate_choose(a, s, key, lane, id, score);
      for (int r = 0; r < a.k; ++r) all += __shfl_sync(0xffffffffu, score, r);
      if (lane < a.k) {
        a.ids[(int64_t)t * a.k + lane] = id;
        if (a.weights) a.weights[(int64_t)t * a.k + lane] = (float)((a.renorm ? score / all : score) * (double)a.scale);
        if (count) atomicAdd(&hist[id], 1);
      }
    }
    __syncthreads();
  }
  if (!count) return;
  if (a.counts) {
    for (int i = threadIdx.x; i < gate_pad(a.E); i += blockDim.x) a.counts[(int64_t)blockIdx.x * gate_pad(a.E) + i] = i < a.E ? hist[i] : 0;
    return;
  }
  if (rows.expert_counts) for (int i = threadIdx.x; i < a.E; i += blockDim.x) rows.expert_counts[i] = hist[i];
  if (!rows.slot_to_row) return;
  if (warp == 0) gate_offsets(hist, next, a.E);
  gate_places(a.ids, 0, (int64_t)a.T * a.k, a.E, next, reinterpret_cast<uint4 *>(sm + 2 * gate_pad(a.E)), rows.slot_to_row);
}

// The slots' places in the stable order by expert, from the counts of the chunks: every CTA adds up those of all chunks (first rows of the experts) and of the chunks
// in front of it, then ranks its own slots inside their experts.
__global__ void __launch_bounds__(kGateThreads) gate_rows_kernel(const GateRowsArgs a) {
  extern __shared__ int sm[];
  const int Ep = gate_pad(a.E);
  int *next = sm, *total = sm + Ep;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, warp = tid >> 5, me = blockIdx.x, chunks = gridDim.x;
  for (int e = tid; e < 2 * Ep; e += kGateThreads) sm[e] = 0;
  __syncthreads();
  {
    // parts of the chunks side by side, a thread per four experts in each
    const int width = Ep / 4, parts = kGateThreads / width, e = tid % width, part = tid / width;      // (E <= 1024)
    if (part < parts) {
      int4 all = make_int4(0, 0, 0, 0), before = make_int4(0, 0, 0, 0);
      const int4 *counts = reinterpret_cast<const int4 *>(a.counts) + e;
#pragma unroll 8
      for (int c = part; c < chunks; c += parts) {
        const int4 n = counts[(int64_t)c * width];
        all.x += n.x; all.y += n.y; all.z += n.z; all.w += n.w;
        if (c < me) { before.x += n.x; before.y += n.y; before.z += n.z; before.w += n.w; }
      }
      const int t[4] = {all.x, all.y, all.z, all.w}, f[4] = {before.x, before.y, before.z, before.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (t[i]) atomicAdd(&total[4 * e + i], t[i]);
        if (f[i]) atomicAdd(&next[4 * e + i], f[i]);
      }
    }
  }
  __syncthreads();
  if (me == 0 && a.expert_counts)
    for (int e = tid; e < a.E; e += kGateThreads) a.expert_counts[e] = total[e];
  if (!a.slot_to_row) return;
  if (warp == 0) gate_offsets(total, next, a.E);
  gate_places(a.ids, (int64_t)me * a.chunk * a.k, min((int64_t)a.T, (int64_t)(me + 1) * a.chunk) * a.k, a.E, next, reinterpret_cast<uint4 *>(sm + 2 * Ep), a.slot_to_row);
}

}  // namespace b200
