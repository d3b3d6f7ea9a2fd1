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

struct GateTop { unsigned long long key; int id; };
// the largest key of the warp, ties to the lower id
__device__ __forceinline__ GateTop gate_best(GateTop t) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const unsigned long long key = __shfl_xor_sync(0xffffffffu, t.key, o);
    const int id = __shfl_xor_sync(0xffffffffu, t.id, o);
    if (key > t.key || (key == t.key && id < t.id)) { t.key = key; t.id = id; }
  }
  return t;
}

// A warp's token in 64 bits.  x[j]: logit of expert 32 j + lane.  Lane i < k returns the i-th choice and its score.
template <int PER>
__device__ __forceinline__ void gate_token(const GateArgs &a, const float (&x)[PER], int lane, int &id, double &score) {
  double s[PER];
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] = 1.0 / (1.0 + exp(-(double)x[j]));
  } else {
    float mx = __int_as_float(0xff800000);
#pragma unroll
    for (int j = 0; j < PER; ++j) if (j * 32 + lane < a.E) mx = fmaxf(mx, x[j]);
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) { s[j] = j * 32 + lane < a.E ? exp((double)x[j] - (double)mx) : 0.0; sum += s[j]; }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] /= sum;
  }
  unsigned long long key[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int e = j * 32 + lane;
    key[j] = e < a.E ? gate_key(a.bias ? s[j] + (double)a.bias[e] : s[j]) : 0ull;
  }
  if (a.groups > 1) {
    // lane g: the score of group g
    unsigned long long mine = 0ull;
    for (int g = 0; g < a.groups; ++g) {
      double total = 0.0;
      int first = -1;
      for (int r = 0; r <= a.top2; ++r) {
        GateTop t{0ull, 0x7fffffff};
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const int e = j * 32 + lane;
          if (e / a.per_group == g && e != first && key[j] > t.key) t = GateTop{key[j], e};
        }
        t = gate_best(t);
        if (t.key == 0ull) break;            // a group of one expert
        first = t.id;
        const double c = t.key == 1ull ? __longlong_as_double(0x7ff8000000000000ll)
                                       : __longlong_as_double((long long)(t.key >> 63 ? t.key & 0x7fffffffffffffffull : ~t.key));
        total = r == 0 ? c : total + c;
      }
      if (lane == g) mine = gate_key(total);
    }
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const unsigned long long other = __shfl_sync(0xffffffffu, mine, g);
      rank += other > mine || (other == mine && g < lane);
    }
    const unsigned chosen = __ballot_sync(0xffffffffu, lane < a.groups && rank < a.top_groups);
#pragma unroll
    for (int j = 0; j < PER; ++j) { const int e = j * 32 + lane; if (e < a.E && !((chosen >> (e / a.per_group)) & 1u)) key[j] = 0ull; }
  }
  id = 0; score = 0.0;
  for (int r = 0; r < a.k; ++r) {
    GateTop t{0ull, 0x7fffffff};
    double v = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) if (key[j] > t.key) { t = GateTop{key[j], j * 32 + lane}; v = s[j]; }
    t = gate_best(t);
    v = __shfl_sync(0xffffffffu, v, t.id & 31);
#pragma unroll
    for (int j = 0; j < PER; ++j) if (t.id == j * 32 + lane) key[j] = 0ull;
    if (lane == r) { id = t.id; score = v; }
  }
}

constexpr int kGateThreads = 256;
template <int PER>
__global__ void __launch_bounds__(kGateThreads) gate_kernel(const GateArgs a) {
  __shared__ int hist[PER * 32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t0 = blockIdx.x * a.chunk, t1 = min(a.T, t0 + a.chunk);
  if (a.counts) {
    for (int i = threadIdx.x; i < a.E; i += kGateThreads) hist[i] = 0;
    __syncthreads();
  }
  for (int t = t0 + warp; t < t1; t += kGateThreads / 32) {
    float x[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = j * 32 + lane;
      x[j] = e < a.E ? load_as_f32(a.logits, a.logits_bf16 ? DT_BF16 : DT_F32, t * a.ld + e) : 0.f;
    }
    int id; double score;
    gate_token<PER>(a, x, lane, id, score);
    double sum = 0.0;
    for (int r = 0; r < a.k; ++r) sum += __shfl_sync(0xffffffffu, score, r);
    if (lane < a.k) {
      a.ids[(int64_t)t * a.k + lane] = id;
      if (a.weights) a.weights[(int64_t)t * a.k + lane] = (float)((a.renorm ? score / sum : score) * (double)a.scale);
      if (a.counts) atomicAdd(&hist[id], 1);
    }
  }
  if (a.counts) {
    __syncthreads();
    for (int i = threadIdx.x; i < a.E; i += kGateThreads) a.counts[(int64_t)blockIdx.x * a.E + i] = hist[i];
  }
}

// The slots' places in the stable order by expert, from the counts of the chunks: every CTA adds up those of all chunks (first rows of the experts) and of the chunks
// in front of it, then ranks its own slots inside their experts.
struct GateRowsArgs { const int32_t *ids, *counts; int T, E, k, chunk; int32_t *expert_counts, *slot_to_row; };
constexpr int kGateRowsThreads = 1024;
__global__ void __launch_bounds__(kGateRowsThreads) gate_rows_kernel(const GateRowsArgs a) {
  extern __shared__ int sm[];
  int *next = sm, *total = sm + a.E, *cnt = sm + 2 * a.E;          // this chunk's next row of each expert; all rows; [32 warps][E]
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, me = blockIdx.x, chunks = gridDim.x;
  const int64_t s_end = min((int64_t)a.T, (int64_t)(me + 1) * a.chunk) * a.k;
  for (int e = tid; e < a.E; e += kGateRowsThreads) { next[e] = 0; total[e] = 0; }
  __syncthreads();
  for (int i = tid; i < chunks * a.E; i += kGateRowsThreads) {
    const int c = i / a.E, e = i - c * a.E, n = a.counts[i];
    if (n) { atomicAdd(&total[e], n); if (c < me) atomicAdd(&next[e], n); }
  }
  __syncthreads();
  if (warp == 0) {
    int carry = 0;
    for (int base = 0; base < a.E; base += 32) {
      const int e = base + lane, n = e < a.E ? total[e] : 0;
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += v; }
      if (e < a.E) next[e] += carry + sum - n;
      carry += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  if (me == 0 && a.expert_counts)
    for (int e = tid; e < a.E; e += kGateRowsThreads) a.expert_counts[e] = total[e];
  if (!a.slot_to_row) return;
  __syncthreads();
  for (int64_t s0 = (int64_t)me * a.chunk * a.k; s0 < s_end; s0 += kGateRowsThreads) {
    for (int i = tid; i < 32 * a.E; i += kGateRowsThreads) cnt[i] = 0;
    __syncthreads();
    const int64_t s = s0 + tid;
    const int e = s < s_end ? a.ids[s] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, e);
    const int before = __popc(same & ((1u << lane) - 1u));
    if (e >= 0 && before == 0) cnt[warp * a.E + e] = __popc(same);
    __syncthreads();
    if (e >= 0) {
      int row = next[e] + before;
      for (int w = 0; w < warp; ++w) row += cnt[w * a.E + e];
      a.slot_to_row[s] = row;
    }
    __syncthreads();
    for (int i = tid; i < a.E; i += kGateRowsThreads) { int n = 0; for (int w = 0; w < 32; ++w) n += cnt[w * a.E + i]; next[i] += n; }
    __syncthreads();
  }
}

}  // namespace b200
