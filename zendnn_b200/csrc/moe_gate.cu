// Entry point of the routing with bias and groups: b200dnn_moe_gate (checks, staging, launches).
#include <algorithm>
#include <cmath>
#include "runtime.cuh"
#include "moe_gate.cuh"

namespace b200 {
namespace {

template <typename... P>
int32_t launch(void (*kern)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t st, const P &...args) {
  // (48 KB without asking, and that holds for what the kernels declare themselves, a word or two, as well)
  if (smem > 47 * 1024) B2_TRY(ensure_max_smem((const void *)kern, (int)smem));
  B2_TRY(launch_pdl(kern, grid, threads, smem, st, true, args...));
  B2_LAUNCHED();
  return B200DNN_SUCCESS;
}

// Tokens of a CTA: all of a small batch, whose places then need no second launch (us, one CTA and two launches: 32 tokens over 64 experts 5.7, 6.3; 24 over 256 in groups 7.7, 8.5; but 32 over
// 256 9.1, 8.2; 64 over 64 8.2, 6.5); else 8 and as many more as leave a CTA for every SM (every CTA of the second launch adds up the counts of all), up to 2048 (they may all be on its list
// of tokens for 64 bits).
constexpr int kGateMostTokens = 2048;
bool gate_one_cta(int T, int E) { return T <= 32 && T * E < 8192; }
int32_t launch_gate(const GateArgs &a, const GateRowsArgs &r, unsigned grid, cudaStream_t st) {
  const unsigned threads = (unsigned)std::min(a.E <= 256 ? kGateTokenThreads<8> : kGateTokenThreads<32>, 32 * a.chunk);
  const size_t smem = (size_t)gate_pad(a.E) * 8 + (size_t)a.E * 32 + (size_t)a.chunk * 4;
  if (a.E <= 32) return launch(gate_kernel<1>, grid, threads, smem, st, a, r);
  if (a.E <= 64) return launch(gate_kernel<2>, grid, threads, smem, st, a, r);
  if (a.E <= 128) return launch(gate_kernel<4>, grid, threads, smem, st, a, r);
  if (a.E <= 256) return launch(gate_kernel<8>, grid, threads, smem, st, a, r);
  if (a.E <= 512) return launch(gate_kernel<16>, grid, threads, smem, st, a, r);
  return launch(gate_kernel<32>, grid, threads, smem, st, a, r);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int32_t b200dnn_moe_gate(const b200dnn_moe_gate_t *d, void *stream) {
  const char *who = "moe gate";
  B2_CHECK(d, B200DNN_FAILURE, "null descriptor");
  const int T = d->num_tokens, E = d->num_experts, k = d->topk, G = d->num_groups;
  B2_CHECK(T >= 0 && E > 0, B200DNN_FAILURE, "%s: num_tokens must be >= 0 and num_experts > 0", who);
  B2_CHECK(E <= 1024, B200DNN_UNIMPLEMENTED, "%s: up to 1024 experts (%d)", who, E);
  B2_CHECK(d->score == B200DNN_GATE_SOFTMAX || d->score == B200DNN_GATE_SIGMOID, B200DNN_FAILURE, "%s: unknown score %d", who, d->score);
  B2_CHECK(G >= 1 && E % G == 0 && d->topk_groups >= 1 && d->topk_groups <= G, B200DNN_FAILURE, "%s: num_groups (%d) must divide num_experts (%d), topk_groups (%d) lie in 1 .. num_groups",
           who, G, E, d->topk_groups);
  B2_CHECK(G <= 32, B200DNN_UNIMPLEMENTED, "%s: up to 32 groups (%d)", who, G);
  B2_CHECK(d->group_score == B200DNN_GROUP_MAX || d->group_score == B200DNN_GROUP_TOP2, B200DNN_FAILURE, "%s: unknown group_score %d", who, d->group_score);
  B2_CHECK(k > 0 && k <= d->topk_groups * (E / G), B200DNN_FAILURE, "%s: topk (%d) must lie in 1 .. the experts of topk_groups groups", who, k);
  B2_CHECK(k <= kGateMaxTopk, B200DNN_UNIMPLEMENTED, "%s: topk up to %d (%d)", who, kGateMaxTopk, k);
  B2_CHECK(std::isfinite(d->scale), B200DNN_FAILURE, "%s: scale must be finite", who);
  B2_CHECK(d->logits_dt == B200DNN_F32 || d->logits_dt == B200DNN_BF16, B200DNN_UNIMPLEMENTED, "%s: logits are f32 or bf16 (dt %d)", who, d->logits_dt);
  // (the last block's tokens, and a step of the loop behind them, are counted in 32 bits)
  B2_CHECK((int64_t)T * k < (1ll << 31) - 2 * kGateMostTokens, B200DNN_UNIMPLEMENTED, "%s: too many slots in one call", who);
  B2_CHECK(T == 0 || (d->logits && d->ids), B200DNN_FAILURE, "%s: logits or ids is null", who);
  B2_CHECK(T == 0 || d->ld >= E, B200DNN_FAILURE, "%s: ld (%lld) must be at least num_experts", who, (long long)d->ld);
  if (T == 0 && !d->expert_counts) return B200DNN_SUCCESS;
  B2_ENTER(stream);
  const Staging g{d->device, st, who};
  B2_TRY(g.check());
  const size_t ns = (size_t)T * k;
  Staged ids{}, weights{}, counts{}, rows{};
  B2_TRY(g.out(d->expert_counts, (size_t)E * 4, 4, &counts));
  if (T == 0) {
    B2_CUDA(cudaMemsetAsync(counts.dev, 0, (size_t)E * 4, st));
    return g.finish({&counts});
  }
  GateArgs a{};
  B2_TRY(g.in(d->logits, span_bytes(T, E, d->ld, d->logits_dt), dt_size(d->logits_dt), &a.logits));
  if (d->bias) B2_TRY(g.in(d->bias, (size_t)E * 4, 4, &a.bias));
  B2_TRY(g.out(d->ids, ns * 4, 4, &ids));
  B2_TRY(g.out(d->weights, ns * 4, 4, &weights));
  B2_TRY(g.out(d->slot_to_row, ns * 4, 4, &rows));
  a.ld = d->ld; a.logits_bf16 = d->logits_dt == B200DNN_BF16;
  a.T = T; a.E = E; a.k = k; a.sigmoid = d->score == B200DNN_GATE_SIGMOID; a.groups = G; a.top_groups = d->topk_groups; a.per_group = E / G;
  a.top2 = d->group_score == B200DNN_GROUP_TOP2; a.renorm = d->renorm ? 1 : 0; a.scale = d->scale;
  a.ids = (int32_t *)ids.dev; a.weights = (float *)weights.dev;
  a.chunk = gate_one_cta(T, E) ? T : std::min(kGateMostTokens, std::max(8, (T + rt().sm_count - 1) / rt().sm_count));
  const unsigned grid = (unsigned)((T + a.chunk - 1) / a.chunk);
  GateRowsArgs r{a.ids, nullptr, T, E, k, a.chunk, (int32_t *)counts.dev, (int32_t *)rows.dev};
  const bool second = grid > 1 && (d->expert_counts || d->slot_to_row);
  if (second) {
    uint32_t *zeros; uint8_t *scratch = nullptr;
    B2_TRY(call_scratch(0, (size_t)grid * gate_pad(E) * 4, st, &zeros, &scratch));
    a.counts = (int32_t *)scratch;
    r.counts = a.counts;
  }
  B2_TRY(launch_gate(a, grid > 1 ? GateRowsArgs{} : r, grid, st));
  if (second) B2_TRY(launch(gate_rows_kernel, grid, kGateThreads, (size_t)gate_pad(E) * 8 + (size_t)E * 32, st, r));
  return g.finish({&ids, &weights, &counts, &rows});
}
