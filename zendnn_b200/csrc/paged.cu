// Entry points of the paged key/value cache: b200dnn_kv_append and b200dnn_paged_attention (checks, staging, launches).
#include <algorithm>
#include <cmath>
#include <cuda_bf16.h>
#include "runtime.cuh"
#include "paged_append.cuh"
#include "paged_attention.cuh"

namespace b200 {

namespace {

template <typename... P>
int32_t launch(void (*kern)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t st, const P &...args) {
  if (smem > 48 * 1024) B2_TRY(ensure_max_smem((const void *)kern, (int)smem));
  B2_TRY(launch_pdl(kern, grid, threads, smem, st, true, args...));
  B2_LAUNCHED();
  return B200DNN_SUCCESS;
}

// Bytes from the first element to behind the last one of rows [n0][n1][dim]
size_t span2(int64_t n0, int64_t n1, int64_t dim, const int64_t (&s)[2], int32_t dt) {
  return n0 <= 0 || n1 <= 0 ? 0 : (size_t)((n0 - 1) * s[0] + (n1 - 1) * s[1] + dim) * dt_size(dt);
}
// Strides of one row from the next: rows do not overlap (an extent of one takes any stride)
bool rows_apart(int64_t n0, int64_t n1, int64_t dim, const int64_t (&s)[2]) {
  return (n0 <= 1 || s[0] >= dim) && (n1 <= 1 || s[1] >= dim) && s[0] < (1ll << 40) && s[1] < (1ll << 40);
}

int32_t check_cache(const char *who, const b200dnn_kv_cache_t &c) {
  B2_CHECK(c.dt == B200DNN_BF16 || c.dt == B200DNN_S8, B200DNN_UNIMPLEMENTED, "%s: the cache is bf16 or s8 (dt %d)", who, c.dt);
  B2_CHECK(c.page_size > 0 && c.kv_heads > 0 && c.head_dim > 0 && c.num_pages > 0, B200DNN_FAILURE, "%s: page_size, kv_heads, head_dim and num_pages must be > 0", who);
  B2_CHECK(c.head_dim <= 256, B200DNN_UNIMPLEMENTED, "%s: head_dim up to 256 (%d)", who, c.head_dim);
  B2_CHECK(c.page_size < (1 << 20) && c.num_pages < (1ll << 31) && c.kv_heads < (1 << 16), B200DNN_UNIMPLEMENTED, "%s: sizes beyond the cache's limits", who);
  B2_CHECK(c.key && c.value, B200DNN_FAILURE, "%s: the cache's key or value pointer is null", who);
  const int64_t n[3] = {c.num_pages, c.page_size, c.kv_heads};
  for (int i = 0; i < 3; ++i) {
    B2_CHECK(n[i] == 1 || (c.key_stride[i] >= c.head_dim && c.value_stride[i] >= c.head_dim), B200DNN_FAILURE, "%s: the cache's rows overlap (stride %d)", who, i);
    B2_CHECK(c.key_stride[i] < (1ll << 31) && c.value_stride[i] < (1ll << 31) && c.key_stride[i] >= 0 && c.value_stride[i] >= 0, B200DNN_UNIMPLEMENTED,
             "%s: cache strides are below 2^31 elements", who);
  }
  if (c.dt == B200DNN_S8) {
    B2_CHECK(c.key_scale && c.value_scale, B200DNN_FAILURE, "%s: an s8 cache needs key_scale and value_scale", who);
    for (int i = 0; i < 3; ++i)
      B2_CHECK((n[i] == 1 || c.scale_stride[i] >= 1) && c.scale_stride[i] >= 0 && c.scale_stride[i] < (1ll << 31), B200DNN_FAILURE, "%s: bad scale stride %d", who, i);
  }
  return B200DNN_SUCCESS;
}

// The kernels use the cache where it lies.
int32_t check_cache_here(const Staging &g, const b200dnn_kv_cache_t &c) {
  B2_TRY(g.here("the cache", c.key, dt_size(c.dt)));
  B2_TRY(g.here("the cache", c.value, dt_size(c.dt)));
  if (c.dt == B200DNN_S8) {
    B2_TRY(g.here("the cache's scales", c.key_scale, 4));
    B2_TRY(g.here("the cache's scales", c.value_scale, 4));
  }
  return B200DNN_SUCCESS;
}

template <typename T, bool S8>
int32_t launch_append(const AppendArgs &a, cudaStream_t st) {
  const int R = a.q_heads + 2 * a.kv_heads;
  // vectors: 16 bytes of every input and of bf16 rows, 8 of s8 rows; a rotary part of whole pairs of pieces
  auto apart = [](const void *p, uintptr_t bytes, int size, int64_t n0, int64_t s0, int64_t n1, int64_t s1) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && (n0 <= 1 || s0 * size % (int64_t)bytes == 0) && (n1 <= 1 || s1 * size % (int64_t)bytes == 0);
  };
  const int ct = S8 ? 1 : 2, cb = S8 ? 8 : 16, it = sizeof(T) == 4 ? 4 : 2;
  auto cache = [&](const void *p, const int64_t (&s)[3]) {
    return apart(p, cb, ct, 2, s[0], a.page_size, s[1]) && apart(p, cb, ct, a.kv_heads, s[2], 1, 0);
  };
  const bool vec = a.dim % 8 == 0 && a.rot % 16 == 0 && cache(a.key, a.ck) && cache(a.value, a.cv) &&
                   apart(a.k, 16, it, a.T, a.ks[0], a.kv_heads, a.ks[1]) && apart(a.v, 16, it, a.T, a.vs[0], a.kv_heads, a.vs[1]) &&
                   (a.q_heads == 0 || (apart(a.q, 16, it, a.T, a.qs[0], a.q_heads, a.qs[1]) && apart(a.q_out, 16, it, a.T, a.os[0], a.q_heads, a.os[1]))) &&
                   (a.rot == 0 || (apart(a.cos_t, 16, 4, a.table_rows, a.table_ld, 1, 0) && apart(a.sin_t, 16, 4, a.table_rows, a.table_ld, 1, 0)));
  if (!vec) return launch(append_rows_kernel<T, S8>, (unsigned)((a.T * R + 7) / 8), 256, 0, st, a);
  const int tpr = a.dim <= 32 ? 2 : a.dim <= 64 ? 4 : a.dim <= 128 ? 8 : 16;
  // a token's rows over as many threads as take kAppendRows of them each
  const unsigned threads = (unsigned)std::min(256, (int)round_up((int64_t)(R + kAppendRows<T> - 1) / kAppendRows<T> * tpr, 32));
  switch (tpr) {
    case 2: return launch(append_token_kernel<T, S8, 2>, (unsigned)a.T, threads, 0, st, a);
    case 4: return launch(append_token_kernel<T, S8, 4>, (unsigned)a.T, threads, 0, st, a);
    case 8: return launch(append_token_kernel<T, S8, 8>, (unsigned)a.T, threads, 0, st, a);
    default: return launch(append_token_kernel<T, S8, 16>, (unsigned)a.T, threads, 0, st, a);
  }
}

// The split form, where rows are 16-byte vectors: B200DNN_UNIMPLEMENTED when the call does not fit.
template <bool S8, int DP, int NT>
int32_t launch_split(PagedSplitArgs &s, bool f32, cudaStream_t st) {
  const bool p8 = s.a.page_size % 8 == 0;
  auto kern = f32 ? (p8 ? paged_split_kernel<S8, DP, NT, true, true> : paged_split_kernel<S8, DP, NT, false, true>)
                  : (p8 ? paged_split_kernel<S8, DP, NT, true, false> : paged_split_kernel<S8, DP, NT, false, false>);
  constexpr size_t smem = paged_smem<S8, DP, NT>();
  // CTAs an SM, by shared memory (2848 to 4128 bytes of a CTA's own and 1 KB of the system's beside the dynamic part: three fit where this says three).  DP 256: one (of bf16 no more
  // fit; of s8 two would by shared memory and registers, not measured).
  const int resident = (int)std::min<size_t>(DP <= 128 ? 3 : 1, (size_t)(227 * 1024) / (smem + 2048));
  constexpr int unit = PagedRing<S8, DP>::KS * kPagedWarps;
  const int64_t most = (int64_t)s.a.B * s.blocks * s.side * ((s.a.n_keys + unit - 1) / unit + 1);      // (a window may begin inside a unit)
  if (most >= (1ll << 31)) return B200DNN_UNIMPLEMENTED;
  const unsigned grid = (unsigned)std::min<int64_t>(most, (int64_t)resident * rt().sm_count / s.side * s.side);
  const size_t part_o = (size_t)grid * 2 * 8 * NT * DP * 4, part_ml = (size_t)grid * 2 * 8 * NT * 8;
  uint8_t *scratch = nullptr;
  B2_TRY(call_scratch(grid, part_o + part_ml, st, &s.counters, &scratch));
  s.part_o = (float *)scratch;
  s.part_ml = (float2 *)(scratch + part_o);
  return launch(kern, grid, 32 * kPagedWarps, smem, st, s);
}
template <bool S8, int DP>
int32_t launch_split_heads(PagedSplitArgs &s, bool f32, cudaStream_t st) {
  const bool two = s.a.group > 8;
  s.tiles = (s.a.group + (two ? 16 : 8) - 1) / (two ? 16 : 8);
  const int rows = s.a.kv_heads * s.tiles;
  // s8: eight rows of a sequence side by side (or as many as divide them), see there; bf16 (32 heads of 128, 64 sequences of 4096 keys): 177 us, one by one 174
  s.side = S8 ? 8 : 1;
  while (rows % s.side) --s.side;
  s.blocks = rows / s.side;
  return two ? launch_split<S8, DP, 2>(s, f32, st) : launch_split<S8, DP, 1>(s, f32, st);
}
template <bool S8>
int32_t paged_split(const PagedArgs &a, bool out_f32, cudaStream_t st) {
  const int vec = S8 ? 16 : 8;          // elements of 16 bytes
  auto rows_vec = [&](const void *p, const int64_t (&s)[3]) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s[0] % vec == 0 && (a.page_size == 1 || s[1] % vec == 0) && (a.kv_heads == 1 || s[2] % vec == 0);
  };
  if (a.dim % vec != 0 || !rows_vec(a.key, a.ck) || !rows_vec(a.value, a.cv)) return B200DNN_UNIMPLEMENTED;
  PagedSplitArgs s{};
  s.a = a;
  s.q_vec = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && a.qs[0] % 8 == 0 && a.qs[1] % 8 == 0;
  const int ov = out_f32 ? 4 : 8;
  s.out_vec = (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 && a.os[0] % ov == 0 && a.os[1] % ov == 0;
  if (a.dim <= 64) return launch_split_heads<S8, 64>(s, out_f32, st);
  if (a.dim <= 128) return launch_split_heads<S8, 128>(s, out_f32, st);
  return launch_split_heads<S8, 256>(s, out_f32, st);
}

}  // namespace

}  // namespace b200

using namespace b200;

extern "C" int32_t b200dnn_kv_append(const b200dnn_kv_append_t *d, void *stream) {
  const char *who = "kv append";
  B2_CHECK(d, B200DNN_FAILURE, "null descriptor");
  const b200dnn_kv_cache_t &c = d->cache;
  B2_TRY(check_cache(who, c));
  const int64_t T = d->num_tokens;
  B2_CHECK(T >= 0 && d->q_heads >= 0, B200DNN_FAILURE, "%s: num_tokens and q_heads must be >= 0", who);
  B2_CHECK(d->dt == B200DNN_BF16 || d->dt == B200DNN_F32, B200DNN_UNIMPLEMENTED, "%s: q, k and v are bf16 or f32 (dt %d)", who, d->dt);
  B2_CHECK(d->rotary_dim >= 0 && d->rotary_dim % 2 == 0 && d->rotary_dim <= c.head_dim, B200DNN_FAILURE, "%s: rotary_dim must be even and at most head_dim (%d)", who, d->rotary_dim);
  if (T == 0) return B200DNN_SUCCESS;
  const int R = d->q_heads + 2 * c.kv_heads;
  B2_CHECK(T < (1ll << 31) && d->q_heads < (1 << 16) && T * R <= (1ll << 34) - 8, B200DNN_UNIMPLEMENTED, "%s: too many rows in one call", who);
  B2_CHECK(d->k && d->v && d->slots, B200DNN_FAILURE, "%s: k, v or slots is null", who);
  B2_CHECK(d->q_heads == 0 || (d->q && d->q_out), B200DNN_FAILURE, "%s: q or q_out is null", who);
  B2_CHECK(rows_apart(T, c.kv_heads, c.head_dim, d->k_stride) && rows_apart(T, c.kv_heads, c.head_dim, d->v_stride) &&
               (d->q_heads == 0 || (rows_apart(T, d->q_heads, c.head_dim, d->q_stride) && rows_apart(T, d->q_heads, c.head_dim, d->q_out_stride))),
           B200DNN_FAILURE, "%s: token and head strides must be at least head_dim", who);
  B2_CHECK(d->q_heads == 0 || d->q != d->q_out || ((T == 1 || d->q_stride[0] == d->q_out_stride[0]) && (d->q_heads == 1 || d->q_stride[1] == d->q_out_stride[1])), B200DNN_FAILURE,
           "%s: q rotated in place must keep its strides", who);
  if (d->rotary_dim > 0)
    B2_CHECK(d->positions && d->cos_table && d->sin_table && d->table_rows > 0 && d->table_ld >= d->rotary_dim / 2 && d->table_ld < (1ll << 31), B200DNN_FAILURE,
             "%s: a rotation needs positions and tables of at least rotary_dim / 2 columns", who);
  B2_ENTER(stream);
  const Staging g{d->device, st, who};
  B2_TRY(g.check());
  B2_TRY(check_cache_here(g, c));
  AppendArgs a{};
  const size_t table_bytes = d->rotary_dim ? (size_t)((d->table_rows - 1) * d->table_ld + d->rotary_dim / 2) * 4 : 0;
  Staged q_out{};
  B2_TRY(g.in(d->k, span2(T, c.kv_heads, c.head_dim, d->k_stride, d->dt), dt_size(d->dt), &a.k));
  B2_TRY(g.in(d->v, span2(T, c.kv_heads, c.head_dim, d->v_stride, d->dt), dt_size(d->dt), &a.v));
  B2_TRY(g.in(d->slots, (size_t)T * 8, 8, &a.slots));
  if (d->q_heads) {
    B2_TRY(g.in(d->q, span2(T, d->q_heads, c.head_dim, d->q_stride, d->dt), dt_size(d->dt), &a.q));
    B2_TRY(g.out(d->q_out, span2(T, d->q_heads, c.head_dim, d->q_out_stride, d->dt), dt_size(d->dt), &q_out, true));
    a.q_out = q_out.dev;
  }
  if (d->rotary_dim) {
    B2_TRY(g.in(d->positions, (size_t)T * 4, 4, &a.positions));
    B2_TRY(g.in(d->cos_table, table_bytes, 4, &a.cos_t));
    B2_TRY(g.in(d->sin_table, table_bytes, 4, &a.sin_t));
  }
  for (int i = 0; i < 2; ++i) { a.qs[i] = d->q_stride[i]; a.ks[i] = d->k_stride[i]; a.vs[i] = d->v_stride[i]; a.os[i] = d->q_out_stride[i]; }
  for (int i = 0; i < 3; ++i) { a.ck[i] = c.key_stride[i]; a.cv[i] = c.value_stride[i]; a.cs[i] = c.scale_stride[i]; }
  a.key = c.key; a.value = c.value; a.key_scale = c.key_scale; a.value_scale = c.value_scale;
  a.table_rows = d->table_rows; a.table_ld = d->table_ld;
  a.n_slots = c.num_pages * c.page_size; a.T = T;
  a.page_size = c.page_size; a.q_heads = d->q_heads; a.kv_heads = c.kv_heads; a.dim = c.head_dim; a.rot = d->rotary_dim; a.interleaved = d->interleaved ? 1 : 0;
  a.bad_index = index_word(st);
  const bool f32 = d->dt == B200DNN_F32, s8 = c.dt == B200DNN_S8;
  B2_TRY(f32 ? (s8 ? launch_append<float, true>(a, st) : launch_append<float, false>(a, st))
             : (s8 ? launch_append<__nv_bfloat16, true>(a, st) : launch_append<__nv_bfloat16, false>(a, st)));
  return g.finish({&q_out});
}

extern "C" int32_t b200dnn_paged_attention(const b200dnn_paged_attention_t *d, void *stream) {
  const char *who = "paged attention";
  B2_CHECK(d, B200DNN_FAILURE, "null descriptor");
  const b200dnn_kv_cache_t &c = d->cache;
  B2_TRY(check_cache(who, c));
  B2_CHECK(d->num_seqs >= 0, B200DNN_FAILURE, "%s: num_seqs must be >= 0", who);
  B2_CHECK(d->q_heads > 0 && d->q_heads % c.kv_heads == 0, B200DNN_FAILURE, "%s: q_heads (%d) must be a multiple of kv_heads (%d)", who, d->q_heads, c.kv_heads);
  B2_CHECK(d->q_dt == B200DNN_BF16, B200DNN_UNIMPLEMENTED, "%s: queries are bf16 (dt %d)", who, d->q_dt);
  B2_CHECK(d->out_dt == B200DNN_BF16 || d->out_dt == B200DNN_F32, B200DNN_UNIMPLEMENTED, "%s: the output is bf16 or f32 (dt %d)", who, d->out_dt);
  B2_CHECK(d->window >= 0, B200DNN_FAILURE, "%s: window must be >= 0", who);
  B2_CHECK(d->softcap >= 0.f && std::isfinite(d->softcap), B200DNN_FAILURE, "%s: softcap must be finite and >= 0", who);
  B2_CHECK(std::isfinite(d->scale), B200DNN_FAILURE, "%s: scale must be finite", who);
  // (times 64 and log2(e), and one over the other, they are finite in f32: an infinity, times a product of zero, is a NaN)
  B2_CHECK(std::fabs(d->scale) <= 0x1p120, B200DNN_UNIMPLEMENTED, "%s: scale up to 2^120", who);
  B2_CHECK(d->softcap <= 0x1p120f, B200DNN_UNIMPLEMENTED, "%s: softcap up to 2^120", who);
  const double scale = d->scale == 0.0 ? 1.0 / std::sqrt((double)c.head_dim) : d->scale;
  B2_CHECK(d->softcap == 0.f || 64.0 * std::fabs(scale) <= 0x1p127 * d->softcap, B200DNN_UNIMPLEMENTED, "%s: scale / softcap up to 2^121", who);
  if (d->num_seqs == 0) return B200DNN_SUCCESS;
  B2_CHECK(d->max_pages > 0 && d->page_table_ld >= d->max_pages && d->page_table_ld < (1ll << 31), B200DNN_FAILURE, "%s: page_table_ld must be at least max_pages > 0", who);
  B2_CHECK(d->q && d->out && d->page_table && d->seq_lens, B200DNN_FAILURE, "%s: q, out, page_table or seq_lens is null", who);
  const int64_t B = d->num_seqs;
  B2_CHECK(rows_apart(B, d->q_heads, c.head_dim, d->q_stride) && rows_apart(B, d->q_heads, c.head_dim, d->out_stride), B200DNN_FAILURE,
           "%s: sequence and head strides must be at least head_dim", who);
  B2_CHECK(B * d->q_heads < (1ll << 31), B200DNN_UNIMPLEMENTED, "%s: too many rows in one call", who);
  B2_CHECK((int64_t)d->max_pages * c.page_size < (1ll << 30), B200DNN_UNIMPLEMENTED, "%s: sequences have less than 2^30 keys", who);
  B2_CHECK(d->q != d->out, B200DNN_FAILURE, "%s: out must not overlap q", who);
  B2_ENTER(stream);
  const Staging g{d->device, st, who};
  B2_TRY(g.check());
  B2_TRY(check_cache_here(g, c));
  PagedArgs a{};
  Staged out{}, lse{};
  B2_TRY(g.in((const uint16_t *)d->q, span2(B, d->q_heads, c.head_dim, d->q_stride, d->q_dt), dt_size(d->q_dt), &a.q));
  B2_TRY(g.in(d->page_table, (size_t)((B - 1) * d->page_table_ld + d->max_pages) * 4, 4, &a.table));
  B2_TRY(g.in(d->seq_lens, (size_t)B * 4, 4, &a.lens));
  if (d->sinks) B2_TRY(g.in(d->sinks, (size_t)d->q_heads * 4, 4, &a.sinks));
  B2_TRY(g.out(d->out, span2(B, d->q_heads, c.head_dim, d->out_stride, d->out_dt), dt_size(d->out_dt), &out, true));
  if (d->lse) B2_TRY(g.out(d->lse, (size_t)B * d->q_heads * 4, 4, &lse, true));
  a.out = out.dev; a.lse = d->lse ? (float *)lse.dev : nullptr;
  for (int i = 0; i < 2; ++i) { a.qs[i] = d->q_stride[i]; a.os[i] = d->out_stride[i]; }
  for (int i = 0; i < 3; ++i) { a.ck[i] = c.key_stride[i]; a.cv[i] = c.value_stride[i]; a.cs[i] = c.scale_stride[i]; }
  a.key = c.key; a.value = c.value; a.key_scale = c.key_scale; a.value_scale = c.value_scale;
  a.table_ld = d->page_table_ld; a.n_pages = c.num_pages; a.n_keys = (int64_t)d->max_pages * c.page_size;
  a.B = (int)B; a.q_heads = d->q_heads; a.kv_heads = c.kv_heads; a.group = d->q_heads / c.kv_heads; a.dim = c.head_dim; a.page_size = c.page_size; a.window = d->window;
  a.scale = d->scale == 0.0 ? 1.0f / std::sqrt((float)c.head_dim) : (float)d->scale;
  a.softcap = d->softcap;
  a.bad_index = index_word(st);
  const int f32 = d->out_dt == B200DNN_F32;
  const int32_t rc = c.dt == B200DNN_S8 ? paged_split<true>(a, f32, st) : paged_split<false>(a, f32, st);
  if (rc != B200DNN_UNIMPLEMENTED) { B2_TRY(rc); return g.finish({&out, &lse}); }
  const unsigned grid = (unsigned)(B * d->q_heads);
  B2_TRY(c.dt == B200DNN_S8 ? launch(paged_rows_kernel<true>, grid, 32 * kPagedRowWarps, 0, st, a, f32) : launch(paged_rows_kernel<false>, grid, 32 * kPagedRowWarps, 0, st, a, f32));
  return g.finish({&out, &lse});
}
