// Attention of one new token per sequence over a paged cache (b200dnn_paged_attention).
//
//   z_j = scale (q . k_j), optionally softcap tanh(z_j / softcap);   m = max z_j;   l = sum exp(z_j - m) (+ exp(sink - m))
//   out = sum exp(z_j - m) v_j / l,   lse = m + log l
//
// over the keys j of [max(0, n - window), n); key j lies on page table[j / page_size] at j % page_size.  Each visible key and value is read once: the
// call is bound by these bytes.
#pragma once
#include <cuda_bf16.h>
#include "common.cuh"
#include "mbar.cuh"

namespace b200 {

struct PagedArgs {
  const uint16_t *q; void *out; float *lse; const float *sinks;
  int64_t qs[2], os[2];                              // elements: sequence, head
  const void *key, *value; const float *key_scale, *value_scale;
  int64_t ck[3], cv[3], cs[3];                       // elements: page, token, head
  const int32_t *table, *lens; int64_t table_ld;
  int64_t n_pages, n_keys;                           // pages of the cache; most keys that a row of the table has room for
  int B, q_heads, kv_heads, group, dim, page_size, window;
  float scale, softcap;
  int32_t *status;
};

// A sequence's visible keys [lo, hi).  False: padding.  Lengths beyond the table's room are cut, and reported.
__device__ __forceinline__ bool paged_range(const PagedArgs &a, int i, int64_t &lo, int64_t &hi) {
  hi = a.lens[i];
  lo = 0;
  if (hi < 0) return false;
  if (hi > a.n_keys) { report_status(a.status, kStatusIndex); hi = a.n_keys; }
  if (a.window > 0 && hi > a.window) lo = hi - a.window;
  return true;
}
__device__ __forceinline__ int64_t paged_page(const PagedArgs &a, int i, int64_t column) {
  int32_t page = a.table[i * a.table_ld + column];
  if (page < 0 || page >= a.n_pages) { report_status(a.status, kStatusIndex); page = 0; }
  return page;
}

// Any sizes, strides and alignment: a CTA per sequence and query head, a warp per key, the head dimension over the lanes, in f32 throughout.
constexpr int kPagedRowWarps = 8;
template <bool S8>
__global__ void __launch_bounds__(32 * kPagedRowWarps) paged_rows_kernel(const PagedArgs a, int out_f32) {
  constexpr int PER = 8;                             // head_dim <= 256
  __shared__ float s_m[kPagedRowWarps], s_l[kPagedRowWarps], s_o[kPagedRowWarps][32 * PER];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int i = blockIdx.x / a.q_heads, h = blockIdx.x - i * a.q_heads, g = h / a.group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t lo, hi;
  if (!paged_range(a, i, lo, hi)) return;
  const float ninf = __int_as_float(0xff800000);
  float q[PER], o[PER], m = ninf, l = 0.f;
#pragma unroll
  for (int e = 0; e < PER; ++e) { const int d = e * 32 + lane; q[e] = d < a.dim ? bf16_bits_to_f32(a.q[i * a.qs[0] + h * a.qs[1] + d]) : 0.f; o[e] = 0.f; }
  auto load = [&](const void *p, int64_t at) { return S8 ? (float)reinterpret_cast<const int8_t *>(p)[at] : bf16_bits_to_f32(reinterpret_cast<const uint16_t *>(p)[at]); };
  for (int64_t j = lo + warp; j < hi; j += kPagedRowWarps) {
    const int64_t column = j / a.page_size, off = j - column * a.page_size, page = paged_page(a, i, column);
    const int64_t kb = page * a.ck[0] + off * a.ck[1] + g * a.ck[2], vb = page * a.cv[0] + off * a.cv[1] + g * a.cv[2], sb = page * a.cs[0] + off * a.cs[1] + g * a.cs[2];
    float z = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) { const int d = e * 32 + lane; if (d < a.dim) z = __fmaf_rn(q[e], load(a.key, kb + d), z); }
#pragma unroll
    for (int w = 16; w; w >>= 1) z += __shfl_xor_sync(0xffffffffu, z, w);
    if (S8) z *= a.key_scale[sb];
    z *= a.scale;
    if (a.softcap > 0.f) z = a.softcap * tanhf(z / a.softcap);
    const float to = fmaxf(m, z), frame = to == ninf ? 0.f : to, keep = expf(m - frame), p = expf(z - frame);
    l = l * keep + p;
    const float pv = S8 ? p * a.value_scale[sb] : p;
#pragma unroll
    for (int e = 0; e < PER; ++e) { const int d = e * 32 + lane; if (d < a.dim) o[e] = __fmaf_rn(pv, load(a.value, vb + d), o[e] * keep); }
    m = to;
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) s_o[warp][e * 32 + lane] = o[e];
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
  __syncthreads();
  const bool any = hi > lo;
  float top = a.sinks && any ? a.sinks[h] : ninf;
  for (int w = 0; w < kPagedRowWarps; ++w) top = fmaxf(top, s_m[w]);
  const float frame = top == ninf ? 0.f : top;
  float total = a.sinks && any ? expf(a.sinks[h] - frame) : 0.f;
  for (int w = 0; w < kPagedRowWarps; ++w) total += s_l[w] * expf(s_m[w] - frame);
  for (int d = threadIdx.x; d < a.dim; d += blockDim.x) {
    float x = 0.f;
    for (int w = 0; w < kPagedRowWarps; ++w) x += s_o[w][d] * expf(s_m[w] - frame);
    x = total == 0.f ? 0.f : x / total;
    const int64_t at = i * a.os[0] + h * a.os[1] + d;
    if (out_f32) reinterpret_cast<float *>(a.out)[at] = x; else reinterpret_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(x);
  }
  if (a.lse && threadIdx.x == 0) a.lse[(int64_t)i * a.q_heads + h] = frame + logf(total);
}

}  // namespace b200
