// Appending rotated keys and values to a paged cache (b200dnn_kv_append).
//
//   y[a] = x[a] c - x[b] s,   y[b] = x[b] c + x[a] s      for the pairs (a, b) of the rotary part of a row of q or k, in f32
//
// and the row goes to its place: q to q_out, k and v to the cache row of the token's slot, rounded to bf16 or quantised to s8 with one
// f32 scale a row.  Bound by the bytes moved: each input row read once, each output row written once.
#pragma once
#include "common.cuh"
#include "mbar.cuh"
#include "quant_codes.cuh"

namespace b200 {

struct AppendArgs {
  const void *q, *k, *v; void *q_out;
  int64_t qs[2], ks[2], vs[2], os[2];               // elements: token, head
  void *key, *value; float *key_scale, *value_scale;
  int64_t ck[3], cv[3], cs[3];                      // elements: page, token, head
  const int32_t *positions; const float *cos_t, *sin_t; int64_t table_rows, table_ld;
  const int64_t *slots; int64_t n_slots;            // page * page_size + token, below n_slots
  int64_t T;
  int page_size, q_heads, kv_heads, dim, rot, interleaved;
  int32_t *status;
};

template <typename T> __device__ __forceinline__ float append_load(const void *p, int64_t i) {
  if constexpr (sizeof(T) == 4) return reinterpret_cast<const float *>(p)[i];
  else return bf16_bits_to_f32(reinterpret_cast<const uint16_t *>(p)[i]);
}
template <typename T> __device__ __forceinline__ void append_store(void *p, int64_t i, float v) {
  if constexpr (sizeof(T) == 4) reinterpret_cast<float *>(p)[i] = v;
  else reinterpret_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

// The token's place: false when nothing of it is to be written (padding, or an index out of range, which is reported).
__device__ __forceinline__ bool append_place(const AppendArgs &a, int64_t t, int64_t &page, int &off, int64_t &pos) {
  const int64_t slot = a.slots[t];
  pos = a.rot ? a.positions[t] : 0;
  if (slot < 0) return false;
  if (slot >= a.n_slots || pos < 0 || (a.rot && pos >= a.table_rows)) {
    report_status(a.status, kStatusIndex);
    return false;
  }
  page = slot / a.page_size;
  off = (int)(slot - page * a.page_size);
  return true;
}

__device__ __forceinline__ void append_turn(float &x, float &y, float c, float s) {
  const float a = x, b = y;
  x = __fmaf_rn(a, c, -__fmul_rn(b, s));
  y = __fmaf_rn(b, c, __fmul_rn(a, s));
}

// Any sizes, strides and alignment: a warp per row of q, k or v, two elements a lane at a time.  Pair p of the row is elements (i0, i1): the rotary pairs first, then
// neighbours.  An s8 row is computed twice, for its largest value and for the codes.
template <typename T, bool S8>
__global__ void __launch_bounds__(256) append_rows_kernel(const AppendArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int R = a.q_heads + 2 * a.kv_heads, lane = threadIdx.x & 31;
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int64_t t = w / R;
  if (t >= a.T) return;
  int h = (int)(w - t * R);
  int64_t page, pos; int off;
  if (!append_place(a, t, page, off, pos)) return;
  const int half = a.rot >> 1, pairs = (a.dim + 1) >> 1;
  const void *src; int64_t at;                      // the row
  void *dst; int64_t to;
  const int kind = h < a.q_heads ? 0 : h < a.q_heads + a.kv_heads ? 1 : 2;
  float *scale_to = nullptr;
  if (kind == 0) { src = a.q; at = t * a.qs[0] + h * a.qs[1]; dst = a.q_out; to = t * a.os[0] + h * a.os[1]; }
  else if (kind == 1) {
    h -= a.q_heads;
    src = a.k; at = t * a.ks[0] + h * a.ks[1]; dst = a.key; to = page * a.ck[0] + off * a.ck[1] + h * a.ck[2];
    scale_to = a.key_scale;
  } else {
    h -= a.q_heads + a.kv_heads;
    src = a.v; at = t * a.vs[0] + h * a.vs[1]; dst = a.value; to = page * a.cv[0] + off * a.cv[1] + h * a.cv[2];
    scale_to = a.value_scale;
  }
  auto load = [&](int p, int &i0, int &i1, float &x, float &y) {
    const bool turned = kind != 2 && p < half;
    i0 = p < half ? (a.interleaved ? 2 * p : p) : 2 * p;
    i1 = p < half ? (a.interleaved ? 2 * p + 1 : p + half) : 2 * p + 1;
    x = append_load<T>(src, at + i0);
    y = i1 < a.dim ? append_load<T>(src, at + i1) : 0.f;
    if (turned) append_turn(x, y, a.cos_t[pos * a.table_ld + p], a.sin_t[pos * a.table_ld + p]);
  };
  int i0, i1; float x, y;
  if (S8 && kind != 0) {
    float most = 0.f;
    for (int p = lane; p < pairs; p += 32) {
      load(p, i0, i1, x, y);
      if (finite_f32(x)) most = fmaxf(most, fabsf(x));
      if (finite_f32(y)) most = fmaxf(most, fabsf(y));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const float scale = scale_from_absmax(most);
    for (int p = lane; p < pairs; p += 32) {
      load(p, i0, i1, x, y);
      reinterpret_cast<int8_t *>(dst)[to + i0] = quant_sym(x, scale);
      if (i1 < a.dim) reinterpret_cast<int8_t *>(dst)[to + i1] = quant_sym(y, scale);
    }
    if (lane == 0) scale_to[page * a.cs[0] + off * a.cs[1] + h * a.cs[2]] = scale;
    return;
  }
  for (int p = lane; p < pairs; p += 32) {
    load(p, i0, i1, x, y);
    if (kind == 0) {
      append_store<T>(dst, to + i0, x);
      if (i1 < a.dim) append_store<T>(dst, to + i1, y);
    } else {
      append_store<__nv_bfloat16>(dst, to + i0, x);
      if (i1 < a.dim) append_store<__nv_bfloat16>(dst, to + i1, y);
    }
  }
}

}  // namespace b200
