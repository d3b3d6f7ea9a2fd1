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
  int32_t *bad_index;
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
__device__ __forceinline__ bool append_place(const AppendArgs &a, int64_t slot, int64_t pos, int64_t &page, int &off) {
  if (slot < 0) return false;
  if (slot >= a.n_slots || pos < 0 || (a.rot && pos >= a.table_rows)) {
    report_index(a.bad_index);
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
// neighbours.  An s8 row is computed twice, for its largest value and for the codes.  Bound by its scattered two-byte accesses: 8192 tokens, 32 / 8 heads of 128, bf16, 125 us.
template <typename T, bool S8>
__global__ void __launch_bounds__(256) append_rows_kernel(const AppendArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int R = a.q_heads + 2 * a.kv_heads, lane = threadIdx.x & 31;
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int64_t t = w / R;
  if (t >= a.T) return;
  int h = (int)(w - t * R);
  int64_t page; int off;
  const int64_t pos = a.rot ? a.positions[t] : 0;
  if (!append_place(a, a.slots[t], pos, page, off)) return;
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


// Rows of 16-byte vectors.  A CTA takes one token, TPR threads a row: thread j of a row holds 16 elements in two pieces of eight, those of a rotary pair where the row is
// rotated (half against half: [8 j, +8) and [rot / 2 + 8 j, +8); interleaved: 16 neighbours), and goes through the token's rows with them, so that a piece of the
// tables is loaded once for all heads.  All of a thread's rows are loaded before the token's place is known.  s8: the row's largest element by shuffles over its threads.
// Bound by HBM: 8192 tokens, 32 / 8 heads of 128, bf16, 37.7 us (5.4 TB/s, 0.83 of the copy rate); 256 tokens into an s8 cache 5 us, a chain of three loads.
struct Append8 { float v[8]; };
// eight elements as they lie in memory
template <typename T> struct AppendRaw { uint4 w[sizeof(T) / 2]; };
// (KEPT: what the kernel does not write.  Queries may be rotated in place, and are not to be read through the read-only path.)
template <typename T, bool KEPT> __device__ __forceinline__ AppendRaw<T> append_raw(const void *p, int64_t i) {
  const uint4 *q = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(p) + i * (int64_t)sizeof(T));
  AppendRaw<T> x;
#pragma unroll
  for (int e = 0; e < (int)sizeof(T) / 2; ++e) x.w[e] = KEPT ? __ldg(q + e) : q[e];
  return x;
}
template <typename T> __device__ __forceinline__ Append8 append_floats(const AppendRaw<T> &x) {
  Append8 y;
#pragma unroll
  for (int e = 0; e < (int)sizeof(T) / 2; ++e) {
    const uint32_t w[4] = {x.w[e].x, x.w[e].y, x.w[e].z, x.w[e].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) y.v[4 * e + i] = __uint_as_float(w[i]);
      else { y.v[2 * i] = __uint_as_float(w[i] << 16); y.v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
  }
  return y;
}
__device__ __forceinline__ uint32_t append_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T> __device__ __forceinline__ void append_store8(void *p, int64_t i, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    float4 *q = reinterpret_cast<float4 *>(reinterpret_cast<float *>(p) + i);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(p) + i) = make_uint4(append_pack(v[0], v[1]), append_pack(v[2], v[3]), append_pack(v[4], v[5]), append_pack(v[6], v[7]));
  }
}

// Rows of a thread in flight: 128 bytes (their registers decide how many CTAs an SM holds, and the call is bound by how much is in flight).
template <typename T> constexpr int kAppendRows = sizeof(T) == 4 ? 2 : 4;
// TPR: threads of a row, a power of two
template <typename T, bool S8, int TPR>
__global__ void __launch_bounds__(256, 3) append_token_kernel(const AppendArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t t = blockIdx.x;
  const int R = a.q_heads + 2 * a.kv_heads, j = threadIdx.x % TPR, row0 = threadIdx.x / TPR, rows = blockDim.x / TPR;
  const int half = a.rot >> 1, turned_threads = a.rot >> 4;
  const bool turns = j < turned_threads;
  // the two pieces: of a rotated row, and of a row of v
  const int c0 = turns && !a.interleaved ? 8 * j : 16 * j, c1 = turns && !a.interleaved ? half + 8 * j : 16 * j + 8;
  const int64_t slot = a.slots[t], pos = a.rot ? a.positions[t] : 0;
  int64_t page = 0; int off = 0;
  Append8 cs, sn;
  bool placed = false;
  for (int first = row0; first < R; first += rows * kAppendRows<T>) {
    AppendRaw<T> x[kAppendRows<T>][2];
    auto source = [&](int row, const void *&p, int64_t &at) {
      if (row < a.q_heads) { p = a.q; at = t * a.qs[0] + row * a.qs[1]; }
      else if (row < a.q_heads + a.kv_heads) { p = a.k; at = t * a.ks[0] + (row - a.q_heads) * a.ks[1]; }
      else { p = a.v; at = t * a.vs[0] + (row - a.q_heads - a.kv_heads) * a.vs[1]; }
    };
#pragma unroll
    for (int i = 0; i < kAppendRows<T>; ++i) {
      const int row = first + i * rows;
      x[i][0] = x[i][1] = AppendRaw<T>{};
      if (row >= R) continue;
      const void *p; int64_t at;
      source(row, p, at);
      const int o0 = row < a.q_heads + a.kv_heads ? c0 : 16 * j, o1 = row < a.q_heads + a.kv_heads ? c1 : 16 * j + 8;
      if (o0 < a.dim) x[i][0] = append_raw<T, false>(p, at + o0);
      if (o1 < a.dim) x[i][1] = append_raw<T, false>(p, at + o1);
    }
    if (!placed) {
      if (!append_place(a, slot, pos, page, off)) return;
      if (turns) {
        cs = append_floats<float>(append_raw<float, true>(a.cos_t, pos * a.table_ld + 8 * j));
        sn = append_floats<float>(append_raw<float, true>(a.sin_t, pos * a.table_ld + 8 * j));
      }
      placed = true;
    }
#pragma unroll
    for (int i = 0; i < kAppendRows<T>; ++i) {
      const int row = first + i * rows;
      const bool on = row < R;
      const bool key = row >= a.q_heads && row < a.q_heads + a.kv_heads, value = row >= a.q_heads + a.kv_heads;
      Append8 x0 = append_floats<T>(x[i][0]), x1 = append_floats<T>(x[i][1]);
      float (&u)[8] = x0.v, (&w)[8] = x1.v;
      if (turns && !value) {
        if (a.interleaved) {
#pragma unroll
          for (int e = 0; e < 4; ++e) { append_turn(u[2 * e], u[2 * e + 1], cs.v[e], sn.v[e]); append_turn(w[2 * e], w[2 * e + 1], cs.v[4 + e], sn.v[4 + e]); }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) append_turn(u[e], w[e], cs.v[e], sn.v[e]);
        }
      }
      const int o0 = value ? 16 * j : c0, o1 = value ? 16 * j + 8 : c1, h = row - a.q_heads - (value ? a.kv_heads : 0);
      if (!key && !value) {
        if (!on) continue;
        const int64_t to = t * a.os[0] + row * a.os[1];
        if (o0 < a.dim) append_store8<T>(a.q_out, to + o0, u);
        if (o1 < a.dim) append_store8<T>(a.q_out, to + o1, w);
        continue;
      }
      void *dst = value ? a.value : a.key;
      const int64_t to = page * (value ? a.cv[0] : a.ck[0]) + off * (value ? a.cv[1] : a.ck[1]) + h * (value ? a.cv[2] : a.ck[2]);
      if constexpr (S8) {
        float most = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (finite_f32(u[e])) most = fmaxf(most, fabsf(u[e]));
          if (finite_f32(w[e])) most = fmaxf(most, fabsf(w[e]));
        }
        const unsigned lanes = TPR == 32 ? 0xffffffffu : ((1u << TPR) - 1u) << ((threadIdx.x & 31) / TPR * TPR);
#pragma unroll
        for (int o = TPR / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(lanes, most, o));
        if (!on) continue;
        const float scale = scale_from_absmax(most), rinv = __frcp_rn(scale);
        auto codes = [&](const float (&v)[8]) {
          uint32_t c[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) c[e] = (uint32_t)(uint8_t)quant_sym_r<float>(v[e], scale, rinv);
          return make_uint2(low_bytes4(c[0], c[1], c[2], c[3]), low_bytes4(c[4], c[5], c[6], c[7]));
        };
        if (o0 < a.dim) *reinterpret_cast<uint2 *>(reinterpret_cast<int8_t *>(dst) + to + o0) = codes(u);
        if (o1 < a.dim) *reinterpret_cast<uint2 *>(reinterpret_cast<int8_t *>(dst) + to + o1) = codes(w);
        if (j == 0) (value ? a.value_scale : a.key_scale)[page * a.cs[0] + off * a.cs[1] + h * a.cs[2]] = scale;
      } else {
        if (!on) continue;
        if (o0 < a.dim) append_store8<__nv_bfloat16>(dst, to + o0, u);
        if (o1 < a.dim) append_store8<__nv_bfloat16>(dst, to + o1, w);
      }
    }
  }
}

}  // namespace b200
