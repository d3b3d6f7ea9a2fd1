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
  int32_t *bad_index;
};

// A sequence's visible keys [lo, hi).  False: padding.  Lengths beyond the table's room are cut, and reported.
__device__ __forceinline__ bool paged_range(const PagedArgs &a, int i, int64_t &lo, int64_t &hi) {
  hi = a.lens[i];
  lo = 0;
  if (hi < 0) return false;
  if (hi > a.n_keys) { report_index(a.bad_index); hi = a.n_keys; }
  if (a.window > 0 && hi > a.window) lo = hi - a.window;
  return true;
}
__device__ __forceinline__ int64_t paged_page(const PagedArgs &a, int i, int64_t column) {
  int32_t page = a.table[i * a.table_ld + column];
  if (page < 0 || page >= a.n_pages) { report_index(a.bad_index); page = 0; }
  return page;
}

// Any sizes, strides and alignment: a CTA per sequence and query head, a warp per key, the head dimension over the lanes, in f32 throughout.  Every query head reads its key head again, from
// L2: 32 sequences of up to 4096 keys, 32 / 8 heads of 128, 835 us.
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


// ---------------------------------------------------------------------------------------------------------------------------------------------
// The split form: rows of 16-byte vectors.
//
// Work.  A row is one sequence and one tile of up to 8 NT query heads of a key head; its visible keys come in units of 128 (of 64 where a row of the cache is longer than 256 bytes).
// The units of all rows, one row after the other, are dealt out evenly: CTA c takes units [c per, (c + 1) per) of a grid that fills the device once, whatever the lengths are (they are on the
// device).  (Except for more than eight heads a key head of up to 64 elements: the grid counts three CTAs an SM by their shared memory, 190 to 218 registers a thread leave two, and the last third
// of the work comes behind; 32 sequences of 8192 keys, 64 / 4 heads of 64, 64 us, 0.64 of the copy rate.)  A row that lies in one CTA is finished there; of the others every CTA leaves a partial result (maximum, sum, unnormalised output), and the last one to arrive joins them, in order.
// With `side` > 1 it is a set of so many CTAs that takes units of so many rows of a sequence, each CTA its own row: they go through the same tokens at the same time.  Short rows that lie
// token after token, head beside head, and the scales beside each other then come from L2 (s8, 8 key heads, pages of 32 tokens: 64 sequences of 8192 keys of 64 elements 204 -> 126 us,
// 105 of 4096 of 128 189 -> 176).
//
// A warp takes 32 keys of a unit at a time (16 of more than 256 bytes), by itself: it copies their rows and those of their values into a ring of its own (cp.async, `ST` steps ahead, across the
// ends of the work's rows), so that no barrier stands between steps.  The products run on mma.m16n8k16 with the keys as the 16 rows:
//   S^T[key][head] = K Q^T     lane (r, c) = (lane / 4, lane % 4) holds pieces of the keys r and r + 8; which element of the head dimension is which index
//                              of the product does not matter as long as Q agrees, so a piece of 8 elements is the operand of two products as it lies
//   O^T[dim][head] = V^T P^T   lane (r, c) holds the same 8 (s8: 16) dims of the keys 2c, 2c + 1, 2c + 8, 2c + 9: a byte permutation pairs two keys of one dim
// P^T comes from S^T by transposing 8 x 8 blocks (movmatrix).  Statistics of heads 2c and 2c + 1 and their columns of O^T are in the same lanes.
// Tensor work is a fifth of what the memory leaves time for, so bf16 tiles of 16 x 8 serve: the call is bound by the bytes of the cache.  bf16, 32 / 8 heads of 128: the same 32 sequences 59 us
// (10 of them start and join, 6.8 TB/s between), two of 131072 keys 171 to 177 us (0.93 to 0.96 of the copy rate).  Head sizes are those of the next form, 64, 128 or 256: of 80 elements a row
// of the ring and the products are those of 128 (32 sequences of 4096 keys 94 us, as long as with 128).
//
// Probabilities enter the second product as the sum of two bf16 (2^-17 relative): one alone would cost as much again as the rounding of a bf16 output.  For an f32 output it is three
// (2^-25).  The row sum has them unrounded.  s8 codes are exact in bf16 (here as 64ths); a key's scale multiplies its scores, a value's scale its probability.
// The running maximum moves only when a score passes it by more than 2^8: probabilities are then at most 256, and few steps meet the exchange.

constexpr float kPagedLog2e = 1.44269504088896340736f;
constexpr int kPagedWarps = 4;
constexpr float kPagedReach = 8.0f;

struct PagedSplitArgs {
  PagedArgs a;
  int tiles;                       // head tiles of a key head
  int blocks, side;                // rows of a sequence, kv_heads * tiles: so many blocks of rows side by side
  int q_vec, out_vec;              // 16-byte rows of q and out
  float *part_o; float2 *part_ml;  // partial results: two slots a CTA
  uint32_t *counters;              // one a CTA, zero between launches
};

__device__ __forceinline__ float paged_exp2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
// BYTES from src, or zeros where size is 0; nothing where go is not set
template <int BYTES>
__device__ __forceinline__ void paged_copy(uint32_t dst, const void *src, uint32_t size, bool go) {
  if constexpr (BYTES == 16)
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %3, 0;\n@p cp.async.cg.shared.global [%0], [%1], 16, %2;\n}" ::"r"(dst), "l"(src), "r"(size), "r"((int)go) : "memory");
  else
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n@p cp.async.ca.shared.global [%0], [%1], %2, %3;\n}" ::"r"(dst), "l"(src), "n"(BYTES), "r"(size), "r"((int)go) : "memory");
}
__device__ __forceinline__ void paged_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void paged_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 paged_lds16(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 paged_lds8(uint32_t p) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t paged_lds_ptr(uint32_t p) {
  uint64_t v;
  asm volatile("ld.shared.b64 %0, [%1];" : "=l"(v) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ float paged_lds4(uint32_t p) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ void paged_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t paged_transpose(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t paged_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t paged_arrive(uint32_t *p) {
  uint32_t n;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(n) : "l"(p) : "memory");
  return n;
}
// Two of a word's four codes as bf16, divided by 64: of its bytes 0 and 2, or 1 and 3.  A byte u with zeros in front is u 2^-133 as a bf16 (below 128 without the leading one, from there on
// with it), so of u = code + 128 one multiplication and addition makes u 2^-6 - 2, exactly.
__device__ __forceinline__ uint32_t paged_codes(uint32_t u) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(u), "r"(0x7f007f00u), "r"(0xc000c000u));
  return r;
}
__device__ __forceinline__ uint32_t paged_codes_even(uint32_t w) { return paged_codes((w ^ 0x80808080u) & 0x00ff00ffu); }
__device__ __forceinline__ uint32_t paged_codes_odd(uint32_t w) { return paged_codes(__byte_perm(w ^ 0x80808080u, 0u, 0x4341)); }
constexpr float kPagedCode = 64.0f;

// What a CTA works on, one piece of a row after the other.
template <bool P8, int UNIT> struct PagedPieces {
  int seq, block, off, n;          // sequence, block of its rows, first unit in the row, units of the row
  int left;                        // units that the CTA still has, this piece included
  int lo, hi, base;                // visible keys of the sequence; where its units begin
  __device__ __forceinline__ int units() const { return min(n - off, left); }
  __device__ __forceinline__ int first_key() const { return base + off * UNIT; }
  __device__ __forceinline__ int end_key() const { return min(hi, base + (off + units()) * UNIT); }
  __device__ __forceinline__ void sequence(const PagedArgs &a) {
    int64_t l, h;
    if (!paged_range(a, seq, l, h)) l = h = 0;
    lo = (int)l; hi = (int)h;
    base = P8 ? lo & ~7 : lo;
    n = hi > lo ? (hi - base + UNIT - 1) / UNIT : 0;
  }
  __device__ __forceinline__ void next(const PagedSplitArgs &s) {
    const int u = units();
    left -= u;
    off += u;
    if (off < n || left <= 0) return;
    off = 0;
    if (++block < s.blocks) return;
    block = 0;
    for (n = 0; n == 0;) {                             // (there are units left, so there is a sequence with some)
      if (++seq >= s.a.B) { left = 0; return; }
      sequence(s.a);
    }
  }
};

template <bool S8, int DP> struct PagedRing {
  static constexpr int kRow = DP * (S8 ? 1 : 2);                             // bytes of a row
  static constexpr int CH = kRow <= 64 ? 4 : kRow <= 128 ? 8 : kRow <= 256 ? 16 : 32;   // lanes of a row, 16 bytes each
  static constexpr int KS = kRow <= 256 ? 32 : 16;                           // keys of a step of one warp
  static constexpr int RI = 32 / CH, IN = KS / RI;                           // rows of one copy instruction, instructions of a step's rows
  static constexpr int kPieceK = kRow / 64;                                  // 16-byte pieces of a key that a lane multiplies
  static constexpr int kWideV = S8 ? (DP % 128 == 0 ? 16 : 8) : 16;          // bytes of a value's pieces
  static constexpr int kPieceV = kRow / (8 * kWideV);
  static constexpr int kRows = KS * CH * 16, kScales = S8 ? KS * 8 : 0;         // bytes of a step's keys (values), and scales
  static constexpr int kStep = 2 * kRows + kScales;
  static constexpr int ST = kRows <= 2048 ? 4 : kRows <= 4096 ? 2 : KS == 32 ? 1 : 2;
  static constexpr int kBytes = kPagedWarps * ST * kStep;
  // 16-byte chunk j of row `key`, as an offset: neither the copies' rows nor the pieces that eight lanes read at a time meet in a bank
  static __device__ __forceinline__ uint32_t at_key(int key, int j) { return (uint32_t)((key * CH + j) ^ (CH >= 8 ? (key & 1) << 2 : 0)) * 16u; }
  static __device__ __forceinline__ uint32_t at_value(int key, int j) { return (uint32_t)((key * CH + j) ^ (((key >> 1) & 3) << 1)) * 16u; }
};
template <bool S8, int DP, int NT> struct PagedJoin {
  static constexpr int kRegs = NT * DP / 4;                                  // unnormalised outputs of a lane
  static constexpr int kBoxes = S8 ? 1 : 2;                                  // warps' outputs in shared memory at a time (with s8 scales in the ring, two would cost an SM its third CTA)
  static constexpr int kBytes = kBoxes * kRegs * 128;
};
template <bool S8, int DP, int NT> constexpr size_t paged_smem() { return PagedRing<S8, DP>::kBytes + PagedJoin<S8, DP, NT>::kBytes; }

// F32: of the output.  P8: pages of a multiple of eight keys.  Units then begin at a multiple of eight, the eight keys of half a step lie on one page, and their places need no lane's
// table entry but two that the whole warp knows; otherwise every lane looks up the key lane % 16.
template <bool S8, int DP, int NT, bool P8, bool F32>
__global__ void __launch_bounds__(32 * kPagedWarps, DP > 128 ? 1 : NT == 1 ? 3 : 2) paged_split_kernel(const PagedSplitArgs s) {
  using Ring = PagedRing<S8, DP>;
  constexpr int KS = Ring::KS, MT = KS / 16, UNIT = KS * kPagedWarps;
  constexpr int ST = Ring::ST, CH = Ring::CH, RI = Ring::RI, IN = Ring::IN, KP = Ring::kPieceK, VP = Ring::kPieceV, VB = Ring::kWideV, REGS = PagedJoin<S8, DP, NT>::kRegs;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float s_m[kPagedWarps][8 * NT], s_l[kPagedWarps][8 * NT];
  __shared__ int s_scan[kPagedWarps], s_before[32 * kPagedWarps];
  __shared__ int s_last;
  __shared__ uint4 s_plan[kPagedWarps][32];
  __shared__ uint64_t s_splan[S8 ? kPagedWarps : 1][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const PagedArgs &a = s.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
  const float ninf = __int_as_float(0xff800000);
  const int beside = (int)blockIdx.x % s.side;

  // ---- sequences without keys: zeros
  for (int i = blockIdx.x; i < a.B; i += gridDim.x) {
    if (a.lens[i] != 0) continue;
    for (int x = tid; x < a.q_heads * a.dim; x += 32 * kPagedWarps) {
      const int h = x / a.dim, d = x - h * a.dim;
      const int64_t at = i * a.os[0] + h * a.os[1] + d;
      if (F32) reinterpret_cast<float *>(a.out)[at] = 0.f; else reinterpret_cast<uint16_t *>(a.out)[at] = 0;
    }
    if (a.lse) for (int h = tid; h < a.q_heads; h += 32 * kPagedWarps) a.lse[(int64_t)i * a.q_heads + h] = ninf;
  }

  // ---- this CTA's units: every thread adds up the sequences of its stretch
  PagedPieces<P8, UNIT> ahead;
  int per, first;
  {
    const int stretch = (a.B + 32 * kPagedWarps - 1) / (32 * kPagedWarps), b0 = min(a.B, tid * stretch), b1 = min(a.B, b0 + stretch);
    int mine = 0;
    for (ahead.seq = b0; ahead.seq < b1; ++ahead.seq) { ahead.sequence(a); mine += ahead.n * s.blocks; }
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += v; }
    if (lane == 31) s_scan[warp] = sum;
    s_before[tid] = sum - mine;                // (of this warp's stretches)
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) total += s_scan[w];
    const int sets = (int)gridDim.x / s.side;
    per = (total + sets - 1) / sets;
    first = min(total, (int)blockIdx.x / s.side * per);
    const int count = min(per, total - first);
    if (count <= 0) return;
    // the stretch: the last one that begins at or before the first unit
    int w = 0, before = 0;
#pragma unroll
    for (int i = 1, begin = 0; i < kPagedWarps; ++i) { begin += s_scan[i - 1]; if (begin <= first) { w = i; before = begin; } }
    const int at = __popc(__ballot_sync(0xffffffffu, before + s_before[w * 32 + lane] <= first)) - 1;
    before += s_before[w * 32 + at];
    ahead.seq = (w * 32 + at) * stretch;
    for (ahead.sequence(a); before + ahead.n * s.blocks <= first && ahead.seq + 1 < a.B; ahead.sequence(a)) { before += ahead.n * s.blocks; ++ahead.seq; }
    ahead.block = (first - before) / ahead.n;
    ahead.off = (first - before) - ahead.block * ahead.n;
    ahead.left = count;
  }
  PagedPieces<P8, UNIT> now = ahead;

  // ---- copies, ST steps ahead
  const uint32_t ring = smem_u32(smem) + (uint32_t)warp * (ST * Ring::kStep);
  constexpr int ES = S8 ? 1 : 2;
  const int dim_bytes = a.dim * ES;
  // what lies behind the head dimension stays zeros: nothing is ever copied there
  if (a.dim < CH * 16 / ES) {
#pragma unroll 1
    for (uint32_t i = lane * 16u; i < ST * Ring::kStep; i += 512u) asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(ring + i), "r"(0) : "memory");
    __syncwarp();
  }
  // The plan: where the rows of the next steps lie, one entry for GK keys that follow each other on a page (P8: eight), found by all lanes together, 32 entries at a time.
  constexpr int GK = P8 ? 8 : 1, EP = KS / GK, SP = 32 / EP;      // keys of an entry, entries of a step, steps of a plan
  const uint32_t plan = smem_u32(s_plan[warp]), splan = S8 ? smem_u32(s_splan[warp]) : 0u;
  const uint32_t k_token = (uint32_t)(a.ck[1] * ES), v_token = (uint32_t)(a.cv[1] * ES);
  int step_key = 0, end_in = 0, lo_in = 0, plan_at = 0, plan_n = 0;
  bool fresh = true;
  auto refill = [&]() {
    __syncwarp();                              // (nobody reads the old one any more)
    plan_at = plan_n = 0;
    while (step_key >= end_in) {               // the next piece in which this warp has steps
      if (!fresh && ahead.left > 0) ahead.next(s);
      fresh = false;
      if (ahead.left <= 0) return;
      step_key = ahead.first_key() + warp * KS;
      end_in = ahead.end_key();
      lo_in = ahead.lo;
    }
    const int g = (ahead.block * s.side + beside) / s.tiles, key = step_key + lane / EP * UNIT + lane % EP * GK;
    uint32_t page = 0, off = 0;                // (behind the end: page 0, token 0; nothing of it is used)
    if (key < end_in) {
      const uint32_t column = (uint32_t)key / (uint32_t)a.page_size;
      off = (uint32_t)key - column * (uint32_t)a.page_size;
      page = (uint32_t)paged_page(a, ahead.seq, column);
    }
    const uint64_t k = reinterpret_cast<uint64_t>(a.key) + (uint64_t)((int64_t)page * a.ck[0] + (int64_t)off * a.ck[1] + g * a.ck[2]) * ES;
    const uint64_t v = reinterpret_cast<uint64_t>(a.value) + (uint64_t)((int64_t)page * a.cv[0] + (int64_t)off * a.cv[1] + g * a.cv[2]) * ES;
    asm volatile("st.shared.v2.b64 [%0], {%1, %2};" ::"r"(plan + (uint32_t)lane * 16u), "l"(k), "l"(v) : "memory");
    if (S8) asm volatile("st.shared.b64 [%0], %1;" ::"r"(splan + (uint32_t)lane * 8u), "l"((int64_t)page * a.cs[0] + (int64_t)off * a.cs[1] + g * a.cs[2]) : "memory");
    plan_n = min(SP, (end_in - step_key + UNIT - 1) / UNIT);
    __syncwarp();
  };
  int slot_in = 0, entry = 0;
  bool cut_in = false;
  unsigned taken = 0;                          // of a cut step: the keys that are visible
  int limit = 0;                               // head_dim in bytes; 0 when there is no step left
  auto take = [&]() {
    if (plan_at == plan_n) refill();
    limit = plan_n > 0 ? dim_bytes : 0;
    entry = plan_at * EP;
    cut_in = step_key + KS > end_in || step_key < lo_in;
    if (cut_in && limit) taken = (0xffffffffu >> max(0, step_key + 32 - end_in)) & (0xffffffffu << max(0, lo_in - step_key));
    if (limit) { ++plan_at; step_key += UNIT; }
  };
  // Copies of whole rows, CH lanes each (a key that the step does not see is zeros: its address is that of a token of the same page, or of page 0).  Measured on their own, 256-byte
  // rows: 6.8 TB/s, with every lane copying the pieces that it multiplies (64 bytes of a row at a time) 4.9.
  const int sub = lane / CH, chunk = lane % CH;
  auto copy_rows = [&](bool value) {
    const uint32_t slot_at = ring + (uint32_t)slot_in * Ring::kStep + (value ? Ring::kRows : 0), token = value ? v_token : k_token;
    const bool go = chunk * 16 < limit;
    auto place = [&](int key) { return slot_at + (value ? Ring::at_value(key, chunk) : Ring::at_key(key, chunk)); };
    auto from = [&](int e) { return paged_lds_ptr(plan + (uint32_t)(entry + e) * 16u + (value ? 8u : 0u)); };
    const uint64_t mine = (P8 ? (uint64_t)sub * token : 0) + chunk * 16;
    if (limit == 0) return;
    if (!cut_in) {
      constexpr int REP_K = RI >= 2 ? 1 : 2, REP_V = RI >= 8 ? 1 : 8 / RI;      // copies after which the swizzle repeats
      const int rep = value ? REP_V : REP_K;
      uint64_t base[P8 ? EP : 1];
      if constexpr (P8) {
#pragma unroll
        for (int e = 0; e < EP; ++e) base[e] = from(e) + mine;
      }
#pragma unroll
      for (int i = 0; i < IN; ++i) {
        const uint64_t p = P8 ? base[P8 ? i * RI / 8 : 0] + (uint64_t)token * (uint32_t)(i * RI % 8) : from(i * RI + sub) + mine;
        paged_copy<16>(place(i % rep * RI + sub) + (uint32_t)(i / rep * rep * RI * CH * 16), reinterpret_cast<const void *>(p), 16u, go);
      }
    } else {
#pragma unroll 1
      for (int i = 0; i < IN; ++i) {
        const int key = i * RI + sub;
        const uint64_t p = P8 ? from(key >> 3) + (uint64_t)token * (uint32_t)(key & 7) + chunk * 16 : from(key) + mine;
        paged_copy<16>(place(key), reinterpret_cast<const void *>(p), (taken >> key) & 1u ? 16u : 0u, go);
      }
    }
  };
  auto copy_keys = [&]() {
    copy_rows(false);
    if (S8) {
#pragma unroll
      for (int i = 0; i < (S8 ? MT : 0); ++i) {
        // keys' scales, then values' (MT 1: sixteen lanes each)
        const int key = MT == 2 ? lane : lane & 15;
        const bool value = MT == 2 ? i == 1 : lane >= 16;
        const int64_t at = (int64_t)paged_lds_ptr(splan + (uint32_t)(entry + key / GK) * 8u) + (int64_t)(key % GK) * a.cs[1];
        paged_copy<4>(ring + (uint32_t)slot_in * Ring::kStep + 2 * Ring::kRows + (uint32_t)(i * 32 + lane) * 4u, (value ? a.value_scale : a.key_scale) + (limit ? at : 0),
                      !cut_in || ((taken >> key) & 1u) ? 4u : 0u, limit > 0);
      }
    }
  };
  auto copy_values = [&]() { copy_rows(true); };
  // where a lane reads: keys r and r + 8 (pieces of an odd t lie 64 bytes from where those of an even t would), values of keys 2c, 2c + 1, 2c + 8, 2c + 9
  const uint32_t k_read[2] = {ring + Ring::at_key(r, c), ring + (CH >= 8 ? Ring::at_key(r, c + 4) : 0u)}, v_read = ring + Ring::kRows + Ring::at_value(2 * c, r);
  auto step_on = [&]() { slot_in = slot_in + 1 == ST ? 0 : slot_in + 1; };
#pragma unroll 1
  for (int i = 0; i < ST; ++i) {
    take();
    copy_keys();
    paged_commit();
    copy_values();
    paged_commit();
    step_on();
  }

  // ---- piece after piece
  int slot = 0;
  int global = first;                         // its first unit among all
#pragma unroll 1
  for (; now.left > 0;) {
    const int units = now.units(), row = now.block * s.side + beside, g = row / s.tiles, h0 = g * a.group + (row - g * s.tiles) * 8 * NT, heads = min(8 * NT, (g + 1) * a.group - h0);
    // queries: the pieces that match the keys'
    uint32_t q[NT][DP / 8];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const bool have = n * 8 + r < heads;
      const uint16_t *qp = a.q + now.seq * a.qs[0] + (int64_t)(have ? h0 + n * 8 + r : h0) * a.qs[1];
#pragma unroll
      for (int t = 0; t < DP / 32; ++t) {
        // eight elements: of piece t for bf16, of half t & 1 of piece t / 2 for s8
        const int d = S8 ? (t >> 1) * 64 + c * 16 + (t & 1) * 8 : t * 32 + c * 8;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (have && d < a.dim) {
          if (s.q_vec) v = *reinterpret_cast<const uint4 *>(qp + d);
          else {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = (uint32_t)qp[d + 2 * e] | ((uint32_t)qp[d + 2 * e + 1] << 16);
            v = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        // (elements of s8 keys are paired as their codes are)
        if constexpr (S8) v = make_uint4(__byte_perm(v.x, v.y, 0x5410), __byte_perm(v.x, v.y, 0x7632), __byte_perm(v.z, v.w, 0x5410), __byte_perm(v.z, v.w, 0x7632));
        q[n][4 * t] = v.x; q[n][4 * t + 1] = v.y; q[n][4 * t + 2] = v.z; q[n][4 * t + 3] = v.w;
      }
    }
    float o[NT][DP / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = ninf; l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int t = 0; t < DP / 16; ++t) o[n][t][0] = o[n][t][1] = o[n][t][2] = o[n][t][3] = 0.f;
    }
    const int end = now.end_key();
    const float unit = S8 ? kPagedCode : 1.f, to_log2 = a.scale * kPagedLog2e * unit, cap_in = a.softcap > 0.f ? a.scale / a.softcap * unit : 0.f, cap_out = a.softcap * kPagedLog2e;
#pragma unroll 1
    for (int key = now.first_key() + warp * KS; key < end; key += UNIT) {
      const uint32_t at = (uint32_t)slot * Ring::kStep;
      slot = slot + 1 == ST ? 0 : slot + 1;
      // ---- scores
      paged_wait<2 * ST - 1>();
      __syncwarp();
      float kscale[MT][2], vscale[MT][2];
      if constexpr (S8) {
        const uint32_t sc = ring + at + 2 * Ring::kRows + 4u * r;
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) { kscale[i >> 1][i & 1] = paged_lds4(sc + 32u * i); vscale[i >> 1][i & 1] = paged_lds4(sc + 4u * KS + 32u * i); }
      }
      float x[MT][NT][4];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) x[i][n][0] = x[i][n][1] = x[i][n][2] = x[i][n][3] = 0.f;
#pragma unroll
      for (int t = 0; t < KP; ++t)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const uint32_t from = at + k_read[t & 1] + (uint32_t)(t >> 1) * 128u + (uint32_t)(i * 16 * CH * 16);
          const uint4 k0 = paged_lds16(from), k1 = paged_lds16(from + 8 * CH * 16);
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
          if constexpr (S8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t a0 = paged_codes_even(w0[e]), a1 = paged_codes_even(w1[e]), a2 = paged_codes_odd(w0[e]), a3 = paged_codes_odd(w1[e]);
#pragma unroll
              for (int n = 0; n < NT; ++n) paged_mma(x[i][n], a0, a1, a2, a3, q[n][8 * t + 2 * e], q[n][8 * t + 2 * e + 1]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; e += 2)
#pragma unroll
              for (int n = 0; n < NT; ++n) paged_mma(x[i][n], w0[e], w1[e], w0[e + 1], w1[e + 1], q[n][4 * t + e], q[n][4 * t + e + 1]);
          }
        }
      __syncwarp();                            // (all lanes have read the slot's keys)
      take();
      copy_keys();
      paged_commit();
      // ---- probabilities
      const bool cut = key + KS > end || key < now.lo;
      bool raise = false;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float z = x[i][n][e];
            if constexpr (S8) z *= kscale[i][e >> 1];
            z = a.softcap > 0.f ? cap_out * tanhf(z * cap_in) : z * to_log2;
            const int at_key = key + 16 * i + r + (e >> 1) * 8;
            if (cut && (at_key >= end || at_key < now.lo)) z = ninf;
            x[i][n][e] = z;
            raise |= z > m[n][e & 1] + kPagedReach;
          }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = m[n][e];
#pragma unroll
            for (int i = 0; i < MT; ++i) top = fmaxf(top, fmaxf(x[i][n][e], x[i][n][e + 2]));
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            const float keep = top == ninf ? 1.f : paged_exp2(m[n][e] - top);
            m[n][e] = top;
            l[n][e] *= keep;
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) { o[n][t][e] *= keep; o[n][t][e + 2] *= keep; }
          }
      }
      uint32_t p[MT][NT][2], pl[MT][NT][2], pr[F32 ? MT : 1][NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float f0 = m[n][0] == ninf ? 0.f : m[n][0], f1 = m[n][1] == ninf ? 0.f : m[n][1];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = paged_exp2(x[i][n][e] - ((e & 1) ? f1 : f0));
          l[n][0] += y[0] + y[2];
          l[n][1] += y[1] + y[3];
          if constexpr (S8) { y[0] *= vscale[i][0]; y[1] *= vscale[i][0]; y[2] *= vscale[i][1]; y[3] *= vscale[i][1]; }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t hi = paged_pack(y[2 * e], y[2 * e + 1]);
            p[i][n][e] = paged_transpose(hi);
            const float r0 = y[2 * e] - __uint_as_float(hi << 16), r1 = y[2 * e + 1] - __uint_as_float(hi & 0xffff0000u);
            const uint32_t lo = paged_pack(r0, r1);
            pl[i][n][e] = paged_transpose(lo);
            if constexpr (F32) pr[i][n][e] = paged_transpose(paged_pack(r0 - __uint_as_float(lo << 16), r1 - __uint_as_float(lo & 0xffff0000u)));
          }
        }
      }
      // ---- outputs
      paged_wait<2 * ST - 1>();
      __syncwarp();
#pragma unroll
      for (int t = 0; t < VP; ++t) {
        constexpr int W = VB / 4;
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          auto product = [&](int d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              paged_mma(o[n][d], a0, a1, a2, a3, p[j][n][0], p[j][n][1]);
              paged_mma(o[n][d], a0, a1, a2, a3, pl[j][n][0], pl[j][n][1]);
              if constexpr (F32) paged_mma(o[n][d], a0, a1, a2, a3, pr[j][n][0], pr[j][n][1]);
            }
          };
          uint32_t v[4][W];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t row = (uint32_t)((16 * j + (i & 1) + 8 * (i >> 1)) * CH * 16);
            if constexpr (VB == 16) { const uint4 w = paged_lds16(at + v_read + row + (uint32_t)t * 128u); v[i][0] = w.x; v[i][1] = w.y; v[i][2] = w.z; v[i][3] = w.w; }
            else {
              const uint2 w = paged_lds8(ring + at + Ring::kRows + Ring::at_value(16 * j + 2 * c + (i & 1) + 8 * (i >> 1), t * 4 + (r >> 1)) + (r & 1) * 8);
              v[i][0] = w.x; v[i][1] = w.y;
            }
          }
#pragma unroll
          for (int w = 0; w < W; ++w) {
            if constexpr (S8) {
              const uint32_t x = __byte_perm(v[0][w], v[1][w], 0x5410), y = __byte_perm(v[2][w], v[3][w], 0x5410);
              const uint32_t x2 = __byte_perm(v[0][w], v[1][w], 0x7632), y2 = __byte_perm(v[2][w], v[3][w], 0x7632);
              product((t * W + w) * 2, paged_codes_even(x), paged_codes_odd(x), paged_codes_even(y), paged_codes_odd(y));
              product((t * W + w) * 2 + 1, paged_codes_even(x2), paged_codes_odd(x2), paged_codes_even(y2), paged_codes_odd(y2));
            } else {
              product(t * W + w, __byte_perm(v[0][w], v[1][w], 0x5410), __byte_perm(v[0][w], v[1][w], 0x7632), __byte_perm(v[2][w], v[3][w], 0x5410),
                      __byte_perm(v[2][w], v[3][w], 0x7632));
            }
          }
        }
      }
      __syncwarp();                            // (and its values)
      copy_values();
      paged_commit();
      step_on();
    }

    // ---- the four warps' results as one, in warp 0: maximum, sum, output of its heads 2c and 2c + 1
    float4 *box = reinterpret_cast<float4 *>(smem + Ring::kBytes);
    auto join_warps = [&]() {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], w);
          if (r == 0) { s_m[warp][n * 8 + 2 * c + e] = m[n][e]; s_l[warp][n * 8 + 2 * c + e] = l[n][e]; }
        }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int h = n * 8 + 2 * c + e;
          float top = s_m[0][h], sum = 0.f;
#pragma unroll
          for (int w = 1; w < kPagedWarps; ++w) top = fmaxf(top, s_m[w][h]);
          const float f = top == ninf ? 0.f : top;
#pragma unroll
          for (int w = 0; w < kPagedWarps; ++w) sum += s_l[w][h] * paged_exp2(s_m[w][h] - f);
          const float keep = paged_exp2(m[n][e] - f);
          m[n][e] = top; l[n][e] = sum;
#pragma unroll
          for (int t = 0; t < DP / 16; ++t) { o[n][t][e] *= keep; o[n][t][e + 2] *= keep; }
        }
      auto put = [&](int b) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int t = 0; t < DP / 16; ++t) box[(b * (REGS / 4) + n * (DP / 16) + t) * 32 + lane] = make_float4(o[n][t][0], o[n][t][1], o[n][t][2], o[n][t][3]);
      };
      auto add = [&](int b) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int t = 0; t < DP / 16; ++t) {
            const float4 v = box[(b * (REGS / 4) + n * (DP / 16) + t) * 32 + lane];
            o[n][t][0] += v.x; o[n][t][1] += v.y; o[n][t][2] += v.z; o[n][t][3] += v.w;
          }
      };
      if constexpr (PagedJoin<S8, DP, NT>::kBoxes == 2) {
        if (warp >= 2) put(warp - 2);
        __syncthreads();
        if (warp < 2) add(warp);
        if (warp == 1) put(1);
        __syncthreads();
        if (warp == 0) add(1);
      } else {
        if (warp == 3) put(0);
#pragma unroll 1
        for (int w = 2; w >= 0; --w) {
          __syncthreads();
          if (warp == w) add(0);
          if (warp == w && w > 0) put(0);
        }
      }
    };
    // the row's result, in warp 0's registers, to where it belongs
    auto finish = [&]() {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int hh = n * 8 + 2 * c + e, h = h0 + hh;
          if (hh >= heads) continue;
          float top = m[n][e], sum = l[n][e], keep = 1.f;
          if (a.sinks) {
            const float sink = a.sinks[h] * kPagedLog2e, to = fmaxf(top, sink), f = to == ninf ? 0.f : to;
            keep = paged_exp2(top - f);
            sum = sum * keep + paged_exp2(sink - f);
            top = to;
          }
          const float by = sum == 0.f ? 0.f : (S8 ? kPagedCode : 1.f) * keep / sum;
          if (a.lse && r == 0) a.lse[(int64_t)now.seq * a.q_heads + h] = sum == 0.f ? ninf : (top + log2f(sum)) * 0.693147180559945309417f;
#pragma unroll
          for (int t = 0; t < DP / 16; t += (S8 && VB == 16 ? 8 : 4)) {
            // S8 with 16-byte pieces: sixteen dims of a lane in eight tiles, else eight in four
            constexpr int TILES = S8 && VB == 16 ? 8 : 4;
            const int d = t * 16 + r * 2 * TILES;
            if (d >= a.dim) continue;
            const int64_t to = now.seq * a.os[0] + h * a.os[1] + d;
            float y[2 * TILES];
#pragma unroll
            for (int w = 0; w < TILES; ++w) { y[2 * w] = o[n][t + w][e] * by; y[2 * w + 1] = o[n][t + w][e + 2] * by; }
            if constexpr (F32) {
              float *out = reinterpret_cast<float *>(a.out) + to;
#pragma unroll
              for (int w = 0; w < TILES / 2; ++w) {
                if (s.out_vec) reinterpret_cast<float4 *>(out)[w] = make_float4(y[4 * w], y[4 * w + 1], y[4 * w + 2], y[4 * w + 3]);
                else for (int i = 0; i < 4; ++i) out[4 * w + i] = y[4 * w + i];
              }
            } else {
              uint16_t *out = reinterpret_cast<uint16_t *>(a.out) + to;
#pragma unroll
              for (int w = 0; w < TILES / 4; ++w) {
                const uint4 v = make_uint4(paged_pack(y[8 * w], y[8 * w + 1]), paged_pack(y[8 * w + 2], y[8 * w + 3]), paged_pack(y[8 * w + 4], y[8 * w + 5]),
                                           paged_pack(y[8 * w + 6], y[8 * w + 7]));
                if (s.out_vec) reinterpret_cast<uint4 *>(out)[w] = v;
                else {
                  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                  for (int i = 0; i < 4; ++i) { out[8 * w + 2 * i] = (uint16_t)(u[i] & 0xffffu); out[8 * w + 2 * i + 1] = (uint16_t)(u[i] >> 16); }
                }
              }
            }
          }
        }
    };
    join_warps();
    if (units == now.n) {
      if (warp == 0) finish();
    } else {
      // a part of a row: slot 1 of the CTA in which the row begins, slot 0 of the others
      const int begin = global - now.off, c0 = begin / per, c1 = (begin + now.n - 1) / per;      // sets
      auto part = [&](int set) { return (int64_t)(set * s.side + beside) * 2 + (set == c0 ? 1 : 0); };
      const int my_set = (int)blockIdx.x / s.side;
      if (warp == 0) {
        float4 *to = reinterpret_cast<float4 *>(s.part_o) + part(my_set) * (REGS / 4) * 32;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int t = 0; t < DP / 16; ++t) __stcg(to + (n * (DP / 16) + t) * 32 + lane, make_float4(o[n][t][0], o[n][t][1], o[n][t][2], o[n][t][3]));
#pragma unroll
          for (int e = 0; e < 2; ++e) if (r == 0) __stcg(s.part_ml + part(my_set) * 8 * NT + n * 8 + 2 * c + e, make_float2(m[n][e], l[n][e]));
        }
        __syncwarp();
        // (the warp's stores in front of it, and the barrier behind it, are ordered by the one atomic; with fences 0.4 us more: one user, 500 keys 9.5 -> 9.05 us)
        if (lane == 0) s_last = paged_arrive(s.counters + c0 * s.side + beside) == (uint32_t)(c1 - c0);
      }
      __syncthreads();
      if (s_last) {
        if (tid == 0) s.counters[c0 * s.side + beside] = 0u;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          m[n][0] = m[n][1] = ninf; l[n][0] = l[n][1] = 0.f;
#pragma unroll
          for (int t = 0; t < DP / 16; ++t) o[n][t][0] = o[n][t][1] = o[n][t][2] = o[n][t][3] = 0.f;
        }
#pragma unroll 1
        for (int i = c0 + warp; i <= c1; i += kPagedWarps) {
          const float4 *from = reinterpret_cast<const float4 *>(s.part_o) + part(i) * (REGS / 4) * 32;
          float4 v[NT][DP / 16];
          float2 ml[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) ml[n][e] = __ldcg(s.part_ml + part(i) * 8 * NT + n * 8 + 2 * c + e);
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) v[n][t] = __ldcg(from + (n * (DP / 16) + t) * 32 + lane);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float mine[2], theirs[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float top = fmaxf(m[n][e], ml[n][e].x), f = top == ninf ? 0.f : top;
              mine[e] = paged_exp2(m[n][e] - f);
              theirs[e] = paged_exp2(ml[n][e].x - f);
              m[n][e] = top;
              l[n][e] = l[n][e] * mine[e] + (r == 0 ? ml[n][e].y * theirs[e] : 0.f);
            }
#pragma unroll
            for (int t = 0; t < DP / 16; ++t) {
              o[n][t][0] = o[n][t][0] * mine[0] + v[n][t].x * theirs[0]; o[n][t][1] = o[n][t][1] * mine[1] + v[n][t].y * theirs[1];
              o[n][t][2] = o[n][t][2] * mine[0] + v[n][t].z * theirs[0]; o[n][t][3] = o[n][t][3] * mine[1] + v[n][t].w * theirs[1];
            }
          }
        }
        join_warps();
        if (warp == 0) finish();
      }
    }
    global += units;
    now.next(s);
  }
}

}  // namespace b200
