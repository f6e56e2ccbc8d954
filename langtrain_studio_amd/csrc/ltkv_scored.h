// What the kernels of scored and tree attention share.
//
// Scored attention (ltkv_scored_attention): row r of a sequence with m rows and
// L positions stands at position p = L - m + r and sees the positions t with
//   t < L, first_r <= t, (t <= p or t < prefix), and, with a window of w,
//   (t > p - w or t < first_r + sinks).
// Its weights are the softmax over these of
//   s = scale q.k;  s <- cap tanh(s / cap) with a cap;  s <- s - slope_h |p - t|,
// and a row that sees nothing (or stands before the context) gives zeros.
//
// The weights are exp2((s - ref) log2(e)) for a reference near the running
// maximum; numerators and sums over several ranges of positions are folded by
// their references.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/ltkv.h"
#include "ltkv_device.h"
#include "ltkv_kernels.h"

namespace ltkv {

// Sequences with more rows than this go to the chunk kernel.
constexpr int kRowsKernelMax = 2;

// The rows kernel (ltkv_scored_rows.hip): sequences of at most `most_rows`
// rows, each row on its own.
bool scored_rows_supported(int elem, int head_dim);
hipError_t launch_scored_rows(const PoolGeom &g, const ScoredArgs &a, int64_t most_rows, hipStream_t s);

// The chunk kernel (ltkv_scored_chunk.hip): sequences of more than `min_rows`
// rows. A work-group takes kChunkColumns (row, query head) pairs of a kv head.
constexpr int kChunkWaves = 4;
constexpr int kChunkColumns = 32 * kChunkWaves;
inline bool scored_chunks_supported(int elem, int head_dim, int group) {
  return elem != 4 && (head_dim == 64 || head_dim == 128) && group <= kChunkColumns;
}
inline int chunk_rows(const ScoredArgs &a) { return kChunkColumns / (a.n_heads / a.n_kv_heads); }
// Rows that share a wave's 16 columns where the rows kernel takes whole chunks.
__host__ __device__ inline int pack_rows(const ScoredArgs &a) {
  const int group = a.n_heads / a.n_kv_heads;
  return group <= 8 ? 16 / group : 1;
}
inline int64_t pack_slots(const ScoredArgs &a) { return a.n_rows / pack_rows(a) + a.n; }
inline int64_t chunk_slots(const ScoredArgs &a) { return a.n_rows / chunk_rows(a) + a.n; }
hipError_t launch_scored_chunks(const PoolGeom &g, const ScoredArgs &a, int64_t min_rows, hipStream_t s);

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

struct Q4 {};  // element tag of q4_0 pools

// A sequence's rows of a call: `count` rows from row `row0`, which stand at
// positions len - count ... len - 1.
struct SeqRows {
  int64_t row0;
  int32_t count, len;
};

__device__ __forceinline__ SeqRows seq_rows(const ScoredArgs &a, int64_t seq) {
  SeqRows s;
  const int64_t len = scalar_read(a.lens, seq);
  s.len = (int32_t)(len < 0 ? 0 : len > a.max_len ? a.max_len : len);
  if (!a.row_starts) {
    s.row0 = seq;
    s.count = 1;
    return s;
  }
  // starts outside [0, n_rows], or falling ones, give fewer rows, never a row
  // outside the call's
  const int64_t lo = scalar_read(a.row_starts, seq), hi = scalar_read(a.row_starts, seq + 1);
  s.row0 = lo < 0 ? 0 : lo > a.n_rows ? a.n_rows : lo;
  const int64_t end = hi > a.n_rows ? a.n_rows : hi;
  s.count = (int32_t)(end > s.row0 ? end - s.row0 : 0);
  return s;
}

// The positions a row sees: [first, sink_end) and [from, end) without those
// before `from` again, masked by sees().
struct RowView {
  int32_t pos;       // the row's position
  int32_t first;     // first position of its document
  int32_t sink_end;  // sink positions lie before it
  int32_t from;      // first position inside the window
  int32_t end;       // positions from here on are not visible
  __device__ __forceinline__ bool sees(int32_t t) const {
    // (no short circuits: a select each, not branches)
    return (t >= first) & (t < end) & ((t >= from) | (t < sink_end));
  }
  // any of the positions of the block that begins at t
  __device__ __forceinline__ bool sees_of_block(int32_t t) const {
    const int32_t lo = max(t, first), hi = min(t + 16, end);
    return (hi > lo) & ((hi > from) | (lo < sink_end));
  }
};

__device__ __forceinline__ RowView row_view(const ScoredArgs &a, const SeqRows &s, int64_t seq, int32_t r) {
  RowView v;
  v.pos = s.len - s.count + r;
  v.first = a.first ? max(a.first[s.row0 + r], 0) : 0;
  int32_t end = v.pos + 1;
  if (a.prefix) end = max(end, min(a.prefix[seq], s.len));
  v.end = v.pos >= 0 ? end : 0;
  v.from = v.first;
  v.sink_end = v.first;
  if (a.window > 0) {
    v.from = max(v.first, (int32_t)max((int64_t)v.pos - a.window + 1, (int64_t)0));
    // (first may be anything: no sum past the last position)
    v.sink_end = v.first < s.len ? v.first + (int32_t)min(a.sinks, (int64_t)(s.len - v.first)) : v.first;
  }
  return v;
}

// Slots of the chunk kernel's tiles (and of the rows kernel's packs): those of sequence i begin at starts[i] /
// rows_per_tile + i, which leaves room for all of its tiles whatever its first
// row's place in a tile.
__device__ __forceinline__ int64_t first_slot(const ScoredArgs &a, int64_t i, int rows_per_tile) {
  const int64_t st = a.row_starts[i];
  return (st < 0 ? 0 : st > a.n_rows ? a.n_rows : st) / rows_per_tile + i;
}

// Sequence of such a slot: the last one whose slots begin at or before it.
__device__ __forceinline__ int64_t seq_of_slot(const ScoredArgs &a, int64_t slot, int rows_per_tile) {
  int64_t lo = 0, hi = a.n;
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (first_slot(a, mid, rows_per_tile) <= slot) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Sequence of launch row `row`: the last one whose first row is not behind it.
__device__ __forceinline__ int64_t seq_of_row(const ScoredArgs &a, int64_t row) {
  if (!a.row_starts) return row;
  int64_t lo = 0, hi = a.n;  // starts[lo] <= row, or lo == 0
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if ((int64_t)scalar_read(a.row_starts, mid) <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ float row_load(const ScoredArgs &a, int64_t i) {
  if (a.row_type == LTKV_ROWS_F32) return static_cast<const float *>(a.q)[i];
  const uint16_t u = static_cast<const uint16_t *>(a.q)[i];
  return a.row_type == LTKV_ROWS_F16 ? (float)__builtin_bit_cast(_Float16, u)
                                     : __builtin_bit_cast(float, (uint32_t)u << 16);
}

__device__ __forceinline__ void row_store(const ScoredArgs &a, int64_t i, float x) {
  if (a.row_type == LTKV_ROWS_F32) static_cast<float *>(a.out)[i] = x;
  else
    static_cast<uint16_t *>(a.out)[i] = a.row_type == LTKV_ROWS_F16 ? (uint16_t)f16_bits(x) : bf16_bits(x);
}


// Element e of the pool row of cell `cell` (block * 16 + slot) as f32.
template <typename T>
__device__ __forceinline__ float cell_value(const void *pool, const void *scales, int64_t cell, int64_t kv_dim,
                                            int64_t e) {
  if constexpr (std::is_same_v<T, Q4>) {
    const int64_t at = (((cell >> 4) * (kv_dim >> 5) + (e >> 5)) << 4) + (cell & 15);
    const int i = (int)e & 31;
    const uint32_t w = static_cast<const uint32_t *>(pool)[at * 4 + (i >> 3)];
    const int q = (int)(w >> (4 * ((i & 7) >> 1) + 16 * (i & 1)) & 15u) - 8;
    return (float)q * (float)static_cast<const _Float16 *>(scales)[at];
  } else if constexpr (std::is_same_v<T, int8_t>) {
    const int q = (int)static_cast<const uint8_t *>(pool)[cell * kv_dim + e] - 128;
    const int64_t at = (((cell >> 4) * (kv_dim >> 5) + (e >> 5)) << 4) + (cell & 15);
    return (float)q * (float)static_cast<const _Float16 *>(scales)[at];
  } else {
    return (float)static_cast<const T *>(pool)[cell * kv_dim + e];
  }
}

// A load at a uniform base plus a 32-bit lane offset. The offset is made opaque
// where it is used: widened outside of the loop it would be added as 64 bits in
// vector registers for every load.
template <typename V>
__device__ __forceinline__ V load_at(const char *base, uint32_t off) {
  asm volatile("" : "+v"(off));
  return *reinterpret_cast<const V *>(base + off);
}

// Quants of q4_0, 8 a dword: a nibble u becomes the low mantissa bits of an f16
// in [1024, 1040) (0x6400 | u) and 1032 is subtracted, or the next ones of an f16
// in [1024, 1280) (1024 + 16 u) that is taken times 1/16 minus 72; then the scale
// is multiplied. All of it is exact (the scale has 8 bits). The bias sits in a
// vector register: an and-or takes only one scalar operand.
__device__ __forceinline__ h8 q4x8_to_h8(uint32_t w, h2 d) {
  uint32_t bias;
  asm("v_mov_b32 %0, 0x64006400" : "=v"(bias));
  const h2 off = {(_Float16)-1032.f, (_Float16)-1032.f}, sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f},
           off16 = {(_Float16)-72.f, (_Float16)-72.f};
  const uint32_t v = w >> 8;
  const h2 p0 = (__builtin_bit_cast(h2, (w & 0x000f000fu) | bias) + off) * d;
  const h2 p1 = __builtin_elementwise_fma(__builtin_bit_cast(h2, (w & 0x00f000f0u) | bias), sixteenth, off16) * d;
  const h2 p2 = (__builtin_bit_cast(h2, (v & 0x000f000fu) | bias) + off) * d;
  const h2 p3 = __builtin_elementwise_fma(__builtin_bit_cast(h2, (v & 0x00f000f0u) | bias), sixteenth, off16) * d;
  return h8{p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
}

// hi + lo f16 parts of x: 22 bits together.
__device__ __forceinline__ void split2(float x, _Float16 &hi, _Float16 &lo) {
  // x as an f32 number: folded into a product's conversion it could be rounded
  // once for hi and twice for what lo is the rest of
  asm("" : "+v"(x));
  hi = (_Float16)x;
  lo = (_Float16)(x - (float)hi);
}

// What the product of a query and a key that entered times powers of two is
// multiplied by to give a score over the cap (or, without one, a score in log2):
// factor 2^e, held between 1e-37 and 1e37. Where caps are tiny or the powers far
// apart it would be infinite or zero, and a product of exactly zero, or a masked
// position's infinity, times that no number. Products lie between 2^-24 and 2^35,
// so a score that the limits change is past any cap, or nothing.
__device__ __forceinline__ float score_factor(float factor, int e) {
  const float f = __builtin_amdgcn_ldexpf(factor, e);
  return __builtin_copysignf(__builtin_amdgcn_fmed3f(__builtin_fabsf(f), 1e-37f, 1e37f), f);
}

// Score references are raised only when a score exceeds them by kSlack (log2),
// so most steps need no exchange between lanes and no rescaling; weights carry
// 2^lift, so that the largest (2^(kSlack + lift)) lie near the top of f16 and the
// lo parts of small ones stay out of its subnormals: kLift for values V that are
// f16 numbers themselves. q8_0 weights are multiplied by V's scales first: the
// lift follows the largest scale met, whatever its magnitude.
constexpr float kSlack = 8.f;
constexpr float kLift = 6.f;

// tanh, to a few units of f32 at any size: odd polynomial below 0.35 (the next
// term is below 2^-26 there), 1 - 2 / (exp(2 |x|) + 1) beyond.
__device__ __forceinline__ float tanh_f32(float x) {
  const float y = x * x;
  float p = __builtin_fmaf(y, -0.008863235529902197f, 0.021869488536155203f);
  p = __builtin_fmaf(y, p, -0.05396825396825397f);
  p = __builtin_fmaf(y, p, 0.13333333333333333f);
  p = __builtin_fmaf(y, p, -0.3333333333333333f);
  const float small = __builtin_fmaf(x * y, p, x);
  const float ax = __builtin_fabsf(x);
  const float e = __builtin_amdgcn_exp2f(ax * (2.f * kLog2e));
  const float large = __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f);
  return ax < 0.35f ? small : __builtin_copysignf(large, x);
}

// Largest cap whose tanh may be off by a few units of f32 in absolute terms
// (tanh_f16, and the chunk kernel's cap - 2 cap / (exp(2 x) + 1)): a score is
// then off by ~3e-7 times the cap, 8e-5 here, a sixth of what the rounding of a
// 16-bit row's weight to f16 may cost (2^-11). Larger caps of such rows take
// f32 rows' way.
constexpr float kShortCap = 256.f;

// tanh to a few units of f32 in absolute terms.
__device__ __forceinline__ float tanh_f16(float x) {
  return __builtin_fmaf(-2.f, __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(x * (2.f * kLog2e)) + 1.f), 1.f);
}

// Elements i ... i + 7 of Q as f32 (zeros where `live` is false).
__device__ __forceinline__ void load_row8(const ScoredArgs &a, int64_t i, bool live, float (&x)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = 0.f;
  if (!live) return;
  if (a.row_type == LTKV_ROWS_F32) {
    const f32x4 *p = reinterpret_cast<const f32x4 *>(static_cast<const float *>(a.q) + i);
    const f32x4 u = p[0], v = p[1];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[k] = u[k];
      x[4 + k] = v[k];
    }
    return;
  }
  const u32x4 u = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(a.q) + i);
  const h8 h = __builtin_bit_cast(h8, u);
#pragma unroll
  for (int k = 0; k < 8; ++k)
    x[k] = a.row_type == LTKV_ROWS_F16
               ? (float)h[k]
               : __builtin_bit_cast(float, k & 1 ? u[k >> 1] & 0xffff0000u : u[k >> 1] << 16);
}

// Elements i ... i + 3 of the output.
__device__ __forceinline__ void store_row4(const ScoredArgs &a, int64_t i, const f32x4 &x) {
  if (a.row_type == LTKV_ROWS_F32) {
    *reinterpret_cast<f32x4 *>(static_cast<float *>(a.out) + i) = x;
    return;
  }
  uint32_t u[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) u[k] = a.row_type == LTKV_ROWS_F16 ? f16_bits(x[k]) : bf16_bits(x[k]);
  *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + i) = u32x2{u[0] | u[1] << 16, u[2] | u[3] << 16};
}

// Two ds_read_b64_tr_b16 as one operand: positions at p and `step` bytes on.
__device__ __forceinline__ h8 read_tr2(const char *p, int step) {
  const h4 x = __builtin_bit_cast(h4, lds_read_tr(p)), y = __builtin_bit_cast(h4, lds_read_tr(p + step));
  return h8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// True if an element is infinite or NaN.
__device__ __forceinline__ bool not_finite(const h8 &x) {
  const u32x4 u = __builtin_bit_cast(u32x4, x);
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, u[i] & 0x7fff7fffu));
  return m.x >= 0x7c00 || m.y >= 0x7c00;
}

// Largest of a value over a position's four lanes, in each of them.
__device__ __forceinline__ float position_max(float x) {
  x = __builtin_fmaxf(x, dpp<0xB1>(x));     // quad_perm [1,0,3,2]
  return __builtin_fmaxf(x, dpp<0x4E>(x));  // quad_perm [2,3,0,1]
}

// Sum / maximum of a value over lanes l and l ^ 32.
template <bool MAX>
__device__ __forceinline__ float halves_reduce(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const float p = __builtin_bit_cast(float, (uint32_t)b[0]), q = __builtin_bit_cast(float, (uint32_t)b[1]);
  return MAX ? __builtin_fmaxf(p, q) : p + q;
}

// Work-group barrier that orders LDS only: loads from global memory stay in
// flight across it.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <typename F>
hipError_t by_element(int elem, F &&f) {
  if (elem == kElemQ4) return f(Q4{});
  if (elem == 1) return f(int8_t{});
  if (elem == 2) return f(_Float16{});
  return f(float{});
}


// Tokens per part of a row's visible positions (rounded up to 32-token steps;
// a multiple of 64): a function of the row's own span, so that a decode
// query's bits do not depend on its batch.
constexpr int64_t kShortSpan = 1024, kLongSpan = 8192;
__host__ __device__ inline int scored_part_tokens(int64_t span, int fixed) {
  if (fixed > 0) return fixed;
  return span <= kShortSpan ? 128 : span <= kLongSpan ? 256 : 512;
}

// Most parts of spans up to `span` tokens.
inline int64_t scored_max_parts(int64_t span, int fixed) {
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  if (fixed > 0) return up(span, fixed);
  int64_t parts = up(std::min<int64_t>(span, kShortSpan), 128);
  if (span > kShortSpan) parts = std::max(parts, up(std::min<int64_t>(span, kLongSpan), 256));
  if (span > kLongSpan) parts = std::max(parts, up(span, 512));
  return parts;
}

// The STEP-position steps over what a row (or rows together) sees: those of the
// sinks, then those of the window (one range where the two meet). Steps begin
// at block borders; a step's positions end at its range's end.
template <int STEP>
struct StepRange {
  int32_t a0, a_end, b0, b_end;
  int32_t n_a, n;
  __device__ __forceinline__ int32_t start(int32_t step) const {
    return step < n_a ? a0 + STEP * step : b0 + STEP * (step - n_a);
  }
  __device__ __forceinline__ int32_t end(int32_t step) const { return step < n_a ? a_end : b_end; }
};

template <int STEP>
__device__ __forceinline__ StepRange<STEP> step_range(const RowView &v) {
  StepRange<STEP> s;
  s.a0 = v.first & ~15;
  s.a_end = min(v.sink_end, v.end);
  s.b0 = v.from & ~15;
  s.b_end = v.end;
  if (s.a_end > v.first && s.b0 <= ((s.a_end + 15) & ~15)) {  // the ranges meet
    s.b0 = s.a0;
    s.a_end = s.a0;
  }
  s.n_a = s.a_end > v.first ? (s.a_end - s.a0 + STEP - 1) / STEP : 0;
  s.n = s.n_a + (s.b_end > v.from || (s.b0 == s.a0 && s.b_end > v.first) ? (s.b_end - s.b0 + STEP - 1) / STEP : 0);
  return s;
}

}  // namespace
}  // namespace ltkv
