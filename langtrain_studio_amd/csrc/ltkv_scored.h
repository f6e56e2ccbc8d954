// What the kernels of scored attention share.
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

namespace {

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
    return t >= first && t < end && (t >= from || t < sink_end);
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

// f32 -> bf16, nearest even (NaN stays NaN).
__device__ __forceinline__ uint16_t bf16_bits(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

__device__ __forceinline__ void row_store(const ScoredArgs &a, int64_t i, float x) {
  if (a.row_type == LTKV_ROWS_F32) static_cast<float *>(a.out)[i] = x;
  else
    static_cast<uint16_t *>(a.out)[i] = a.row_type == LTKV_ROWS_F16 ? (uint16_t)f16_bits(x) : bf16_bits(x);
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
__host__ __device__ inline int scored_part_tokens(int64_t span, int fixed) {
  if (fixed > 0) return fixed;
  return span <= 2048 ? 256 : span <= 8192 ? 512 : 1024;
}

// Most parts of spans up to `span` tokens.
inline int64_t scored_max_parts(int64_t span, int fixed) {
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  if (fixed > 0) return up(span, fixed);
  int64_t parts = up(std::min<int64_t>(span, 2048), 256);
  if (span > 2048) parts = std::max(parts, up(std::min<int64_t>(span, 8192), 512));
  if (span > 8192) parts = std::max(parts, up(span, 1024));
  return parts;
}

// The 32-token steps over a row's visible positions: those of its sinks, then
// those of its window (one range where the two meet). Steps begin at block
// borders; a step's positions end at its range's end.
struct StepRange {
  int32_t a0, a_end, b0, b_end;
  int32_t n_a, n;
  __device__ __forceinline__ int32_t start(int32_t step) const {
    return step < n_a ? a0 + 32 * step : b0 + 32 * (step - n_a);
  }
  __device__ __forceinline__ int32_t end(int32_t step) const { return step < n_a ? a_end : b_end; }
};

__device__ __forceinline__ StepRange step_range(const RowView &v) {
  StepRange s;
  s.a0 = v.first & ~15;
  s.a_end = min(v.sink_end, v.end);
  s.b0 = v.from & ~15;
  s.b_end = v.end;
  if (s.a_end > v.first && s.b0 <= ((s.a_end + 15) & ~15)) {  // the ranges meet
    s.b0 = s.a0;
    s.a_end = s.a0;
  }
  s.n_a = s.a_end > v.first ? (s.a_end - s.a0 + 31) / 32 : 0;
  s.n = s.n_a + (s.b_end > v.from || (s.b0 == s.a0 && s.b_end > v.first) ? (s.b_end - s.b0 + 31) / 32 : 0);
  return s;
}

}  // namespace
}  // namespace ltkv
