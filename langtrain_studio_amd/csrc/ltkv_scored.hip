// gfx950 (MI355X, CDNA4) kernels of scored attention and of q4_0 pools.
//
//   scored_any_kernel       scored attention and q4_0 decode attention of any shape
//   scored_merge_kernel     fold of the parts of rows that were split
//   gather_values_kernel    rows behind block tables as f32 values
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/ltkv.h"
#include "ltkv_device.h"
#include "ltkv_kernels.h"
#include "ltkv_scored.h"

namespace ltkv {
namespace {

// The score of a visible position from q.k, in the log2 domain.
__device__ __forceinline__ float score_of(float qk, float scale, float softcap, float slope, int32_t dist) {
  float s = qk * scale;
  if (softcap > 0.f) s = softcap * tanhf(s / softcap);
  return (s - slope * (float)dist) * kLog2e;
}

constexpr int kAnyThreads = 256;
constexpr int kAnyMaxHeadDim = 1024;  // four output elements per thread
constexpr int kAnyD = kAnyMaxHeadDim / kAnyThreads;

// Any shape and pool. Work-group = (row, query head): 256 positions a round,
// one score a thread, the softmax of the round against the running maximum
// (exp2 domain), then each thread accumulates up to four output elements over
// the round's positions. Positions a row does not see are skipped, not
// multiplied by zero: they may hold infinities or NaN. It serves shapes that
// the matrix-core kernels do not, and is bound by its scalar loads.
template <typename T>
__global__ void __launch_bounds__(kAnyThreads) scored_any_kernel(ScoredArgs a, int64_t n_blocks, int64_t kv_dim) {
  __shared__ float sq[kAnyMaxHeadDim];
  __shared__ float sp[kAnyThreads];
  __shared__ int32_t sblk[kAnyThreads / 16];
  __shared__ float red[4];
  const int t = (int)threadIdx.x;
  const int h = (int)(blockIdx.x % a.n_heads);
  const int64_t row = blockIdx.x / a.n_heads;
  const int64_t seq = seq_of_row(a, row);
  const SeqRows s = seq_rows(a, seq);
  if (row < s.row0 || row >= s.row0 + s.count) return;  // no sequence's row: left as it is
  const RowView view = row_view(a, s, seq, (int32_t)(row - s.row0));
  const int64_t head_off = (int64_t)(h / (a.n_heads / a.n_kv_heads)) * a.head_dim;
  const int64_t qh = (row * a.n_heads + h) * a.head_dim;
  for (int d = t; d < a.head_dim; d += kAnyThreads) sq[d] = row_load(a, qh + d);
  const int32_t *tab = table_of(a.tables, a.table_stride, a.rows, a.table_rows, seq);
  if (t < 64) {
    const int32_t sinks = min(view.sink_end, view.end);
    if (sinks > view.first)
      check_table(tab, view.first >> 4, (sinks + 15) >> 4, n_blocks, a.rows, a.table_rows, seq, a.status);
    if (view.end > view.from)
      check_table(tab, view.from >> 4, (view.end + 15) >> 4, n_blocks, a.rows, a.table_rows, seq, a.status);
  }
  const float slope = a.slopes ? a.slopes[h] : 0.f;
  float m = -INFINITY, l = 0.f, o[kAnyD];
#pragma unroll
  for (int k = 0; k < kAnyD; ++k) o[k] = 0.f;
  // rounds of 16-position blocks, from the sinks on to the window
  int32_t t0 = (view.sink_end > view.first ? view.first : view.from) & ~15;
  for (; t0 < view.end; t0 += kAnyThreads) {
    if (t0 >= view.sink_end && t0 + 16 <= view.from) t0 = view.from & ~15;
    const int n_tok = min(view.end - t0, kAnyThreads);
    if (t < (n_tok + 15) / 16) {
      int32_t blk = tab[(t0 >> 4) + t];
      if (blk < 0 || blk >= n_blocks) blk = 0;  // reported by check_table
      sblk[t] = blk;
    }
    __syncthreads();
    float sc = -INFINITY;
    const bool seen = t < n_tok && view.sees(t0 + t);
    if (seen) {
      const int64_t cell = (int64_t)sblk[t >> 4] * 16 + (t & 15);
      float acc = 0.f;
      for (int d = 0; d < a.head_dim; ++d)
        acc += sq[d] * cell_value<T>(a.k_layer, a.k_scale, cell, kv_dim, head_off + d);
      sc = score_of(acc, a.scale, a.softcap, slope, abs(view.pos - (t0 + t)));
    }
    const float mx = block_reduce<true>(sc, red);
    const float mn = __builtin_fmaxf(m, mx);
    const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen yet
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    const float p = seen ? __builtin_amdgcn_exp2f(sc - ref) : 0.f;
    const float sum = l * alpha + block_reduce<false>(p, red);
    // o: the average over the positions so far, no larger than their V
    const float inv = sum != 0.f ? 1.f / sum : 0.f;  // (a NaN sum stays one)
    sp[t] = seen ? p * inv : -1.f;
    const float keep = l * alpha * inv;
    l = sum;
    m = mn;
#pragma unroll
    for (int k = 0; k < kAnyD; ++k) o[k] *= keep;
    __syncthreads();
    for (int j = 0; j < n_tok; ++j) {
      const float pj = sp[j];
      if (pj < 0.f) continue;
      const int64_t cell = (int64_t)sblk[j >> 4] * 16 + (j & 15);
#pragma unroll
      for (int k = 0; k < kAnyD; ++k) {
        const int d = t + kAnyThreads * k;
        if (d < a.head_dim) o[k] += pj * cell_value<T>(a.v_layer, a.v_scale, cell, kv_dim, head_off + d);
      }
    }
    __syncthreads();  // sblk and sp are rewritten next round
  }
#pragma unroll
  for (int k = 0; k < kAnyD; ++k) {
    const int d = t + kAnyThreads * k;
    if (d < a.head_dim) row_store(a, qh + d, o[k]);
  }
}

// Rows whose positions were taken in several parts (or splits): their numerators
// and sums folded in order by their references. VEC elements of a row a thread:
// first the part slots of the rows kernel (ScoredArgs::part_n), then the rows
// that the chunk kernel's split tile slots may hold.
// ROWS: only part slots of sequences' rows: a thread an element, 16 parts' loads
// at a time, since latency counts (one context's fold 4.6 us, 5.8 with four
// elements a thread), and no searches. Else four elements a thread: the splits
// are many (27 -> 15 us for six chunks of 512 rows, 9.4 by the call's rows instead
// of the tiles').
constexpr int kMergeThreads = 256;
constexpr int merge_vec(bool rows) { return rows ? 1 : 4; }

template <bool ROWS>
__global__ void __launch_bounds__(kMergeThreads) scored_merge_kernel(ScoredArgs a, int slices, int64_t part_slots,
                                                                     int64_t min_rows, int rows_per_tile) {
  constexpr int VEC = merge_vec(ROWS), AHEAD = ROWS ? 16 : 8;
  using vec = std::conditional_t<ROWS, float, f32x4>;
  const int64_t item = blockIdx.x / (uint32_t)slices;
  const int i = ((int)(blockIdx.x % (uint32_t)slices) * kMergeThreads + (int)threadIdx.x) * VEC;
  if (i >= a.n_heads * a.head_dim) return;  // (head_dim is a multiple of 8 here)
  const int h = i / a.head_dim, e = i - h * a.head_dim;
  // row of a slot of the packs, -1 for slots without one
  auto slot_row = [&](int64_t slot) -> int64_t {
    const int64_t pack = slot / rows_per_tile, seq = seq_of_slot(a, pack, rows_per_tile);
    const SeqRows s = seq_rows(a, seq);
    const int64_t r = (pack - first_slot(a, seq, rows_per_tile)) * rows_per_tile + slot % rows_per_tile;
    return r < 0 || r >= s.count ? -1 : s.row0 + r;
  };
  int64_t row, slot;
  int n_parts, stride;
  const float *o, *ml;
  if (ROWS || item < part_slots) {
    slot = item;
    if (!ROWS && a.packs) {
      row = slot_row(slot);
    } else {
      const int64_t seq = item / a.max_rows;
      const SeqRows s = seq_rows(a, seq);
      row = s.row0 + (item - seq * a.max_rows);
      // (slots of rows that no kernel took hold nothing)
      if (row >= s.row0 + s.count || s.count > min_rows) row = -1;
    }
    if (row < 0) return;
    n_parts = scalar_read(a.part_n, slot);
    stride = a.max_parts;
    o = a.part_o;
    ml = a.part_ml;
  } else {
    slot = row = item - part_slots;
    const int64_t seq = seq_of_row(a, row);
    const SeqRows s = seq_rows(a, seq);
    const int64_t r = row - s.row0;
    if (r < 0 || r >= s.count || s.count <= min_rows ||
        first_slot(a, seq, rows_per_tile) + r / rows_per_tile >= a.split_slots)
      return;
    n_parts = scalar_read(a.chunk_n, row);
    stride = a.splits;
    o = a.chunk_o;
    ml = a.chunk_ml;
  }
  if (n_parts <= 1) return;
  const int64_t at = (slot * a.n_heads + h) * stride;
  ml += 2 * at;
  o += at * a.head_dim + e;
  // AHEAD parts' loads at a time, folded one by one in order
  float mx = -INFINITY, l = 0.f;
  vec x = {};
  for (int p0 = 0; p0 < n_parts; p0 += AHEAD) {
    float pm[AHEAD], pl[AHEAD];
    vec po[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int p = p0 + k < n_parts ? p0 + k : n_parts - 1;
      const f32x2 v = *reinterpret_cast<const f32x2 *>(ml + 2 * p);
      po[k] = *reinterpret_cast<const vec *>(o + (int64_t)p * a.head_dim);
      pm[k] = p0 + k < n_parts ? v.x : -INFINITY;
      pl[k] = p0 + k < n_parts ? v.y : 0.f;
      if (p0 + k >= n_parts) po[k] = vec{};
    }
    float next = mx;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) next = __builtin_fmaxf(next, pm[k]);
    const float base = next == -INFINITY ? 0.f : next, f = __builtin_amdgcn_exp2f(mx - base);
    l *= f;
    x *= f;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const float g = __builtin_amdgcn_exp2f(pm[k] - base);
      l = __builtin_fmaf(pl[k], g, l);
      x += po[k] * g;
    }
    mx = next;
  }
  x = l != 0.f ? x / l : vec{};
  if constexpr (ROWS) row_store(a, row * a.n_heads * a.head_dim + i, x);
  else store_row4(a, row * a.n_heads * a.head_dim + i, x);
}

// Rows of a block as f32 values: a work-group per (table entry, K or V), four
// elements a thread and 16-byte stores (one element where kv_dim is not a
// multiple of four), consecutive threads on consecutive elements of a row. ~9 500
// q4_0 rows of 2 x 1024 elements: 18.8 us (89 MB, 4.7 TB/s), bound by the
// stores; stores past the caches (nontemporal) took 21 us.
constexpr int kValuesThreads = 256;

template <typename T, int VEC>
__global__ void __launch_bounds__(kValuesThreads)
gather_values_kernel(const void *__restrict__ kpool, const void *__restrict__ vpool, const void *__restrict__ kscale,
                     const void *__restrict__ vscale, const int32_t *__restrict__ tables, int64_t table_stride,
                     const int32_t *__restrict__ lens, const int64_t *__restrict__ out_offsets,
                     float *__restrict__ kout, float *__restrict__ vout, int64_t n_blocks, int64_t kv_dim,
                     int32_t *__restrict__ status) {
  const int is_v = (int)(blockIdx.x & 1);
  const int64_t entry = blockIdx.x >> 1;
  const int64_t seq = entry / table_stride;
  const int64_t j = entry - seq * table_stride;
  int64_t len = lens[seq];
  if (len > table_stride * 16) len = table_stride * 16;
  const int64_t start = j * 16;
  if (start >= len) return;
  const int rows = (int)(len - start < 16 ? len - start : 16);
  const int32_t blk = tables[entry];
  if (blk < 0 || blk >= n_blocks) {
    if (threadIdx.x == 0) report_fault(status, kFaultTable, seq);
    return;
  }
  const void *pool = is_v ? vpool : kpool, *scale = is_v ? vscale : kscale;
  float *dst = (is_v ? vout : kout) + (out_offsets[seq] + start) * kv_dim;
  const int per_row = (int)(kv_dim / VEC);
  int slot = (int)threadIdx.x / per_row, unit = (int)threadIdx.x - slot * per_row;
  const int step = kValuesThreads / per_row, left = kValuesThreads - step * per_row;
  for (; slot < rows; slot += step, unit += left) {
    if (unit >= per_row) {
      unit -= per_row;
      if (++slot >= rows) break;
    }
    const int64_t e = (int64_t)unit * VEC, cell = (int64_t)blk * 16 + slot;
    float x[VEC];
    if constexpr (VEC == 4 && std::is_same_v<T, Q4>) {
      const int64_t at = (((cell >> 4) * (kv_dim >> 5) + (e >> 5)) << 4) + (cell & 15);
      const uint32_t w = static_cast<const uint32_t *>(pool)[at * 4 + (((int)e & 31) >> 3)] >> (2 * ((int)e & 4));
      const float d = (float)static_cast<const _Float16 *>(scale)[at];
      x[0] = (float)((int)(w & 15u) - 8) * d;
      x[1] = (float)((int)(w >> 16 & 15u) - 8) * d;
      x[2] = (float)((int)(w >> 4 & 15u) - 8) * d;
      x[3] = (float)((int)(w >> 20 & 15u) - 8) * d;
    } else if constexpr (VEC == 4 && std::is_same_v<T, int8_t>) {
      const uint32_t w = *reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(pool) + cell * kv_dim + e);
      const float d =
          (float)static_cast<const _Float16 *>(scale)[(((cell >> 4) * (kv_dim >> 5) + (e >> 5)) << 4) + (cell & 15)];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (float)((int)(w >> (8 * i) & 255u) - 128) * d;
    } else if constexpr (VEC == 4 && std::is_same_v<T, _Float16>) {
      const h4 w = *reinterpret_cast<const h4 *>(static_cast<const _Float16 *>(pool) + cell * kv_dim + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (float)w[i];
    } else if constexpr (VEC == 4) {
      const f32x4 w = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(pool) + cell * kv_dim + e);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = w[i];
    } else {
      x[0] = cell_value<T>(pool, scale, cell, kv_dim, e);
    }
    if constexpr (VEC == 4) *reinterpret_cast<f32x4 *>(dst + slot * kv_dim + e) = f32x4{x[0], x[1], x[2], x[3]};
    else dst[slot * kv_dim + e] = x[0];
  }
}

}  // namespace

namespace {

// Rows from the first on among which those of the split tile slots are: row r is
// in slot r / (rows of a tile) - 1 or a later one.
int64_t split_rows(const ScoredArgs &a) {
  return a.split_slots > 0 ? std::min<int64_t>(a.n_rows, (int64_t)(a.split_slots + 1) * chunk_rows(a)) : 0;
}

// Most positions that the steps of a row cover.
int64_t span_bound(const ScoredArgs &a) {
  int64_t span = a.max_len;
  // (a prefix may show more than the window)
  if (a.window > 0 && !a.prefix) span = std::min(span, a.window + std::min(a.sinks, a.max_len) + 2 * 16);
  return (span + 31) / 32 * 32 + 32;
}

// Which kernels a call takes: the rows kernel where no sequence is expected to
// have more than kRowsKernelMax rows (or packs of rows where the chunk kernel
// does not serve the shape), the chunk kernel else, with the rows kernel
// for the short sequences beside it; the generic kernel for the other shapes.
struct Kernels {
  bool rows, packs, chunks;
};

Kernels kernels_of(int elem, const ScoredArgs &a) {
  const int group = a.n_heads / a.n_kv_heads;
  if (!scored_rows_supported(elem, a.head_dim)) return {false, false, false};
  if (a.max_rows <= kRowsKernelMax) return {true, false, false};
  if (!scored_chunks_supported(elem, a.head_dim, group)) return {true, true, false};
  return {a.n > 1, false, true};
}

}  // namespace

ScoredWorkspace scored_workspace(int elem, ScoredArgs &a) {
  ScoredWorkspace w{};
  const Kernels k = kernels_of(elem, a);
  a.packs = k.packs;
  a.chunks = k.chunks;
  if (k.chunks && k.rows) a.max_rows = kRowsKernelMax;  // of the sequences that the rows kernel takes
  a.max_parts = a.splits = 1;
  a.split_slots = 0;
  const int64_t span = span_bound(a);
  int64_t at = 0;
  if (k.rows) a.max_parts = (int)scored_max_parts(span, a.part_tokens);
  // Rows with starts: no more parts a sequence than 128 waves a CU make in all, or
  // eight. Tables may be far wider than the contexts: 64 rows beside 255 single
  // tokens on tables of 131 072 positions, 32 / 8 heads of 128, took 526 000 waves,
  // most of them empty, and 2.2 GB of partials (677 us); so 33 000 and 136 MB (119
  // us; with half as many 104, but 540 instead of 364 where one of the sequences
  // has 60 000 positions and the others 200).
  if (a.row_starts && !a.packs)
    a.max_parts = (int)std::min<int64_t>(a.max_parts, std::max<int64_t>(8, 128 * a.cu_count / (a.n * a.n_kv_heads)));
  // packs are many where a chunk is long: no more parts than fill the chip a few
  // times (they cost partials)
  if (a.packs)
    a.max_parts = (int)std::max<int64_t>(
        1, std::min<int64_t>(a.max_parts, 32 * a.cu_count / (pack_slots(a) * a.n_kv_heads)));
  if (a.max_parts > 1) {
    const int64_t slots = a.packs ? pack_slots(a) * pack_rows(a) : a.n * a.max_rows;
    const int64_t parts = slots * a.n_heads * (int64_t)a.max_parts;
    w.part_o_off = at;
    w.part_ml_off = at + parts * a.head_dim * 4;
    w.part_n_off = w.part_ml_off + parts * 2 * 4;
    at = (w.part_n_off + slots * 4 + 255) / 256 * 256;
  }
  if (k.chunks) {
    // The work-groups that whole rounds of the resident ones (two a CU) leave over
    // are split over their positions, to fill a round as well (at least 256
    // positions each): partials cost their traffic only there.
    const int rows = chunk_rows(a);
    const int64_t tiles = (a.n_rows + rows - 1) / rows * a.n_kv_heads, resident = 2 * a.cu_count;
    const int64_t over = tiles % resident;
    // (a few left over cost less than the merge of their splits)
    if (over >= resident / 8 || (over > 0 && tiles < resident))
      a.splits = (int)std::max<int64_t>(1, std::min<int64_t>({resident / over, span / 256, 32}));
    if (a.splits > 1) {
      // (slots may be empty: a sequence's tiles need not fill its slots)
      a.split_slots = (int)std::min<int64_t>((over + a.n_kv_heads - 1) / a.n_kv_heads + a.n, chunk_slots(a));
      const int64_t parts = split_rows(a) * a.n_heads * a.splits;
      w.chunk_o_off = at;
      w.chunk_ml_off = at + parts * a.head_dim * 4;
      w.chunk_n_off = w.chunk_ml_off + parts * 2 * 4;
      at = w.chunk_n_off + split_rows(a) * 4;
    }
  }
  w.bytes = at;
  return w;
}

hipError_t launch_scored_attention(const PoolGeom &g, const ScoredArgs &a, hipStream_t s) {
  if (a.n <= 0 || a.n_rows <= 0) return hipSuccess;
  if (!scored_rows_supported(g.elem, a.head_dim)) {
    const int64_t grid = a.n_rows * a.n_heads;
    if (grid * kAnyThreads >= (int64_t{1} << 32)) return hipErrorInvalidValue;
    return by_element(g.elem, [&](auto tag) {
      scored_any_kernel<decltype(tag)><<<(unsigned)grid, kAnyThreads, 0, s>>>(a, g.n_blocks, g.kv_dim);
      return hipGetLastError();
    });
  }
  const int64_t all = INT64_MAX;
  const int64_t border = a.chunks ? (a.n > 1 ? kRowsKernelMax : 0) : all;  // most rows of the rows kernel's sequences
  if (a.chunks)
    if (const hipError_t e = launch_scored_chunks(g, a, border, s); e != hipSuccess) return e;
  if (border > 0)
    if (const hipError_t e = launch_scored_rows(g, a, border, s); e != hipSuccess) return e;
  const int64_t part_slots = border > 0 && a.max_parts > 1 ? (a.packs ? pack_slots(a) * pack_rows(a) : a.n * a.max_rows) : 0;
  const int rows_per_tile = a.chunks ? chunk_rows(a) : pack_rows(a);
  const int64_t items = part_slots + split_rows(a);
  if (items == 0) return hipSuccess;
  const bool rows_only = !a.packs && a.split_slots == 0;
  const int per_group = kMergeThreads * merge_vec(rows_only);
  const int slices = (a.n_heads * a.head_dim + per_group - 1) / per_group;
  if (items * slices * kMergeThreads >= (int64_t{1} << 32)) return hipErrorInvalidValue;
  const auto merge = rows_only ? scored_merge_kernel<true> : scored_merge_kernel<false>;
  merge<<<(unsigned)(items * slices), kMergeThreads, 0, s>>>(a, slices, part_slots, border, rows_per_tile);
  return hipGetLastError();
}

hipError_t launch_gather_values(const PoolGeom &g, const void *k_layer, const void *v_layer, const void *k_scale,
                                const void *v_scale, const int32_t *tables, int64_t table_stride,
                                const int32_t *lens, const int64_t *out_offsets, int64_t n, float *k_out,
                                float *v_out, int32_t *status, hipStream_t s) {
  if (n <= 0 || table_stride <= 0) return hipSuccess;
  const int64_t wgs = n * table_stride * 2;
  if (wgs * kValuesThreads >= (int64_t{1} << 32)) return hipErrorInvalidValue;
  return by_element(g.elem, [&](auto tag) {
    using T = decltype(tag);
    const auto kernel = g.kv_dim % 4 == 0 ? gather_values_kernel<T, 4> : gather_values_kernel<T, 1>;
    kernel<<<(unsigned)wgs, kValuesThreads, 0, s>>>(k_layer, v_layer, k_scale, v_scale, tables, table_stride, lens,
                                                    out_offsets, k_out, v_out, g.n_blocks, g.kv_dim, status);
    return hipGetLastError();
  });
}

}  // namespace ltkv
