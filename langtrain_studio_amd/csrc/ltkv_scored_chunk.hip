// gfx950 (MI355X, CDNA4) kernel of scored attention for prompt chunks: many rows
// of a sequence against tiles of its positions that they share, on the matrix
// cores.

#include "ltkv_scored.h"

namespace ltkv {
namespace {

constexpr int kChunkTokens = 64;  // positions of a tile

// A thread's share of a tile on its way from the pool to LDS: a quarter of the
// head (NC = HD / 32 chunks of 8 elements) of one position, K and V. get() and
// get2() give a chunk as f16 numbers: f16 and q4_0 cells are f16 numbers; q8_0
// cells times a power of two (see TileRange) as f16 hi + lo pairs.
template <typename T, int NC>
struct Share;

// A wave stages the 16 positions of one block: its address is uniform, a lane's
// place in a block always the same (load_at).
template <int NC>
struct Share<_Float16, NC> {
  u32x4 x[NC];
  // chunk of the head that x[j] is: 64 consecutive bytes of a position a load
  __device__ static __forceinline__ int chunk(int part, int j) { return part + 4 * j; }
  static __device__ __forceinline__ int64_t block_bytes(int64_t kv_dim) { return kv_dim * 32; }
  static __device__ __forceinline__ uint32_t place(int64_t kv_dim, int64_t head_off, int slot, int part) {
    return (uint32_t)((slot * kv_dim + head_off + part * 8) * 2);
  }
  __device__ __forceinline__ void load(const void *pool, const void *, int64_t at, uint32_t place) {
    const char *base = static_cast<const char *>(pool) + at;
#pragma unroll
    for (int j = 0; j < NC; ++j) x[j] = load_at<u32x4>(base, place + 64 * j);
  }
  __device__ __forceinline__ h8 get(int j) const { return __builtin_bit_cast(h8, x[j]); }
};

template <int NC>
struct Share<Q4, NC> {
  uint32_t x[NC];
  uint32_t s;  // (as 32 bits: a 16-bit value would be waited for to be moved)
  __device__ static __forceinline__ int chunk(int part, int j) { return part * NC + j; }
  static __device__ __forceinline__ int64_t block_bytes(int64_t kv_dim) { return kv_dim * 8; }
  // of the quants; the scale lies at an eighth of their group's place
  static __device__ __forceinline__ uint32_t place(int64_t, int64_t head_off, int slot, int part) {
    const uint32_t e = (uint32_t)head_off + part * NC * 8;
    return ((e >> 5) * 16 + slot) * 16 + ((e & 31) >> 3) * 4;
  }
  __device__ __forceinline__ void load(const void *pool, const void *scales, int64_t at, uint32_t place) {
    const char *base = static_cast<const char *>(pool) + at;
    s = load_at<uint16_t>(static_cast<const char *>(scales) + (at >> 3), (place >> 4) * 2);
    if constexpr (NC == 4) {
      const u32x4 w = load_at<u32x4>(base, place);
      x[0] = w.x;
      x[1] = w.y;
      x[2] = w.z;
      x[3] = w.w;
    } else {
      const u32x2 w = load_at<u32x2>(base, place);
      x[0] = w.x;
      x[1] = w.y;
    }
  }
  __device__ __forceinline__ h8 get(int j) const {
    const _Float16 d = __builtin_bit_cast(_Float16, (uint16_t)s);
    return q4x8_to_h8(x[j], h2{d, d});
  }
};

template <int NC>
struct Share<int8_t, NC> {
  u32x2 x[NC];
  uint32_t s;
  __device__ static __forceinline__ int chunk(int part, int j) { return part * NC + j; }
  static __device__ __forceinline__ int64_t block_bytes(int64_t kv_dim) { return kv_dim * 16; }
  static __device__ __forceinline__ uint32_t place(int64_t kv_dim, int64_t head_off, int slot, int part) {
    return (uint32_t)(slot * kv_dim + head_off + part * NC * 8);
  }
  static __device__ __forceinline__ uint32_t scale_place(int64_t head_off, int slot, int part) {
    return (uint32_t)((((head_off + part * NC * 8) >> 5) * 16 + slot) * 2);
  }
  __device__ __forceinline__ void load(const void *pool, const void *scales, int64_t at, uint32_t place,
                                       uint32_t scale_place) {
    const char *base = static_cast<const char *>(pool) + at;
    s = load_at<uint16_t>(static_cast<const char *>(scales) + (at >> 4), scale_place);
#pragma unroll
    for (int j = 0; j < NC; j += 2) {
      const u32x4 w = load_at<u32x4>(base, place + 8 * j);
      x[j] = u32x2{w.x, w.y};
      x[j + 1] = u32x2{w.z, w.w};
    }
  }
  __device__ __forceinline__ float scale() const { return (float)__builtin_bit_cast(_Float16, (uint16_t)s); }
  // chunk j times d (the scale times a power of two), as hi + lo parts
  __device__ __forceinline__ void get2(int j, float d, h8 &hi, h8 &lo) const {
    const h8 q = i8x8_to_h8(x[j]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      _Float16 a, b;
      split2((float)q[i] * d, a, b);
      hi[i] = a;
      lo[i] = b;
    }
  }
};

__device__ __forceinline__ h8 finite_or_zero(const h8 &x) {
  h8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = __builtin_fabsf((float)x[i]) <= 65504.f ? x[i] : (_Float16)0.f;
  return r;
}

// The same over a wave's 16 positions, of values that a position's lanes share.
__device__ __forceinline__ float positions_max(float x) {
  x = __builtin_fmaxf(x, dpp<0x141>(x));  // row_half_mirror
  x = __builtin_fmaxf(x, dpp<0x140>(x));  // row_mirror
  return rows_reduce<true>(x);
}

// e such that quants of up to 128 times the scale d stay below 2^15 times 2^e.
__device__ __forceinline__ int scale_exponent(float d) { return d > 0.f ? __builtin_amdgcn_frexp_expf(d) - 8 : 0; }

// K and V of a q8_0 tile enter the products times powers of two. K: one for the
// tile where every row sees all of it, else one for each position, which the
// scores are multiplied by. V: one for the tile. A row must not lose bits to a
// scale that it does not see, so V's power follows the largest scale that some
// row sees only while that stays within 2^12 of a scale that every row has to do
// with: the largest one that all of them see, or, where they share no position,
// the least. (2^12: such a row's V still has f32's bits, since hi + lo parts keep
// 22 bits down to 2^16 below the largest.) Else it follows that scale, and what
// then passes the top of f16 is added apart, for the rows that see it
// (kLeftOut). Positions that no row sees have no part in it. (Against one power
// for all 64 positions, whoever sees them: chunks of 2 x 1024 f32 rows 176 -> 171
// us, of bf16 rows 110 -> 126.)
struct TileRange {
  float k_top;               // largest scale of K
  float top, shared, least;  // V's (least: negative, as a maximum)
  __device__ __forceinline__ void add(const TileRange &o) {
    k_top = __builtin_fmaxf(k_top, o.k_top);
    top = __builtin_fmaxf(top, o.top);
    shared = __builtin_fmaxf(shared, o.shared);
    least = __builtin_fmaxf(least, o.least);
  }
  __device__ __forceinline__ int v_exponent() const {
    const float base = shared > 0.f ? shared : -least;
    return __builtin_amdgcn_readfirstlane(scale_exponent(top <= 4096.f * base ? top : 16.f * base));
  }
};
constexpr float kLeftOut = 511.f;  // scales (times the power of two) from here on could pass f16's largest number

// The least and largest of what the rows of a wave (or work-group) see. (No short
// circuits, as in RowView::sees.)
struct Bounds {
  int32_t first_min, first_max, from_min, from_max, sink_min, sink_max, end_min, end_max;
  __device__ __forceinline__ bool none(int32_t t, int32_t n) const {  // of positions [t, t + n)
    return (t >= end_max) | (t + n <= first_min) | ((t + n <= from_min) & (t >= sink_max));
  }
  __device__ __forceinline__ bool all(int32_t t, int32_t n) const {
    return (t >= first_max) & (t + n <= end_min) & ((t >= from_max) | (t + n <= sink_min));
  }
};

// A work-group takes 128 columns, which are (row, query head) pairs of one kv
// head: 128 / group rows; each of its four waves 32 of them. Tiles of 64
// positions go through LDS as f16 numbers, on 32x32x16 products (two chains of
// dependent ones for the scores, one per 32 positions): scores^T = K Q^T, weights
// in place, numerators^T += V^T W (a lane's scores are positions 8 (r / 4) + 4
// (lane / 32) + r % 4 of its column, which is the second product's operand layout
// when its 16 positions are taken as 4 (lane / 32) ... + 3 and 8 + 4 (lane / 32)
// ... + 3: no exchange). FULL
// (f32 rows, and any rows with a cap over kShortCap): Q and the weights as hi +
// lo pairs; else Q as it is (times a power of two), the weights rounded to f16, and
// V of q8_0 pools by its hi parts alone (one f16 rounding, as the weights': a third
// of the products less).
//
// A prompt of 4096 bf16 rows at 32 / 8 heads of 128 with capped scores takes 224
// us (137 GFLOP, 615 TFLOP/s): per tile and wave 32 products (~1000 cycles) stand
// beside 32 scores a lane of two exp2, one reciprocal and ~5 other vector
// instructions each, which the two work-groups of a CU only partly overlap (MFMA
// busy 27%, VALU 48%). Six chunks of up to 512 f32 rows behind 4-bit contexts at
// 28 / 4 heads: 188 us with their merge (149 GFLOP of hi and lo products, 790
// TFLOP/s; MFMA busy 44%, VALU 45%).
template <typename T, int HD, bool FULL>
__global__ void __launch_bounds__(64 * kChunkWaves, 2)
scored_chunk_kernel(ScoredArgs a, int64_t n_blocks, int64_t kv_dim, int rows_per_tile, int64_t min_rows,
                    int64_t n_slots) {
  constexpr int NC = HD / 32, NK = HD / 16;
  constexpr bool Q8 = std::is_same_v<T, int8_t>;
  constexpr int K_PLANES = Q8 ? 2 : 1, V_PLANES = Q8 && FULL ? 2 : 1;
  constexpr int K_PITCH = HD * 2 + 16;  // rows 4 banks apart: 16-byte reads of 16 rows without conflicts
  constexpr int V_PITCH = HD * 2 + 64;  // rows 16 banks apart, for the transposing reads
  constexpr int K_BYTES = kChunkTokens * K_PITCH, V_BYTES = kChunkTokens * V_PITCH;
  __shared__ __align__(16) char lds[K_PLANES * K_BYTES + V_PLANES * V_BYTES];
  __shared__ Bounds s_bounds[kChunkWaves];
  __shared__ TileRange s_range[kChunkWaves];                     // q8_0: scales of the next tile
  __shared__ __align__(16) float s_kpow[Q8 ? kChunkTokens : 4];  // q8_0: K of a position entered divided by this
  __shared__ uint64_t s_bad[kChunkWaves];  // lanes whose share of V is left out (positions 16 wave + lane / 4)
  char *const lds_k = lds, *const lds_v = lds + K_PLANES * K_BYTES;

  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int group = a.n_heads / a.n_kv_heads;
  const int kvh = (int)(blockIdx.x % (uint32_t)a.n_kv_heads);
  const uint32_t b = blockIdx.x / (uint32_t)a.n_kv_heads;
  // late slots first: under a causal mask a chunk's last rows see most; the
  // first split_slots slots, which come last, in `splits` work-groups each
  const uint32_t whole_slots = (uint32_t)(n_slots - a.split_slots);
  int split = 0, splits = 1;
  int64_t slot = n_slots - 1 - (int64_t)b;
  if (b >= whole_slots) {
    splits = a.splits;
    split = (int)((b - whole_slots) % (uint32_t)splits);
    slot = a.split_slots - 1 - (int64_t)((b - whole_slots) / (uint32_t)splits);
  }
  auto slot0 = [&](int64_t i) { return first_slot(a, i, rows_per_tile); };
  int64_t seq = 0;
  for (int64_t size = a.n; size > 1;) {  // the last sequence whose slots begin at or before this one
    const int64_t step = (size + 63) / 64, i = seq + lane * step;
    const bool before = i < seq + size && slot0(i) <= slot;
    const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before));
    if (n == 0) return;
    const int64_t skip = (n - 1) * step;
    seq += skip;
    size = size - skip < step ? size - skip : step;
  }
  seq = ((int64_t)__builtin_amdgcn_readfirstlane((int)(seq >> 32)) << 32) |
        (uint32_t)__builtin_amdgcn_readfirstlane((int)seq);
  const SeqRows rows = seq_rows(a, seq);
  const int64_t tile64 = slot - slot0(seq);
  if (rows.count <= min_rows || tile64 < 0 || tile64 * rows_per_tile >= rows.count) return;
  const int32_t r0 = (int32_t)tile64 * rows_per_tile;

  // the lane's column
  const int c128 = wave * 32 + col, rr = c128 / group;
  const bool live = rr < rows_per_tile && r0 + rr < rows.count;
  const int head = kvh * group + c128 - rr * group;
  const int64_t row = rows.row0 + r0 + (live ? rr : 0);
  RowView view = row_view(a, rows, seq, r0 + (live ? rr : 0));
  if (!live) view.end = 0;
  Bounds wb, gb;
  {
    auto reduce = [](int32_t x, bool most) {
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) {
        const int32_t y = __shfl_xor(x, off, 64);
        x = most ? max(x, y) : min(x, y);
      }
      return __builtin_amdgcn_readfirstlane(x);
    };
    const int32_t lo = INT32_MIN, hi = INT32_MAX;
    // rows that see nothing bound nothing
    const bool any = live && view.end > view.first;
    wb.first_min = reduce(any ? view.first : hi, false);
    wb.first_max = reduce(any ? view.first : lo, true);
    wb.from_min = reduce(any ? view.from : hi, false);
    wb.from_max = reduce(any ? view.from : lo, true);
    wb.sink_min = reduce(any ? view.sink_end : hi, false);
    wb.sink_max = reduce(any ? view.sink_end : lo, true);
    wb.end_min = reduce(any ? view.end : live ? lo : hi, false);  // (but they keep tiles from being whole)
    wb.end_max = reduce(any ? view.end : lo, true);
    if (lane == 0) s_bounds[wave] = wb;
    __syncthreads();
    gb = s_bounds[0];
#pragma unroll
    for (int w = 1; w < kChunkWaves; ++w) {
      const Bounds o = s_bounds[w];
      gb.first_min = min(gb.first_min, o.first_min);
      gb.first_max = max(gb.first_max, o.first_max);
      gb.from_min = min(gb.from_min, o.from_min);
      gb.from_max = max(gb.from_max, o.from_max);
      gb.sink_min = min(gb.sink_min, o.sink_min);
      gb.sink_max = max(gb.sink_max, o.sink_max);
      gb.end_min = min(gb.end_min, o.end_min);
      gb.end_max = max(gb.end_max, o.end_max);
    }
    // (the same in every lane: scalar registers)
    int32_t *const g = reinterpret_cast<int32_t *>(&gb);
#pragma unroll
    for (int i = 0; i < (int)(sizeof gb / 4); ++i) g[i] = __builtin_amdgcn_readfirstlane(g[i]);
  }
  StepRange<kChunkTokens> range{0, 0, 0, 0, 0, 0};
  if (gb.end_max > 0) {
    const RowView all{0, gb.first_min, gb.sink_max, gb.from_min, gb.end_max};
    range = step_range<kChunkTokens>(all);
  }
  const int per_part = (range.n + splits - 1) / splits;
  const int n_parts = per_part > 0 ? (range.n + per_part - 1) / per_part : 1;
  if (split >= n_parts) return;
  const int s_begin = split * per_part, s_end = min(range.n, s_begin + per_part);

  // Table entries outside the pool are reported where some row sees a position of
  // their block (between the rows' ranges may lie blocks that none of them sees):
  // once, in front of the loop, which only reads block 0 in their place. The first
  // come with Q.
  const int32_t *tab = table_of(a.tables, a.table_stride, a.rows, a.table_rows, seq);
  auto entry_of = [&](int32_t i) {  // i counts blocks from step s_begin on
    if (i >= 4 * (s_end - s_begin)) return 0;
    const int32_t t = range.start(s_begin + i / 4) + 16 * (i % 4);
    return t < range.end(s_begin + i / 4) ? tab[t >> 4] : 0;
  };
  int32_t entry = entry_of(tid);

  // Q columns (as scored_rows_kernel's)
  h8 qh[NK], ql[FULL ? NK : 1];
  int q_exp;  // Q entered times 2^q_exp
  {
    float x[NK][8], amax = 0.f;
    const int64_t at = (row * a.n_heads + head) * (int64_t)HD;
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      load_row8(a, at + 16 * j + 8 * half, live, x[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) amax = __builtin_fmaxf(amax, __builtin_fabsf(x[j][i]));
    }
    amax = halves_reduce<true>(amax);
    // (at most 100: a smaller row's scores are nothing beside their rounding)
    q_exp = amax > 0.f && amax < INFINITY ? min(10 - __builtin_amdgcn_frexp_expf(amax), 100) : 0;
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        _Float16 hi, lo;
        split2(__builtin_amdgcn_ldexpf(x[j][i], q_exp), hi, lo);
        qh[j][i] = hi;
        if constexpr (FULL) ql[j][i] = lo;
      }
  }
  const bool cap = a.softcap > 0.f;
  const float factor = cap ? a.scale / a.softcap : a.scale * kLog2e, in_scale = score_factor(factor, -q_exp);
  const float cap_scale = a.softcap * kLog2e;
  const float slope = a.slopes && live ? a.slopes[head] * kLog2e : 0.f;
  // scores are an affine function of the products (or of the capped rows' c),
  // which falls with it where its factor is negative
  const bool affine = !a.slopes && !(FULL && cap) && a.scale != 0.f;
  const bool falling = affine && (cap || a.scale < 0.f);

  f32x16 o[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) o[i] = f32x16{};
  float ref = -INFINITY, sum = 0.f;
  int v_exp = -1000;  // q8_0: V enters the products times 2^-v_exp

  // staging
  const int64_t head_off = (int64_t)kvh * HD;
  const int tok = tid >> 2, part = tid & 3;
  for (int32_t i = tid; i < 4 * (s_end - s_begin); entry = entry_of(i += 64 * kChunkWaves)) {
    if ((uint32_t)entry < (uint32_t)n_blocks) continue;
    const int32_t t = range.start(s_begin + i / 4) + 16 * (i % 4);
    bool needed = false;
    for (int32_t r = 0; r < rows_per_tile && r0 + r < rows.count; ++r)
      needed |= row_view(a, rows, seq, r0 + r).sees_of_block(t);
    if (needed) report_fault(a.status, kFaultTable, seq);
  }
  // The wave's block of a tile, read a tile ahead of its cells (past the end:
  // block 0, read and masked).
  auto block_of = [&](int s) {
    const int32_t t = range.start(s) + 16 * wave;
    int32_t e = s < s_end && t < range.end(s) ? scalar_read(tab, t >> 4) : 0;
    return (uint32_t)e < (uint32_t)n_blocks ? e : 0;
  };
  const int64_t block_bytes = Share<T, NC>::block_bytes(kv_dim);
  const uint32_t place = Share<T, NC>::place(kv_dim, head_off, tok & 15, part);
  uint32_t scale_place = 0;
  if constexpr (Q8) scale_place = Share<T, NC>::scale_place(head_off, tok & 15, part);
  Share<T, NC> ks, vs;
  auto load = [&](int32_t block) {
    const int64_t at = (int64_t)(uint32_t)block * block_bytes;
    if constexpr (Q8) {
      ks.load(a.k_layer, a.k_scale, at, place, scale_place);
      vs.load(a.v_layer, a.v_scale, at, place, scale_place);
    } else {
      ks.load(a.k_layer, a.k_scale, at, place);
      vs.load(a.v_layer, a.v_scale, at, place);
    }
  };
  int32_t next = 0;
  if (s_begin < s_end) {
    load(block_of(s_begin));
    next = block_of(s_begin + 1);
  }

  for (int s = s_begin; s < s_end; ++s) {
    const int32_t t0 = range.start(s), t_end = range.end(s);
    // a row of the work-group does not see the whole tile
    const bool partial = t0 + kChunkTokens > t_end || !gb.all(t0, kChunkTokens);
    bool inside = false;  // q8_0: some row sees the thread's position
    int k_exp = 0;
    if constexpr (Q8) {
      const float d = __builtin_fminf(position_max(vs.scale()), 65504.f);
      TileRange r;
      r.k_top = positions_max(__builtin_fminf(position_max(ks.scale()), 65504.f));
      if (!partial) {
        inside = true;
        r.top = r.shared = positions_max(d);
        r.least = -INFINITY;
      } else {
        inside = (t0 + tok < t_end) & !gb.none(t0 + tok, 1);
        const bool shared = inside & gb.all(t0 + tok, 1);
        r.top = positions_max(inside ? d : 0.f);
        r.shared = positions_max(shared ? d : 0.f);
        r.least = positions_max((inside & !shared & (d > 0.f)) ? -d : -INFINITY);
      }
      if (lane == 0) s_range[wave] = r;
    }
    lds_barrier();  // the last tile has been read
    if constexpr (Q8) {
      TileRange r = s_range[0];
#pragma unroll
      for (int w = 1; w < kChunkWaves; ++w) r.add(s_range[w]);
      if (!partial) k_exp = __builtin_amdgcn_readfirstlane(scale_exponent(r.k_top));
      const int e = r.v_exponent();
      // (the numerators are f32 numbers: their power of two may fall as well)
      if (__builtin_amdgcn_readfirstlane(r.top > 0.f) && (e > v_exp || e < v_exp - 2)) {
        if (v_exp > -1000) {
          const float f = __builtin_amdgcn_ldexpf(1.f, v_exp - e);
#pragma unroll
          for (int i = 0; i < NC; ++i) o[i] *= f;
        }
        v_exp = e;
      }
    }
    // Infinities and NaN in V (and q8_0 elements beyond the tile's power of two)
    // may reach only the rows that see them: looked for in partial tiles.
    bool bad = false;
    {
      float dk = 0.f, dv = 0.f;
      if constexpr (Q8) {
        int e = k_exp;
        if (partial) {
          e = scale_exponent(__builtin_fminf(position_max(ks.scale()), 65504.f));
          if (part == 0) s_kpow[tok] = __builtin_amdgcn_ldexpf(1.f, e);
        }
        dk = __builtin_amdgcn_ldexpf(ks.scale(), -e);
        dv = __builtin_amdgcn_ldexpf(vs.scale(), -(v_exp > -1000 ? v_exp : 0));
      }
      const bool left_out = Q8 & partial & !(dv < kLeftOut);
      bad = left_out & inside;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int c = Share<T, NC>::chunk(part, j) * 16;
        if constexpr (Q8) {
          h8 hi, lo;
          ks.get2(j, dk, hi, lo);
          *reinterpret_cast<h8 *>(lds_k + tok * K_PITCH + c) = hi;
          *reinterpret_cast<h8 *>(lds_k + K_BYTES + tok * K_PITCH + c) = lo;
          vs.get2(j, dv, hi, lo);
          if (left_out) {
            hi = h8{};
            lo = h8{};
          }
          *reinterpret_cast<h8 *>(lds_v + tok * V_PITCH + c) = hi;
          if constexpr (V_PLANES == 2) *reinterpret_cast<h8 *>(lds_v + V_BYTES + tok * V_PITCH + c) = lo;
        } else {
          *reinterpret_cast<h8 *>(lds_k + tok * K_PITCH + c) = ks.get(j);
          *reinterpret_cast<h8 *>(lds_v + tok * V_PITCH + c) = vs.get(j);
        }
      }
      if constexpr (std::is_same_v<T, _Float16>) {
        if (partial) {
#pragma unroll
          for (int j = 0; j < NC; ++j) bad = bad || not_finite(vs.get(j));
        }
        if (bad) {  // once more, without them
#pragma unroll
          for (int j = 0; j < NC; ++j)
            *reinterpret_cast<h8 *>(lds_v + tok * V_PITCH + Share<T, NC>::chunk(part, j) * 16) = finite_or_zero(vs.get(j));
        }
      }
    }
    if constexpr (!std::is_same_v<T, Q4>) {
      const uint64_t lanes = __builtin_amdgcn_ballot_w64(bad);
      if (lane == 0) s_bad[wave] = lanes;
    }
    if (s + 1 < s_end) {
      load(next);
      next = block_of(s + 2);
    }
    lds_barrier();
    if (wb.none(t0, kChunkTokens)) continue;
    // scores of positions t0 + 32 u + 8 (i / 4) + 4 half + i % 4
    f32x16 c[2] = {};
    const char *kp = lds_k + col * K_PITCH + 16 * half;
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int j = 0; j < NK; ++j) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const h8 x = *reinterpret_cast<const h8 *>(kp + 32 * u * K_PITCH + 32 * j);
        c[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qh[j], c[u], 0, 0, 0);
        if constexpr (FULL) c[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, ql[j], c[u], 0, 0, 0);
        if constexpr (Q8) {
          const h8 y = *reinterpret_cast<const h8 *>(kp + K_BYTES + 32 * u * K_PITCH + 32 * j);
          c[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, qh[j], c[u], 0, 0, 0);
        }
      }
    }
    __builtin_amdgcn_s_setprio(0);
    if (Q8 && partial) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const f32x4 f = *reinterpret_cast<const f32x4 *>(s_kpow + 8 * i + 4 * half);
#pragma unroll
        for (int k = 0; k < 4; ++k) c[i >> 2][4 * (i & 3) + k] *= f[k];
      }
    }
    const int32_t tl = t0 + 4 * half;
    // Scores in the log2 domain as m c + m0: the multiplication is left to the
    // fused one before exp2. Capped rows of 16 bits take c = 1 / (exp(2 x) + 1),
    // since cap tanh(x) = cap - 2 cap c: five instructions a score.
    float m = Q8 ? score_factor(factor, k_exp - q_exp) : in_scale, m0 = 0.f;
    if (affine) {
      if (cap) {
        const float to_e = m * (2.f * kLog2e);
#pragma unroll
        for (int i = 0; i < 32; ++i)
          c[i >> 4][i & 15] = __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(c[i >> 4][i & 15] * to_e) + 1.f);
        m = -2.f * cap_scale;
        m0 = cap_scale;
      }
    } else {
      float to_x = m;  // opaque: the products would be taken before the branch, for both sides
      asm("" : "+v"(to_x));
      if (cap) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float x = c[i >> 4][i & 15] * to_x;
          if constexpr (FULL) c[i >> 4][i & 15] = tanh_f32(x) * cap_scale;
          else c[i >> 4][i & 15] = tanh_f16(x) * cap_scale;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) c[i >> 4][i & 15] *= to_x;
      }
      const float d0 = (float)(view.pos - tl);
#pragma unroll
      for (int i = 0; i < 32; ++i)
        c[i >> 4][i & 15] =
            __builtin_fmaf(-slope, __builtin_fabsf(d0 - (float)(8 * (i / 4) + i % 4)), c[i >> 4][i & 15]);
      m = 1.f;
    }
    if (t0 + kChunkTokens > t_end || !wb.all(t0, kChunkTokens)) {
      const float none = falling ? INFINITY : -INFINITY;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const int32_t t = tl + 8 * (i / 4) + i % 4;
        c[i >> 4][i & 15] = (view.sees(t) & (t < t_end)) ? c[i >> 4][i & 15] : none;
      }
    }
    float top = c[0][0];
    if (falling) {
#pragma unroll
      for (int i = 1; i < 32; ++i) top = __builtin_fminf(top, c[i >> 4][i & 15]);
    } else {
#pragma unroll
      for (int i = 1; i < 32; ++i) top = __builtin_fmaxf(top, c[i >> 4][i & 15]);
    }
    top = __builtin_fmaf(top, m, m0);
    if (__builtin_amdgcn_ballot_w64(top > ref + kSlack)) {
      const float nr = __builtin_fmaxf(ref, halves_reduce<true>(top));
      const float f = nr == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref - nr);
      sum *= f;
#pragma unroll
      for (int i = 0; i < NC; ++i) o[i] *= f;
      ref = nr;
    }
    const float base = m0 - ((ref == -INFINITY ? 0.f : ref) - kLift);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      c[i >> 4][i & 15] = __builtin_amdgcn_exp2f(__builtin_fmaf(c[i >> 4][i & 15], m, base));
      if constexpr (FULL) sum += c[i >> 4][i & 15];
    }
#pragma unroll
    for (int p = 0; p < kChunkTokens / 16; ++p) {
      h8 wh, wl;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // (an exponential is no product that a conversion could fold: no copy of it
        // as split2 makes)
        const float w = c[p >> 1][8 * (p & 1) + i];
        wh[i] = (_Float16)w;
        if constexpr (FULL) wl[i] = (_Float16)(w - (float)wh[i]);
      }
      if constexpr (!FULL) {  // the weights as they enter the product, two an instruction
        const h2 one = {(_Float16)1.f, (_Float16)1.f};
#pragma unroll
        for (int i = 0; i < 8; i += 2) sum = __builtin_amdgcn_fdot2(h2{wh[i], wh[i + 1]}, one, sum, false);
      }
      const char *vp = lds_v + (16 * p + 4 * half + ((lane & 15) >> 2)) * V_PITCH +
                       (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const h8 x = read_tr2(vp + 64 * i, 8 * V_PITCH);
        o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, wh, o[i], 0, 0, 0);
        if constexpr (FULL) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, wl, o[i], 0, 0, 0);
        if constexpr (V_PLANES == 2) {
          const h8 y = read_tr2(vp + V_BYTES + 64 * i, 8 * V_PITCH);
          o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, wh, o[i], 0, 0, 0);
        }
      }
    }
    if constexpr (!std::is_same_v<T, Q4>) {
      if (__builtin_amdgcn_readfirstlane((s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3]) != 0)) {
        // V elements that are infinite or NaN (q8_0: too large for the tile's
        // power of two) entered as zeros: the rows that see their positions get
        // them here, the others do not
        for (int j = 0; j < kChunkTokens; ++j) {
          const int32_t t = t0 + j;
          if (t >= t_end) break;
          if ((s_bad[j >> 4] >> (4 * (j & 15)) & 15) == 0) continue;
          int32_t e = scalar_read(tab, t >> 4);
          if (e < 0 || e >= n_blocks) e = 0;
          const int64_t cell = (int64_t)e * 16 + (t & 15);
          float w = 0.f;
#pragma unroll
          for (int i = 0; i < 32; ++i)  // position j is score i of lane (column, j / 4 % 2)
            if (i == (j >> 3) * 4 + (j & 3)) w = __shfl(c[i >> 4][i & 15], col + 32 * ((j >> 2) & 1), 64);
          if (!view.sees(t)) continue;
          if constexpr (Q8) {
#pragma unroll
            for (int i = 0; i < NC; ++i) {  // a tile of the numerators is a group
              const _Float16 scale = static_cast<const _Float16 *>(
                  a.v_scale)[scale_index((int32_t)cell, (int)(head_off >> 5) + i, (int)(kv_dim >> 5))];
              const float d = __builtin_amdgcn_ldexpf((float)scale, -(v_exp > -1000 ? v_exp : 0));
              if (d < kLeftOut) continue;
              const char *const row = static_cast<const char *>(a.v_layer) + cell * kv_dim + head_off + 32 * i;
#pragma unroll
              for (int k = 0; k < 16; k += 4) {
                const uint32_t u = load_at<uint32_t>(row + 2 * k, 4 * half);
#pragma unroll
                for (int b = 0; b < 4; ++b) o[i][k + b] += w * ((float)((int)(u >> (8 * b) & 255u) - 128) * d);
              }
            }
          } else {
            for (int k = 0; k < NC * 16; ++k) {
              const int64_t d = head_off + 32 * (k / 16) + 8 * (k % 16 / 4) + 4 * half + k % 4;
              const float x = cell_value<T>(a.v_layer, a.v_scale, cell, kv_dim, d);
              if (__builtin_fabsf(x) < INFINITY) continue;
#pragma unroll
              for (int i = 0; i < NC * 16; ++i)
                if (i == k) o[i / 16][i % 16] += w * x;
            }
          }
        }
      }
    }
  }

  sum = halves_reduce<false>(sum);
  if constexpr (Q8) {
    const float f = __builtin_amdgcn_ldexpf(1.f, v_exp > -1000 ? v_exp : 0);
#pragma unroll
    for (int i = 0; i < NC; ++i) o[i] *= f;
  }
  if (live) {
    const int64_t rh = row * a.n_heads + head;
    if (n_parts == 1) {
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int k = 0; k < 16; k += 4)
          store_row4(a, rh * HD + 32 * i + 2 * k + 4 * half,
                     f32x4{o[i][k] * inv, o[i][k + 1] * inv, o[i][k + 2] * inv, o[i][k + 3] * inv});
    } else {
      const int64_t at = rh * a.splits + split;
      float *dst = a.chunk_o + at * HD + 4 * half;
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int k = 0; k < 16; k += 4)
          *reinterpret_cast<f32x4 *>(dst + 32 * i + 2 * k) = f32x4{o[i][k], o[i][k + 1], o[i][k + 2], o[i][k + 3]};
      if (half == 0) {
        a.chunk_ml[2 * at] = ref;
        a.chunk_ml[2 * at + 1] = sum;
      }
    }
    if (splits > 1 && split == 0 && half == 0 && kvh == 0 && c128 - rr * group == 0)
      a.chunk_n[row] = n_parts;
  }
}

template <typename T, int HD>
hipError_t launch_chunk_t(const PoolGeom &g, const ScoredArgs &a, int64_t min_rows, hipStream_t s) {
  const int rows_per_tile = chunk_rows(a);
  const int64_t n_slots = chunk_slots(a);
  const int64_t wgs = (n_slots - a.split_slots + (int64_t)a.split_slots * a.splits) * a.n_kv_heads;
  if (wgs * 64 * kChunkWaves >= (int64_t{1} << 32)) return hipErrorInvalidValue;
  // (a second tanh in the kernel of 16-bit rows took registers that it does not
  // have: 12 to 22 spilled at head_dim 128)
  const bool full = a.row_type == LTKV_ROWS_F32 || a.softcap > kShortCap;
  const auto kernel = full ? scored_chunk_kernel<T, HD, true> : scored_chunk_kernel<T, HD, false>;
  kernel<<<(unsigned)wgs, 64 * kChunkWaves, 0, s>>>(a, g.n_blocks, g.kv_dim, rows_per_tile, min_rows, n_slots);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_chunk_hd(const PoolGeom &g, const ScoredArgs &a, int64_t min_rows, hipStream_t s) {
  return a.head_dim == 64 ? launch_chunk_t<T, 64>(g, a, min_rows, s) : launch_chunk_t<T, 128>(g, a, min_rows, s);
}

}  // namespace

hipError_t launch_scored_chunks(const PoolGeom &g, const ScoredArgs &a, int64_t min_rows, hipStream_t s) {
  if (g.elem == kElemQ4) return launch_chunk_hd<Q4>(g, a, min_rows, s);
  if (g.elem == 1) return launch_chunk_hd<int8_t>(g, a, min_rows, s);
  return launch_chunk_hd<_Float16>(g, a, min_rows, s);
}

}  // namespace ltkv
