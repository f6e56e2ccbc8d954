// gfx950 (MI355X, CDNA4) kernel of scored attention for single rows (decodes),
// and of decode attention over q4_0 pools, on the matrix cores.

#include "ltkv_scored.h"

namespace ltkv {
namespace {

constexpr int kRowsWaves = 4;
constexpr int kTopExp = 15;  // q8_0 weights times V scales stay below 2^kTopExp

// K or V of 16 positions as a wave loads them: lane (t, quad) = (lane & 15,
// lane >> 4) holds NC chunks of 8 elements of position t. Chunk j of a lane is
// head elements chunk_at(quad, j) ... + 7: a contiguous quarter of the head
// where that makes loads of 16 bytes (SPAN), else 32 j + 8 quad.
template <typename T, int NC, bool SPAN>
struct Cells;

template <int NC, bool SPAN>
struct Cells<_Float16, NC, SPAN> {
  u32x4 x[NC];
  __device__ __forceinline__ void load(const ScoredArgs &a, const void *pool, const void *, int64_t kv_dim, int32_t blk,
                                       int t, int quad, int64_t head_off) {
    const _Float16 *row = static_cast<const _Float16 *>(pool) + ((int64_t)blk * 16 + t) * kv_dim + head_off;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int c = SPAN ? quad * NC + j : 4 * j + quad;
      if (SPAN || c * 8 < a.head_dim) x[j] = *reinterpret_cast<const u32x4 *>(row + c * 8);
      else x[j] = u32x4{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ h8 get(int j) const { return __builtin_bit_cast(h8, x[j]); }
};

template <int NC, bool SPAN>
struct Cells<Q4, NC, SPAN> {
  static constexpr int NS = SPAN ? (NC + 3) / 4 : NC;  // scales a lane needs
  uint32_t x[NC];
  uint16_t s[NS];
  __device__ __forceinline__ void load(const ScoredArgs &a, const void *pool, const void *scales, int64_t kv_dim,
                                       int32_t blk, int t, int quad, int64_t head_off) {
    const int64_t tile0 = (int64_t)blk * (kv_dim >> 5);
    if constexpr (SPAN) {
      // the quarter lies in one group, or is whole groups (16 bytes each)
      const int e = (int)head_off + quad * NC * 8;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int64_t at = (tile0 + (e >> 5) + i) * 16 + t;
        s[i] = static_cast<const uint16_t *>(scales)[at];
        const uint32_t *p = static_cast<const uint32_t *>(pool) + at * 4 + ((e & 31) >> 3);
        constexpr int W = NC < 4 ? NC : 4;
        if constexpr (W == 4) {
          const u32x4 w = *reinterpret_cast<const u32x4 *>(p);
          x[4 * i] = w.x;
          x[4 * i + 1] = w.y;
          x[4 * i + 2] = w.z;
          x[4 * i + 3] = w.w;
        } else {
          const u32x2 w = *reinterpret_cast<const u32x2 *>(p);
          x[0] = w.x;
          x[1] = w.y;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int c = 4 * j + quad;
        x[j] = 0;
        s[j] = 0;
        if (c * 8 < a.head_dim) {
          const int e = (int)head_off + c * 8;
          const int64_t at = (tile0 + (e >> 5)) * 16 + t;
          x[j] = static_cast<const uint32_t *>(pool)[at * 4 + ((e & 31) >> 3)];
          s[j] = static_cast<const uint16_t *>(scales)[at];
        }
      }
    }
  }
  __device__ __forceinline__ h8 get(int j) const {
    const _Float16 d = __builtin_bit_cast(_Float16, s[SPAN ? j / 4 : j]);
    return q4x8_to_h8(x[j], h2{d, d});
  }
};

// q8_0 elements enter the products as their quants; the scales multiply the
// scores of a 32-element group and the weights of its numerators (SPAN false:
// chunk j of every lane is group j). s[j]: the scales of the lane's four score
// positions 4 quad ... + 3.
template <int NC, bool SPAN>
struct Cells<int8_t, NC, SPAN> {
  u32x2 x[NC];
  u32x2 s[NC];
  __device__ __forceinline__ void load(const ScoredArgs &, const void *pool, const void *scales, int64_t kv_dim,
                                       int32_t blk, int t, int quad, int64_t head_off) {
    static_assert(!SPAN, "a product must stay inside a group");
    const uint8_t *row = static_cast<const uint8_t *>(pool) + ((int64_t)blk * 16 + t) * kv_dim + head_off;
    const uint16_t *sc =
        static_cast<const uint16_t *>(scales) + ((int64_t)blk * (kv_dim >> 5) + (head_off >> 5)) * 16 + quad * 4;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      x[j] = *reinterpret_cast<const u32x2 *>(row + 32 * j + 8 * quad);
      s[j] = *reinterpret_cast<const u32x2 *>(sc + 16 * j);
    }
  }
  __device__ __forceinline__ h8 get(int j) const { return i8x8_to_h8(x[j]); }
  __device__ __forceinline__ h4 scale(int j) const { return __builtin_bit_cast(h4, s[j]); }
};

// A work-group takes one part of one row's visible positions for one kv head:
// its four waves take 32-position steps in turn. Per step and wave, on 16x16x32
// products: scores^T = K Q^T (16 positions x the group's query heads as
// columns, twice), weights from the scores in place, numerators^T += V^T W: the
// score tiles' lane layout (4 quad + r, column) is the operand layout of the
// second product when its 32 positions are taken as (tile 0: 4 quad ... + 3,
// tile 1: 4 quad ... + 3), so weights move between no lanes. V is transposed on
// its way through LDS (ds_read_b64_tr_b16). Q and the weights enter as f16
// hi + lo pairs: f32 accuracy for twice the matrix-core work, which is idle
// here otherwise.
template <typename T, int HDP, bool SPAN, bool MODS>
__global__ void __launch_bounds__(64 * kRowsWaves)
scored_rows_kernel(ScoredArgs a, int64_t n_blocks, int64_t kv_dim, int head_tiles, int64_t most_rows) {
  constexpr int NC = HDP / 32;     // chunks of 8 elements a lane, products per score tile
  constexpr int ND = HDP / 16;     // 16-element tiles of the numerators
  constexpr int PITCH = HDP * 2 + 32;  // bytes of a V row in LDS: rows of a read start 8 banks apart
  constexpr bool Q8 = std::is_same_v<T, int8_t>;
  constexpr int RED = HDP + 4;  // floats of a (wave, column) in the final fold: numerators, reference, sum
  constexpr int V_BYTES = 32 * PITCH, RED_BYTES = 16 * RED * 4;
  __shared__ __align__(16) char lds[kRowsWaves * (V_BYTES > RED_BYTES ? V_BYTES : RED_BYTES)];

  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int group = a.n_heads / a.n_kv_heads;
  uint32_t b = blockIdx.x;
  const int head_tile = (int)(b % (uint32_t)head_tiles);
  b /= (uint32_t)head_tiles;
  const int kvh = (int)(b % (uint32_t)a.n_kv_heads);
  b /= (uint32_t)a.n_kv_heads;
  const int part = (int)(b % (uint32_t)a.max_parts);
  const int64_t item = b / (uint32_t)a.max_parts;
  // an item is a sequence, whose rows are taken one after the other, or a row
  const int64_t seq = a.row_items ? seq_of_row(a, item) : item;
  const SeqRows rows = seq_rows(a, seq);
  if (rows.count > most_rows) return;
  if (a.row_items && (item < rows.row0 || item >= rows.row0 + rows.count)) return;
  const int r_begin = a.row_items ? (int)(item - rows.row0) : 0, r_end = a.row_items ? r_begin + 1 : rows.count;
  const int cols = min(16, group - head_tile * 16);
  const int head0 = kvh * group + head_tile * 16;
  const bool live = col < cols;
  const int64_t head_off = (int64_t)kvh * a.head_dim;
  const int32_t *tab = table_of(a.tables, a.table_stride, a.rows, a.table_rows, seq);
  if (a.rows && part == 0 && wave == 0 && rows.len > 0) {
    const int32_t r = scalar_read(a.rows, seq);
    if (r < 0 || r >= a.table_rows) report_fault(a.status, kFaultTable, seq);
  }
  char *const my = lds + wave * V_BYTES;

  for (int r = r_begin; r < r_end; ++r) {
    const RowView view = row_view(a, rows, seq, r);
    const StepRange<32> range = step_range<32>(view);
    int per_part = scored_part_tokens((int64_t)range.n * 32, a.part_tokens) >> 5;
    // no memory for the parts of rows past the expected most: one part
    const bool parted = a.row_items || r < a.max_rows;
    if (!parted) per_part = range.n;
    else if ((int64_t)per_part * a.max_parts < range.n) per_part = (range.n + a.max_parts - 1) / a.max_parts;
    const int n_parts = range.n > per_part ? (range.n + per_part - 1) / per_part : 1;
    if (part >= n_parts) continue;
    const int s_end = min(range.n, (part + 1) * per_part);
    const int s_first = part * per_part + wave;
    const int64_t row = rows.row0 + r, slot = a.row_items ? row : seq * a.max_rows + r;

    // block ids of the wave's next 32 steps, two a step, one a lane
    int entry = 0;
    auto fill = [&](int s0) {
      const int s = s0 + kRowsWaves * (lane >> 1);
      const int32_t t = range.start(s) + 16 * (lane & 1);
      const bool valid = s < s_end && t < range.end(s);
      entry = valid ? tab[t >> 4] : 0;
      const bool bad = entry < 0 || entry >= n_blocks;
      if (bad) entry = 0;
      if (__builtin_amdgcn_ballot_w64(bad)) report_fault(a.status, kFaultTable, seq);
    };

    // Q columns, scaled by a power of two so that the head's largest element
    // lies in [2^9, 2^10): any magnitude enters f16 with 22 bits
    h8 qh[NC], ql[NC];
    float qscale;
    {
      float x[NC][8], amax = 0.f;
      const int64_t at = (row * a.n_heads + head0 + col) * (int64_t)a.head_dim;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int e = (SPAN ? quad * NC + j : 4 * j + quad) * 8;
        load_row8(a, at + e, live && (SPAN || e < a.head_dim), x[j]);
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = __builtin_fmaxf(amax, __builtin_fabsf(x[j][i]));
      }
      amax = rows_reduce<true>(amax);
      const int up = amax > 0.f && amax < INFINITY ? 10 - __builtin_amdgcn_frexp_expf(amax) : 0;
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          _Float16 hi, lo;
          split2(__builtin_amdgcn_ldexpf(x[j][i], up), hi, lo);
          qh[j][i] = hi;
          ql[j][i] = lo;
        }
      qscale = __builtin_amdgcn_ldexpf(a.scale, -up);
    }
    const bool cap = MODS && a.softcap > 0.f;
    const float in_scale = cap ? qscale / a.softcap : qscale * kLog2e;
    const float cap_scale = a.softcap * kLog2e;
    const float slope = MODS && a.slopes && live ? a.slopes[head0 + col] * kLog2e : 0.f;

    f32x4 o[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float ref = -INFINITY, sum = 0.f;
    float lift = Q8 ? 0.f : kLift, scale_top = 0.f;  // q8_0: no scale has exceeded scale_top

    Cells<T, NC, SPAN> k[2], v[2];
    auto load = [&](Cells<T, NC, SPAN> (&c)[2], const void *pool, const void *scales, int i) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        c[u].load(a, pool, scales, kv_dim, __builtin_amdgcn_readlane(entry, 2 * i + u), col, quad, head_off);
    };
    int held = 0;  // step of `entry`'s window
    if (s_first < s_end) {
      fill(s_first);
      load(k, a.k_layer, a.k_scale, 0);
      load(v, a.v_layer, a.v_scale, 0);
    }
    for (int s = s_first; s < s_end; s += kRowsWaves) {
      const int32_t t0 = range.start(s), t_end = range.end(s);
      const bool more = s + kRowsWaves < s_end;
      ++held;
      if (more && held == 32) {
        fill(s + kRowsWaves);
        held = 0;
      }
      // scores
      f32x4 c[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        c[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (Q8) {
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            const h8 x = k[u].get(j);
            f32x4 g = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qh[j], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            g = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ql[j], g, 0, 0, 0);
            const h4 d = k[u].scale(j);
#pragma unroll
            for (int i = 0; i < 4; ++i) c[u][i] = __builtin_fmaf((float)d[i], g[i], c[u][i]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            const h8 x = k[u].get(j);
            c[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qh[j], c[u], 0, 0, 0);
            c[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, ql[j], c[u], 0, 0, 0);
          }
        }
      }
      if (more) load(k, a.k_layer, a.k_scale, held);

      const bool whole = t0 + 32 <= t_end && t0 >= view.first && (t0 >= view.from || t0 + 32 <= view.sink_end);
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int32_t t = t0 + 16 * u + 4 * quad + i;
          float x = c[u][i] * in_scale;
          if constexpr (MODS) {
            if (cap) x = tanh_f32(x) * cap_scale;
            x = __builtin_fmaf(-slope, (float)abs(view.pos - t), x);
          }
          c[u][i] = x;
        }
      if (!whole)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int32_t t = t0 + 16 * u + 4 * quad + i;
            if (!(view.sees(t) && t < t_end)) c[u][i] = -INFINITY;
          }
      float top = __builtin_fmaxf(__builtin_fmaxf(c[0][0], c[0][1]), __builtin_fmaxf(c[0][2], c[0][3]));
      top = __builtin_fmaxf(
          top, __builtin_fmaxf(__builtin_fmaxf(c[1][0], c[1][1]), __builtin_fmaxf(c[1][2], c[1][3])));
      if (__builtin_amdgcn_ballot_w64(top > ref + kSlack)) {
        const float next = __builtin_fmaxf(ref, rows_reduce<true>(top));
        const float f = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref - next);
        sum *= f;
#pragma unroll
        for (int i = 0; i < ND; ++i) o[i] *= f;
        ref = next;
      }
      h4 dv[2][Q8 ? NC : 1];
      if constexpr (Q8) {
        h4 most = {};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            dv[u][j] = v[u].scale(j);
            if (!whole)  // a scale of an unseen position may be infinite
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int32_t t = t0 + 16 * u + 4 * quad + i;
                if (!(view.sees(t) && t < t_end)) dv[u][j][i] = (_Float16)0.f;
              }
            most = __builtin_elementwise_max(most, dv[u][j]);
          }
        const float top_d = __builtin_fmaxf(__builtin_fmaxf((float)most[0], (float)most[1]),
                                            __builtin_fmaxf((float)most[2], (float)most[3]));
        if (__builtin_amdgcn_ballot_w64(top_d > scale_top)) {
          const float d = __builtin_fminf(rows_reduce<true>(top_d), 65504.f);  // the same in every column
          const int ex = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_frexp_expf(d));
          const float next = (float)(kTopExp - ex) - kSlack, f = __builtin_amdgcn_exp2f(next - lift);
          sum *= f;
#pragma unroll
          for (int i = 0; i < ND; ++i) o[i] *= f;
          lift = next;
          scale_top = __builtin_amdgcn_ldexpf(1.f, ex);
        }
      }
      const float base = (ref == -INFINITY ? 0.f : ref) - lift;
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = __builtin_amdgcn_exp2f(c[i >> 2][i & 3] - base);
        sum += w[i];
      }

      // V through LDS: positions that the row does not see as zeros
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int32_t t = t0 + 16 * u + col;
        const bool seen = whole || (view.sees(t) && t < t_end);
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          h8 x = v[u].get(j);
          if constexpr (std::is_same_v<T, _Float16>)
            if (!seen) x = h8{};
          const int e = (SPAN ? quad * NC + j : 4 * j + quad) * 8;
          *reinterpret_cast<h8 *>(my + (16 * u + col) * PITCH + e * 2) = x;
        }
      }
      if (more) load(v, a.v_layer, a.v_scale, held);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      h8 wh, wl;
      if constexpr (!Q8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          _Float16 hi, lo;
          split2(w[i], hi, lo);
          wh[i] = hi;
          wl[i] = lo;
        }
      }
#pragma unroll
      for (int i = 0; i < ND; ++i) {
        if constexpr (Q8) {
          if (i % 2 == 0) {  // a group's two tiles share its weights
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              _Float16 hi, lo;
              split2(w[e] * (float)dv[e >> 2][i / 2][e & 3], hi, lo);
              wh[e] = hi;
              wl[e] = lo;
            }
          }
        }
        const char *p = my + (4 * quad + (col >> 2)) * PITCH + (16 * i + 4 * (col & 3)) * 2;
        const h8 x = read_tr2(p, 16 * PITCH);
        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, wh, o[i], 0, 0, 0);
        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, wl, o[i], 0, 0, 0);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }

    // fold the waves: numerators [column][element], reference and sum
    sum = rows_reduce<false>(sum);
    __syncthreads();  // every wave is done with its V rows
    float *const red = reinterpret_cast<float *>(lds);
    if (live) {
      float *dst = red + (wave * 16 + col) * RED;
#pragma unroll
      for (int i = 0; i < ND; ++i) *reinterpret_cast<f32x4 *>(dst + 16 * i + 4 * quad) = o[i];
      if (quad == 0) {
        dst[HDP] = ref - lift;
        dst[HDP + 1] = sum;
      }
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < cols * HDP; i += 64 * kRowsWaves) {
      const int cc = i / HDP, e = i - cc * HDP;
      const float *src = red + cc * RED;
      float m[kRowsWaves], mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < kRowsWaves; ++w) {
        m[w] = src[w * 16 * RED + HDP];
        mx = __builtin_fmaxf(mx, m[w]);
      }
      const float base = mx == -INFINITY ? 0.f : mx;
      float l = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < kRowsWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(m[w] - base);
        l = __builtin_fmaf(src[w * 16 * RED + HDP + 1], f, l);
        x = __builtin_fmaf(src[w * 16 * RED + e], f, x);
      }
      if (e >= a.head_dim) continue;
      const int64_t rh = row * a.n_heads + head0 + cc;
      if (n_parts == 1) {
        row_store(a, rh * a.head_dim + e, l != 0.f ? x / l : 0.f);
      } else {
        const int64_t at = (slot * a.n_heads + head0 + cc) * a.max_parts + part;
        a.part_o[at * a.head_dim + e] = x;
        if (e == 0) {
          a.part_ml[2 * at] = mx;
          a.part_ml[2 * at + 1] = l;
        }
      }
    }
    if (a.part_n && parted && part == 0 && threadIdx.x == 0) a.part_n[slot] = n_parts;
    __syncthreads();  // the fold's memory is the next row's V rows
  }
}

template <typename T, int HDP, bool SPAN>
hipError_t launch_rows_t(const PoolGeom &g, const ScoredArgs &a, int64_t most_rows, hipStream_t s) {
  const int group = a.n_heads / a.n_kv_heads, head_tiles = (group + 15) / 16;
  const int64_t wgs = (a.row_items ? a.n_rows : a.n) * a.max_parts * a.n_kv_heads * head_tiles;
  if (wgs * 64 * kRowsWaves >= (int64_t{1} << 32)) return hipErrorInvalidValue;
  const bool mods = a.softcap > 0.f || a.slopes;
  const auto kernel = mods ? scored_rows_kernel<T, HDP, SPAN, true> : scored_rows_kernel<T, HDP, SPAN, false>;
  kernel<<<(unsigned)wgs, 64 * kRowsWaves, 0, s>>>(a, g.n_blocks, g.kv_dim, head_tiles, most_rows);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_rows_hd(const PoolGeom &g, const ScoredArgs &a, int64_t most_rows, hipStream_t s) {
  constexpr bool span = !std::is_same_v<T, int8_t>;
  if (a.head_dim == 64) return launch_rows_t<T, 64, span>(g, a, most_rows, s);
  if (a.head_dim == 128) return launch_rows_t<T, 128, span>(g, a, most_rows, s);
  if (a.head_dim <= 32) return launch_rows_t<T, 32, false>(g, a, most_rows, s);
  if (a.head_dim <= 64) return launch_rows_t<T, 64, false>(g, a, most_rows, s);
  if (a.head_dim <= 96) return launch_rows_t<T, 96, false>(g, a, most_rows, s);
  if (a.head_dim <= 128) return launch_rows_t<T, 128, false>(g, a, most_rows, s);
  if (a.head_dim <= 192) return launch_rows_t<T, 192, false>(g, a, most_rows, s);
  return launch_rows_t<T, 256, false>(g, a, most_rows, s);
}

}  // namespace

// q8_0: a head's 32-element products are whole groups, and none is padded.
bool scored_rows_supported(int elem, int head_dim) {
  if (elem == 4 || head_dim % 8 != 0 || head_dim > 256) return false;
  return elem != 1 || head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 192 ||
         head_dim == 256;
}

hipError_t launch_scored_rows(const PoolGeom &g, const ScoredArgs &a, int64_t most_rows, hipStream_t s) {
  if (g.elem == kElemQ4) return launch_rows_hd<Q4>(g, a, most_rows, s);
  if (g.elem == 1) return launch_rows_hd<int8_t>(g, a, most_rows, s);
  return launch_rows_hd<_Float16>(g, a, most_rows, s);
}

}  // namespace ltkv
