// gfx950 (MI355X, CDNA4) kernels around the attention of a step with drafted
// tokens.
//
//   rope_table_kernel       cosines and sines of scaled rotary frequencies
//   write_rope_rows_kernel  K rotated into its cells, V appended, Q rotated, for rows of any type
//   step_layout_kernel      row starts, lengths, tables, slots, positions and masks of a step
//   window_masks_kernel     a step's masks for a layer with a window
//   accept_tree_kernel      the accepted path of every tree, and its rows moved together
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/ltkv.h"
#include "ltkv_device.h"
#include "ltkv_kernels.h"

namespace ltkv {
namespace {

// A thread a (position, pair): the angle in 64 bits, since an f32 product of a
// position near 10^5 is off by up to 2^-7 radians. The magnitude is a factor of
// both, rounded with them once.
__global__ void __launch_bounds__(256)
rope_table_kernel(const double *__restrict__ inv_freq, float magnitude, int half, int64_t n, float *__restrict__ table) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t pos = i / half;
  const double angle = (double)pos * inv_freq[i - pos * half];
  table[2 * i] = (float)(cos(angle) * (double)magnitude);
  table[2 * i + 1] = (float)(sin(angle) * (double)magnitude);
}

// ---- rotary appends of rows of any type --------------------------------------

struct F16Row {};
struct Bf16Row {};

// N (4 or 8) elements of a row as they lie in memory, read as f32 values.
template <typename R, int N>
struct Elements {
  static constexpr int WORDS = std::is_same_v<R, float> ? N : N / 2;
  uint32_t w[WORDS];
  __device__ __forceinline__ void load(const char *row, int64_t e) {
    const char *src = row + e * (std::is_same_v<R, float> ? 4 : 2);
    if constexpr (WORDS == 2) {
      const u32x2 u = *reinterpret_cast<const u32x2 *>(src);
      w[0] = u.x;
      w[1] = u.y;
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; i += 4) {
        const u32x4 u = *reinterpret_cast<const u32x4 *>(src + 4 * i);
#pragma unroll
        for (int k = 0; k < 4; ++k) w[i + k] = u[k];
      }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (std::is_same_v<R, float>) return __builtin_bit_cast(float, w[i]);
    if constexpr (std::is_same_v<R, Bf16Row>)
      return __builtin_bit_cast(float, i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    const h2 h = __builtin_bit_cast(h2, w[i >> 1]);
    return i & 1 ? (float)h.y : (float)h.x;
  }
};

// 8 f32 values as elements of a row.
template <typename R>
__device__ __forceinline__ void store_row(void *row, int64_t e, const float (&x)[8]) {
  if constexpr (std::is_same_v<R, float>) {
    f32x4 *dst = reinterpret_cast<f32x4 *>(static_cast<float *>(row) + e);
    dst[0] = f32x4{x[0], x[1], x[2], x[3]};
    dst[1] = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = std::is_same_v<R, F16Row> ? pack_f16x2(x[2 * k], x[2 * k + 1])
                                       : (uint32_t)bf16_bits(x[2 * k]) | (uint32_t)bf16_bits(x[2 * k + 1]) << 16;
    *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(row) + e) = w;
  }
}

// 8 f32 values into elements e ... e + 7 of cell s of a pool. Quantised pools: the
// four lanes of a group of 32 elements call it together.
template <int ELEM>
__device__ __forceinline__ void store_cell(void *pool, void *scales, int32_t s, int e, int kv_dim, const float (&x)[8]) {
  if constexpr (ELEM == 2) store_row<F16Row>(pool, (int64_t)s * kv_dim + e, x);
  else if constexpr (ELEM == 4) store_row<float>(pool, (int64_t)s * kv_dim + e, x);
  else store_quants<ELEM == kElemQ4 ? 4 : 8>(x, s, e, kv_dim, static_cast<int8_t *>(pool), static_cast<uint16_t *>(scales));
}

// How a head's elements pair up: (2i, 2i+1); (i, i + rope_dim/2), where 8
// consecutive elements have 8 consecutive partners, or where only 4 have.
constexpr int kInterleaved = 0, kHalves = 1, kHalvesOfFour = 2;

// A team of waves takes a token; a lane takes 8 elements at one place in a head
// (a slice) for several heads, so that their cosines and sines are read once, and
// a wave whole heads: with d_q_out == d_q every element of a head is read before
// one is written. Every lane of the four that share a group of a quantised row
// takes the same path. Pairs' partners are read a second time, through L1. The loads
// of kHeads heads come before the first is needed. Bound by HBM: 13 047 bf16 rows of
// 28 + 2 x 4 heads of 128 into f16 cells in 41-44 us (240 MB, 5.5-5.9 TB/s, the last
// level cache's hits in it); a few tokens take 4.6 us of latency.
constexpr int kHeads = 4;

template <int ELEM, typename R, int PAIRS>
__global__ void __launch_bounds__(256)
write_rope_rows_kernel(void *__restrict__ kpool, void *__restrict__ vpool, void *__restrict__ kscale,
                       void *__restrict__ vscale, RopeRows a, RopeGeom r, int kv_dim, int64_t n_cells, int team) {
#pragma clang fp contract(off)
  constexpr int SIZE = std::is_same_v<R, float> ? 4 : 2;
  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int waves = team >> 6, wave_of_team = wave % waves;
  const int64_t row = (int64_t)blockIdx.x * (4 / waves) + wave / waves;
  if (row >= a.n) return;
  const int32_t pos = scalar_read(a.positions, row), s = scalar_read(a.slots, row);
  if (pos < 0 || pos >= r.max_pos) return;
  const bool cell = s >= 0 && (int64_t)s < n_cells;
  const int slices = r.head_dim >> 3, per_wave = 64 / slices;
  const int hl = lane / slices, slice = lane - hl * slices, e = slice * 8;
  const int half = r.rope_dim >> 1;
  const char *const krow = static_cast<const char *>(a.k) + row * a.src_stride * SIZE;
  const char *const vrow = static_cast<const char *>(a.v) + row * a.src_stride * SIZE;
  const char *const qrow = static_cast<const char *>(a.q) + row * a.q_stride * SIZE;
  char *const orow = static_cast<char *>(a.q_out) + row * a.out_stride * SIZE;
  const int v0 = wave_of_team * 64 + lane, v_end = cell ? kv_dim >> 3 : 0;
  Elements<R, 8> v;
  if (v0 < v_end) v.load(vrow, 8 * v0);
  if (hl < per_wave) {
    const bool turns = e < r.rope_dim;
    // (cosine, sine) of element i's pair, sine negative where the element is its first member
    float c[8], sn[8];
    if (turns) {
      const float *cs = r.table + (int64_t)pos * half * 2;
      if constexpr (PAIRS == kInterleaved) {
        const f32x4 u = *reinterpret_cast<const f32x4 *>(cs + e), w = *reinterpret_cast<const f32x4 *>(cs + e + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const f32x4 &x = i < 4 ? u : w;
          c[i] = x[2 * (i >> 1 & 1)];
          sn[i] = i & 1 ? x[2 * (i >> 1 & 1) + 1] : -x[2 * (i >> 1 & 1) + 1];
        }
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {  // 4 elements on one side each
          const int x = e + 4 * q;
          const bool low = x < half;
          const float *const at = cs + 2 * (low ? x : x - half);
          const f32x4 u = *reinterpret_cast<const f32x4 *>(at), w = *reinterpret_cast<const f32x4 *>(at + 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float y = i < 2 ? u[2 * i + 1] : w[2 * i - 3];
            c[4 * q + i] = i < 2 ? u[2 * i] : w[2 * i - 4];
            sn[4 * q + i] = low ? -y : y;
          }
        }
      }
    }
    const int n_kv = kv_dim / r.head_dim, heads = n_kv + (a.q ? a.n_heads : 0);
    const int step = waves * per_wave;
    for (int h = (cell ? 0 : n_kv) + wave_of_team * per_wave + hl; h < heads; h += kHeads * step) {
      Elements<R, 8> x[kHeads], y[kHeads];
      Elements<R, 4> z[kHeads][2];
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        const int mine = h + k * step;
        if (mine >= heads) break;
        const char *src = mine >= n_kv ? qrow : krow;
        const int64_t at = (int64_t)(mine >= n_kv ? mine - n_kv : mine) * r.head_dim + e;
        x[k].load(src, at);
        if (turns) {  // the elements' partners
          if constexpr (PAIRS == kHalves) y[k].load(src, at + (e < half ? half : -half));
          if constexpr (PAIRS == kHalvesOfFour) {
#pragma unroll
            for (int q = 0; q < 2; ++q) z[k][q].load(src, at + 4 * q + (e + 4 * q < half ? half : -half));
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        const int mine = h + k * step;
        if (mine >= heads) break;
        const bool is_q = mine >= n_kv;
        const int64_t at = (int64_t)(is_q ? mine - n_kv : mine) * r.head_dim + e;
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = x[k].get(i);
        if (turns) {
          // first members a c - b s, second ones a s + b c = b c + a s
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float p = PAIRS == kInterleaved ? x[k].get(i ^ 1)
                            : PAIRS == kHalves    ? y[k].get(i)
                                                  : z[k][i >> 2].get(i & 3);
            o[i] = o[i] * c[i] + p * sn[i];
          }
        }
        if (is_q) store_row<R>(orow, at, o);
        else store_cell<ELEM>(kpool, kscale, s, (int)at, kv_dim, o);
      }
    }
  }
  for (int u = v0; u < v_end; u += team) {
    if (u != v0) v.load(vrow, 8 * u);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = v.get(i);
    store_cell<ELEM>(vpool, vscale, s, 8 * u, kv_dim, x);
  }
}

// ---- the layout of a step ----------------------------------------------------

constexpr int kStepThreads = 256;

__device__ __forceinline__ int64_t block_sum(int64_t x, int64_t *red) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}

// New tokens that request i asks for (none without a live table).
__device__ __forceinline__ int32_t asked(const LayoutArgs &a, int64_t i) {
  const int32_t r = a.rows[i];
  if (r < 0 || r >= a.n_table_rows) return 0;
  return a.news ? max(a.news[i], 0) : 1;
}

// A work-group takes a slice of a request's tokens and table entries; it adds up
// the requests in front of its own by itself, so that the step is one launch (for up
// to some thousand requests: 4096 13 us, 16 384 93 us, growing with the square). The
// last ones write the rows behind the last token. A token's mask is its way up
// the tree: its bits fall from word to word, so no word is written twice. Bound by
// latency (counts, then tables): 64 trees of 16 to 64 tokens 6.4 us, 48 prompts 4.3.
constexpr int kParentsHeld = 1024;

__global__ void __launch_bounds__(kStepThreads) step_layout_kernel(LayoutArgs a, int slices) {
  __shared__ int64_t red[4];
  __shared__ int32_t held[kParentsHeld];
  const int t = (int)threadIdx.x;
  const int64_t i = blockIdx.x / (uint32_t)slices;
  const int slice = (int)(blockIdx.x % (uint32_t)slices);
  int64_t before = 0;
  for (int64_t j = t; j < min(i, a.n); j += kStepThreads) before += asked(a, j);
  before = block_sum(before, red);
  if (i >= a.n) {  // behind the last token
    if (slice == 0 && t == 0) a.row_starts[a.n] = (int32_t)min(before, a.n_tokens);
    for (int64_t j = before + slice * kStepThreads + t; j < a.n_tokens; j += (int64_t)slices * kStepThreads) {
      a.slots[j] = -1;
      a.positions[j] = -1;
      for (int64_t w = 0; a.masks && w < a.mask_words; ++w) a.masks[j * a.mask_words + w] = 0;
    }
    return;
  }
  const int32_t row = a.rows[i];
  const bool live = row >= 0 && row < a.n_table_rows;
  const int64_t len = live ? max(a.lens[i], 0) : 0, want = asked(a, i);
  const int64_t start = min(before, a.n_tokens), room = min(a.n_tokens - start, (int64_t)INT32_MAX - len);
  const int32_t m = (int32_t)min(want, room);
  const int32_t have = live ? (int32_t)min((int64_t)a.counts[row], a.width) : 0;  // blocks of the table
  const int64_t need = (len + m + 15) >> 4;
  const int32_t *tab = a.tables + (live ? row : 0) * a.width;
  if (slice == 0 && t == 0) {
    a.row_starts[i] = (int32_t)start;
    a.new_lens[i] = (int32_t)(len + m);
    if (m < want || need > have || need > a.stride) report_fault(a.status, kFaultLayout, i);
  }
  for (int64_t j = slice * kStepThreads + t; j < a.stride; j += (int64_t)slices * kStepThreads)
    a.out_tables[i * a.stride + j] = j < need && j < have ? tab[j] : -1;
  const int32_t *up = a.parents ? a.parents + start : nullptr;
  if (up && m <= kParentsHeld) {
    for (int j = t; j < m; j += kStepThreads) held[j] = up[j];
    __syncthreads();
  }
  for (int32_t j = slice * kStepThreads + t; j < m; j += slices * kStepThreads) {
    const int64_t p = len + j;
    a.slots[start + j] = (p >> 4) < have ? tab[p >> 4] * 16 + (int32_t)(p & 15) : -1;
    int32_t depth = j;
    if (up) {
      depth = -1;
      int64_t word = a.mask_words - 1;
      uint32_t bits = 0;
      int32_t *const mask = a.masks + (start + j) * a.mask_words;
      for (int32_t node = j; node >= 0;) {
        ++depth;
        for (; word > node >> 5; --word, bits = 0) mask[word] = (int32_t)bits;
        if (word == node >> 5) bits |= 1u << (node & 31);  // (rows past the words have no bit)
        const int32_t above = m <= kParentsHeld ? held[node] : up[node];
        node = above < node ? above : -1;  // a parent comes before its children
      }
      for (; word >= 0; --word, bits = 0) mask[word] = (int32_t)bits;
    }
    a.positions[start + j] = (int32_t)min(len + depth, (int64_t)INT32_MAX);
  }
}

// ---- masks of a layer with a window --------------------------------------------

// A thread a word: the sequence by bisection, then the positions of the rows whose
// bits are set. Bound by latency: 5 us.
__global__ void __launch_bounds__(256) window_masks_kernel(WindowMasks a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.n_rows * a.words) return;
  const int64_t row = i / a.words, word = i - row * a.words;
  int64_t lo = 0, hi = a.n;  // the last sequence whose first row is not behind the row
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if ((int64_t)a.row_starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  const int64_t row0 = a.row_starts[lo], row1 = a.row_starts[lo + 1];
  uint32_t kept = 0;
  if (row0 >= 0 && row >= row0 && row < row1) {
    const int64_t from = (int64_t)a.positions[row] - a.window;  // positions up to it are not seen
    for (uint32_t bits = (uint32_t)a.masks[i]; bits; bits &= bits - 1) {
      const int64_t other = row0 + 32 * word + __builtin_ctz(bits);
      if (other < row1 && other < a.n_rows && a.positions[other] > from) kept |= bits & -bits;
    }
  }
  a.out[i] = (int32_t)kept;
}

// ---- acceptance --------------------------------------------------------------

// Rows moved at a time: all of them are read before one is written, which is safe
// in any order of the cells, since a path's k-th node is at place k or behind it.
constexpr int kMoves = 8;

// A work-group takes a request's rows in one layer's K or V pool and finds the
// path by itself (a wave's lanes hold 64 drafts; a step down the tree is one
// ballot), so that the walk and the moves are one launch. Bound by latency: a
// single tree 6.0 us, 48 trees of 20 to 64 drafts in four layers 10 us.
template <typename U>
__global__ void __launch_bounds__(256)
accept_tree_kernel(AcceptArgs a, int64_t n_blocks, int kv_dim, int elem) {
  const int t = (int)threadIdx.x, lane = t & 63;
  const int64_t per_seq = 2 * a.n_layers, seq = blockIdx.x / per_seq;
  const int part = (int)(blockIdx.x - seq * per_seq), layer = part >> 1;
  const bool is_v = part & 1, first = part == 0;
  const int64_t lo = scalar_read(a.row_starts, seq), hi = scalar_read(a.row_starts, seq + 1);
  // starts outside [0, n_rows], or falling ones, give fewer rows, never a row
  // outside the call's or one that another request has in front
  const int64_t row0 = lo < 0 ? 0 : lo > a.n_rows ? a.n_rows : lo;
  const int64_t row1 = hi > a.n_rows ? a.n_rows : hi < row0 ? row0 : hi;
  const int32_t m = (int32_t)(row1 - row0);
  const int64_t len = scalar_read(a.lens, seq), base = len - m;
  const int32_t *tab = a.tables + seq * a.table_stride;
  if (first) {  // rows of no request
    if (seq == 0)
      for (int64_t j = t; j < row0; j += 256) a.path[j] = -1;
    if (seq == a.n - 1)
      for (int64_t j = row1 + t; j < a.n_rows; j += 256) a.path[j] = -1;
  }
  char *const pool = static_cast<char *>(is_v ? a.v : a.k) + layer * a.layer_bytes;
  uint16_t *const scales = elem > 1 ? nullptr : static_cast<uint16_t *>(is_v ? a.v_scale : a.k_scale) + layer * a.layer_scales;
  const int kg = kv_dim >> 5;
  const int row_bytes = elem == kElemQ4 ? kv_dim / 2 : kv_dim * elem;
  // (lanes of a draft behind the last: no draft's child)
  int32_t parent = -2, token = 0, target = 0;
  if (lane < m) {
    parent = a.parents[row0 + lane];
    token = a.tokens[row0 + lane];
    target = a.targets[row0 + lane];
  }
  int32_t cur = m > 0 ? 0 : -1, count = 0, next = -1;
  while (cur >= 0) {
    int32_t src[kMoves];  // the next nodes of the path
    int n = 0;
    const int32_t at = count;
#pragma unroll
    for (int k = 0; k < kMoves; ++k) {
      src[k] = cur;
      if (cur < 0) continue;
      ++n;
      const int32_t want = cur < 64 ? __builtin_amdgcn_readlane(target, cur) : scalar_read(a.targets, row0 + cur);
      next = want;
      int32_t found = -1;
      uint64_t hits = __builtin_amdgcn_ballot_w64((parent == cur) & (token == want) & (lane > cur));
      if (hits) found = (int32_t)__builtin_ctzll(hits);
      for (int32_t c = cur < 64 ? 64 : cur & ~63; c < m && found < 0; c += 64) {
        const int32_t j = c + lane;
        hits = __builtin_amdgcn_ballot_w64(j > cur && j < m && a.parents[row0 + j] == cur && a.tokens[row0 + j] == want);
        if (hits) found = c + (int32_t)__builtin_ctzll(hits);
      }
      cur = found;
    }
    count += n;
    if (first && t < n) {
      int32_t node = src[0];
#pragma unroll
      for (int k = 1; k < kMoves; ++k) node = t == k ? src[k] : node;
      a.path[row0 + at + t] = node;
    }
    int64_t from[kMoves], to[kMoves];  // cells; -1: nothing to move
#pragma unroll
    for (int k = 0; k < kMoves; ++k) {
      from[k] = to[k] = -1;
      const int64_t p = base + src[k], d = base + at + k;
      if (k >= n || src[k] == at + k || d < 0) continue;
      const int32_t e = (p >> 4) < a.table_stride ? scalar_read(tab, p >> 4) : -1;
      const int32_t f = (d >> 4) < a.table_stride ? scalar_read(tab, d >> 4) : -1;
      if (e < 0 || e >= n_blocks || f < 0 || f >= n_blocks) {
        report_fault(a.status, kFaultTable, seq);
        continue;
      }
      from[k] = (int64_t)e * 16 + (p & 15);
      to[k] = (int64_t)f * 16 + (d & 15);
    }
    auto place = [&](int64_t cell, int u) -> int64_t {  // of unit u of a cell
      return elem == kElemQ4 ? (((cell >> 4) * kg + u) * 16 + (cell & 15)) * 16
                             : cell * row_bytes + (int64_t)u * (int)sizeof(U);
    };
    for (int u = t; u < row_bytes / (int)sizeof(U); u += 256) {
      U x[kMoves];
#pragma unroll
      for (int k = 0; k < kMoves; ++k)
        if (from[k] >= 0) x[k] = *reinterpret_cast<const U *>(pool + place(from[k], u));
#pragma unroll
      for (int k = 0; k < kMoves; ++k)
        if (from[k] >= 0) *reinterpret_cast<U *>(pool + place(to[k], u)) = x[k];
    }
    if (scales) {
      for (int g = t; g < kg; g += 256) {
        uint16_t x[kMoves];
#pragma unroll
        for (int k = 0; k < kMoves; ++k)
          if (from[k] >= 0) x[k] = scales[((from[k] >> 4) * kg + g) * 16 + (from[k] & 15)];
#pragma unroll
        for (int k = 0; k < kMoves; ++k)
          if (from[k] >= 0) scales[((to[k] >> 4) * kg + g) * 16 + (to[k] & 15)] = x[k];
      }
    }
  }
  if (!first) return;
  for (int32_t j = count + t; j < m; j += 256) a.path[row0 + j] = -1;
  if (t == 0) {
    a.accepted[seq] = count;
    a.next[seq] = next;
    a.new_lens[seq] = (int32_t)max(base + count, (int64_t)0);
  }
}

}  // namespace

hipError_t launch_rope_table(const double *inv_freq, float magnitude, int half, int64_t max_pos, float *table,
                             hipStream_t s) {
  const int64_t n = max_pos * half;
  if ((n + 255) / 256 >= (int64_t{1} << 24)) return hipErrorInvalidValue;
  rope_table_kernel<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(inv_freq, magnitude, half, n, table);
  return hipGetLastError();
}

namespace {

template <int ELEM, typename R>
hipError_t launch_rope_rows_t(const PoolGeom &g, void *k_layer, void *v_layer, void *k_scale, void *v_scale,
                              const RopeRows &a, const RopeGeom &r, hipStream_t s) {
  // A token's waves: four while the tokens are few (a wave's loads then wait for one
  // another), two where they begin to fill the chip, one behind that, which short rows
  // gain by. Whole calls, us with four, two and one:
  //              32/8 x 128 bf16, f16    32/8 x 96 f32, q8_0   32/4 x 64 bf16   9/3 x 64 f32
  //   512 tokens  7.9   7.9   8.4         8.0   8.2   9.0      7.9  8.1  8.0    8.0  8.1  7.9
  //   1024        7.9   7.9   9.1         9.3   9.6  10.6      7.9  7.9  7.9    7.9  7.7  8.2
  //   2048       12.8  11.2  12.3        16.3  14.7  15.9      9.1  8.0  8.0    8.3  8.1  8.0
  //   4800       24.9  22.2  21.2        31.9  29.5  28.5     17.6 13.9 12.7   14.9 11.2 10.8
  //   13 000     64.7  57.2  57.4         103  89.0  88.5     39.7 28.5 25.9   36.8 25.1 22.7
  //   24 000      123   108   114         184   153   153     70.1 48.8 43.0   64.5 42.8 35.6
  const int team = a.n <= 1024 ? 256 : a.n <= 2560 ? 128 : 64;
  const int64_t wgs = (a.n + 256 / team - 1) / (256 / team);
  if (wgs >= (int64_t{1} << 24)) return hipErrorInvalidValue;
  const auto kernel = !r.neox                ? write_rope_rows_kernel<ELEM, R, kInterleaved>
                      : r.rope_dim % 16 == 0 ? write_rope_rows_kernel<ELEM, R, kHalves>
                                             : write_rope_rows_kernel<ELEM, R, kHalvesOfFour>;
  kernel<<<(unsigned)wgs, 256, 0, s>>>(k_layer, v_layer, k_scale, v_scale, a, r, g.kv_dim, g.n_blocks * 16, team);
  return hipGetLastError();
}

template <int ELEM>
hipError_t launch_rope_rows_e(const PoolGeom &g, void *k_layer, void *v_layer, void *k_scale, void *v_scale,
                              const RopeRows &a, const RopeGeom &r, hipStream_t s) {
  if (a.row_type == LTKV_ROWS_F16) return launch_rope_rows_t<ELEM, F16Row>(g, k_layer, v_layer, k_scale, v_scale, a, r, s);
  if (a.row_type == LTKV_ROWS_BF16)
    return launch_rope_rows_t<ELEM, Bf16Row>(g, k_layer, v_layer, k_scale, v_scale, a, r, s);
  return launch_rope_rows_t<ELEM, float>(g, k_layer, v_layer, k_scale, v_scale, a, r, s);
}

}  // namespace

hipError_t launch_write_rope_rows(const PoolGeom &g, void *k_layer, void *v_layer, void *k_scale, void *v_scale,
                                  const RopeRows &a, const RopeGeom &r, hipStream_t s) {
  if (a.n <= 0) return hipSuccess;
  if (g.elem == kElemQ4) return launch_rope_rows_e<kElemQ4>(g, k_layer, v_layer, k_scale, v_scale, a, r, s);
  if (g.elem == 1) return launch_rope_rows_e<1>(g, k_layer, v_layer, k_scale, v_scale, a, r, s);
  if (g.elem == 2) return launch_rope_rows_e<2>(g, k_layer, v_layer, k_scale, v_scale, a, r, s);
  return launch_rope_rows_e<4>(g, k_layer, v_layer, k_scale, v_scale, a, r, s);
}

hipError_t launch_step_layout(const LayoutArgs &a, hipStream_t s) {
  if (a.n <= 0) return hipSuccess;
  // slices of a request: one unless few requests have many tokens or wide tables
  const int64_t units = std::max((a.n_tokens + a.n - 1) / a.n, a.stride);
  const int64_t most = std::max<int64_t>(1, 1024 / a.n);
  const int slices = (int)std::min((units + kStepThreads - 1) / kStepThreads, most);
  const int64_t wgs = (a.n + 1) * std::max(slices, 1);
  if (wgs >= (int64_t{1} << 24)) return hipErrorInvalidValue;
  step_layout_kernel<<<(unsigned)wgs, kStepThreads, 0, s>>>(a, std::max(slices, 1));
  return hipGetLastError();
}

hipError_t launch_window_masks(const WindowMasks &a, hipStream_t s) {
  const int64_t wgs = (a.n_rows * a.words + 255) / 256;
  if (wgs <= 0) return hipSuccess;
  if (wgs >= (int64_t{1} << 24)) return hipErrorInvalidValue;
  window_masks_kernel<<<(unsigned)wgs, 256, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_accept_tree(const PoolGeom &g, const AcceptArgs &a, hipStream_t s) {
  if (a.n <= 0) return hipSuccess;
  const int64_t wgs = a.n * 2 * a.n_layers;
  if (wgs >= (int64_t{1} << 24)) return hipErrorInvalidValue;
  const bool wide = g.elem == kElemQ4 || (int64_t)g.kv_dim * g.elem % 16 == 0;
  const auto kernel = wide ? accept_tree_kernel<u32x4> : accept_tree_kernel<uint16_t>;
  kernel<<<(unsigned)wgs, 256, 0, s>>>(a, g.n_blocks, g.kv_dim, g.elem);
  return hipGetLastError();
}

}  // namespace ltkv
