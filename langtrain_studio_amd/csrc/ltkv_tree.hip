// gfx950 (MI355X, CDNA4) kernels of attention for trees of drafted tokens.
//
//   tree_tile_kernel   tiles of rows against tiles of positions, on the matrix cores
//   tree_merge_kernel  fold of the tiles that several work-groups share
//   tree_any_kernel    any shape
//
// Row j of a sequence with m rows and L positions (context C = L - m) is the cell
// at position C + j. It sees the context positions t < C, with a window of w only t
// > p - w (p: the row's position in its sequence, at least C), and the rows' own
// cells C + i whose bit i its mask holds. Weights are the softmax over these of s =
// scale q.k, capped to cap tanh(s / cap) with a cap; a row that sees nothing gives
// zeros.
#include "ltkv_scored.h"

namespace ltkv {
namespace {

// What a row sees of 32 positions at a time.
struct TreeView {
  const int32_t *mask;  // its words, or nullptr: the rows up to its own
  int64_t words;
  int32_t row;        // the row among its sequence's
  int32_t from, ctx;  // visible context: [from, ctx)
  int32_t len;

  // bit b: position t + b
  __device__ __forceinline__ uint32_t sees32(int32_t t) const {
    const int32_t lo = min(max(from - t, 0), 32), hi = min(max(ctx - t, 0), 32);
    uint32_t bits = low_bits(hi) & ~low_bits(lo);
    if (t + 32 > ctx && t < len) {
      const int32_t j = t - ctx;  // first drafted row of the word (below 0: later bits)
      uint32_t drafted;
      if (mask) {
        // (both words loaded in any case: conditions would wait for one after the other)
        const int32_t w = j >> 5, last = (int32_t)words - 1;  // (floor)
        const uint32_t x = (uint32_t)mask[min(max(w, 0), last)], y = (uint32_t)mask[min(max(w + 1, 0), last)];
        const uint32_t a = w >= 0 && w <= last ? x : 0u, b = w + 1 <= last ? y : 0u;
        drafted = (uint32_t)((((uint64_t)b << 32) | a) >> (j & 31));
      } else {
        drafted = low_bits(min(max(row + 1 - j, 0), 32));
        if (j < 0) drafted &= ~low_bits(min(-j, 32));
      }
      bits |= drafted & low_bits(min(len - t, 32));
    }
    return bits;
  }
  static __device__ __forceinline__ uint32_t low_bits(int32_t n) {  // 0 <= n <= 32
    return n >= 32 ? ~0u : (1u << n) - 1u;
  }
};

__device__ __forceinline__ TreeView tree_view(const TreeArgs &a, const SeqRows &s, int32_t r) {
  TreeView v;
  v.words = a.mask_words;
  v.mask = a.masks ? a.masks + (s.row0 + r) * a.mask_words : nullptr;
  v.row = r;
  v.len = s.len;
  v.ctx = max(s.len - s.count, 0);
  v.from = 0;
  if (a.window > 0) v.from = (int32_t)max((int64_t)max(a.positions[s.row0 + r], v.ctx) - a.window + 1, (int64_t)0);
  return v;
}

constexpr int kAnyThreads = 256;
constexpr int kAnyMaxHeadDim = 1024;
constexpr int kAnyD = kAnyMaxHeadDim / kAnyThreads;

// Any shape and pool: a work-group takes a (row, query head), 256 positions a
// round, a score a thread, then each thread up to four output elements over the
// round's visible positions. It serves shapes that the tile kernel does not, and
// is bound by its scalar loads (8 trees of 8 rows behind 2000 positions: 71 heads of 64
// over one 2.0 ms, where 64 heads on the tile kernel take 27 us; 8/2 heads of 320 1.3 ms).
template <typename T>
__global__ void __launch_bounds__(kAnyThreads) tree_any_kernel(TreeArgs a, int64_t n_blocks, int64_t kv_dim) {
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
  TreeView view = tree_view(a, s, (int32_t)(row - s.row0));
  // (rows in front of position 0: their cells do not exist)
  const int32_t shift = s.len - s.count;
  const int64_t head_off = (int64_t)(h / (a.n_heads / a.n_kv_heads)) * a.head_dim;
  const int64_t qh = (row * a.n_heads + h) * a.head_dim;
  for (int d = t; d < a.head_dim; d += kAnyThreads) sq[d] = row_load(a, qh + d);
  const int32_t *tab = table_of(a.tables, a.table_stride, nullptr, 0, seq);
  view.ctx = shift;  // (negative where the rows outnumber the positions)
  float m = -INFINITY, l = 0.f, o[kAnyD];
#pragma unroll
  for (int k = 0; k < kAnyD; ++k) o[k] = 0.f;
  // (the window bounds the context alone: a row's drafts lie behind its end, however
  // far behind them the row's position is)
  for (int32_t t0 = min(view.from, max(shift, 0)) & ~15; t0 < view.len; t0 += kAnyThreads) {
    const int n_tok = min(view.len - t0, kAnyThreads);
    const bool seen = t < n_tok && (view.sees32(t0 + (t & ~31)) >> (t & 31) & 1);
    __syncthreads();  // sblk and sp of the last round have been read
    if (t < kAnyThreads / 16) sblk[t] = 0;
    __syncthreads();
    // the entries of blocks that some thread sees (a wave holds four blocks)
    const uint64_t any = __builtin_amdgcn_ballot_w64(seen);
    if (any >> (t & 48) & 0xffffu) {
      int32_t blk = tab[(t0 + t) >> 4];
      if (blk < 0 || blk >= n_blocks) {
        report_fault(a.status, kFaultTable, seq);
        blk = 0;
      }
      sblk[t >> 4] = blk;
    }
    __syncthreads();
    float sc = -INFINITY;
    if (seen) {
      const int64_t cell = (int64_t)sblk[t >> 4] * 16 + (t & 15);
      float acc = 0.f;
      for (int d = 0; d < a.head_dim; ++d)
        acc += sq[d] * cell_value<T>(a.k_layer, a.k_scale, cell, kv_dim, head_off + d);
      sc = acc * a.scale;
      if (a.softcap > 0.f) sc = a.softcap * tanhf(sc / a.softcap);
      sc *= kLog2e;
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
      if (pj < 0.f) continue;  // (a position that is not seen may hold infinities or NaN)
      const int64_t cell = (int64_t)sblk[j >> 4] * 16 + (j & 15);
#pragma unroll
      for (int k = 0; k < kAnyD; ++k) {
        const int d = t + kAnyThreads * k;
        if (d < a.head_dim) o[k] += pj * cell_value<T>(a.v_layer, a.v_scale, cell, kv_dim, head_off + d);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kAnyD; ++k) {
    const int d = t + kAnyThreads * k;
    if (d < a.head_dim) row_store(a, qh + d, o[k]);
  }
}

// ---- the tile kernel ----------------------------------------------------------
//
// Its work is laid out as one line of steps: sequence by sequence, of each the tiles
// of rows (rows_per_tile rows by the group's query heads are the columns of a
// work-group), of each the steps of 64 positions. The line is cut into equal
// shares, wherever they begin and end, so that a ragged batch, one long context and
// a short step all load the chip evenly, and a table wider than its contexts costs
// nothing. A share has a work-group for each kv head, next to each other on one XCD:
// they read whole pool rows together. A tile that lies in several shares leaves an
// average per share, which tree_merge_kernel folds.
constexpr int kTreeWaves = 4, kTreeThreads = 64 * kTreeWaves;
constexpr int kTreeTokens = 64;  // positions of a step
// Instruction classes of sched_group_barrier: LDS reads, matrix products.
constexpr int kSchedReads = 0x100, kSchedProducts = 0x8;

struct TreeSeq {
  SeqRows rows;
  int32_t ctx;    // below 0 where the rows outnumber the positions
  int32_t first;  // position of the first step
  int32_t steps, tiles;
};

__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs &a, const SeqRows &rows) {
  TreeSeq s;
  s.rows = rows;
  s.ctx = s.rows.len - s.rows.count;
  // no row sees a position in front of the window of the context's end
  s.first = a.window > 0 ? (int32_t)max((int64_t)s.ctx - a.window + 1, (int64_t)0) & ~15 : 0;
  s.steps = max((s.rows.len - s.first + kTreeTokens - 1) / kTreeTokens, 1);  // (rows that see nothing: zeros)
  s.tiles = (s.rows.count + a.rows_per_tile - 1) / a.rows_per_tile;
  return s;
}

__device__ __forceinline__ int64_t tree_steps(const TreeArgs &a, const SeqRows &rows) {
  const TreeSeq s = tree_seq(a, rows);
  return (int64_t)s.steps * s.tiles;
}

__device__ __forceinline__ void keep_rows(int32_t (&to)[3], const SeqRows &r) {
  to[0] = (int32_t)r.row0;
  to[1] = r.count;
  to[2] = r.len;
}

__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return ((int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) |
         (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}

// What a position's K and V hold as products' operands: f16 and q4_0 cells are f16
// numbers; q8_0 and f32 cells enter as f16 hi + lo pairs (a q8_0 element exactly, an
// f32 one but for its last bit at most) times a power of two of the position's own, so that
// no row loses bits to a position that it does not see.
template <typename T>
constexpr bool kPairs = std::is_same_v<T, int8_t> || std::is_same_v<T, float>;

// A load at a uniform base plus a 32-bit lane offset (see load_at). NT: past the
// caches, for rows that one work-group reads alone; each line in one instruction, else
// it is fetched twice.
template <bool NT, typename V>
__device__ __forceinline__ V pool_load(const char *base, uint32_t off) {
  if constexpr (!NT) return load_at<V>(base, off);
  asm volatile("" : "+v"(off));
  return __builtin_nontemporal_load(reinterpret_cast<const V *>(base + off));
}

// Largest of a value over aligned groups of N lanes (a power of two), in each of them.
template <int N>
__device__ __forceinline__ float lanes_max(float x) {
  if constexpr (N > 1) x = __builtin_fmaxf(x, dpp<0xB1>(x));    // quad_perm [1,0,3,2]
  if constexpr (N > 2) x = __builtin_fmaxf(x, dpp<0x4E>(x));    // quad_perm [2,3,0,1]
  if constexpr (N > 4) x = __builtin_fmaxf(x, dpp<0x141>(x));   // row_half_mirror
  if constexpr (N > 8) x = __builtin_fmaxf(x, dpp<0x140>(x));   // row_mirror
  if constexpr (N > 16) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t p = a[0], q = a[1];
    x = __builtin_fmaxf(__builtin_bit_cast(float, p), __builtin_bit_cast(float, q));
  }
  if constexpr (N > 32) x = halves_reduce<true>(x);
  return x;
}

// A wave's share of a step on its way from the pool to LDS: K or V of the 16
// positions of one block, whose address is uniform. A load takes whole rows of the
// head, ROW lanes each, 64 / ROW rows an instruction: with 64 bytes of 16 rows an
// instruction, lines were fetched in two pieces (64 trees of up to 16 rows, f16: the
// kernel with nothing but its loads 197 us; so, past the caches, 160). EXACT: head_dim is HD, 64 or 128; else
// elements past head_dim are zeros, and 8-bit and 4-bit chunks of 8 bring a scale
// each (a head may begin inside a group of 32).
// put() writes the positions' rows in LDS; `bad` has a bit for each load whose V
// enters as zeros (bad()). Types of pairs give each position's power of two too.
template <typename T, int HD, bool EXACT, bool NT>
struct Cells;

template <int HD, bool EXACT, bool NT>
struct Cells<_Float16, HD, EXACT, NT> {
  static constexpr int ROW = HD / 8, ROWS = 64 / ROW, N = 16 / ROWS;
  u32x4 x[N];
  static __device__ __forceinline__ int64_t block_bytes(int64_t kv_dim) { return kv_dim * 32; }
  static __device__ __forceinline__ int row(int lane, int j) { return lane / ROW + ROWS * j; }
  __device__ __forceinline__ void load(const void *pool, const void *, int64_t at, int64_t kv_dim, uint32_t head_off,
                                       int lane, int head_dim) {
    const char *base = static_cast<const char *>(pool) + at;
    const uint32_t e = lane % ROW * 8, place = ((lane / ROW) * (uint32_t)kv_dim + head_off + e) * 2;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (EXACT || (int)e < head_dim) x[j] = pool_load<NT, u32x4>(base, place + (uint32_t)(2 * ROWS * j) * (uint32_t)kv_dim);
      else x[j] = u32x4{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ uint32_t bad() const {
    uint32_t b = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) b |= not_finite(__builtin_bit_cast(h8, x[j])) ? 1u << j : 0u;
    return b;
  }
  __device__ __forceinline__ void put(char *lds, int pitch, int lane, uint32_t bad) const {
#pragma unroll
    for (int j = 0; j < N; ++j)
      *reinterpret_cast<u32x4 *>(lds + row(lane, j) * pitch + lane % ROW * 16) =
          bad >> j & 1 ? u32x4{0, 0, 0, 0} : x[j];
  }
};

template <int HD, bool EXACT, bool NT>
struct Cells<Q4, HD, EXACT, NT> {
  // a lane takes a quarter of one position's head: of a head of whole groups, the
  // lanes of a load take a contiguous piece of the block's tiles
  static constexpr int ROW = 4, ROWS = 16, N = 1, NC = HD / 32, NS = EXACT ? 1 : NC;
  uint32_t x[NC];
  uint32_t s[NS];  // (as 32 bits: a 16-bit value would be waited for to be moved)
  static __device__ __forceinline__ int64_t block_bytes(int64_t kv_dim) { return kv_dim * 8; }
  static __device__ __forceinline__ int row(int lane, int) { return lane >> 2; }
  static __device__ __forceinline__ int chunk(int lane, int j) {
    return EXACT ? (lane & 3) * NC + j : (lane & 3) + 4 * j;
  }
  __device__ __forceinline__ void load(const void *pool, const void *scales, int64_t at, int64_t, uint32_t head_off,
                                       int lane, int head_dim) {
    const char *base = static_cast<const char *>(pool) + at, *sbase = static_cast<const char *>(scales) + (at >> 3);
    const uint32_t slot = lane >> 2;
    if constexpr (EXACT) {
      static_assert(NC == 2 || NC == 4, "a lane's chunks lie in one group");
      const uint32_t e = head_off + chunk(lane, 0) * 8, place = ((e >> 5) * 16 + slot) * 16 + ((e & 31) >> 3) * 4;
      s[0] = load_at<uint16_t>(sbase, (place >> 4) * 2);
      if constexpr (NC == 4) {
        const u32x4 w = pool_load<NT, u32x4>(base, place);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = w[j];
      } else {
        const u32x2 w = pool_load<NT, u32x2>(base, place);
        x[0] = w.x;
        x[1] = w.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        x[j] = 0;
        s[j] = 0;
        if (chunk(lane, j) * 8 >= head_dim) continue;
        const uint32_t e = head_off + chunk(lane, j) * 8, tile = (e >> 5) * 16 + slot;
        x[j] = load_at<uint32_t>(base, tile * 16 + ((e & 31) >> 3) * 4);
        s[j] = load_at<uint16_t>(sbase, tile * 2);
      }
    }
  }
  __device__ __forceinline__ uint32_t bad() const { return 0; }
  __device__ __forceinline__ void put(char *lds, int pitch, int lane, uint32_t) const {
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const _Float16 d = __builtin_bit_cast(_Float16, (uint16_t)s[EXACT ? 0 : j]);
      *reinterpret_cast<h8 *>(lds + row(lane, 0) * pitch + chunk(lane, j) * 16) = q4x8_to_h8(x[j], h2{d, d});
    }
  }
};

template <int HD, bool EXACT, bool NT>
struct Cells<int8_t, HD, EXACT, NT> {
  static constexpr int E = EXACT ? 16 : 8;  // elements a load and lane
  static constexpr int ROW = HD / E, ROWS = 64 / ROW, N = 16 / ROWS;
  typedef std::conditional_t<EXACT, u32x4, u32x2> Quants;
  Quants x[N];
  uint32_t s[N];
  static __device__ __forceinline__ int64_t block_bytes(int64_t kv_dim) { return kv_dim * 16; }
  static __device__ __forceinline__ int row(int lane, int j) { return lane / ROW + ROWS * j; }
  __device__ __forceinline__ void load(const void *pool, const void *scales, int64_t at, int64_t kv_dim,
                                       uint32_t head_off, int lane, int head_dim) {
    const char *base = static_cast<const char *>(pool) + at, *sbase = static_cast<const char *>(scales) + (at >> 4);
    const uint32_t e = head_off + lane % ROW * E, place = lane / ROW * (uint32_t)kv_dim + e;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (EXACT || lane % ROW * E < head_dim) {
        s[j] = load_at<uint16_t>(sbase, ((e >> 5) * 16 + row(lane, j)) * 2);
        x[j] = pool_load<NT, Quants>(base, place + (uint32_t)(ROWS * j) * (uint32_t)kv_dim);
      } else {
        s[j] = 0;
#pragma unroll
        for (int i = 0; i < E / 4; ++i) x[j][i] = 0x80808080u;  // (quants are stored offset by 128)
      }
    }
  }
  __device__ __forceinline__ float scale(int j) const {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)s[j]);
  }
  __device__ __forceinline__ uint32_t bad() const {
    uint32_t b = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) b |= scale(j) <= 65504.f ? 0u : 1u << j;
    return b;
  }
  // Elements times 2^-e stay below 2^15. q d as hi + lo parts in packed f16: q has 8
  // bits and d 11, so what the rounding of the product leaves is an f16 number, which
  // the fused multiply-add gives exactly (d times a power of two is one too, down to
  // 2^-22 of the largest scale).
  // Returns the largest power of the lane's positions.
  __device__ __forceinline__ float put(char *lds, int plane, int pitch, int lane, uint32_t bad, float *pow,
                                       bool) const {
    float most = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d0 = scale(j), top = lanes_max<ROW>(__builtin_fminf(d0, 65504.f));
      const int e = top > 0.f ? __builtin_amdgcn_frexp_expf(top) - 8 : -32;
      const _Float16 d = bad >> j & 1 ? (_Float16)0.f : (_Float16)__builtin_amdgcn_ldexpf(d0, -e);
      const h8 d8 = {d, d, d, d, d, d, d, d};
      if (lane % ROW == 0) pow[row(lane, j)] = __builtin_amdgcn_ldexpf(1.f, e);
      most = __builtin_fmaxf(most, __builtin_amdgcn_ldexpf(1.f, e));
#pragma unroll
      for (int i = 0; i < E / 8; ++i) {
        const h8 q = i8x8_to_h8(u32x2{x[j][2 * i], x[j][2 * i + 1]}), hi = q * d8;
        char *const to = lds + row(lane, j) * pitch + lane % ROW * (2 * E) + 16 * i;
        *reinterpret_cast<h8 *>(to) = hi;
        *reinterpret_cast<h8 *>(to + plane) = __builtin_elementwise_fma(q, d8, -hi);
      }
    }
    return most;
  }
};

template <int HD, bool EXACT, bool NT>
struct Cells<float, HD, EXACT, NT> {
  static constexpr int ROW = HD / 4, ROWS = 64 / ROW, N = 16 / ROWS;
  u32x4 x[N];
  static __device__ __forceinline__ int64_t block_bytes(int64_t kv_dim) { return kv_dim * 64; }
  static __device__ __forceinline__ int row(int lane, int j) { return lane / ROW + ROWS * j; }
  __device__ __forceinline__ void load(const void *pool, const void *, int64_t at, int64_t kv_dim, uint32_t head_off,
                                       int lane, int head_dim) {
    const char *base = static_cast<const char *>(pool) + at;
    const uint32_t e = lane % ROW * 4, place = ((lane / ROW) * (uint32_t)kv_dim + head_off + e) * 4;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (EXACT || (int)e < head_dim) x[j] = pool_load<NT, u32x4>(base, place + (uint32_t)(4 * ROWS * j) * (uint32_t)kv_dim);
      else x[j] = u32x4{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ uint32_t top_bits(int j) const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, x[j][i] & 0x7fffffffu);
    return m;
  }
  __device__ __forceinline__ uint32_t bad() const {
    uint32_t b = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) b |= top_bits(j) >= 0x7f800000u ? 1u << j : 0u;
    return b;
  }
  // Powers of at least 2^-100: smaller values are nothing beside their products'
  // rounding. Each position has its own where a row does not see all of the step;
  // else the block's 16 share one (a reduction instead of eight). Parts to nearest: by
  // truncation the largest term of the result's error (8 trees of 8 f32 rows behind
  // 8000 positions: 7.2e-7, so 5.8e-7; 155 us, 160).
  __device__ __forceinline__ float put(char *lds, int plane, int pitch, int lane, uint32_t bad, float *pow,
                                       bool apart) const {
    int e[N];
    if (apart) {
#pragma unroll
      for (int j = 0; j < N; ++j) e[j] = exponent(lanes_max<ROW>(__builtin_bit_cast(float, min(top_bits(j), 0x7f7fffffu))));
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) top = max(top, top_bits(j));
      const int all = exponent(lanes_max<64>(__builtin_bit_cast(float, min(top, 0x7f7fffffu))));
#pragma unroll
      for (int j = 0; j < N; ++j) e[j] = all;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (lane % ROW == 0) pow[row(lane, j)] = __builtin_amdgcn_ldexpf(1.f, e[j]);
      h2 hi[2], lo[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t u = bad >> j & 1 ? 0u : x[j][2 * i + k];
          v[k] = __builtin_amdgcn_ldexpf(__builtin_bit_cast(float, u), -e[j]);
        }
        hi[i] = h2{(_Float16)v[0], (_Float16)v[1]};
        lo[i] = h2{(_Float16)__builtin_fmaf((float)hi[i].x, -1.f, v[0]),
                   (_Float16)__builtin_fmaf((float)hi[i].y, -1.f, v[1])};
      }
      char *const to = lds + row(lane, j) * pitch + lane % ROW * 8;
      *reinterpret_cast<h4 *>(to) = h4{hi[0].x, hi[0].y, hi[1].x, hi[1].y};
      *reinterpret_cast<h4 *>(to + plane) = h4{lo[0].x, lo[0].y, lo[1].x, lo[1].y};
    }
    return 0.f;
  }
  static __device__ __forceinline__ int exponent(float top) {
    return top > 0.f ? max(__builtin_amdgcn_frexp_expf(top) - 15, -100) : -100;
  }
};

// A lane's part of a row of Q as it lies in memory: elements 16 j ... + 7 of row type R
// (float, _Float16, or uint16_t for bf16), zeros from element `n` on and where `live`
// is false. All loads come before the first value is needed.
template <typename R, int NK, bool EXACT>
struct Column {
  static constexpr int V = std::is_same_v<R, float> ? 2 : 1;
  u32x4 u[NK][V];
  __device__ __forceinline__ Column(const void *q, int64_t i, bool live, int n) {
    const R *const row = static_cast<const R *>(q) + i;
#pragma unroll
    for (int j = 0; j < NK; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        u[j][v] = u32x4{0, 0, 0, 0};
        if (live && (EXACT || 16 * j < n)) u[j][v] = *reinterpret_cast<const u32x4 *>(row + 16 * j + 4 * v);
      }
  }
  __device__ __forceinline__ float get(int j, int k) const {
    const uint32_t w = V == 2 ? u[j][k >> 2][k & 3] : u[j][0][k >> 1];
    if constexpr (std::is_same_v<R, float>) return __builtin_bit_cast(float, w);
    if constexpr (std::is_same_v<R, uint16_t>) return __builtin_bit_cast(float, k & 1 ? w & 0xffff0000u : w << 16);
    const h2 h = __builtin_bit_cast(h2, w);
    return k & 1 ? (float)h.y : (float)h.x;
  }
};

// WC waves share a step's columns, 32 each; 4 / WC waves its positions. Steps go
// through LDS as f16 numbers, on 32x32x16 products: scores^T = K Q^T, weights in
// place, numerators^T += V^T W (a lane's scores are positions 8 (r / 4) + 4 (lane /
// 32) + r % 4 of its column, which is the second product's operand layout when its
// 16 positions are taken as 4 (lane / 32) ... + 3 and 8 + 4 (lane / 32) ... + 3: no
// exchange). The weights enter as hi + lo pairs for rows of any type: rounded to f16,
// they took f16 rows' error from 2.07e-4, the output's own rounding, to 2.44e-4 (16
// trees of 64 rows over a 4-bit cache, capped; 104 us, 94 so) and bf16 rows' from
// 1.66e-3 to 1.68e-3, and either off what f32 arithmetic gives by as much as its
// rounding. FULL (f32 rows, and any rows with a cap over kShortCap): Q as hi + lo pairs
// and the cap's tanh to f32 accuracy; else Q as it is, times a power of two, and on pools
// that are no pairs the tanh off by up to 3e-7, below a sixth of a 16-bit row's rounding.
// Of pairs (kPairs) the scores are multiplied by their position's power of two, and
// so are the weights. f32 pools: a column's numerators have a reference of their own
// (`top_o`): the largest weight times V, not the largest weight, lies near the top of
// f16. 8-bit pools, whose powers lie between 2^-32 and 2^8: weights carry the inverse
// of the largest power that the column has seen (`v_exp`), one instruction a score.
// f32 pools, and heads of more than 128 elements, take one work-group a CU: two left
// their waves too few registers (f32, one step of 8 rows: 18 us with spills).
//
// Measured (32/8 heads of 128 unless said): 64 trees of 10 to 16 bf16 rows behind 2048
// to 4096 positions of an f16 cache 172-184 us (842 MB read, 26 MB of parts written),
// bound by the reads: a kernel of the same loads alone takes 138 us, and a tile's end
// costs a work-group 7 to 10 us (Q is read behind the K and V on their way). 8 trees of
// 40 to 48 f32 rows behind 32 000 positions of a q8_0 cache (28/4 heads) 570-620 us:
// three products of pairs (486 GFLOP: products 42% of the cycles, vector instructions
// 41%, partly overlapped). 16 trees of 64 f16 rows, capped, over a 4-bit cache in a
// window of 2048: 102 us (vector instructions 53% of the cycles, products 25%, one after
// the other; waves wait a third of their time; 85 parts of 32 tiles, 44 MB written). One
// tree of 8 rows behind 400 positions: 8.7 us, latency.
constexpr int tree_groups_a_cu(bool wide, int hd) { return wide || hd > 128 ? 1 : 2; }

template <typename T, int HD, bool EXACT, bool FULL, int WC>
__global__ void __launch_bounds__(kTreeThreads, tree_groups_a_cu(std::is_same_v<T, float>, HD))
tree_tile_kernel(TreeArgs a, int64_t n_blocks, int64_t kv_dim) {
  constexpr int NC = HD / 32, NK = HD / 16, WP = kTreeWaves / WC, U = 2 / WP;
  constexpr bool PAIRS = kPairs<T>, BYTES = std::is_same_v<T, int8_t>, WIDE = PAIRS && !BYTES;
  constexpr int PLANES = PAIRS ? 2 : 1;
  constexpr int K_PITCH = HD * 2 + 16;  // rows 4 banks apart: 16-byte reads of 16 rows without conflicts
  constexpr int V_PITCH = HD * 2 + 64;  // rows 16 banks apart, for the transposing reads
  constexpr int K_BYTES = kTreeTokens * K_PITCH, V_BYTES = kTreeTokens * V_PITCH;
  constexpr int STEP_BYTES = PLANES * (K_BYTES + V_BYTES);
  constexpr int FOLD = NC * 16 + 4;  // floats that a lane hands over where waves share columns
  // Few columns (WC 2) are bound by the pool's bytes: two steps ahead of the products,
  // in registers that Q leaves free in LDS.
  constexpr int AHEAD = WC == 2 && !BYTES ? 2 : 1;
  constexpr bool Q_LDS = WC == 2 && !PAIRS && HD > 64;
  constexpr int Q_BYTES = Q_LDS ? 32 * WC * K_PITCH : 16;
  static_assert(WP == 1 || (kTreeWaves - WC) * 64 * FOLD * 4 <= STEP_BYTES, "the fold fits the step's memory");
  __shared__ __align__(16) char lds[STEP_BYTES];
  __shared__ __align__(16) char lds_q[(FULL ? 2 : 1) * Q_BYTES];
  __shared__ __align__(16) float s_kpow[PAIRS ? kTreeTokens : 4], s_vpow[PAIRS ? kTreeTokens : 4];
  __shared__ uint32_t s_bad[kTreeWaves];  // bit p: V of position 16 wave + p has an infinity or NaN
  __shared__ int64_t s_begin[kTreeThreads + 1];
  __shared__ int64_t s_sum[kTreeWaves];
  __shared__ int64_t s_found[3];
  __shared__ int32_t s_rows[kTreeThreads][3];  // of the last sequence that a thread looked at: first row, rows, length
  __shared__ int32_t s_from[kTreeWaves];
  __shared__ float s_top[kTreeWaves];  // 8-bit pools: the largest power of a wave's positions' V
  char *const lds_k = lds, *const lds_v = lds + PLANES * K_BYTES;

  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cw = wave % WC, pw = wave / WC;
  const int col = lane & 31, half = lane >> 5;
  const int group = a.n_heads / a.n_kv_heads;

  // the line: a thread's sequences [i0, i1) begin at s_begin[tid]
  const int64_t each = (a.n + kTreeThreads - 1) / kTreeThreads;
  const int64_t i0 = min((int64_t)tid * each, a.n), i1 = min(i0 + each, a.n);
  {
    int64_t sum = 0;
    for (int64_t i = i0; i < i1; ++i) {
      const SeqRows r = seq_rows(a, i);
      keep_rows(s_rows[tid], r);
      sum += tree_steps(a, r);
    }
    int64_t upto = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int64_t y = __shfl_up(upto, off, 64);
      if (lane >= off) upto += y;
    }
    if (lane == 63) s_sum[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; ++w) upto += s_sum[w];
    s_begin[tid] = upto - sum;
    if (tid == kTreeThreads - 1) s_begin[kTreeThreads] = upto;
    __syncthreads();
  }
  const int64_t total = uniform64(s_begin[kTreeThreads]);
  const int64_t per = (total + a.shares - 1) / a.shares;
  // (shares: a multiple of 8; neighbours on the line lie on one XCD too, of eight)
  const uint32_t place = blockIdx.x >> 3;
  const int kvh = (int)(place % (uint32_t)a.n_kv_heads);
  const int64_t share = (int64_t)(blockIdx.x & 7) * (a.shares >> 3) + place / (uint32_t)a.n_kv_heads;
  const int64_t me = share * a.n_kv_heads + kvh;
  int64_t at = share * per;
  const int64_t end = min(total, at + per);
  if (tid == 0) a.ends[8 * me] = a.ends[8 * me + 4] = -1;  // (none, until one is met)

  while (at < end) {
    __syncthreads();  // s_found, and the step's memory, have been read
    if (s_begin[tid] <= at && at < s_begin[tid + 1]) {
      int64_t begin = s_begin[tid], i = i0;
      for (; i + 1 < i1; ++i) {  // (a single sequence lies there already)
        const SeqRows r = seq_rows(a, i);
        keep_rows(s_rows[tid], r);
        const int64_t next = begin + tree_steps(a, r);
        if (at < next) break;
        begin = next;
      }
      if (i0 + 1 < i1 && i + 1 == i1) keep_rows(s_rows[tid], seq_rows(a, i));
      s_found[0] = i;
      s_found[1] = begin;
      s_found[2] = tid;
    }
    __syncthreads();
    const int64_t seq = uniform64(s_found[0]), off = at - uniform64(s_found[1]);
    const int32_t *const found = s_rows[s_found[2]];
    const TreeSeq ts = tree_seq(a, SeqRows{__builtin_amdgcn_readfirstlane(found[0]), __builtin_amdgcn_readfirstlane(found[1]),
                                           __builtin_amdgcn_readfirstlane(found[2])});
    const SeqRows rows = ts.rows;
    const int tile = (int)(off / ts.steps);
    const int s_first = (int)(off - (int64_t)tile * ts.steps);
    const int s_last = (int)min((int64_t)ts.steps, s_first + (end - at));
    const int32_t r0 = tile * a.rows_per_tile;
    if (tid == 0 && s_last - s_first < ts.steps) {
      const int64_t begin = at - s_first;
      reinterpret_cast<i32x4 *>(a.ends)[2 * me + (s_first > 0 ? 0 : 1)] =
          i32x4{(int)rows.row0 + r0, min(a.rows_per_tile, rows.count - r0), (int)(begin / per),
                (int)((begin + ts.steps - 1) / per)};
    }
    at += s_last - s_first;

    // the first steps, on their way while Q is laid out
    const int32_t *tab = table_of(a.tables, a.table_stride, nullptr, 0, seq);
    auto block_of = [&](int s) {  // the wave's block of a step (past the end: block 0, read and masked)
      const int32_t t = ts.first + kTreeTokens * s + 16 * wave;
      const int32_t e = s < s_last && t < rows.len ? scalar_read(tab, t >> 4) : 0;
      return (uint32_t)e < (uint32_t)n_blocks ? e : 0;
    };
    const uint32_t head_off = (uint32_t)(kvh * a.head_dim);
    // (rows of one tile are read by one work-group alone)
    typedef Cells<T, HD, EXACT, WC == 2> Rows;
    struct Step {
      Rows k, v;
    };
    Step steps[AHEAD];
    auto load = [&](Step &x, int32_t block) {
      const int64_t b = (int64_t)(uint32_t)block * Rows::block_bytes(kv_dim);
      x.k.load(a.k_layer, a.k_scale, b, kv_dim, head_off, lane, a.head_dim);
      x.v.load(a.v_layer, a.v_scale, b, kv_dim, head_off, lane, a.head_dim);
    };
    int32_t next = block_of(s_first + AHEAD);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) load(steps[k], block_of(s_first + k));

    // Table entries outside the pool are reported where a row sees a position of
    // their block; the steps read block 0 in their place.
    const int32_t blocks_end = (min(rows.len, ts.first + kTreeTokens * s_last) + 15) >> 4;
    int32_t block = ((ts.first + kTreeTokens * s_first) >> 4) + tid;
    int32_t entry = block < blocks_end ? tab[block] : 0;

    // the lane's column
    const int c = cw * 32 + col, rr = c / group;
    const bool live = rr < a.rows_per_tile && r0 + rr < rows.count;
    const int head = kvh * group + c - rr * group;
    const int64_t row = rows.row0 + r0 + (live ? rr : 0);
    TreeView view = tree_view(a, rows, r0 + (live ? rr : 0));
    view.ctx = ts.ctx;
    const bool wave_live = __builtin_amdgcn_ballot_w64(live) != 0;
    int32_t from_max = 0;  // positions in front of it some row does not see
    if (a.window > 0) {
      from_max = live ? view.from : 0;
#pragma unroll
      for (int x = 16; x >= 1; x >>= 1) from_max = max(from_max, __shfl_xor(from_max, x, 64));
      if (lane == 0) s_from[wave] = from_max;
      __syncthreads();
      from_max = __builtin_amdgcn_readfirstlane(max(max(s_from[0], s_from[1]), max(s_from[2], s_from[3])));
    }

    // Q columns, times a power of two and the scale's sign
    h8 qh[Q_LDS ? 1 : NK], ql[FULL && !Q_LDS ? NK : 1];
    char *const qp = lds_q + (Q_LDS ? (32 * cw + col) * K_PITCH + 16 * half : 0);
    int q_exp = 0;
    auto lay_out = [&](auto tag) {
      const Column<decltype(tag), NK, EXACT> x(a.q, (row * a.n_heads + head) * (int64_t)a.head_dim + 8 * half, live,
                                               a.head_dim - 8 * half);
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < NK; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = __builtin_fmaxf(amax, __builtin_fabsf(x.get(j, i)));
      amax = halves_reduce<true>(amax);
      // (at most 100: a smaller row's scores are nothing beside their rounding)
      q_exp = amax > 0.f && amax < INFINITY ? min(10 - __builtin_amdgcn_frexp_expf(amax), 100) : 0;
#pragma unroll
      for (int j = 0; j < NK; ++j) {
        h8 hi8, lo8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = __builtin_amdgcn_ldexpf(x.get(j, i), q_exp);
          _Float16 hi, lo;
          split2(a.scale < 0.f ? -y : y, hi, lo);
          hi8[i] = hi;
          lo8[i] = lo;
        }
        if constexpr (Q_LDS) {  // (waves of the same columns write the same; the loop's barriers come first)
          *reinterpret_cast<h8 *>(qp + 32 * j) = hi8;
          if constexpr (FULL) *reinterpret_cast<h8 *>(qp + Q_BYTES + 32 * j) = lo8;
        } else {
          qh[j] = hi8;
          if constexpr (FULL) ql[j] = lo8;
        }
      }
    };
    if (FULL && a.row_type == LTKV_ROWS_F32) lay_out(float{});
    else if (a.row_type == LTKV_ROWS_F16) lay_out(_Float16{});
    else lay_out(uint16_t{});
    for (; block < blocks_end; block += kTreeThreads, entry = block < blocks_end ? tab[block] : 0) {
      if ((uint32_t)entry < (uint32_t)n_blocks) continue;
      bool needed = false;
      for (int32_t r = 0; r < a.rows_per_tile && r0 + r < rows.count; ++r) {
        TreeView v = tree_view(a, rows, r0 + r);
        v.ctx = ts.ctx;
        needed |= (v.sees32(16 * block) & 0xffffu) != 0;
      }
      if (needed) report_fault(a.status, kFaultTable, seq);
    }
    const bool cap = a.softcap > 0.f;
    const float scale = __builtin_fabsf(a.scale);
    const float in_scale = score_factor(cap ? scale / a.softcap : scale * kLog2e, -q_exp);
    const float cap_scale = a.softcap * kLog2e;

    f32x16 o[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) o[i] = f32x16{};
    float ref = -INFINITY, sum = 0.f;      // weights are 2^(score - ref + kLift)
    float top_o = -INFINITY, to_o = 0.f;   // pairs: numerators are taken times 2^(ref - top_o) = to_o
    float v_exp = -1000.f;                 // 8-bit pools: weights and sums are taken times 2^-v_exp
    bool poisoned = false;                 // the column sees an infinity or NaN in V

    auto step = [&](Step &cells, int s) __attribute__((always_inline)) {
      const int32_t t0 = ts.first + kTreeTokens * s;
      const bool partial = t0 + kTreeTokens > ts.ctx || t0 < from_max;  // some row does not see all of it
      lds_barrier();  // the last step has been read
      uint32_t bad = 0, bad_rows = 0;  // infinities and NaN of V may reach only the rows that see them
      if (partial) {
        bad = cells.v.bad();
        if (__builtin_amdgcn_ballot_w64(bad != 0)) {
#pragma unroll
          for (int j = 0; j < Rows::N; ++j) {
            const uint64_t lanes = __builtin_amdgcn_ballot_w64(bad >> j & 1);
            for (int r = 0; r < Rows::ROWS; ++r)
              if (lanes >> (r * Rows::ROW) & (~0ull >> (64 - Rows::ROW))) bad_rows |= 1u << (r + Rows::ROWS * j);
          }
        }
      }
      if constexpr (PAIRS) {
        cells.k.put(lds_k + 16 * wave * K_PITCH, K_BYTES, K_PITCH, lane, 0, s_kpow + 16 * wave, partial);
        const float v_top =
            cells.v.put(lds_v + 16 * wave * V_PITCH, V_BYTES, V_PITCH, lane, bad, s_vpow + 16 * wave, partial);
        if constexpr (BYTES) {
          const float x = lanes_max<64>(v_top);
          if (lane == 0) s_top[wave] = x;
        }
      } else {
        cells.k.put(lds_k + 16 * wave * K_PITCH, K_PITCH, lane, 0);
        cells.v.put(lds_v + 16 * wave * V_PITCH, V_PITCH, lane, bad);
      }
      if (lane == 0) s_bad[wave] = bad_rows;
      // (without a condition: it would have the loads of all steps waited for)
      load(cells, next);
      next = block_of(s + AHEAD + 1);
      lds_barrier();
      if (!wave_live) return;

      // scores of positions t0 + 32 (pw U + u) + 8 (i / 4) + 4 half + i % 4
      f32x16 sc[U];
#pragma unroll
      for (int u = 0; u < U; ++u) sc[u] = f32x16{};
      const char *kp = lds_k + (32 * pw * U + col) * K_PITCH + 16 * half;
#pragma unroll
      for (int j = 0; j < NK; ++j) {
        h8 qhi, qlo;
        if constexpr (Q_LDS) {
          qhi = *reinterpret_cast<const h8 *>(qp + 32 * j);
          if constexpr (FULL) qlo = *reinterpret_cast<const h8 *>(qp + Q_BYTES + 32 * j);
        } else {
          qhi = qh[j];
          if constexpr (FULL) qlo = ql[j];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const h8 x = *reinterpret_cast<const h8 *>(kp + 32 * u * K_PITCH + 32 * j);
          sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qhi, sc[u], 0, 0, 0);
          if constexpr (FULL) sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qlo, sc[u], 0, 0, 0);
          if constexpr (PAIRS) {
            const h8 y = *reinterpret_cast<const h8 *>(kp + K_BYTES + 32 * u * K_PITCH + 32 * j);
            sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, qhi, sc[u], 0, 0, 0);
          }
        }
      }
      {  // operands two products ahead
        constexpr int READS = U * (PAIRS ? 2 : 1) + (Q_LDS ? (FULL ? 2 : 1) : 0);
        constexpr int PRODUCTS = U * (1 + (FULL ? 1 : 0) + (PAIRS ? 1 : 0));
        __builtin_amdgcn_sched_group_barrier(kSchedReads, 2 * READS, 0);
#pragma unroll
        for (int j = 0; j < NK - 2; ++j) {
          __builtin_amdgcn_sched_group_barrier(kSchedProducts, PRODUCTS, 0);
          __builtin_amdgcn_sched_group_barrier(kSchedReads, READS, 0);
        }
        __builtin_amdgcn_sched_group_barrier(kSchedProducts, 2 * PRODUCTS, 0);
      }
      float m = in_scale;  // scores are m sc
      if constexpr (PAIRS) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const f32x4 f = *reinterpret_cast<const f32x4 *>(s_kpow + 32 * (pw * U + u) + 2 * i + 4 * half);
#pragma unroll
            for (int k = 0; k < 4; ++k) sc[u][i + k] *= BYTES ? f[k] : __builtin_fminf(f[k] * in_scale, 1e37f);
          }
        if constexpr (WIDE) m = 1.f;
      }
      if (cap) {
        float to_x = m;  // opaque: the products would be taken before the branch, for both sides
        asm("" : "+v"(to_x));
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float x = sc[u][i] * to_x;
            sc[u][i] = (FULL || PAIRS ? tanh_f32(x) : tanh_f16(x)) * cap_scale;
          }
        m = 1.f;
      }
      float most_v = 0.f;  // 8-bit pools: the largest power of the positions that the column sees
      if (partial) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t seen = live ? view.sees32(t0 + 32 * (pw * U + u)) : 0u, mine = seen >> (4 * half);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            sc[u][i] = mine >> (8 * (i / 4) + i % 4) & 1 ? sc[u][i] : -INFINITY;
          if constexpr (BYTES) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              const f32x4 f = *reinterpret_cast<const f32x4 *>(s_vpow + 32 * (pw * U + u) + 2 * i + 4 * half);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                most_v = __builtin_fmaxf(most_v, mine >> (2 * i + k) & 1 ? f[k] : 0.f);
            }
          }
          // the infinities and NaN of V entered as zeros
          poisoned |= (seen & (s_bad[2 * (pw * U + u)] | s_bad[2 * (pw * U + u) + 1] << 16)) != 0;
        }
      }
      if constexpr (BYTES) {
        most_v = partial ? halves_reduce<true>(most_v)
                         : __builtin_fmaxf(__builtin_fmaxf(s_top[0], s_top[1]), __builtin_fmaxf(s_top[2], s_top[3]));
        const float e = most_v > 0.f ? (float)(__builtin_amdgcn_frexp_expf(most_v) - 1) : -1000.f;
        if (__builtin_amdgcn_ballot_w64(e > v_exp)) {
          const float ne = __builtin_fmaxf(e, v_exp), f = __builtin_amdgcn_exp2f(v_exp - ne);
          sum *= f;
#pragma unroll
          for (int i = 0; i < NC; ++i) o[i] *= f;
          v_exp = ne;
        }
      }
      float top = sc[0][0];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, sc[u][i]);
      top *= m;
      if (__builtin_amdgcn_ballot_w64(top > ref + kSlack)) {
        const float nr = __builtin_fmaxf(ref, halves_reduce<true>(top));
        const float f = nr == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ref - nr);
        sum *= f;
        if constexpr (WIDE) {
          if (top_o > -INFINITY) to_o = __builtin_fminf(__builtin_amdgcn_exp2f(nr - top_o), 3e38f);
        } else {
#pragma unroll
          for (int i = 0; i < NC; ++i) o[i] *= f;
        }
        ref = nr;
      }
      const float base = kLift - (ref == -INFINITY ? 0.f : ref) - (BYTES ? v_exp : 0.f);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          sc[u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[u][i], m, base));
          sum += sc[u][i];
        }
      if constexpr (BYTES) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const f32x4 f = *reinterpret_cast<const f32x4 *>(s_vpow + 32 * (pw * U + u) + 2 * i + 4 * half);
#pragma unroll
            for (int k = 0; k < 4; ++k) sc[u][i + k] *= f[k];
          }
      }
      if constexpr (WIDE) {
        float most = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            const f32x4 f = *reinterpret_cast<const f32x4 *>(s_vpow + 32 * (pw * U + u) + 2 * i + 4 * half);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              sc[u][i + k] *= f[k];
              most = __builtin_fmaxf(most, sc[u][i + k]);
            }
          }
        // (kLift + kSlack: the largest weights times V stay below 2^14)
        const bool first = top_o == -INFINITY && most > 0.f;
        if (__builtin_amdgcn_ballot_w64(first || most * to_o > 16384.f)) {
          const float z = halves_reduce<true>(__builtin_amdgcn_logf(most)) + ref - kLift;
          const float nt = __builtin_fmaxf(top_o, z);
          const float f = top_o > -INFINITY ? __builtin_amdgcn_exp2f(top_o - nt) : 1.f;
#pragma unroll
          for (int i = 0; i < NC; ++i) o[i] *= f;
          top_o = nt;
          if (nt > -INFINITY) to_o = __builtin_fminf(__builtin_amdgcn_exp2f(ref - nt), 3e38f);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[u][i] *= to_o;
      }
#pragma unroll
      for (int p = 0; p < 2 * U; ++p) {  // 16 positions each
        // hi and lo parts of the weights. By truncation: the lo parts take what is left
        // of hi, and 21 bits are past every other rounding but those of f32 pools.
        h8 wh, wl;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          float x = sc[p >> 1][8 * (p & 1) + i], y = sc[p >> 1][8 * (p & 1) + i + 1];
          h2 hi, lo;
          if constexpr (WIDE) {
            asm("" : "+v"(x), "+v"(y));  // (f32 numbers, as in split2)
            hi = h2{(_Float16)x, (_Float16)y};
            lo = h2{(_Float16)__builtin_fmaf((float)hi.x, -1.f, x), (_Float16)__builtin_fmaf((float)hi.y, -1.f, y)};
          } else {
            hi = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(x, y));
            lo = __builtin_bit_cast(h2, __builtin_amdgcn_cvt_pkrtz(__builtin_fmaf((float)hi.x, -1.f, x),
                                                                   __builtin_fmaf((float)hi.y, -1.f, y)));
          }
          wh[i] = hi.x;
          wh[i + 1] = hi.y;
          wl[i] = lo.x;
          wl[i + 1] = lo.y;
        }
        const char *vp = lds_v + (32 * pw * U + 16 * p + 4 * half + ((lane & 15) >> 2)) * V_PITCH +
                         (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const h8 x = read_tr2(vp + 64 * i, 8 * V_PITCH);
          o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, wh, o[i], 0, 0, 0);
          o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, wl, o[i], 0, 0, 0);
          if constexpr (PAIRS) {
            const h8 y = read_tr2(vp + V_BYTES + 64 * i, 8 * V_PITCH);
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, wh, o[i], 0, 0, 0);
          }
        }
      }
    };
    for (int s = s_first; s < s_last; s += AHEAD) {
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (s + k < s_last) step(steps[k], s + k);
    }

    // the column's average
    sum = halves_reduce<false>(sum);
    if constexpr (BYTES) ref += v_exp;  // (a column that has seen nothing: -inf)
    if (poisoned) sum = __builtin_nanf("");
    if constexpr (WP > 1) {
      __syncthreads();  // the last step has been read
      float *const fold = reinterpret_cast<float *>(lds) + (wave - WC) * 64 * FOLD + lane;
      if (pw > 0) {
#pragma unroll
        for (int i = 0; i < NC * 16; ++i) fold[64 * i] = o[i >> 4][i & 15];
        fold[64 * (NC * 16)] = ref;
        fold[64 * (NC * 16 + 1)] = sum;
        fold[64 * (NC * 16 + 2)] = top_o;
      }
      __syncthreads();
      if (pw > 0) continue;
#pragma unroll
      for (int w = 1; w < WP; ++w) {
        const float *const other = reinterpret_cast<const float *>(lds) + (w * WC + cw - WC) * 64 * FOLD + lane;
        const float ref2 = other[64 * (NC * 16)], sum2 = other[64 * (NC * 16 + 1)], top2 = other[64 * (NC * 16 + 2)];
        const float nr = __builtin_fmaxf(ref, ref2), r = nr == -INFINITY ? 0.f : nr;
        float f = __builtin_amdgcn_exp2f(ref - r), g = __builtin_amdgcn_exp2f(ref2 - r);
        sum = sum * f + sum2 * g;
        ref = nr;
        if constexpr (WIDE) {
          const float nt = __builtin_fmaxf(top_o, top2), t = nt == -INFINITY ? 0.f : nt;
          f = __builtin_amdgcn_exp2f(top_o - t);
          g = __builtin_amdgcn_exp2f(top2 - t);
          top_o = nt;
        }
#pragma unroll
        for (int i = 0; i < NC * 16; ++i) o[i >> 4][i & 15] = o[i >> 4][i & 15] * f + other[64 * i] * g;
      }
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;  // (a NaN sum stays one)
    const float back = WIDE && top_o > -INFINITY ? __builtin_amdgcn_exp2f(top_o - ref) : 1.f;
    const bool whole = s_first == 0 && s_last == ts.steps;
    // (a share's last tile may go on in the next one, its first come from the last)
    const int64_t slot = 2 * me + (s_first == 0 ? 1 : 0);
    const int64_t column = slot * (a.rows_per_tile * group) + c;
    const int64_t out0 = (row * a.n_heads + head) * (int64_t)a.head_dim;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int k = 0; k < 16; k += 4) {
        const int d = 32 * i + 2 * k + 4 * half;
        if (!live || (!EXACT && d >= a.head_dim)) continue;
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = o[i][k + e] * inv * back;
        if (whole) store_row4(a, out0 + d, x);
        else *reinterpret_cast<f32x4 *>(a.part_o + column * a.head_dim + d) = x;
      }
    if (live && !whole && half == 0) {
      a.part_ml[2 * column] = ref;
      a.part_ml[2 * column + 1] = sum;
    }
  }
}

// A running average of the parts of a tile, weighted by their sums against the
// largest reference. (x stays an average, no larger than its V.)
struct TreeFold {
  float mx = -INFINITY, l = 0.f;
  f32x4 x = {};
  __device__ __forceinline__ void add(float m, float sum, const f32x4 &o) {
    const float next = __builtin_fmaxf(mx, m), ref = next == -INFINITY ? 0.f : next;
    const float kept = l * __builtin_amdgcn_exp2f(mx - ref), p = sum * __builtin_amdgcn_exp2f(m - ref);
    l = kept + p;
    const float inv = l != 0.f ? 1.f / l : 0.f;
    x = x * (kept * inv) + o * (p * inv);
    mx = next;
  }
};

// The parts of a tile are folded by the work-groups that have them, each an equal
// piece of its elements (kMergeGroups work-groups a share and kv head; a share has at
// most two such tiles, its first and its last). A thread takes four elements of some
// parts, in order; where the parts are many and the elements few, threads share the
// parts and their averages are folded in LDS. One tree of 8 rows over 4000 positions
// lies in 63 shares: 7.9 us (one work-group a share 6.8, four 11.6); 64 trees of up to
// 16 rows in two or three: 10.2 us (10.6, 10.6).
constexpr int kMergeGroups = 2;

__global__ void __launch_bounds__(kTreeThreads) tree_merge_kernel(TreeArgs a) {
  __shared__ float s_fold[6][kTreeThreads];
  const int tid = (int)threadIdx.x;
  const int tile = (int)(blockIdx.x / kMergeGroups), me = tile >> 1, share = me / a.n_kv_heads;
  const i32x4 r = reinterpret_cast<const i32x4 *>(a.ends)[tile];
  const int kvh = me - share * a.n_kv_heads, group = a.n_heads / a.n_kv_heads, columns = a.rows_per_tile * group;
  const int row0 = r.x, first = r.z, parts = r.w - first + 1;
  if (row0 < 0) return;
  const int all = r.y * group * a.head_dim / 4, pieces = parts * kMergeGroups;
  const int piece = (share - first) * kMergeGroups + (int)(blockIdx.x % kMergeGroups);
  const int v0 = all * piece / pieces, n = all * (piece + 1) / pieces - v0;
  if (n == 0) return;
  // `lanes` elements by `sets` of parts
  int shift = 0;
  while (1 << shift < n && 1 << shift < kTreeThreads) ++shift;
  const int lanes = 1 << shift, sets = kTreeThreads >> shift, set = tid >> shift, lane = tid & (lanes - 1);
  const int each = (parts + sets - 1) >> (8 - shift), w0 = first + set * each, w1 = min(w0 + each, first + parts);
  static_assert(kTreeThreads == 256, "sets are 2^(8 - shift)");
  for (int v = lane; v < ((n + lanes - 1) & ~(lanes - 1)); v += lanes) {
    const int x0 = 4 * (v0 + min(v, n - 1)), c = x0 / a.head_dim, d = x0 - c * a.head_dim;
    constexpr int AHEAD = 4;
    TreeFold fold;
    for (int w = w0; w < w1; w += AHEAD) {
      f32x2 ml[AHEAD];
      f32x4 o[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int p = min(w + i, w1 - 1);
        const int64_t column = (2 * (p * a.n_kv_heads + kvh) + (p == first ? 1 : 0)) * columns + c;
        ml[i] = *reinterpret_cast<const f32x2 *>(a.part_ml + 2 * column);
        o[i] = *reinterpret_cast<const f32x4 *>(a.part_o + column * a.head_dim + d);
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (w + i < w1) fold.add(ml[i].x, ml[i].y, o[i]);
    }
    for (int half = sets >> 1; half > 0; half >>= 1) {
      __syncthreads();  // the last round has been read
      s_fold[0][tid] = fold.mx;
      s_fold[1][tid] = fold.l;
#pragma unroll
      for (int i = 0; i < 4; ++i) s_fold[2 + i][tid] = fold.x[i];
      __syncthreads();
      if (set < half) {
        const int t = tid + half * lanes;
        fold.add(s_fold[0][t], s_fold[1][t], f32x4{s_fold[2][t], s_fold[3][t], s_fold[4][t], s_fold[5][t]});
      }
    }
    if (set == 0 && v < n) {
      const int rr = c / group;
      store_row4(a, (((int64_t)row0 + rr) * a.n_heads + (int64_t)kvh * group + (c - rr * group)) * a.head_dim + d, fold.x);
    }
  }
}

bool tree_tiles_supported(const TreeArgs &a) {
  const int group = a.n_heads / a.n_kv_heads;
  return a.head_dim % 8 == 0 && a.head_dim <= 256 && group <= 64;
}

// Waves that share a step's columns: two where a tile has up to 64 (the other two
// take half of the positions), else four.
int tile_waves(const TreeArgs &a) {
  return a.head_dim <= 128 && (int64_t)a.rows_per_tile * (a.n_heads / a.n_kv_heads) <= 64 ? 2 : 4;
}

template <typename T, int HD, bool EXACT, int WC>
hipError_t launch_tiles(const PoolGeom &g, const TreeArgs &a, hipStream_t s) {
  // (16-bit rows' Q has no lo part. 8 trees of 44 f16 rows behind 32 000 positions of
  // a q8_0 cache, 28/4 heads: 550 us with the products of zeros, 510 without)
  const bool full = a.row_type == LTKV_ROWS_F32 || a.softcap > kShortCap;
  const auto kernel = full ? tree_tile_kernel<T, HD, EXACT, true, WC> : tree_tile_kernel<T, HD, EXACT, false, WC>;
  kernel<<<(unsigned)(a.shares * a.n_kv_heads), kTreeThreads, 0, s>>>(a, g.n_blocks, g.kv_dim);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_tiles_of(const PoolGeom &g, const TreeArgs &a, hipStream_t s) {
  const bool two = tile_waves(a) == 2;
  if (a.head_dim > 128) return launch_tiles<T, 256, false, 4>(g, a, s);
  if (a.head_dim == 64) return two ? launch_tiles<T, 64, true, 2>(g, a, s) : launch_tiles<T, 64, true, 4>(g, a, s);
  if (a.head_dim == 128) return two ? launch_tiles<T, 128, true, 2>(g, a, s) : launch_tiles<T, 128, true, 4>(g, a, s);
  return two ? launch_tiles<T, 128, false, 2>(g, a, s) : launch_tiles<T, 128, false, 4>(g, a, s);
}

}  // namespace

int64_t tree_workspace(int elem, TreeArgs &a) {
  a.rows_per_tile = a.shares = 0;
  if (!tree_tiles_supported(a) || a.max_len == 0) return 0;  // (max_len 0: a cache without blocks)
  const int group = a.n_heads / a.n_kv_heads;
  a.rows_per_tile = (int)std::min<int64_t>(a.max_rows, 32 * kTreeWaves / group);
  // as many work-groups as a CU holds at a time, or as there can be steps
  const int64_t tiles = a.n_rows / a.rows_per_tile + a.n;
  const int64_t steps = tiles * std::max<int64_t>((a.max_len + kTreeTokens - 1) / kTreeTokens, 1);
  const int64_t resident =
      std::max<int64_t>(tree_groups_a_cu(elem == 4, a.head_dim) * a.cu_count / a.n_kv_heads / 8 * 8, 8);
  a.shares = (int)std::min<int64_t>(resident, (steps + 7) / 8 * 8);
  const int64_t groups = (int64_t)a.shares * a.n_kv_heads;
  return 2 * groups * a.rows_per_tile * group * (a.head_dim + 2) * 4 + groups * 8 * 4;
}

void tree_partials(TreeArgs &a, uint8_t *base) {
  a.ends = reinterpret_cast<int32_t *>(base);
  const int64_t groups = (int64_t)a.shares * a.n_kv_heads;
  a.part_o = reinterpret_cast<float *>(base + groups * 8 * 4);
  a.part_ml = a.part_o + 2 * groups * a.rows_per_tile * (a.n_heads / a.n_kv_heads) * a.head_dim;
}

hipError_t launch_tree_attention(const PoolGeom &g, const TreeArgs &a, hipStream_t s) {
  if (a.n <= 0 || a.n_rows <= 0) return hipSuccess;
  if (a.shares == 0) {
    const int64_t grid = a.n_rows * a.n_heads;
    if (grid * kAnyThreads >= (int64_t{1} << 32)) return hipErrorInvalidValue;
    return by_element(g.elem, [&](auto tag) {
      tree_any_kernel<decltype(tag)><<<(unsigned)grid, kAnyThreads, 0, s>>>(a, g.n_blocks, g.kv_dim);
      return hipGetLastError();
    });
  }
  if (const hipError_t e = by_element(g.elem, [&](auto tag) { return launch_tiles_of<decltype(tag)>(g, a, s); });
      e != hipSuccess)
    return e;
  tree_merge_kernel<<<(unsigned)(2 * a.shares * a.n_kv_heads * kMergeGroups), kTreeThreads, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace ltkv
