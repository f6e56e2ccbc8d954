// gfx950 (MI355X, CDNA4) kernel of scored attention for single rows (decodes),
// and of decode attention over q4_0 pools, on the matrix cores.

#include "ltkv_scored.h"

namespace ltkv {
namespace {

constexpr int kRowsWaves = 4;
constexpr int kAllButVmem = 0x78f;  // sched_barrier: what may move across (not accesses to global memory)
constexpr int kTopExp = 15;  // f16 operands stay below 2^kTopExp
constexpr int kNoExp = -10000;

// K or V of 16 positions (a block) as a wave loads them: lane (t, quad) =
// (lane & 15, lane >> 4) holds NC chunks of 8 elements of position t. Chunk j of a
// lane is head elements 8 chunk_of(quad, j) ... + 7: a contiguous quarter of the
// head where that makes loads of 16 bytes (SPAN), else 32 j + 8 quad. A block's
// address is uniform over the wave, a lane's place in a block the same for every
// block (load_at).
template <int NC, bool SPAN>
__device__ __forceinline__ int chunk_of(int quad, int j) {
  return SPAN ? quad * NC + j : 4 * j + quad;
}

template <typename T, int NC, bool SPAN>
struct Cells;

template <int NC, bool SPAN>
struct Cells<_Float16, NC, SPAN> {
  u32x4 x[NC];
  struct Place {
    uint32_t at;
    int chunks;  // chunks of the lane inside the head
    __device__ __forceinline__ Place(const ScoredArgs &a, int64_t kv_dim, int64_t head_off, int t, int quad) {
      at = (uint32_t)((t * kv_dim + head_off + chunk_of<NC, SPAN>(quad, 0) * 8) * 2);
      chunks = SPAN ? NC : (a.head_dim / 8 - quad + 3) / 4;
    }
  };
  static __device__ __forceinline__ int64_t block_bytes(int64_t kv_dim) { return kv_dim * 32; }
  __device__ __forceinline__ void load(const char *pool, const char *, int64_t at, const Place &p) {
    const char *base = pool + at;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      if (SPAN || j < p.chunks) x[j] = load_at<u32x4>(base, p.at + j * (SPAN ? 16 : 64));
      else x[j] = u32x4{0, 0, 0, 0};
    }
  }
  __device__ __forceinline__ h8 get(int j) const { return __builtin_bit_cast(h8, x[j]); }
};

template <int NC, bool SPAN>
struct Cells<Q4, NC, SPAN> {
  static constexpr int NS = SPAN ? (NC + 3) / 4 : NC;  // scales a lane needs
  uint32_t x[NC];
  uint32_t s[NS];  // (as 32 bits: a 16-bit value would be waited for to be moved)
  struct Place {
    uint32_t at[SPAN ? 1 : NC];  // of quants; scales lie at an eighth of the group's place
    uint32_t sc[SPAN ? 1 : NC];
    int chunks;
    __device__ __forceinline__ Place(const ScoredArgs &a, int64_t, int64_t head_off, int t, int quad) {
      chunks = SPAN ? NC : (a.head_dim / 8 - quad + 3) / 4;
#pragma unroll
      for (int j = 0; j < (SPAN ? 1 : NC); ++j) {
        const uint32_t e = (uint32_t)head_off + chunk_of<NC, SPAN>(quad, j) * 8, cell = (e >> 5) * 16 + t;
        at[j] = cell * 16 + ((e & 31) >> 3) * 4;
        sc[j] = cell * 2;
      }
    }
  };
  static __device__ __forceinline__ int64_t block_bytes(int64_t kv_dim) { return kv_dim * 8; }
  __device__ __forceinline__ void load(const char *pool, const char *scales, int64_t at, const Place &p) {
    const char *base = pool + at, *sbase = scales + (at >> 3);
    if constexpr (SPAN) {  // the quarter lies in one group, or is whole groups (16 bytes each)
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        s[i] = load_at<uint16_t>(sbase, p.sc[0] + 32 * i);
        if constexpr (NC >= 4) {
          const u32x4 w = load_at<u32x4>(base, p.at[0] + 256 * i);
          x[4 * i] = w.x;
          x[4 * i + 1] = w.y;
          x[4 * i + 2] = w.z;
          x[4 * i + 3] = w.w;
        } else {
          const u32x2 w = load_at<u32x2>(base, p.at[0]);
          x[0] = w.x;
          x[1] = w.y;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        x[j] = 0;
        s[j] = 0;
        if (j < p.chunks) {
          x[j] = load_at<uint32_t>(base, p.at[j]);
          s[j] = load_at<uint16_t>(sbase, p.sc[j]);
        }
      }
    }
  }
  __device__ __forceinline__ h8 get(int j) const {
    const _Float16 d = __builtin_bit_cast(_Float16, (uint16_t)s[SPAN ? j / 4 : j]);
    return q4x8_to_h8(x[j], h2{d, d});
  }
};

// q8_0 elements enter the products as their quants; the scales multiply the
// scores of a 32-element group and the weights of its numerators (SPAN false:
// chunk j of every lane is group j). s[j]: the scales of the lane's four score
// positions 4 quad ... + 3.
template <int NC, bool SPAN>
struct Cells<int8_t, NC, SPAN> {
  static_assert(!SPAN, "a product must stay inside a group");
  u32x2 x[NC];
  u32x2 s[NC];
  struct Place {
    uint32_t at, sc;
    __device__ __forceinline__ Place(const ScoredArgs &, int64_t kv_dim, int64_t head_off, int t, int quad) {
      at = (uint32_t)(t * kv_dim + head_off + 8 * quad);
      sc = (uint32_t)((head_off >> 5) * 32 + quad * 8);
    }
  };
  static __device__ __forceinline__ int64_t block_bytes(int64_t kv_dim) { return kv_dim * 16; }
  __device__ __forceinline__ void load(const char *pool, const char *scales, int64_t at, const Place &p) {
    const char *base = pool + at, *sbase = scales + (at >> 4);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      x[j] = load_at<u32x2>(base, p.at + 32 * j);
      s[j] = load_at<u32x2>(sbase, p.sc + 32 * j);
    }
  }
  __device__ __forceinline__ h8 get(int j) const { return i8x8_to_h8(x[j]); }
  __device__ __forceinline__ h4 scale(int j) const { return __builtin_bit_cast(h4, s[j]); }
};

// f32 elements enter the products as f16 hi + lo parts of the element times a
// power of two, which brings the step's largest below 2^kTopExp (22 bits down to
// 2^16 below it, fewer for smaller elements).
template <int NC, bool SPAN>
struct Cells<float, NC, SPAN> {
  f32x4 x[NC][2];
  struct Place {
    uint32_t at;
    int chunks;
    __device__ __forceinline__ Place(const ScoredArgs &a, int64_t kv_dim, int64_t head_off, int t, int quad) {
      at = (uint32_t)((t * kv_dim + head_off + chunk_of<NC, SPAN>(quad, 0) * 8) * 4);
      chunks = SPAN ? NC : (a.head_dim / 8 - quad + 3) / 4;
    }
  };
  static __device__ __forceinline__ int64_t block_bytes(int64_t kv_dim) { return kv_dim * 64; }
  __device__ __forceinline__ void load(const char *pool, const char *, int64_t at, const Place &p) {
    const char *base = pool + at;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      if (SPAN || j < p.chunks) {
        x[j][0] = load_at<f32x4>(base, p.at + j * (SPAN ? 32 : 128));
        x[j][1] = load_at<f32x4>(base, p.at + j * (SPAN ? 32 : 128) + 16);
      } else {
        x[j][0] = x[j][1] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < NC; ++j) x[j][0] = x[j][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  template <bool FINITE>
  __device__ __forceinline__ float largest() const {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = __builtin_fabsf(x[j][i >> 2][i & 3]);
        m = __builtin_fmaxf(m, FINITE && !(y < INFINITY) ? 0.f : y);
      }
    return m;
  }
  __device__ __forceinline__ void get2(int j, int e, h8 &hi, h8 &lo) const {  // times 2^e
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      _Float16 a, b;
      split2(__builtin_amdgcn_ldexpf(x[j][i >> 2][i & 3], e), a, b);
      hi[i] = a;
      lo[i] = b;
    }
  }
};

// Maximum over the wave, in every lane.
__device__ __forceinline__ float wave_max(float x) {
  x = __builtin_fmaxf(x, dpp<0xB1>(x));   // quad_perm [1,0,3,2]
  x = __builtin_fmaxf(x, dpp<0x4E>(x));   // quad_perm [2,3,0,1]
  x = __builtin_fmaxf(x, dpp<0x141>(x));  // row_half_mirror
  x = __builtin_fmaxf(x, dpp<0x140>(x));  // row_mirror
  return rows_reduce<true>(x);
}

// Steps of a part of a row that takes n steps.
__device__ __forceinline__ int steps_per_part(const ScoredArgs &a, int n) {
  const int per_part = scored_part_tokens((int64_t)n * 32, a.part_tokens) >> 5;
  // (never more parts than there is memory for)
  return (int64_t)per_part * a.max_parts < n ? (n + a.max_parts - 1) / a.max_parts : per_part;
}

// What a launch of the rows kernel takes: plain decode attention, one row per
// sequence over its whole context; rows of short sequences with any scoring; or
// packs of consecutive rows of a sequence, which share the columns.
enum class Take { kDecode, kRows, kPacks };

// Parts of a sequence of one row.
template <bool MODS>
__device__ __forceinline__ int parts_of(const ScoredArgs &a, int64_t seq) {
  const int64_t len = a.lens[seq];
  const int32_t cut = (int32_t)(len < 0 ? 0 : len > a.max_len ? a.max_len : len);
  int n = (cut + 31) / 32;
  if constexpr (MODS) n = step_range<32>(row_view(a, SeqRows{seq, 1, cut}, seq, 0)).n;
  const int per_part = steps_per_part(a, n);
  return n > per_part ? (n + per_part - 1) / per_part : 1;
}

// A wave takes a run of parts of one row's visible positions for one kv head
// (four waves of a work-group: neighbouring kv heads, whose cells lie together).
// It streams through 32-position steps, the next one in flight, and writes each
// part's numerators, reference and sum (one part: the output). Per step, on
// 16x16x32 products: scores^T = K Q^T (16 positions x the group's query heads as
// columns, twice), weights from the scores in place, numerators^T += V^T W: the
// score tiles' lane layout (4 quad + r, column) is the operand layout of the
// second product when its 32 positions are taken as (tile 0: 4 quad ... + 3,
// tile 1: 4 quad ... + 3), so weights move between no lanes. V is transposed on
// its way through LDS (ds_read_b64_tr_b16). Q and the weights enter as f16
// hi + lo pairs: f32 accuracy for twice the matrix-core work, which is idle
// here otherwise. A pack's steps that some row sees in part are taken once for
// each row, with the other rows' columns masked and unseen values as zeros: no
// row's values meet another's infinities, or its powers of two.
// OCC: waves a SIMD that the registers are cut to.
//
// Bound by the vector ALU: a step of 32 q4_0 positions of 128 elements is ~300
// vector instructions (11 a dword of quants), 16 stores to LDS and 32 products,
// ~3100 cycles for a wave alone. 64 decodes of 2048 .. 4096 tokens at 32 / 8
// heads of 128 take 62.7 us + 5.9 us of merge (226 MB, 3.3 TB/s; 4.5 TB/s inside
// the loop, the rest is the start of the waves and their uneven end), 8 of 32 700
// at 28 / 4 heads 47 us (151 MB). One context of 5 003 tokens is 160 waves of 8
// steps: 15.2 us. Four waves that shared a part and folded it in LDS were faster
// where there are few parts (12 short q8_0 rows in 17 us instead of 21) and
// slower for full batches (81 us against 71 for these 64).
template <typename T, int HDP, bool SPAN, Take TAKE, int OCC>
__global__ void __launch_bounds__(64 * kRowsWaves, OCC)
scored_rows_kernel(ScoredArgs a, int64_t n_blocks, int64_t kv_dim, int head_tiles, int64_t waves, int64_t share,
                   int64_t most_rows) {
  constexpr bool MODS = TAKE != Take::kDecode, PACK = TAKE == Take::kPacks;
  constexpr int NC = HDP / 32;     // chunks of 8 elements a lane, products per score tile
  constexpr int ND = HDP / 16;     // 16-element tiles of the numerators
  constexpr int PITCH = HDP * 2 + 32;  // bytes of a V row in LDS: rows of a read start 8 banks apart
  constexpr bool Q8 = std::is_same_v<T, int8_t>, F32 = std::is_same_v<T, float>;
  constexpr int V_BYTES = 32 * PITCH * (F32 ? 2 : 1);  // f32: hi parts, then lo parts
  __shared__ __align__(16) char lds[kRowsWaves * V_BYTES];

  const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int group = a.n_heads / a.n_kv_heads;
  uint32_t b = blockIdx.x * kRowsWaves + (uint32_t)wave;
  if ((int64_t)b >= waves) return;
  const int head_tile = (int)(b % (uint32_t)head_tiles);
  b /= (uint32_t)head_tiles;
  const int kvh = (int)(b % (uint32_t)a.n_kv_heads);
  b /= (uint32_t)a.n_kv_heads;
  // Few parts: a wave for each that a sequence (or row) could have, the last
  // ones slowest, so that those past the end of shorter contexts come last. Many
  // (share > 0): every sequence has one row, and wave b of `share` takes the
  // b-th of as many equal stretches of all parts in sequence order.
  const int pack = PACK ? pack_rows(a) : 1;
  const uint32_t items = (uint32_t)(PACK ? a.n_rows / pack + a.n : a.n);
  int64_t item = b % items;
  int p_first = (int)(b / items), p_count = 1;
  if (share > 0) {
    auto scan = [&](int64_t i0, int &own) {  // inclusive sums of 64 sequences' parts, from i0 on
      own = i0 + lane < a.n ? parts_of<MODS>(a, i0 + lane) : 0;
      int x = own;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(x, off, 64);
        if (lane >= off) x += y;
      }
      return x;
    };
    int own, x = scan(0, own);
    int64_t total = __builtin_amdgcn_readlane(x, 63);
    for (int64_t i0 = 64; i0 < a.n; i0 += 64) {
      int rest;
      total += __builtin_amdgcn_readlane(scan(i0, rest), 63);
    }
    const int64_t p0 = total * b / share, p1 = total * (b + 1) / share;
    if (p0 == p1) return;
    // the sequence of part p0
    int64_t before = 0;
    for (item = 0; item < a.n; item += 64) {
      if (item > 0) x = scan(item, own);
      const int sum = __builtin_amdgcn_readlane(x, 63);
      if (before + sum > p0) {
        const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(before + x > p0));
        p_first = (int)(p0 - before) - (__builtin_amdgcn_readlane(x, at) - __builtin_amdgcn_readlane(own, at));
        item += at;
        break;
      }
      before += sum;
    }
    p_count = (int)(p1 - p0);
  }
  const int cols = min(16, group - head_tile * 16);
  const int head0 = kvh * group + head_tile * 16;
  const int sub = pack > 1 ? col / group : 0;  // the column's row of a pack
  const int head = head0 + col - sub * group;
  const int64_t head_off = (int64_t)kvh * a.head_dim;
  char *const my = lds + wave * V_BYTES;
  const typename Cells<T, NC, SPAN>::Place place(a, kv_dim, head_off, col, quad);

  // an item is a sequence, whose rows are taken one after the other, or a pack
  for (int r_next = -1; p_count > 0;) {
    const int64_t seq = PACK ? seq_of_slot(a, item, pack) : item;
    SeqRows rows = seq_rows(a, seq);
    if constexpr (!MODS) {
      rows.row0 = seq;
      rows.count = 1;
    }
    if constexpr (PACK) r_next = (int)(item - first_slot(a, seq, pack)) * pack;
    else ++r_next;
    if (rows.count > most_rows || r_next < 0 || r_next >= rows.count) return;
    const int r = r_next;
    const int n_pack = PACK ? min(pack, rows.count - r) : 1;
    const bool live = PACK && pack > 1 ? sub < n_pack : col < cols;
    const int32_t *tab = table_of(a.tables, a.table_stride, a.rows, a.table_rows, seq);
    if (a.rows && p_first == 0 && rows.len > 0) {
      const int32_t t = scalar_read(a.rows, seq);
      if (t < 0 || t >= a.table_rows) report_fault(a.status, kFaultTable, seq);
    }
    // a pack: all that its rows see (seen), and what each of them sees (whole_*)
    RowView view = MODS ? row_view(a, rows, seq, r) : RowView{rows.len - 1, 0, 0, 0, rows.len};
    RowView seen = view;
    int32_t whole_first = view.first, whole_from = view.from, whole_sink_end = view.sink_end, whole_end = view.end;
    if constexpr (PACK)
      for (int i = 1; i < n_pack; ++i) {
        const RowView w = row_view(a, rows, seq, r + i);
        whole_first = max(whole_first, w.first);
        whole_from = max(whole_from, w.from);
        whole_sink_end = min(whole_sink_end, w.sink_end);
        whole_end = min(whole_end, w.end);
        if (w.end <= w.first) continue;
        if (seen.end <= seen.first) {
          seen = w;
          continue;
        }
        seen.first = min(seen.first, w.first);
        seen.from = min(seen.from, w.from);
        seen.sink_end = max(seen.sink_end, w.sink_end);
        seen.end = max(seen.end, w.end);
      }
    const int32_t pos = view.pos + sub;  // of the column's row
    const StepRange<32> range =
        MODS ? step_range<32>(seen) : StepRange<32>{0, 0, 0, rows.len, 0, (rows.len + 31) / 32};
    int per_part = steps_per_part(a, range.n);
    // no memory for the parts of rows past the expected most: one part
    const bool parted = !MODS || PACK || r < a.max_rows;
    if (!parted) per_part = max(range.n, 1);
    const int n_parts = range.n > per_part ? (range.n + per_part - 1) / per_part : 1;
    const int64_t row = rows.row0 + r + sub;  // the column's
    const int64_t slot = PACK ? item * pack + sub : MODS ? seq * a.max_rows + r : row;
    if (a.part_n && parted && p_first == 0 && kvh == 0 && head_tile == 0 &&
        (PACK ? live && quad == 0 && head == 0 : lane == 0))
      a.part_n[slot] = n_parts;
    int part = p_first;
    // this item's stretch, and what follows it
    const int here = min(p_count, n_parts - p_first);
    if (share > 0) {
      p_count -= here;
      p_first = 0;
      ++item;
      r_next = -1;
    } else if (PACK) {
      p_count = 0;
    }
    if (here <= 0) continue;
    const int s_first = part * per_part, s_end = min(range.n, (part + here) * per_part);

    // block ids of the next 32 steps, two a step, one a lane
    int entry = 0, entry_step = s_first;
    auto fill = [&](int s0) {
      const int s = s0 + (lane >> 1);
      const int32_t t = range.start(s) + 16 * (lane & 1);
      const bool valid = s < s_end && t < range.end(s);
      entry = valid ? tab[t >> 4] : 0;
      entry_step = s0;
      bool bad = entry < 0 || entry >= n_blocks;
      if (bad) entry = 0;
      if constexpr (PACK)
        if (__builtin_amdgcn_ballot_w64(bad)) {  // (between the rows' ranges may lie blocks that none of them sees)
          bool needed = false;
          for (int i = 0; i < n_pack; ++i) needed |= row_view(a, rows, seq, r + i).sees_of_block(t);
          bad &= needed;
        }
      if (__builtin_amdgcn_ballot_w64(bad)) report_fault(a.status, kFaultTable, seq);
    };
    Cells<T, NC, SPAN> k[2], v[2];
    int64_t at[2];  // byte offsets of the next step's blocks
    const int64_t block_bytes = Cells<T, NC, SPAN>::block_bytes(kv_dim);
    auto find = [&](int s) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
        at[u] = (int64_t)(uint32_t)__builtin_amdgcn_readlane(entry, 2 * (s - entry_step) + u) * block_bytes;
    };
    auto load = [&](Cells<T, NC, SPAN> (&c)[2], const void *pool, const void *scales) {
      // not before the last use of what it replaces (the loaded registers would be
      // copied, and so waited for)
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < 2; ++u)
        c[u].load(static_cast<const char *>(pool), static_cast<const char *>(scales), at[u], place);
      // V, K, V, K ... in this order everywhere: a wait then leaves the later ones
      // in flight
      __builtin_amdgcn_sched_barrier(kAllButVmem);
    };
    if (s_first < s_end) {
      fill(s_first);
      find(s_first);
      load(v, a.v_layer, a.v_scale);
      load(k, a.k_layer, a.k_scale);
    }

    // Q columns, scaled by a power of two so that the head's largest element
    // lies in [2^9, 2^10): any magnitude enters f16 with 22 bits
    h8 qh[NC], ql[NC];
    int q_exp;  // Q entered times 2^q_exp
    {
      float x[NC][8], amax = 0.f;
      const int64_t at = (row * a.n_heads + head) * (int64_t)a.head_dim;
#pragma unroll
      for (int j = 0; j < NC; ++j) {
        const int e = chunk_of<NC, SPAN>(quad, j) * 8;
        load_row8(a, at + e, live && (SPAN || e < a.head_dim), x[j]);
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = __builtin_fmaxf(amax, __builtin_fabsf(x[j][i]));
      }
      amax = rows_reduce<true>(amax);
      // (at most 100: a smaller row's scores are nothing beside their rounding)
      q_exp = amax > 0.f && amax < INFINITY ? min(10 - __builtin_amdgcn_frexp_expf(amax), 100) : 0;
#pragma unroll
      for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          _Float16 hi, lo;
          split2(__builtin_amdgcn_ldexpf(x[j][i], q_exp), hi, lo);
          qh[j][i] = hi;
          ql[j][i] = lo;
        }
    }
    const bool cap = MODS && a.softcap > 0.f;
    const float factor = cap ? a.scale / a.softcap : a.scale * kLog2e, in_scale = score_factor(factor, -q_exp);
    const float cap_scale = a.softcap * kLog2e;
    const float slope = MODS && a.slopes && live ? a.slopes[head] * kLog2e : 0.f;

    f32x4 o[ND];
    float ref, sum, lift, scale_top;
    int v_exp;  // f32: numerators are sums of V times 2^-v_exp (a pack: of the column's row)
    auto reset = [&]() {
#pragma unroll
      for (int i = 0; i < ND; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      ref = -INFINITY;
      sum = 0.f;
      lift = Q8 ? 0.f : kLift;
      scale_top = 0.f;  // q8_0: no scale has exceeded it
      v_exp = kNoExp;
    };
    auto flush = [&]() {
      float total = rows_reduce<false>(sum);
      if (!live) return;
      const int64_t rh = row * a.n_heads + head;
      float inv = n_parts == 1 ? total != 0.f ? 1.f / total : 0.f : 1.f;
      int lower = 0;
      if constexpr (F32) {
        // Numerators are up to 2^23 and more times their V: of values near f32's
        // largest they are divided first (one part), or lowered with their sum, as
        // weights of a reference that much higher.
        const int e = v_exp == kNoExp ? 0 : v_exp;
        if (n_parts > 1 && e > 60) lower = 40;
        total = __builtin_amdgcn_ldexpf(total, -lower);
        const float f = __builtin_amdgcn_ldexpf(1.f, (e - lower) / 2);
        const float g = __builtin_amdgcn_ldexpf(1.f, e - lower - (e - lower) / 2);
#pragma unroll
        for (int i = 0; i < ND; ++i) o[i] = o[i] * inv * f * g;
        inv = 1.f;
      }
      if (n_parts == 1) {
#pragma unroll
        for (int i = 0; i < ND; ++i)
          if (SPAN || 16 * i + 4 * quad < a.head_dim)
            store_row4(a, rh * a.head_dim + 16 * i + 4 * quad, o[i] * inv);
        return;
      }
      const int64_t at = (slot * a.n_heads + head) * a.max_parts + part;
      float *dst = a.part_o + at * a.head_dim + 4 * quad;
#pragma unroll
      for (int i = 0; i < ND; ++i)
        if (SPAN || 16 * i + 4 * quad < a.head_dim) *reinterpret_cast<f32x4 *>(dst + 16 * i) = o[i];
      if (quad == 0) {
        a.part_ml[2 * at] = ref - lift + (float)lower;
        a.part_ml[2 * at + 1] = total;
      }
    };

    int turn = 0;  // row of a pack that a step in part is taken for
    auto step = [&](int s) {  // true: done
      const int32_t t0 = range.start(s), t_end = range.end(s);
      const bool whole = t0 + 32 <= (PACK ? min(t_end, whole_end) : t_end) && t0 >= whole_first &&
                         (t0 >= whole_from || t0 + 32 <= whole_sink_end);
      auto visible = [&](int32_t t) { return MODS ? view.sees(t) & (t < t_end) : t < t_end; };
      const bool again = PACK && !whole && turn + 1 < n_pack;
      const bool mine = !PACK || whole || sub == turn;
      if constexpr (PACK)
        if (!whole) view = row_view(a, rows, seq, r + turn);
      turn = again ? turn + 1 : 0;
      // always loaded, so that the loads in flight are counted exactly: past the
      // end the last step again
      const int s_next = again ? s : min(s + 1, s_end - 1);
      if (s_next - entry_step == 32) fill(s_next);
      find(s_next);
      // f32: powers of two that bring K and V below 2^kTopExp (positions that the
      // row does not see count as zeros)
      int k_exp = 0, stage_exp = 0;
      float v_share = 1.f;  // a pack's weights times this: what V entered divided by over the column's 2^v_exp
      if constexpr (F32) {
        if (!whole)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int32_t t = t0 + 16 * u + col;
            if (!visible(t)) {
              k[u].clear();
              v[u].clear();
            }
          }
        auto most = [](const Cells<T, NC, SPAN> (&c)[2]) {  // of the finite elements
          float m = wave_max(__builtin_fmaxf(c[0].template largest<false>(), c[1].template largest<false>()));
          if (__builtin_amdgcn_readfirstlane(m == INFINITY))
            m = wave_max(__builtin_fmaxf(c[0].template largest<true>(), c[1].template largest<true>()));
          return m;
        };
        auto exponent = [](float m) {  // m < 2^e
          return __builtin_amdgcn_readfirstlane(m > 0.f ? __builtin_amdgcn_frexp_expf(m) : 0);
        };
        k_exp = exponent(most(k)) - kTopExp;
        const float m = most(v);
        const int e = exponent(m) - kTopExp;
        if constexpr (PACK) {
          // Each row keeps a power of its own: one that follows what another row
          // sees would cost it its bits.
          if (__builtin_amdgcn_readfirstlane(m > 0.f)) {
            stage_exp = e;
            const int to = mine ? max(v_exp, e) : v_exp;
            if (__builtin_amdgcn_ballot_w64(to > v_exp)) {
              const float f = __builtin_amdgcn_ldexpf(1.f, v_exp - to);  // (0 the first time: no numerators yet)
#pragma unroll
              for (int i = 0; i < ND; ++i) o[i] *= f;
              v_exp = to;
            }
            v_share = mine ? __builtin_amdgcn_ldexpf(1.f, e - v_exp) : 0.f;
          }
        } else if (__builtin_amdgcn_readfirstlane(m > 0.f) && e > v_exp) {
          if (v_exp != kNoExp) {
            const float f = __builtin_amdgcn_ldexpf(1.f, v_exp - e);
#pragma unroll
            for (int i = 0; i < ND; ++i) o[i] *= f;
          }
          v_exp = e;
        }
        if constexpr (!PACK) stage_exp = v_exp == kNoExp ? 0 : v_exp;
      }
      // V into LDS (positions that the row does not see as zeros); the scores are
      // computed while it settles
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int32_t t = t0 + 16 * u + col;
        const bool seen = whole || visible(t);
        if constexpr (F32) {
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            h8 hi, lo;
            v[u].get2(j, -stage_exp, hi, lo);
            char *p = my + (16 * u + col) * PITCH + chunk_of<NC, SPAN>(quad, j) * 16;
            *reinterpret_cast<h8 *>(p) = hi;
            *reinterpret_cast<h8 *>(p + 32 * PITCH) = lo;
          }
          continue;
        } else
#pragma unroll
        for (int j = 0; j < NC; ++j) {
          h8 y = v[u].get(j);
          if constexpr (std::is_same_v<T, _Float16>)
            if (!seen) y = h8{};
          *reinterpret_cast<h8 *>(my + (16 * u + col) * PITCH + chunk_of<NC, SPAN>(quad, j) * 16) = y;
        }
      }
      h4 dv[2][Q8 ? NC : 1];
      if constexpr (Q8) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            dv[u][j] = v[u].scale(j);
            if (!whole)  // a scale of an unseen position may be infinite
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int32_t t = t0 + 16 * u + 4 * quad + i;
                if (!visible(t)) dv[u][j][i] = (_Float16)0.f;
              }
          }
      }
      load(v, a.v_layer, a.v_scale);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");

      // scores
      f32x4 c[2], cl[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        c[u] = cl[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (Q8) {
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            const h8 y = k[u].get(j);
            f32x4 g = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, qh[j], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            g = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, ql[j], g, 0, 0, 0);
            const h4 d = k[u].scale(j);
#pragma unroll
            for (int i = 0; i < 4; ++i) c[u][i] = __builtin_fmaf((float)d[i], g[i], c[u][i]);
          }
        } else if constexpr (F32) {
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            h8 hi, lo;
            k[u].get2(j, -k_exp, hi, lo);
            c[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, qh[j], c[u], 0, 0, 0);
            cl[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, ql[j], cl[u], 0, 0, 0);
            cl[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, qh[j], cl[u], 0, 0, 0);
          }
        } else {  // (two chains of dependent products)
#pragma unroll
          for (int j = 0; j < NC; ++j) {
            const h8 y = k[u].get(j);
            c[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, qh[j], c[u], 0, 0, 0);
            cl[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y, ql[j], cl[u], 0, 0, 0);
          }
        }
      }
      load(k, a.k_layer, a.k_scale);
      // V^T operands: on their way during the softmax (f32: too many registers)
      const char *const my_t = my + (4 * quad + (col >> 2)) * PITCH + 4 * (col & 3) * 2;
      h8 vt[F32 ? 1 : ND];
      if constexpr (!F32) {
#pragma unroll
        for (int i = 0; i < ND; ++i) vt[i] = read_tr2(my_t + 32 * i, 16 * PITCH);
      }
      const float to_y = F32 ? score_factor(factor, k_exp - q_exp) : in_scale;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y = (Q8 ? c[u][i] : c[u][i] + cl[u][i]) * to_y;
          if constexpr (MODS) {
            if (cap) y = tanh_f32(y) * cap_scale;
            y = __builtin_fmaf(-slope, (float)abs(pos - (t0 + 16 * u + 4 * quad + i)), y);
          }
          c[u][i] = y;
        }
      if (!whole)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int32_t t = t0 + 16 * u + 4 * quad + i;
            if constexpr (!MODS) {
              if (!(t < t_end)) c[u][i] = -INFINITY;
            } else {
              c[u][i] = (mine & visible(t)) ? c[u][i] : -INFINITY;
            }
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
      if constexpr (Q8) {
        h4 most = {};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < NC; ++j) most = __builtin_elementwise_max(most, dv[u][j]);
        const float top_d = __builtin_fmaxf(__builtin_fmaxf((float)most[0], (float)most[1]),
                                            __builtin_fmaxf((float)most[2], (float)most[3]));
        if (__builtin_amdgcn_ballot_w64((top_d > scale_top) & mine)) {
          const float d = __builtin_fminf(rows_reduce<true>(top_d), 65504.f);  // the same in every column
          const int ex = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_frexp_expf(d));
          // (a pack: only of the rows that see the scale, and not met a larger one)
          const float to_top = __builtin_amdgcn_ldexpf(1.f, ex);
          const bool raise = !PACK | (mine & (to_top > scale_top));
          const float next = raise ? (float)(kTopExp - ex) - kSlack : lift, f = __builtin_amdgcn_exp2f(next - lift);
          sum *= f;
#pragma unroll
          for (int i = 0; i < ND; ++i) o[i] *= f;
          lift = next;
          scale_top = raise ? to_top : scale_top;
        }
      }
      const float base = (ref == -INFINITY ? 0.f : ref) - lift;
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = __builtin_amdgcn_exp2f(c[i >> 2][i & 3] - base);
        sum += w[i];
      }
      // a column whose row is not taken keeps its numerators: values that another
      // row sees may be infinite, and zero weights would not hide that
      auto keep = [&](f32x4 &to, const f32x4 &x) {
        if constexpr (!PACK) to = x;
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) to[e] = mine ? x[e] : to[e];
      };
      h8 wh, wl;
      if constexpr (!Q8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          _Float16 hi, lo;
          split2(F32 && PACK ? w[i] * v_share : w[i], hi, lo);
          wh[i] = hi;
          wl[i] = lo;
        }
        if constexpr (F32) {
#pragma unroll
          for (int i = 0; i < ND; ++i) {
            const h8 hi = read_tr2(my_t + 32 * i, 16 * PITCH), lo = read_tr2(my_t + 32 * PITCH + 32 * i, 16 * PITCH);
            f32x4 x = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, wh, o[i], 0, 0, 0);
            x = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, wl, x, 0, 0, 0);
            x = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, wh, x, 0, 0, 0);
            keep(o[i], x);
          }
        } else if constexpr (PACK) {
#pragma unroll
          for (int i = 0; i < ND; ++i) {
            f32x4 x = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt[i], wh, o[i], 0, 0, 0);
            x = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt[i], wl, x, 0, 0, 0);
            keep(o[i], x);
          }
        } else {
#pragma unroll
          for (int i = 0; i < ND; ++i) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt[i], wh, o[i], 0, 0, 0);
#pragma unroll
          for (int i = 0; i < ND; ++i) o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt[i], wl, o[i], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          if (i % 2 == 0) {  // a group's two tiles share its weights
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              _Float16 hi, lo;
              split2(w[e] * (float)dv[e >> 2][i / 2][e & 3], hi, lo);
              wh[e] = hi;
              wl[e] = lo;
            }
          }
          f32x4 x = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt[i], wh, o[i], 0, 0, 0);
          x = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt[i], wl, x, 0, 0, 0);
          keep(o[i], x);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      return !again;
    };

    reset();
    int left = per_part;  // steps until the part ends
    for (int s = s_first; s < s_end; ++s) {
      if constexpr (PACK) {
        while (!step(s)) {
        }
      } else {
        step(s);
      }
      if (--left == 0 && s + 1 < s_end) {
        flush();
        reset();
        left = per_part;
        ++part;
      }
    }
    flush();
  }
}

template <typename T, int HDP, bool SPAN>
hipError_t launch_rows_t(const PoolGeom &g, const ScoredArgs &a, int64_t most_rows, hipStream_t s) {
  const int group = a.n_heads / a.n_kv_heads, head_tiles = (group + 15) / 16;
  constexpr int occ = HDP <= 64 ? 3 : HDP <= 128 ? (std::is_same_v<T, Q4> ? 3 : 2) : 1;
  // a wave for each possible part, or all parts shared by as many as are resident
  const int64_t lanes = (int64_t)a.n_kv_heads * head_tiles, slots = std::max<int64_t>(a.cu_count * 4 * occ / lanes, 1);
  int64_t waves = (a.packs ? pack_slots(a) : a.n) * a.max_parts, share = 0;
  if (waves > slots && !a.row_starts) waves = share = slots;
  waves *= lanes;
  const int64_t wgs = (waves + kRowsWaves - 1) / kRowsWaves;
  if (wgs * 64 * kRowsWaves >= (int64_t{1} << 32)) return hipErrorInvalidValue;
  const bool mods = a.softcap > 0.f || a.slopes || a.window > 0 || a.prefix || a.first || a.row_starts;
  const auto kernel = a.packs ? scored_rows_kernel<T, HDP, SPAN, Take::kPacks, occ>
                      : mods  ? scored_rows_kernel<T, HDP, SPAN, Take::kRows, occ>
                              : scored_rows_kernel<T, HDP, SPAN, Take::kDecode, occ>;
  kernel<<<(unsigned)wgs, 64 * kRowsWaves, 0, s>>>(a, g.n_blocks, g.kv_dim, head_tiles, waves, share, most_rows);
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
  if constexpr (!std::is_same_v<T, float>) {
    if (a.head_dim <= 192) return launch_rows_t<T, 192, false>(g, a, most_rows, s);
    return launch_rows_t<T, 256, false>(g, a, most_rows, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

// q8_0: a head's 32-element products are whole groups, and none is padded. f32:
// wider heads would leave no registers for the next step.
bool scored_rows_supported(int elem, int head_dim) {
  if (head_dim % 8 != 0 || head_dim > (elem == 4 ? 128 : 256)) return false;
  return elem != 1 || head_dim == 32 || head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 192 ||
         head_dim == 256;
}

hipError_t launch_scored_rows(const PoolGeom &g, const ScoredArgs &a, int64_t most_rows, hipStream_t s) {
  if (g.elem == kElemQ4) return launch_rows_hd<Q4>(g, a, most_rows, s);
  if (g.elem == 1) return launch_rows_hd<int8_t>(g, a, most_rows, s);
  if (g.elem == 4) return launch_rows_hd<float>(g, a, most_rows, s);
  return launch_rows_hd<_Float16>(g, a, most_rows, s);
}

}  // namespace ltkv
