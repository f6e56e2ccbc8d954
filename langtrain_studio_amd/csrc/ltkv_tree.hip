// gfx950 (MI355X, CDNA4) kernels of attention for trees of drafted tokens.
//
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
        const int32_t w = j >> 5;  // (floor)
        const uint32_t a = w >= 0 && w < words ? (uint32_t)mask[w] : 0u;
        const uint32_t b = w + 1 < words ? (uint32_t)mask[w + 1] : 0u;
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
// is bound by its scalar loads.
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
  for (int32_t t0 = view.from & ~15; t0 < view.len; t0 += kAnyThreads) {
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

}  // namespace

int64_t tree_workspace(int elem, TreeArgs &a) {
  (void)elem;
  a.rows_per_tile = a.groups = 0;
  return 0;
}

void tree_partials(TreeArgs &, uint8_t *) {}

hipError_t launch_tree_attention(const PoolGeom &g, const TreeArgs &a, hipStream_t s) {
  if (a.n <= 0 || a.n_rows <= 0) return hipSuccess;
  const int64_t grid = a.n_rows * a.n_heads;
  if (grid * kAnyThreads >= (int64_t{1} << 32)) return hipErrorInvalidValue;
  return by_element(g.elem, [&](auto tag) {
    tree_any_kernel<decltype(tag)><<<(unsigned)grid, kAnyThreads, 0, s>>>(a, g.n_blocks, g.kv_dim);
    return hipGetLastError();
  });
}

}  // namespace ltkv
