// Device helpers shared by the kernel sources (ltkv_kernels.hip and
// ltkv_scored.hip): vector types, fault reports, block tables, wave and
// work-group reductions, conversions of stored elements.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace ltkv {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef __fp16 hf4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
typedef __attribute__((address_space(3))) hf4 lds_hf4;
typedef __attribute__((address_space(3))) char lds_char;

// Fault bits of a cache's status word (reported by ltkv_synchronize).
constexpr int kFaultTable = 1;      // a block-table entry outside the pool
constexpr int kFaultFusedCell = 2;  // a fused append's cell is not position len - 1 of its table

// ds_read_b64_tr_b16: within each 16-lane group, lane i receives element
// i % 4 of the 8 bytes addressed by lane 4 j + i / 4 as its element j.
__device__ __forceinline__ hf4 lds_read_tr(const char *p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4f16((lds_hf4 *)(lds_char *)p);
}

// ----------------------------------------------------------------------------
// f32 -> f16, IEEE round-to-nearest-even (the conversion of f16::from_f32).
// v_cvt_f16_f32 rounds to nearest even in the default mode; NaN is rewritten
// explicitly so the result is sign | 0x7e00 | top payload bits on every part.
// ----------------------------------------------------------------------------
__device__ __forceinline__ uint32_t f16_bits(float x) {
  const _Float16 h = (_Float16)x;
  uint32_t b = (uint32_t)__builtin_bit_cast(uint16_t, h);
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  if ((u & 0x7fffffffu) > 0x7f800000u) b = ((u >> 16) & 0x8000u) | 0x7e00u | ((u >> 13) & 0x3ffu);
  return b;
}

__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  return f16_bits(a) | (f16_bits(b) << 16);
}

// DPP move of x (row_mask and bank_mask all set).
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(
      float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}

// Scale entry of (cell s, group g): layout [block][kv_dim / 32][16 slots],
// so the scales of one kv head of a block are one contiguous run.
__device__ __forceinline__ int64_t scale_index(int32_t s, int g, int kg) {
  return (((int64_t)(s >> 4) * kg + g) << 4) + (s & 15);
}

constexpr float kLog2e = 1.4426950408889634f;

// Block table of query qi: row qi of `tables`, or, with resident tables, row
// rows[qi] (a row outside [0, n_rows) reads row 0: such a query must have
// length 0, and nothing is read then).
__device__ __forceinline__ const int32_t *table_of(const int32_t *tables, int64_t stride,
                                                   const int32_t *rows, int64_t n_rows, int64_t qi) {
  int64_t r = qi;
  if (rows) {
    r = ((const __attribute__((address_space(4))) int32_t *)rows)[qi];  // uniform: the scalar cache
    if (r < 0 || r >= n_rows) r = 0;
  }
  return tables + r * stride;
}

// Faults a device op met, for ltkv_synchronize to report (the reference
// panics at the same places): status[0] ORs the fault bits, status[1] holds
// the query of one of them. The op goes on safely (a bad entry reads block
// 0), so nothing faults on the GPU.
// A wave-uniform read of memory no thread writes during the launch (block
// tables, lengths), through the scalar cache: the constant address space
// tells the compiler so, where stores elsewhere in the kernel would keep it
// from proving it.
__device__ __forceinline__ int32_t scalar_read(const int32_t *p, int64_t i) {
  return ((const __attribute__((address_space(4))) int32_t *)p)[i];
}

// Every calling lane stores the same bits and query: no lane test, so values
// the caller computes around a report stay uniform over the wave.
__device__ __forceinline__ void report_fault(int32_t *status, int code, int64_t qi) {
  if (!status) return;
  __hip_atomic_fetch_or(status, code, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  status[1] = (int32_t)qi;
}

// Checks the table entries of blocks [b0, b1) (the positions a work-group
// reads: kv.rs:147 indexes the sequence's blocks with them) and the query's
// row in the resident tables; run once before the tile loop, one wave.
__device__ __forceinline__ void check_table(const int32_t *tab, int b0, int b1, int64_t n_blocks,
                                            const int32_t *rows, int64_t n_rows, int64_t qi, int32_t *status) {
  if (!status || b1 <= b0) return;
  bool bad = false;
  if (rows) {
    const int32_t r = rows[qi];
    bad = r < 0 || r >= n_rows;  // such a query must have length 0
  }
  for (int b = b0 + (int)(threadIdx.x & 63); b < b1 && !bad; b += 64) {
    const int32_t blk = tab[b];
    bad = blk < 0 || blk >= n_blocks;
  }
  if (__builtin_amdgcn_ballot_w64(bad)) report_fault(status, kFaultTable, qi);
}

// Stored quants x 8 (bytes u = x + 128) -> f16 x 8 of x, exact: each byte
// becomes the mantissa of an f16 in [1024, 1280) (bits 0x6400 | u, value
// 1024 + u), and 1152 is subtracted: two v_perm_b32 and two packed f16
// subtractions per four elements.
__device__ __forceinline__ h8 i8x8_to_h8(const u32x2 &w) {
  constexpr uint32_t kHi = 0x64646464u;
  const uint32_t a = w.x, b = w.y;
  const h2 bias = {(_Float16)1152.f, (_Float16)1152.f};
  const h2 p0 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(kHi, a, 0x04010400u)) - bias;
  const h2 p1 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(kHi, a, 0x04030402u)) - bias;
  const h2 p2 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(kHi, b, 0x04010400u)) - bias;
  const h2 p3 = __builtin_bit_cast(h2, __builtin_amdgcn_perm(kHi, b, 0x04030402u)) - bias;
  return h8{p0.x, p0.y, p1.x, p1.y, p2.x, p2.y, p3.x, p3.y};
}

// Sum / maximum of a value over the four lanes l, l ^ 16, l ^ 32, l ^ 48 (the
// four 16-lane rows of the wave), in every lane: v_permlane16_swap and
// v_permlane32_swap of x with itself give the even and odd rows (the lower
// and upper halves) in both places, so no exchange goes through LDS.
template <bool MAX>
__device__ __forceinline__ float rows_reduce(float x) {
  auto op = [](float a, float b) { return MAX ? __builtin_fmaxf(a, b) : a + b; };
  uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  x = op(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
  u = __builtin_bit_cast(uint32_t, x);
  const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return op(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}

// Block-wide max / sum over the 256 threads (every thread gets it).
template <bool MAX>
__device__ __forceinline__ float block_reduce(float x, float *red) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const float y = __shfl_xor(x, off, 64);
    x = MAX ? __builtin_fmaxf(x, y) : x + y;
  }
  __syncthreads();  // red may still be read by the previous reduction
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  const float a = red[0], b = red[1], c = red[2], d = red[3];
  return MAX ? __builtin_fmaxf(__builtin_fmaxf(a, b), __builtin_fmaxf(c, d)) : (a + b) + (c + d);
}

}  // namespace
}  // namespace ltkv
