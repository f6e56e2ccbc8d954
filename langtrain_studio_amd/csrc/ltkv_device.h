// Device helpers shared by the kernel sources: vector types, fault reports, block
// tables, wave and work-group reductions, conversions of stored elements.
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
constexpr int kFaultLayout = 4;     // a step's layout has a token without a cell or a place in its arrays

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

// f32 -> bf16, nearest even (NaN stays NaN).
__device__ __forceinline__ uint16_t bf16_bits(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
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

// quant.rs:785-791 on one 32-element group spread over 4 aligned lanes of
// a wave, 8 elements each (lane j of the group holds elements 8j .. 8j+7):
// amax folded with fmaxf from 0 (a NaN element is skipped, as f32::max; an
// all-NaN group gives 0 as the sequential fold does), then across the 4
// lanes with quad_perm DPP (max is order-free); d = amax / 127, id = 1/d (0
// when d is 0), q = roundf(x * id) (half away from zero) saturated to int8
// with NaN -> 0 (Rust's `as i8`); every lane stores its 8 quants, lane 0 d
// as f16. Quants are stored offset by 128 (byte q + 128, so int8 -128..127
// is 0..255): the readers turn a byte into an f16 without a sign fix-up.
__device__ __forceinline__ void quantize_store4(const float (&x)[8], int j, int8_t *__restrict__ dq,
                                                uint16_t *__restrict__ ds) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = __builtin_fmaxf(amax, __builtin_fabsf(x[i]));
  amax = __builtin_fmaxf(amax, dpp<0xB1>(amax));  // quad_perm [1,0,3,2]: lane ^ 1
  amax = __builtin_fmaxf(amax, dpp<0x4E>(amax));  // quad_perm [2,3,0,1]: lane ^ 2
  const float d = amax / 127.f;
  const float id = d > 0.f ? 1.f / d : 0.f;
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float r = __builtin_roundf(x[i] * id);  // half away from zero
    int qv = 0;
    if (r == r) qv = r > 127.f ? 127 : (r < -128.f ? -128 : (int)r);
    w[i >> 2] |= (uint32_t)((qv + 128) & 0xff) << (8 * (i & 3));
  }
  *reinterpret_cast<u32x2 *>(dq + 8 * j) = u32x2{w[0], w[1]};
  if (j == 0) *ds = (uint16_t)f16_bits(d);
}

// A 32-element group as 4-bit quants, spread over 4 aligned lanes like
// quantize_store4's. The scale is minus an eighth of the element of largest
// magnitude (the positive one where both signs reach it), so that element
// becomes -8 exactly and the levels -8 .. 7 are all used; magnitudes over
// 65280 count as 65280 and NaN as 0. The scale is rounded to 8 significant
// bits (bf16, nearest even) before it becomes an f16: q then has at most 3
// bits (or is -8) and d at most 8, so q * d is exactly an f16 number (subnormal
// ones too) and the readers multiply in f16 without rounding. q is the nearest
// integer to x / d, ties to even: the division is correctly rounded and d has
// 8 bits, so its rounding never moves a quotient onto or across a tie. Quants
// are stored offset by 8, element 2 i of a lane's 8 at bits 4 i of its dword
// and element 2 i + 1 at bits 16 + 4 i: a shift and a mask give two f16 lanes.
// A group's 16 bytes lie in its block's tile [kv_dim / 32][16 slots][16 bytes]
// (a head's rows of a block are one contiguous run, as its scales are).
__device__ __forceinline__ void quantize_store4_q4(const float (&x)[8], int j, uint8_t *__restrict__ tile,
                                                   uint16_t *__restrict__ ds) {
  constexpr float kLimit = 65280.f;  // 8 * the largest 8-bit scale whose products are finite f16 numbers
  float c[8], top = -kLimit, low = kLimit;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = x[i] == x[i] ? __builtin_amdgcn_fmed3f(x[i], -kLimit, kLimit) : 0.f;
    top = __builtin_fmaxf(top, c[i]);
    low = __builtin_fminf(low, c[i]);
  }
  top = __builtin_fmaxf(top, dpp<0xB1>(top));
  low = __builtin_fminf(low, dpp<0xB1>(low));
  top = __builtin_fmaxf(top, dpp<0x4E>(top));
  low = __builtin_fminf(low, dpp<0x4E>(low));
  const float e = (top >= -low ? top : low) * -0.125f;
  const uint32_t u = __builtin_bit_cast(uint32_t, e);
  const _Float16 dh = (_Float16)__builtin_bit_cast(float, (u + 0x7fffu + ((u >> 16) & 1u)) & 0xffff0000u);
  const float d = (float)dh;
  // One division a lane: x * (1 / d) and one step on its exact remainder give
  // the correctly rounded x / d (every significand of x against the 128 of d
  // agrees). The nibbles of a half dword add up exactly as a float.
  const float id = d != 0.f ? 1.f / d : 0.f;
  float half[2] = {8.f * 0x1111, 8.f * 0x1111};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = c[i] * id, r = __builtin_fmaf(__builtin_fmaf(-y, d, c[i]), id, y);
    const float q = __builtin_rintf(__builtin_amdgcn_fmed3f(r, -8.f, 7.f));
    half[i & 1] = __builtin_fmaf(q, (float)(1 << (4 * (i >> 1))), half[i & 1]);
  }
  reinterpret_cast<uint32_t *>(tile)[j] = (uint32_t)half[0] | (uint32_t)half[1] << 16;
  if (j == 0) *ds = d != 0.f ? __builtin_bit_cast(uint16_t, dh) : (uint16_t)0;
}

// A lane's 8 elements of row element e (K or V row of cell s) into the pools of
// BITS-bit quants.
template <int BITS>
__device__ __forceinline__ void store_quants(const float (&x)[8], int32_t s, int e, int kv_dim, int8_t *pool,
                                             uint16_t *scales) {
  const int64_t at = scale_index(s, e >> 5, kv_dim >> 5);
  if constexpr (BITS == 8)
    quantize_store4(x, (e >> 3) & 3, pool + (int64_t)s * kv_dim + (e & ~31), scales + at);
  else
    quantize_store4_q4(x, (e >> 3) & 3, reinterpret_cast<uint8_t *>(pool) + at * 16, scales + at);
}

// Four rotation pairs by (cosine, sine) pairs, without fused multiply-adds: the
// products and sums of the reference's f32 rotation (model.rs:299-306).
__device__ __forceinline__ void rope_pairs(const float *__restrict__ cs, float (&x0)[4], float (&x1)[4]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const float c = cs[2 * p], sn = cs[2 * p + 1];
    const float a = x0[p], b = x1[p];
    x0[p] = a * c - b * sn;
    x1[p] = a * sn + b * c;
  }
}

}  // namespace
}  // namespace ltkv
