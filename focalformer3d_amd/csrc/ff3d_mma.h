// 32 x 32 matrix-core tiles in bf16, fp16 and fp32 for the kernels that take all three types.
//
// One step multiplies 32 x 16 by 16 x 32.  A lane l holds 8 elements of each operand, element e being
//   A[l % 32][8 * (l / 32) + e]   and   B[8 * (l / 32) + e][l % 32],
// in every type: 16-bit types feed them to one v_mfma_f32_32x32x16; an fp32 number is the sum of three bf16 numbers (hi, mid, lo, each
// the rest rounded to nearest: 8 bits and a sign more every time, so 24 bits and more in all, over the whole range of exponents) and the
// step is six bf16 products, all but mid * lo, lo * mid and lo * lo, which together are at most 2^-23 of the product and of either
// sign.  Six times 32 cycles against eight v_mfma_f32_32x32x2 of 64, and the vector unit, which splits, works beside the matrix unit.
// (Infinities split into NaN; numbers above 3.39e38 round to infinity.)  The order of k inside a step
// is free as long as both operands agree, which the callers use: the accumulator layout
//   reg r of lane l  =  C[8 * (r / 4) + 4 * (l / 32) + r % 4][l % 32]
// read as the operand of a following product has element e of step s = reg 8 s + e, i.e. k = 16 s + 8 (e / 4) + 4 (l / 32) + e % 4
// (col_frag_acc below): a score tile becomes the next operand without leaving its lanes.
#pragma once
#include "ff3d_common.h"

namespace mma {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Type {
  typedef T vec8 __attribute__((ext_vector_type(8)));
  static constexpr int PER16 = 16 / sizeof(T);     // elements in a 16-byte granule
};
template <typename T>
using vec8 = typename Type<T>::vec8;

__device__ __forceinline__ f32x16 mfma16(vec8<__bf16> a, vec8<__bf16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma16(vec8<_Float16> a, vec8<_Float16> b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// An operand of a step, ready for the matrix unit: itself, or the three parts of fp32.
template <typename T>
struct Op {
  vec8<T> v;
};
template <>
struct Op<float> {
  vec8<__bf16> h, m, l;
};
// two values rounded to bf16 in one register, the first one in the low half
__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 v = __builtin_convertvector((f32x2){a, b}, bf16x2);
  return __builtin_bit_cast(unsigned, v);
}
template <typename T>
__device__ __forceinline__ Op<T> op(vec8<T> x) {
  if constexpr (sizeof(T) == 2) {
    return {x};
  } else {
    Op<float> o;
    unsigned *h = (unsigned*)&o.h, *m = (unsigned*)&o.m, *l = (unsigned*)&o.l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {                    // in pairs: one conversion per plane, 5.5 instructions per element instead of 7.5
      const float x0 = x[2 * e], x1 = x[2 * e + 1];
      h[e] = pack_bf16(x0, x1);
      const float r0 = x0 - __uint_as_float(h[e] << 16), r1 = x1 - __uint_as_float(h[e] & 0xffff0000u);     // exact
      m[e] = pack_bf16(r0, r1);
      l[e] = pack_bf16(r0 - __uint_as_float(m[e] << 16), r1 - __uint_as_float(m[e] & 0xffff0000u));
    }
    return o;
  }
}
// part 0 .. PARTS - 1 of a step, the smallest terms first; the caller may run the parts of several tiles in turn
template <typename T>
constexpr int PARTS = sizeof(T) == 4 ? 6 : 1;
template <int PART, typename T>
__device__ __forceinline__ f32x16 mfma_part(const Op<T>& a, const Op<T>& b, f32x16 c) {
  if constexpr (sizeof(T) == 2) return mfma16(a.v, b.v, c);
  else if constexpr (PART == 0) return mfma16(a.l, b.h, c);
  else if constexpr (PART == 1) return mfma16(a.h, b.l, c);
  else if constexpr (PART == 2) return mfma16(a.m, b.m, c);
  else if constexpr (PART == 3) return mfma16(a.m, b.h, c);
  else if constexpr (PART == 4) return mfma16(a.h, b.m, c);
  else return mfma16(a.h, b.h, c);
}
template <typename T>
__device__ __forceinline__ f32x16 mfma_step(const Op<T>& a, const Op<T>& b, f32x16 c) {
  if constexpr (sizeof(T) == 4) {
    c = mfma_part<0>(a, b, c), c = mfma_part<1>(a, b, c), c = mfma_part<2>(a, b, c);
    c = mfma_part<3>(a, b, c), c = mfma_part<4>(a, b, c), c = mfma_part<5>(a, b, c);
    return c;
  } else {
    return mfma16(a.v, b.v, c);
  }
}

__device__ __forceinline__ int acc_row(int r, int half) { return 8 * (r / 4) + 4 * half + r % 4; }

template <typename T>
__device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f(float v) { return (T)v; }      // round to nearest even

// ---- LDS tiles -----------------------------------------------------------------------------------------------------------
// A tile is a number of rows of GR 16-byte granules.  Two kinds of reads: along a row (the rows are rows of the operand, k runs along
// them) and down the columns (k runs over the rows; ds_read_b64_tr_b16 hands each lane of a group of 16 the 4 elements of its column
// from a 4 x 16 block, lane 4 i + j of the group addressing row i, columns 4 j .. 4 j + 3).  LDS serves a ds_read_b128 in groups of 16
// lanes ({0-3, 12-15, 20-27}, {4-11, 16-19, 28-31} and the same of the upper half) and a transposing read in halves of the wave; a
// group has to touch 16 different granules modulo 256 bytes.  Granule g of row r lies at place(r, g): xor with the row's number modulo
// 256 bytes, its bits rotated so that 4 consecutive rows differ above the 4 granules a transposing read takes of each.  (With the
// plain xor of 8 consecutive rows half of all row reads waited: SQ_LDS_BANK_CONFLICT = 0.5 SQ_LDS_IDX_ACTIVE.)
template <int GR>
__device__ __forceinline__ int place(int r, int g) {
  if constexpr (GR >= 16) return g ^ (((r & 3) << 2) | ((r >> 2) & 3));
  else if constexpr (GR == 8) return g ^ ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
  else if constexpr (GR == 4) return g ^ ((r >> 2) & 3);
  else return g;
}

// elements k0 + 8 half .. + 7 of a row (k0 a multiple of 16)
template <typename T, int GR>
__device__ __forceinline__ vec8<T> row_frag(const char* tile, int row, int k0, int half) {
  vec8<T> v;
  if constexpr (sizeof(T) == 2) {
    v = *(const vec8<T>*)(tile + (row * GR + place<GR>(row, k0 / 8 + half)) * 16);
  } else {
    const int g = k0 / 4 + 2 * half;
    *(u32x4*)&v = *(const u32x4*)(tile + (row * GR + place<GR>(row, g)) * 16);
    *((u32x4*)&v + 1) = *(const u32x4*)(tile + (row * GR + place<GR>(row, g + 1)) * 16);
  }
  return v;
}

// column col0 + lane % 32 (col0 a multiple of 32): elements 0..3 = rows k_lo .. k_lo + 3, 4..7 = rows k_hi .. k_hi + 3 (multiples of 4)
template <typename T, int GR>
__device__ __forceinline__ vec8<T> col_frag_at(const char* tile, int k_lo, int k_hi, int col0, int lane) {
  vec8<T> v;
  if constexpr (sizeof(T) == 2) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int i = (lane & 15) >> 2, c = col0 + (lane & 16) + 4 * (lane & 3);
    const int g = c >> 3, in = (c & 7) * 2, r0 = k_lo + i, r1 = k_hi + i;
    *(s16x4*)&v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + (r0 * GR + place<GR>(r0, g)) * 16 + in));
    *((s16x4*)&v + 1) = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + (r1 * GR + place<GR>(r1, g)) * 16 + in));
  } else {
    const int c = col0 + (lane & 31), g = c >> 2, in = (c & 3) * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = *(const T*)(tile + ((k_lo + e) * GR + place<GR>(k_lo + e, g)) * 16 + in);
      v[4 + e] = *(const T*)(tile + ((k_hi + e) * GR + place<GR>(k_hi + e, g)) * 16 + in);
    }
  }
  return v;
}
// rows k0 .. k0 + 15 in their plain order: k = k0 + 8 half + e
template <typename T, int GR>
__device__ __forceinline__ vec8<T> col_frag(const char* tile, int k0, int col0, int lane) {
  const int k = k0 + 8 * (lane >> 5);
  return col_frag_at<T, GR>(tile, k, k + 4, col0, lane);
}
// in the accumulator's order: k = k0 + 8 (e / 4) + 4 half + e % 4
template <typename T, int GR>
__device__ __forceinline__ vec8<T> col_frag_acc(const char* tile, int k0, int col0, int lane) {
  const int k = k0 + 4 * (lane >> 5);
  return col_frag_at<T, GR>(tile, k, k + 8, col0, lane);
}
// accumulator registers 8 step .. 8 step + 7 (rows 16 step .. 16 step + 15) as the operand that col_frag_acc's k order goes with
template <typename T>
__device__ __forceinline__ vec8<T> acc_frag(const f32x16& c, int step) {
  vec8<T> v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = from_f<T>(c[8 * step + e]);
  return v;
}

// ---- global -> LDS ---------------------------------------------------------------------------------------------------------
// 16 bytes per lane straight into LDS: lane i's granule lands at lds + 16 i (lds uniform in the wave).  Offsets at or beyond
// `bytes` (the descriptor's limit) deliver zeros, which is how tile edges are padded.
typedef __amdgpu_buffer_rsrc_t rsrc_t;
constexpr unsigned OUT = 0x80000000u;                              // an offset that is never inside
__device__ __forceinline__ rsrc_t make_rsrc(const void* p, long long bytes) {
  const unsigned n = bytes > 0x7fffffffll ? 0x7fffffffu : bytes < 0 ? 0u : (unsigned)bytes;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, n, 0x00020000);
}
__device__ __forceinline__ void load_lds16(rsrc_t r, char* lds, unsigned off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, (int)off, 0, 0, 0);
}

// the other half's value of the same column (lane ^ 32), by a register swap: no trip through LDS and no wait for the reads before it
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Waits until at most N of this wave's loads are outstanding and its LDS reads are done, then for the other waves.
// What load_lds16 fetched is read only behind this: a plain __syncthreads() waits for LDS accesses, and whether it also waits for loads on
// their way to LDS is left to where the compiler puts its own waits - behind the barrier or before a loop, as well.
template <int N>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

}  // namespace mma
