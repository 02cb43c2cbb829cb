#pragma once
// Rows held in 8 bits: e4m3 codes with one power-of-two scale for each block of 128 elements of a
// row (the last block may be short). Row r: codes q[r * sq + k], zeros up to the next multiple of 128;
// scale bytes s[r * ss + k / 128], zeros up to the next multiple of 4. An element is
// code * 2^(byte - 127).
//
// Why powers of two: the block-scaled MFMA of gfx950 takes such bytes as an operand, so a product needs
// no multiplication of its own for them, scaling rounds nothing, and e4m3 is as precise everywhere
// between its smallest and largest normal number, so a scale up to 2 too large costs one binade of range.
#include "common.h"

namespace sff8 {

constexpr int BLOCK = 128;         // elements per scale, and bytes of their codes: one cache line
constexpr uint32_t E4M3_TOP = 0x600000u;  // mantissa of 448 = 1.75 * 2^8, the largest e4m3 number

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

__host__ __device__ inline int64_t blocks_of(int64_t K) { return (K + BLOCK - 1) / BLOCK; }
__host__ __device__ inline int64_t code_bytes(int64_t K) { return blocks_of(K) * BLOCK; }
__host__ __device__ inline int64_t scale_bytes(int64_t K) { return (blocks_of(K) + 3) / 4 * 4; }

// Scale byte of a block whose largest finite |element| has the bits `top`: the smallest e >= -127 with
// |element| <= 448 * 2^e, plus 127. At most 247; 0 for a block of zeros.
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
  const int b = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > E4M3_TOP ? 1 : 0);
  return (uint32_t)max(b, 0);
}
// 2^(byte - 127) (2^-127 is subnormal) and its inverse (bytes that scale_byte gives: 0 to 247)
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __uint_as_float(byte > 0 ? byte << 23 : 1u << 22);
}
__device__ __forceinline__ float inverse_of(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }

// Magnitude bits for the maximum: those of NaN and infinities count as zero.
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
  return u >= 0x7f800000u ? 0u : u;
}
// What is converted: v scaled (exact: a power of two); e4m3 has no infinity, so one becomes NaN.
__device__ __forceinline__ float scaled(float v, float inv) {
  const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
  return u == 0x7f800000u ? __builtin_nanf("") : v * inv;
}
// four e4m3 codes, round to nearest even (v_cvt_pk_fp8_f32)
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int r = 0;
  r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  return (uint32_t)r;
}

// Maximum of u over aligned groups of 16 lanes, in every lane (rotations within a DPP row).
__device__ __forceinline__ uint32_t max16(uint32_t u) {
  u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x128, 0xf, 0xf, true));  // row_ror:8
  u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x124, 0xf, 0xf, true));
  u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x122, 0xf, 0xf, true));
  return max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x121, 0xf, 0xf, true));
}
// Maximum over aligned groups of 4 lanes (quad permutations).
__device__ __forceinline__ uint32_t max4(uint32_t u) {
  u = max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0xB1, 0xf, 0xf, true));  // quad_perm 1,0,3,2
  return max(u, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, 0x4E, 0xf, 0xf, true));  // 2,3,0,1
}

// Eight consecutive elements from 16-B aligned memory (32 B of fp32), as fp32.
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&v)[8]) {
  if constexpr (DT == SF_F32) {
    const u32x4 a = *(const u32x4*)((const float*)p + i), b = *(const u32x4*)((const float*)p + i + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = __uint_as_float(a[e]);
      v[4 + e] = __uint_as_float(b[e]);
    }
  } else {
    const u32x4 a = *(const u32x4*)((const u16*)p + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t h = (a[e >> 1] >> ((e & 1) * 16)) & 0xffffu;
      v[e] = DT == SF_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
    }
  }
}

// How the source of a quantisation lies: rows contiguous and 16-B aligned, or anything (element by element).
enum Src { SRC_ROWS = 0, SRC_ANY = 1 };

// Elements k0 .. k0 + 7 of row m minus the shift, in fp32; zeros past K.
template <int DT, int SRC>
__device__ __forceinline__ void load_shifted(const void* x, int64_t sxm, int64_t sxk, const void* shift, int shift_dt,
                                             int shift_vec, int64_t K, int64_t m, int64_t k0, float (&v)[8]) {
  if (SRC == SRC_ROWS && k0 + 8 <= K) {
    load8<DT>(x, m * sxm + k0, v);
    if (shift_vec) {  // shift of x's type, 16-B aligned
      float c[8];
      load8<DT>(shift, k0, c);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] -= c[e];
    } else if (shift) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] -= load_as_f32(shift, shift_dt, k0 + e);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = 0.f;
      if (k0 + e < K) {
        v[e] = load_as_f32(x, DT, m * sxm + (k0 + e) * sxk);
        if (shift) v[e] -= load_as_f32(shift, shift_dt, k0 + e);
      }
    }
  }
}
// The codes of eight elements of a block that sixteen lanes hold together, and the block's scale byte.
__device__ __forceinline__ u32x2 quantize8(float (&v)[8], uint32_t& byte) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, finite_bits(v[e]));
  byte = scale_byte(max16(top));
  const float inv = inverse_of(byte);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = scaled(v[e], inv);
  return u32x2{pack4(v[0], v[1], v[2], v[3]), pack4(v[4], v[5], v[6], v[7])};
}

// Quantises x [M, K] (any strides) minus shift (or NULL) into rows (row0 + m) % R; the arguments have
// been checked. ctr (or NULL): 8 ints, 16 apart, that are set to zero on the way. Defined in fp8_rows.hip.
int launch_quantize(const void* x, int64_t sxm, int64_t sxk, int x_dt, const void* shift, int shift_dt, int64_t M,
                    int64_t K, void* q, int64_t sq, void* scale, int64_t ss, int64_t row0, int64_t R, int32_t* ctr,
                    hipStream_t s);

}  // namespace sff8
