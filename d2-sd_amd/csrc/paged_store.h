// Device helpers of the kernels that put keys and values into a paged cache
// (paged_cache.hip, which has the formats; cache_append.hip): eight head dims of a
// row, as bf16 or as 32-bit values, to their codes and block scales.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "d2sd_internal.h"
#include "kernel_common.h"

namespace d2sd {

// e4m3fn byte pairs of f0..f3, |f| <= 448, rounded to nearest even
__device__ __forceinline__ unsigned fp8x4(float f0, float f1, float f2, float f3) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(f0, f1, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(f2, f3, w, true);
  return (unsigned)w;
}

__device__ __forceinline__ void expand8(const u32x4& u, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_lo(u[i]);
    x[2 * i + 1] = bf16_hi(u[i]);
  }
}

// Maximum over the four threads of a block (threads 4b .. 4b + 3 of a wave).
__device__ __forceinline__ unsigned quad_max(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true));  // quad_perm [1,0,3,2]
  return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true));  // [2,3,0,1]
}

// Eight values as e4m3fn bytes of their quotients by `sc`, each correctly rounded
// in fp32, clamped and rounded to nearest even; a NaN becomes a NaN byte.
__device__ __forceinline__ u32x2 fp8_codes(const float (&x)[8], float sc) {
  u32x2 b;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float q[4];
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float r = __fdiv_rn(x[4 * i + e], sc);
      bad = bad || isnan(r);
      q[e] = fminf(fmaxf(r, -448.f), 448.f);
    }
    b[i] = fp8x4(q[0], q[1], q[2], q[3]);
    if (bad) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (isnan(__fdiv_rn(x[4 * i + e], sc))) b[i] |= 0x7Fu << (8 * e);
    }
  }
  return b;
}

// Exponent of a block's scale from its largest magnitude's bits (finite):
// amax = f 2^k: k + 127 in bits 30..23, f's fraction below (a subnormal's
// k reads as -127, below the range all the same).  over: beyond the largest scale.
template <bool FP4>
__device__ __forceinline__ int block_exponent(unsigned amax, bool& over) {
  constexpr unsigned FM = FP4 ? 0x00400000u : 0x00600000u;  // fraction bits of 1.5, 1.75
  constexpr int KM = FP4 ? 2 : 8, TOP = FP4 ? 125 : 119;
  const int e = (int)(amax >> 23) - 127 - KM + ((amax & 0x007FFFFFu) > FM ? 1 : 0);
  over = amax < 0x7F800000u && e > TOP;
  return min(max(e, -117), TOP);
}

// Elements of eight 32-bit values times 2^-e, exactly, rounded to nearest even,
// saturating (beyond the largest scale).
template <bool FP4>
__device__ __forceinline__ u32x2 block_codes(float (&x)[8], int e) {
  const float inv = __uint_as_float((unsigned)(127 - e) << 23);
  constexpr float M = FP4 ? 6.f : 448.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fminf(fmaxf(x[i] * inv, -M), M);
  u32x2 w = {0u, 0u};
  if constexpr (FP4) {
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], x[0], x[1], 1.f, 0);
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], x[2], x[3], 1.f, 1);
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], x[4], x[5], 1.f, 2);
    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], x[6], x[7], 1.f, 3);
  } else {
    w = (u32x2){fp8x4(x[0], x[1], x[2], x[3]), fp8x4(x[4], x[5], x[6], x[7])};
  }
  return w;
}

// One 8-element piece of a new row into its cache row.  Threads that share a
// block call it together.
template <int FMT>
__device__ __forceinline__ void store_piece(const CacheSide& s, int fmt_head, long long row, long long srow, int d,
                                            const u32x4& val) {
  if constexpr (FMT == CACHE_BF16) {
    *(u32x4*)((uint16_t*)s.codes + row + d) = val;
  } else {
    if constexpr (FMT == CACHE_FP8) {
      float x[8];
      expand8(val, x);
      *(u32x2*)((uint8_t*)s.codes + row + d) = fp8_codes(x, ((const float*)s.scale)[fmt_head]);
    } else {
      constexpr bool FP4 = FMT == CACHE_MXFP4;
      unsigned amax = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) amax = max(amax, max(val[i] << 16 & 0x7FFF0000u, val[i] & 0x7FFF0000u));
      amax = quad_max(amax);
      const bool finite = amax < 0x7F800000u;
      bool over;
      const int e = block_exponent<FP4>(amax, over);
      u32x2 w = {0u, 0u};
      if (!__any(over)) {
        // the converters divide by 2^e, exactly, and round to nearest even
        typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
        typedef short s16x2_t __attribute__((ext_vector_type(2)));
        const float two_e = __uint_as_float((unsigned)(127 + e) << 23);
        const unsigned u[4] = {val[0], val[1], val[2], val[3]};
        auto pair = [&](int i) { return __builtin_bit_cast(bf16x2_t, u[i]); };
        if constexpr (FP4) {
          w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w[0], pair(0), two_e, 0);
          w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w[0], pair(1), two_e, 1);
          w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w[0], pair(2), two_e, 2);
          w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w[0], pair(3), two_e, 3);
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            s16x2_t x = {0, 0};
            x = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(x, pair(2 * i), two_e, false);
            x = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(x, pair(2 * i + 1), two_e, true);
            w[i] = __builtin_bit_cast(unsigned, x);
          }
        }
      } else {
        float x[8];
        expand8(val, x);
        w = block_codes<FP4>(x, e);
      }
      if (!finite) w = (u32x2){0u, 0u};
      if constexpr (FP4)
        *(unsigned*)((uint8_t*)s.codes + row + d / 2) = w[0];
      else
        *(u32x2*)((uint8_t*)s.codes + row + d) = w;
      if ((d & 31) == 0) ((uint8_t*)s.scale)[srow + d / 32] = (uint8_t)(finite ? e + 127 : 255);
    }
  }
}

// The same of eight 32-bit values, rounded once: for rows that a kernel computes.
template <int FMT>
__device__ __forceinline__ void store_values(const CacheSide& s, int fmt_head, long long row, long long srow, int d,
                                             float (&x)[8], bool on) {
  if constexpr (FMT == CACHE_BF16) {
    if (on)
      *(u32x4*)((uint16_t*)s.codes + row + d) =
          (u32x4){pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
  } else if constexpr (FMT == CACHE_FP8) {
    if (on) *(u32x2*)((uint8_t*)s.codes + row + d) = fp8_codes(x, ((const float*)s.scale)[fmt_head]);
  } else {
    constexpr bool FP4 = FMT == CACHE_MXFP4;
    unsigned amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    amax = quad_max(amax);
    const bool finite = amax < 0x7F800000u;
    bool over;
    const int e = block_exponent<FP4>(amax, over);
    u32x2 w = block_codes<FP4>(x, e);
    if (!finite) w = (u32x2){0u, 0u};
    if (!on) return;
    if constexpr (FP4)
      *(unsigned*)((uint8_t*)s.codes + row + d / 2) = w[0];
    else
      *(u32x2*)((uint8_t*)s.codes + row + d) = w;
    if ((d & 31) == 0) ((uint8_t*)s.scale)[srow + d / 32] = (uint8_t)(finite ? e + 127 : 255);
  }
}

}  // namespace d2sd
