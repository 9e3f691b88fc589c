// The fp8 quantisation rule of one 128-element row held by 16 lanes (8
// elements each), shared by the operand-preparation and prefill kernels
// (the 4-bit rule of the latent cache and typed loads and stores are below):
//   scale = max(amax, 1e-6) / 448,  code = e4m3_rne(clamp(x / scale, +-448)),
// the division IEEE fp32 (the reference harness's quantize_e4m3_rowwise,
// K:2969-2974).
#pragma once

#include "dsa_common.h"

namespace dsa {

// Element types of an input: 0 fp32, 1 bf16, 2 fp16.
constexpr int kF32 = 0, kBF16 = 1, kF16 = 2;

template <int DT>
__device__ __forceinline__ float load_elem(const void* p, long i) {
  if constexpr (DT == kF32) return static_cast<const float*>(p)[i];
  const uint16_t v = static_cast<const uint16_t*>(p)[i];
  if constexpr (DT == kBF16) return __uint_as_float((uint32_t)v << 16);
  return (float)__builtin_bit_cast(_Float16, v);
}

// Elements i .. i + 7; WIDE: by 16-byte loads (p 16-byte aligned, i a
// multiple of 8), otherwise one by one.
template <int DT, bool WIDE = true>
__device__ __forceinline__ void load8(const void* p, long i, float* x) {
  if constexpr (!WIDE) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = load_elem<DT>(p, i + e);
  } else if constexpr (DT == kF32) {
    const v4f* f = reinterpret_cast<const v4f*>(static_cast<const float*>(p) + i);
    const v4f a = f[0], b = f[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == kBF16) {
        x[2 * e] = bf16_lo(w[e]);
        x[2 * e + 1] = bf16_hi(w[e]);
      } else {
        x[2 * e] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[e]);
        x[2 * e + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e] >> 16));
      }
    }
  }
}

// max |x| of a lane's 8 elements as integer bits: NaN above infinity above
// every finite value.  NANS false: NaN is passed over.
template <bool NANS>
__device__ __forceinline__ uint32_t amax_bits(const float* x) {
  uint32_t am = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t a = __float_as_uint(x[e]) & 0x7fffffffu;
    am = max(am, NANS || a <= 0x7f800000u ? a : 0u);
  }
  return am;
}

// max over the 16-lane DPP row: rotations by 1, 2, 4, 8
__device__ __forceinline__ uint32_t row16_max(uint32_t am) {
  am = max(am, dpp_u32<0x121, 0xf>(am, 0u));
  am = max(am, dpp_u32<0x122, 0xf>(am, 0u));
  am = max(am, dpp_u32<0x124, 0xf>(am, 0u));
  return max(am, dpp_u32<0x128, 0xf>(am, 0u));
}

__device__ __forceinline__ float scale_of_amax(uint32_t am) {
  const float amax = __uint_as_float(am);
  return (amax < 1e-6f ? 1e-6f : amax) / 448.f;
}

// Row scale from each lane's 8 elements.  NANS: a NaN among the row's 128
// makes the scale NaN; otherwise it is passed over (its own code is -448's).
template <bool NANS>
__device__ __forceinline__ float row_scale(const float* x) {
  return scale_of_amax(row16_max(amax_bits<NANS>(x)));
}

// The 8 codes (two words, element e in byte e).  The quotients are x times
// the correctly rounded reciprocal, corrected twice by the exact remainder:
// the first correction is within an ulp, the second then rounds correctly
// (Markstein's theorem), at 5 instructions a quotient where the compiler's
// general division takes about 10 and a quarter-rate reciprocal.  A scale
// that is not finite takes the division.  scale is the row's own: a quotient is
// at most 448 (1 + 2^-23), which converts to 448 without a clamp; only where a
// NaN was passed over (NANS false) does one turn it into -448.
template <bool NANS>
__device__ __forceinline__ v2u_t quant8(const float* x, float scale) {
  float y[8];
  if (scale < INFINITY) {
    const float r = 1.f / scale;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float q = x[e] * r;
      q = __builtin_fmaf(__builtin_fmaf(-q, scale, x[e]), r, q);
      q = __builtin_fmaf(__builtin_fmaf(-q, scale, x[e]), r, q);
      y[e] = __builtin_copysignf(q, x[e]);  // the corrections turn -0 into +0
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = x[e] / scale;
  }
  int c[4];
  if constexpr (!NANS) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = fminf(fmaxf(y[e], -448.f), 448.f);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) c[e] = __builtin_amdgcn_cvt_pk_fp8_f32(y[2 * e], y[2 * e + 1], 0, false);
  v2u_t w;
  w[0] = ((uint32_t)c[0] & 0xffffu) | (uint32_t)c[1] << 16;
  w[1] = ((uint32_t)c[2] & 0xffffu) | (uint32_t)c[3] << 16;
  return w;
}

// ---- the 4-bit rule of a 32-element group held by 4 lanes (8 each) ----
//   e = the smallest integer with max(amax, 1e-6) <= 6 * 2^e (no value
//   saturates), scale byte e + 127, code = e2m1_rne(x * 2^-e), ties to the
//   even code; a group with a NaN or an infinity has the byte 255, which
//   reads back as NaN (v_cvt_scalef32_* take an exponent of 255 as NaN).
constexpr uint32_t kFp4Nan = 255;

__device__ __forceinline__ uint32_t fp4_scale_byte(const float* x) {
  uint32_t am = amax_bits<true>(x);
  am = max(am, dpp_u32<0xb1, 0xf>(am, 0u));  // quad_perm: lane ^ 1, lane ^ 2
  am = max(am, dpp_u32<0x4e, 0xf>(am, 0u));
  if (am >= 0x7f800000u) return kFp4Nan;
  am = max(am, __float_as_uint(1e-6f));
  // amax = 1.f * 2^(E - 127); 6 * 2^e = 1.5 * 2^(e + 2)
  return (am >> 23) - 2 + ((am & 0x7fffffu) > 0x400000u ? 1u : 0u);
}

// The 8 codes of a lane, element e in bits 4e .. 4e + 3.  The hardware's
// conversion divides by the scale exactly (a power of two) and rounds once.
__device__ __forceinline__ uint32_t quant8_fp4(const float* x, uint32_t scale_byte) {
  const float sc = __uint_as_float((scale_byte == kFp4Nan ? 127u : scale_byte) << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], sc, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], sc, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], sc, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], sc, 3);
  return w;
}

// 8 codes (one word) at a scale -> 8 bf16, exactly (a 2-bit significand
// times a power of two; the smallest scale byte written is 105).
__device__ __forceinline__ uint4 dequant8_fp4(uint32_t w, float sc) {
  uint4 o;
  o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 0));
  o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 1));
  o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 2));
  o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, sc, 3));
  return o;
}

// A pair turned by an angle: (a, b) -> (a c - b s, b c + a s).  The fused
// form is spelled out, so that every path gives the same bits.
__device__ __forceinline__ void turn(float a, float b, float c, float s, float& ya, float& yb) {
  ya = __builtin_fmaf(-b, s, a * c);
  yb = __builtin_fmaf(a, s, b * c);
}

// Elements i .. i + 7 of an output of type DT; WIDE: by 16-byte stores,
// otherwise one by one, those below `end`.
template <int DT, bool WIDE>
__device__ __forceinline__ void store8(void* p, long i, const float* x, long end) {
  if constexpr (!WIDE) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (i + e >= end) break;
      if constexpr (DT == kF32) static_cast<float*>(p)[i + e] = x[e];
      else if constexpr (DT == kBF16) static_cast<uint16_t*>(p)[i + e] = (uint16_t)pack_bf16x2(x[e], 0.f);
      else static_cast<_Float16*>(p)[i + e] = (_Float16)x[e];
    }
  } else if constexpr (DT == kF32) {
    v4f* f = reinterpret_cast<v4f*>(static_cast<float*>(p) + i);
    f[0] = v4f{x[0], x[1], x[2], x[3]};
    f[1] = v4f{x[4], x[5], x[6], x[7]};
  } else {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == kBF16) {
        w[e] = pack_bf16x2(x[2 * e], x[2 * e + 1]);
      } else {
        w[e] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[2 * e]) |
               (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)x[2 * e + 1]) << 16;
      }
    }
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace dsa
