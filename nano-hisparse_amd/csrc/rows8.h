// Rows of a KV cache held in 8 bits. In each of its two planes a row is
// kv_heads x head_dim codes, then (at the next multiple of 4) an fp32 scale
// for every KV head, padded to whole 16-byte chunks. Of the elements x of one
// token, plane and head, with Q the type's largest value:
//   scale = max(max|x| / Q, 2^-80)   the quotient rounded to fp32
//   code  = the type's value nearest to x / scale, ties to even
//   value = code * scale             rounded to fp32
// A slice with an element that is not finite has a NaN for its scale (all of
// it reads as NaN) and codes of 0. One scale per token: rows are gathered one
// by one from any page and appended one by one, so a scale that several
// tokens share would have to be carried beside them, and every append into a
// started block would round what is there a second time.
#pragma once

#include "nhs_common.h"

namespace nhs {

struct Row8 {
  int kv_heads, head_dim;
  int64_t scales_at, bytes;  // of a plane's row
};

inline Row8 row8(int kv_heads, int head_dim) {
  Row8 f;
  f.kv_heads = kv_heads;
  f.head_dim = head_dim;
  f.scales_at = ((int64_t)kv_heads * head_dim + 3) / 4 * 4;
  f.bytes = (f.scales_at + 4 * (int64_t)kv_heads + 15) / 16 * 16;
  return f;
}

inline bool valid_code(int code) { return code == NHS_CODE_I8 || code == NHS_CODE_E4M3; }

constexpr float kLeastScale = 0x1p-80f;  // keeps every quotient and remainder below far from fp32's subnormals

struct I8 {
  static constexpr int code = NHS_CODE_I8;
  static constexpr float largest = 127.f;
};
struct E4M3 {
  static constexpr int code = NHS_CODE_E4M3;
  static constexpr float largest = 448.f;
};

// The scale of a slice from the largest |x| of it, given as bits: as unsigned
// numbers they order as the values do, NaN and infinity on top.
template <typename C>
__device__ __forceinline__ float scale8(uint32_t largest_bits) {
  const float scale = fmaxf(__fdiv_rn(__uint_as_float(largest_bits), C::largest), kLeastScale);
  return largest_bits >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : scale;
}

// |x / scale| rounded so that rounding it once more, to fewer bits, gives what
// the exact quotient gives: the nearest fp32 value, or its neighbour towards
// the exact one where that has an odd last bit (no border between two codes
// has). inv = 1 / scale.
__device__ __forceinline__ float quotient8(float x, float scale, float inv) {
  const float ax = fabsf(x);
  float q = ax * inv;
  q = __builtin_fmaf(__builtin_fmaf(-q, scale, ax), inv, q);
  const float rest = __builtin_fmaf(-q, scale, ax);
  uint32_t bits = __float_as_uint(q);
  if (!(bits & 1u)) bits += rest > 0.f ? 1u : rest < 0.f ? 0xffffffffu : 0u;
  return __uint_as_float(bits);
}

// The codes (one byte each, in order) of four elements of a slice.
template <typename C>
__device__ __forceinline__ uint32_t codes8(const float (&x)[4], float scale, float inv) {
  if (!(scale == scale)) return 0;
  if constexpr (C::code == NHS_CODE_I8) {
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = (int)__builtin_rintf(quotient8(x[i], scale, inv));
      word |= ((uint32_t)(x[i] < 0.f ? -n : n) & 0xffu) << (8 * i);
    }
    return word;
  } else {
    float q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = __builtin_copysignf(quotient8(x[i], scale, inv), x[i]);
    int word = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], word, true);
  }
}

// A code's number.
template <typename C>
__device__ __forceinline__ float decode8(uint32_t byte) {
  if constexpr (C::code == NHS_CODE_I8)
    return (float)(int8_t)byte;
  else
    return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0);
}

// The numbers of four codes.
template <typename C>
__device__ __forceinline__ void decode8(uint32_t word, float (&out)[4]) {
  if constexpr (C::code == NHS_CODE_I8) {
    out[0] = (float)(int8_t)word;
    out[1] = (float)(int8_t)(word >> 8);
    out[2] = (float)(int8_t)(word >> 16);
    out[3] = (float)(int8_t)(word >> 24);
  } else {
    out[0] = __builtin_amdgcn_cvt_f32_fp8((int)word, 0);
    out[1] = __builtin_amdgcn_cvt_f32_fp8((int)word, 1);
    out[2] = __builtin_amdgcn_cvt_f32_fp8((int)word, 2);
    out[3] = __builtin_amdgcn_cvt_f32_fp8((int)word, 3);
  }
}

// A held value: the product as fp32. The barrier keeps the compiler from
// rounding it to fp16 only (v_fma_mixlo_f16), which would be another value
// than the one that is rounded from fp32.
__device__ __forceinline__ float value8(float code, float scale) {
  float v = code * scale;
  asm("" : "+v"(v));
  return v;
}

}  // namespace nhs
