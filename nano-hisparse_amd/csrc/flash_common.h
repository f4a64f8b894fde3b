// What the attention kernels on 32x32x16 MFMA share: the matrix instruction,
// weights packed as its operands, and K and V tiles in LDS. The lane layout
// and the reasons for it stand in prefill.hip.
#pragma once

#include "nhs_common.h"

namespace nhs {

typedef __bf16 pf_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 pf_f16x8 __attribute__((ext_vector_type(8)));
typedef float pf_f32x16 __attribute__((ext_vector_type(16)));
typedef float pf_f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 pf_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 pf_f16x2 __attribute__((ext_vector_type(2)));

template <typename T>
__device__ __forceinline__ pf_f32x16 mfma32x32x16(uint4 a, uint4 b, pf_f32x16 c) {
  if constexpr (T::dtype == NHS_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(pf_bf16x8, a), __builtin_bit_cast(pf_bf16x8, b),
                                                  c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(pf_f16x8, a), __builtin_bit_cast(pf_f16x8, b), c,
                                                 0, 0, 0);
}

// two fp32 weights as a packed pair of the input dtype (round to nearest
// even, by the hardware conversions)
template <typename T>
__device__ __forceinline__ uint32_t pf_pack(float lo, float hi) {
  if constexpr (T::dtype == NHS_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((pf_f32x2){lo, hi}, pf_bf16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((pf_f32x2){lo, hi}, pf_f16x2));
}

// acc + both halves of a packed pair, in fp32
template <typename T>
__device__ __forceinline__ float pf_add_pair(uint32_t pair, float acc) {
  if constexpr (T::dtype == NHS_BF16)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pf_bf16x2, pair),
                                           __builtin_bit_cast(pf_bf16x2, 0x3f803f80u), acc, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(pf_f16x2, pair), __builtin_bit_cast(pf_f16x2, 0x3c003c00u), acc,
                                  false);
}

// LDS slot of 16-byte chunk c of K row r: any 16 consecutive rows at one chunk fall on distinct banks
template <int D>
__device__ __forceinline__ int pf_k_slot(int r, int c) {
  return D == 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7);
}
// and of V row (key) r: the 4 rows of a transposing read fall on distinct banks
template <int D>
__device__ __forceinline__ int pf_v_slot(int r, int c) {
  return D == 128 ? c ^ (4 * (r & 3)) : c ^ (4 * ((r >> 1) & 1));
}

// s_waitcnt vmcnt(n), the other counters left alone; with kPfLgkmcnt0: & lgkmcnt(0)
constexpr int pf_vmcnt(int n) { return 0x0f70 | (n & 15) | (n >> 4) << 14; }
constexpr int kPfVmcnt0 = pf_vmcnt(0);
constexpr int kPfLgkmcnt0 = 0xc07f | 0xf;

// 16 bytes per lane from global memory to LDS at `dst` (uniform over the wave) + 16 * lane
__device__ __forceinline__ void pf_load_lds(const char* src, char* dst) {
  __builtin_amdgcn_global_load_lds((const NHS_GLOBAL void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

typedef short pf_i16x4 __attribute__((ext_vector_type(4)));

// Transposing read: of each 16 lanes, lanes 4r .. 4r+3 name 16 elements of row r; lane i receives column i of the four
// rows.
__device__ __forceinline__ uint2 pf_read_tr(const char* p) {
  return __builtin_bit_cast(
      uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pf_i16x4*)const_cast<char*>(p)));
}

}  // namespace nhs
