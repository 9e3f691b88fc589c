// What the attention kernels of many query rows share (prefill.hip,
// chunk_attention.hip): tile shape, LDS layout, operand fragments.
#pragma once

#include "dsa_common.h"

namespace dsa {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef int v4i __attribute__((ext_vector_type(4)));

constexpr int kPfWaves = 4;                 // one per SIMD: the accumulators take half its registers
constexpr int kPfThreads = kPfWaves * kWave;
constexpr int kPfRowsPerWave = 32;
constexpr int kPfRows = kPfWaves * kPfRowsPerWave;  // 128 rows (8 queries of 16 heads) a workgroup
constexpr int kPfKeys = 32;                 // keys a tile
constexpr int kPfDepth = 8;                 // operand fragments read ahead of their MFMA
constexpr int kPfRowChunks = DSA_QK_DIM / 8;        // 72 16-byte chunks of a key row
constexpr int kPfTileBytes = kPfKeys * DSA_QK_DIM * 2;  // 36864
constexpr int kPfLoads = kPfKeys * kPfRowChunks / kPfThreads; // 9 direct-to-LDS loads a thread and tile
static_assert(kPfLoads * kPfThreads == kPfKeys * kPfRowChunks, "whole loads");

constexpr float kPfRise = 32.f;
// A wave takes the second bf16 term of a tile's probabilities too when one of
// its rows has a probability above this share of the row's sum so far; with
// fewer keys a split than kPfBothKeys it always does.
constexpr float kPfSecond = 1.f / 24.f;
constexpr int kPfBothKeys = 512;

// LDS position of 16-byte chunk j of key row r: rows are 72 chunks apart (8
// mod 16), so chunk j of 16 consecutive rows would fall on two 16-byte bank
// groups; the low three bits of j are xored with the bit-reversed row / 2,
// which spreads a column over all 16 groups, and a transposed read (8 rows x
// 4 chunks) over 16 as well.
__device__ __forceinline__ int pf_swz(int r) {
  const int x = (r >> 1) & 7;
  return ((x & 1) << 2) | (x & 2) | (x >> 2);
}

__device__ __forceinline__ v4i as_v4i(const uint4& a) { return v4i{(int)a.x, (int)a.y, (int)a.z, (int)a.w}; }
__device__ __forceinline__ v8bf as_bf8(const uint4& a) {
  v8bf v;
  __builtin_memcpy(&v, &a, 16);
  return v;
}

typedef short v4s_t __attribute__((ext_vector_type(4)));
typedef v4s_t __attribute__((address_space(3)))* lds_v4s_ptr;
typedef __attribute__((address_space(1))) const void* gvoid_ptr;
typedef __attribute__((address_space(3))) void* lvoid_ptr;

// max of a value over the two half-waves (lane l and l ^ 32)
__device__ __forceinline__ float half_swap_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_swap_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

}  // namespace dsa
