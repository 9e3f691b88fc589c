// Matrix products of e4m3 rows with e4m3 weights (gfx950), scales by block:
//
//   out[t, o] = sum_b sa[t, b] sw[o / 128, b] sum_{k in block b} a[t, k] w[o, k]
//
// over the blocks b of 128 values of k (the last one may be short), for the
// tokens t and outputs o; sa is one scale a token instead, if the rows were
// quantised whole.  With offsets, token t's weights are those of the expert e
// with offsets[e] <= t < offsets[e + 1].  Reference: fp8_gemm
// (inference/modeling/kernels.py:120-221).
//
// A block of 128 is one v_mfma_f32_16x16x128 over a 16 x 16 tile, whose 4
// results a lane enter the fp32 sums by one fma each, with the two scales'
// product: the outputs are the product's rows, so a lane holds 4 outputs of one
// token and one scale serves them all.  Per MFMA (32 clocks) that is 16 clocks
// of VALU, which run beside the matrix unit.
//
// That instruction's own sums keep 13 bits below the largest of 8 products:
// 1.5e-5 of a result's size, nothing beside the rounding to bf16 (1.7e-3) or
// fp16 (2.1e-4).  For fp32 outputs a block is four bf16 MFMAs of the same
// values, at half the rate, with fp32's own error.
//
// Two kernels.  Up to 64 rows (of an expert, by the average) the weights are
// read once and are the cost: rows_kernel, whose waves divide k and stream the
// weights from memory into registers.  More rows: tile_kernel, tiles of
// outputs x tokens through LDS.
#include <algorithm>

#include "dsa_kernels.h"
#include "quant_core.h"

namespace dsa {

typedef __attribute__((address_space(3))) void* mm_lds_ptr;

// The product of a block of 128, by the matrix unit's 8-bit products or, for
// outputs that show their error (EXACT: fp32), by its bf16 ones.
template <bool EXACT>
struct Operand {
  std::conditional_t<EXACT, Bf32, v8i> v;
  __device__ __forceinline__ void set(const v8i& x) {
    if constexpr (EXACT) v = e4m3x32_to_bf16(x);
    else v = x;
  }
};
template <bool EXACT>
__device__ __forceinline__ v4f block_product(const Operand<EXACT>& a, const Operand<EXACT>& b) {
  if constexpr (EXACT) {
    return mfma_bf16_128(a.v, b.v);
  } else {
    const v4f z = {0.f, 0.f, 0.f, 0.f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, z, 0, 0, 0, 0, 0, 0);
  }
}

__device__ __forceinline__ v8i two16(const uint4& x, const uint4& y) {
  return v8i{(int)x.x, (int)x.y, (int)x.z, (int)x.w, (int)y.x, (int)y.y, (int)y.z, (int)y.w};
}

// 4 neighbouring outputs o .. o + 3 of a token (those below N), rounded once.
__device__ __forceinline__ void store_out4(const MatmulArgs& A, long token, int o, const float* v) {
  const long at = token * A.N + o;
  if (A.wide_out && o + 4 <= A.N) {
    if (A.out_dtype == kF32) {
      *reinterpret_cast<v4f*>(static_cast<float*>(A.out) + at) = v4f{v[0], v[1], v[2], v[3]};
    } else {
      v2u_t w;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (A.out_dtype == kBF16) w[e] = pack_bf16x2(v[2 * e], v[2 * e + 1]);
        else
          w[e] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * e]) |
                 (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * e + 1]) << 16;
      }
      *reinterpret_cast<v2u_t*>(static_cast<uint16_t*>(A.out) + at) = w;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (o + e >= A.N) break;
    if (A.out_dtype == kF32) static_cast<float*>(A.out)[at + e] = v[e];
    else if (A.out_dtype == kBF16) static_cast<uint16_t*>(A.out)[at + e] = (uint16_t)pack_bf16x2(v[e], 0.f);
    else static_cast<_Float16*>(A.out)[at + e] = (_Float16)v[e];
  }
}

// The rows of expert e, whatever the offsets hold: inside [0, rows).
__device__ __forceinline__ int2 expert_rows(const MatmulArgs& A, int e) {
  if (!A.offsets) return int2{0, A.rows};
  const int lo = min(max(A.offsets[e], 0), A.rows), hi = min(max(A.offsets[e + 1], lo), A.rows);
  return int2{lo, hi};
}

// ---- few rows ----

constexpr int kRwWaves = 8;
constexpr int kRwThreads = kRwWaves * kWave;

// One workgroup: 16 MT outputs of one expert, 16 TT of its rows at a time.
// Wave w takes the blocks w, w + 8, ... of k: it reads its operands from memory
// straight in the product's layout (lane (r, c) holds bytes [32 c, + 32) of row
// r: whole 128-byte lines), the next block's while this one multiplies; the
// waves' sums meet in LDS, in the order of the waves.
template <int MT, int TT, bool EXACT>
__global__ __launch_bounds__(kRwThreads, TT * MT > 4 || EXACT ? 2 : 4) void rows_kernel(const MatmulArgs A) {
  __shared__ v4f part[kRwWaves][MT * TT][kWave];
  const int lane = threadIdx.x & (kWave - 1), wv = wave_id();
  const int r = lane & 15, c = lane >> 4;
  const int ot = (int)(blockIdx.x % (unsigned)A.otiles), e = (int)(blockIdx.x / (unsigned)A.otiles);
  const int2 range = expert_rows(A, e);
  const int o0 = ot * 16 * MT;
  const uint8_t* wbase = A.w + (long)e * A.N * A.K;
  const float* sw = A.w_scale + ((long)e * A.nblocks + o0 / 128) * A.kblocks;  // (16 MT outputs share a block)
  const uint8_t* wrow[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) wrow[m] = wbase + (long)min(o0 + 16 * m + r, A.N - 1) * A.K + 32 * c;

  struct Block {
    v8i w[MT], a[TT];
    float s[TT];
  };
  for (int t0 = range.x; t0 < range.y; t0 += 16 * TT) {
    const uint8_t* arow[TT];
    const float* srow[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const long row = min(t0 + 16 * t + r, range.y - 1);
      arow[t] = A.a + row * A.K + 32 * c;
      srow[t] = A.a_scale + row * A.a_groups;
    }
    const auto load = [&](int b, Block& x) {
      const int left = A.K - b * 128 - 32 * c;  // bytes of the row from this lane's on
      const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint4* p = reinterpret_cast<const uint4*>(wrow[m] + (long)b * 128);
        x.w[m] = two16(left > 0 ? p[0] : z, left > 16 ? p[1] : z);
      }
      const float ws = sw[b];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const uint4* p = reinterpret_cast<const uint4*>(arow[t] + (long)b * 128);
        x.a[t] = two16(left > 0 ? p[0] : z, left > 16 ? p[1] : z);
        x.s[t] = srow[t][A.a_groups == 1 ? 0 : b] * ws;
      }
    };
    v4f acc[MT][TT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[m][t] = v4f{0.f, 0.f, 0.f, 0.f};
    Block cur, nxt;
    if (wv < A.kblocks) load(wv, cur);
    for (int b = wv; b < A.kblocks; b += kRwWaves) {
      if (b + kRwWaves < A.kblocks) load(b + kRwWaves, nxt);
      Operand<EXACT> wf[MT], af;
#pragma unroll
      for (int m = 0; m < MT; ++m) wf[m].set(cur.w[m]);
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        af.set(cur.a[t]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const v4f d = block_product(wf[m], af);
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][t][i] = __builtin_fmaf(cur.s[t], d[i], acc[m][t][i]);
        }
      }
      cur = nxt;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < TT; ++t) part[wv][m * TT + t][lane] = acc[m][t];
    __syncthreads();
    // tile i of 64 lanes' sums to wave i (mod 8)
    for (int i = wv; i < MT * TT; i += kRwWaves) {
      v4f s = part[0][i][lane];
#pragma unroll
      for (int w = 1; w < kRwWaves; ++w) s += part[w][i][lane];
      const int row = t0 + 16 * (i % TT) + r, o = o0 + 16 * (i / TT) + 4 * c;
      const float v[4] = {s[0], s[1], s[2], s[3]};
      if (row < range.y && o < A.N) store_out4(A, row, o, v);
    }
    __syncthreads();
  }
}

// ---- many rows ----

// Which expert's which tile of BT rows the workgroup's row tile is; rows y > x
// if there is one.  Every wave looks it up for itself: 64 experts at a time.
template <int BT>
__device__ __forceinline__ int2 find_rows(const MatmulArgs& A, int tile, int& expert) {
  expert = 0;
  if (!A.offsets) return int2{tile * BT, min(A.rows, (tile + 1) * BT)};
  const int lane = threadIdx.x & (kWave - 1);
  for (int e0 = 0; e0 < A.experts; e0 += kWave) {
    int2 x = {0, 0};
    if (e0 + lane < A.experts) x = expert_rows(A, e0 + lane);
    const int mine = (x.y - x.x + BT - 1) / BT;
    const int incl = (int)wave_scan_incl<0>((uint32_t)mine);
    const uint64_t at = __ballot(tile < incl);
    if (at) {
      const int l = __builtin_ctzll(at);
      expert = e0 + l;
      const int lo = __builtin_amdgcn_readlane(x.x, l), hi = __builtin_amdgcn_readlane(x.y, l);
      const int before = __builtin_amdgcn_readlane(incl - mine, l);
      const int first = lo + (tile - before) * BT;
      return int2{first, min(hi, first + BT)};
    }
    tile -= __builtin_amdgcn_readlane(incl, kWave - 1);
  }
  return int2{0, 0};
}

// One workgroup: BO outputs x BT rows, WO x WT waves of (16 MO) x (16 TT).
// A block of 128 k at a time goes from memory straight to LDS, two places, the
// next block's on its way while this one multiplies.  A row's 8 16-byte chunks
// lie with their low bits xored with row / 2, so that the 16 rows of an operand
// read fall in distinct banks.
template <int WO, int WT, int MO, int TT, bool EXACT>
__global__ __launch_bounds__(WO* WT* kWave, 2) void tile_kernel(const MatmulArgs A) {
  constexpr int BO = WO * MO * 16, BT = WT * TT * 16, kThreads = WO * WT * kWave;
  constexpr uint32_t kStage = (BO + BT) * 128;
  constexpr int kLoads = (BO + BT) * 8 / kThreads;
  static_assert(kLoads * kThreads == (BO + BT) * 8, "whole loads");
  static_assert((BO * 8) % kThreads == 0, "a load is of weights or of rows");
  __shared__ __align__(16) uint8_t lds[2 * kStage];
  const int t = threadIdx.x, lane = t & (kWave - 1), wv = wave_id();
  const int r = lane & 15, c = lane >> 4;
  const int wo = wv % WO, wt = wv / WO;

  // Workgroups go round the 8 XCDs; each XCD takes a contiguous range of tiles,
  // in bands of 4 row tiles, so that what runs on it at one time shares rows
  // and weights in its L2.
  const unsigned total = (unsigned)A.rtiles * (unsigned)A.otiles;
  const unsigned per = (total + 7) / 8;
  const unsigned id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= per || id >= total) return;
  const unsigned band = id / (4u * A.otiles), in = id % (4u * A.otiles);
  const unsigned height = min(4u, (unsigned)A.rtiles - 4u * band);
  const int ot = (int)(in / height);
  int e;
  const int2 rows = find_rows<BT>(A, (int)(4u * band + in % height), e);
  if (rows.x >= rows.y) return;
  const int o0 = ot * BO;

  const uint8_t* wbase = A.w + (long)e * A.N * A.K;
  const uint8_t* abase = A.a + (long)rows.x * A.K;
  uint32_t off[kLoads];  // of this thread's chunks from wbase + o0 * K or abase
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int p = i * kThreads + t, row = p >> 3, j = (p & 7) ^ ((row >> 1) & 7);
    const int src = row < BO ? min(row, A.N - 1 - o0) : min(row - BO, rows.y - 1 - rows.x);
    off[i] = (uint32_t)src * (uint32_t)A.K + 16u * j;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(mm_lds_ptr)lds;
  const auto issue = [&](int b, uint32_t buf) {
    // in the last, short block a chunk behind the row's end reads the row's
    // last instead; the product masks it
    const int jmax = min(8, (A.K - b * 128) / 16) - 1;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint8_t* base = (i * kThreads < BO * 8 ? wbase + (long)o0 * A.K : abase) + (long)b * 128;
      uint32_t o = off[i];
      if (jmax < 7) {  // uniform
        const int p = i * kThreads + t, j = (p & 7) ^ ((p >> 4) & 7);
        o -= 16u * (uint32_t)max(0, j - jmax);
      }
      const uint32_t dst = __builtin_amdgcn_readfirstlane(lds0 + buf + (uint32_t)(i * kThreads + wv * kWave) * 16u);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                   :
                   : "s"(dst), "v"(o), "s"(base)
                   : "memory", "m0");
    }
  };
  // scales: this lane's token of each row tile, and the wave's outputs' block
  const float* srow[TT];
#pragma unroll
  for (int i = 0; i < TT; ++i)
    srow[i] = A.a_scale + (long)min(rows.x + (wt * TT + i) * 16 + r, rows.y - 1) * A.a_groups;
  const float* sw = A.w_scale + ((long)e * A.nblocks + min(o0 + wo * MO * 16, A.N - 1) / 128) * A.kblocks;
  static_assert(MO * 16 <= 128 && 128 % (MO * 16) == 0, "a wave's outputs share a block");

  const uint32_t swz0 = (uint32_t)(((2 * c) ^ ((r >> 1) & 7)) * 16), swz1 = (uint32_t)(((2 * c + 1) ^ ((r >> 1) & 7)) * 16);
  const uint32_t wofs = (uint32_t)(wo * MO * 16 + r) * 128u, aofs = (uint32_t)(BO + wt * TT * 16 + r) * 128u;
  v4f acc[MO][TT];
#pragma unroll
  for (int m = 0; m < MO; ++m)
#pragma unroll
    for (int i = 0; i < TT; ++i) acc[m][i] = v4f{0.f, 0.f, 0.f, 0.f};
  const bool idle = rows.x + wt * TT * 16 >= rows.y || o0 + wo * MO * 16 >= A.N;  // none of the wave's tiles is needed

  const auto compute = [&](const uint8_t* buf, const float* s, auto tail, int left) {
    const auto frag = [&](uint32_t at) {
      uint4 x = *reinterpret_cast<const uint4*>(buf + at + swz0), y = *reinterpret_cast<const uint4*>(buf + at + swz1);
      if constexpr (decltype(tail)::value) {
        const uint4 z = make_uint4(0, 0, 0, 0);
        x = left > 0 ? x : z;
        y = left > 16 ? y : z;
      }
      Operand<EXACT> f;
      f.set(two16(x, y));
      return f;
    };
    Operand<EXACT> a[TT];
#pragma unroll
    for (int i = 0; i < TT; ++i) a[i] = frag(aofs + (uint32_t)i * (16 * 128));
#pragma unroll
    for (int m = 0; m < MO; ++m) {
      const Operand<EXACT> w = frag(wofs + (uint32_t)m * (16 * 128));
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        const v4f d = block_product(w, a[i]);
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[m][i][q] = __builtin_fmaf(s[i], d[q], acc[m][i][q]);
      }
    }
  };

  float s[TT], ns[TT];
  const auto scales = [&](int b, float* x) {
    const float ws = sw[b];
#pragma unroll
    for (int i = 0; i < TT; ++i) x[i] = srow[i][A.a_groups == 1 ? 0 : b] * ws;
  };
  scales(0, ns);
  issue(0, 0u);
  uint32_t cur = 0;
  for (int b = 0; b < A.kblocks; ++b) {
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      s[i] = ns[i];
      asm volatile("" : "+v"(s[i]));  // waited for here, before the next block's loads
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // block b has landed (every wave's loads), the other place is free
    if (b + 1 < A.kblocks) {
      scales(b + 1, ns);
      issue(b + 1, kStage - cur);
    }
    if (!idle) {
      const int left = A.K - b * 128;
      if (left >= 128) compute(lds + cur, s, std::false_type{}, 0);
      else compute(lds + cur, s, std::true_type{}, left - 32 * c);
    }
    cur = kStage - cur;
  }
  if (idle) return;
#pragma unroll
  for (int m = 0; m < MO; ++m) {
    const int o = o0 + (wo * MO + m) * 16 + 4 * c;
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      const int row = rows.x + (wt * TT + i) * 16 + r;
      const float v[4] = {acc[m][i][0], acc[m][i][1], acc[m][i][2], acc[m][i][3]};
      if (row < rows.y && o < A.N) store_out4(A, row, o, v);
    }
  }
}

template <int MT, int TT, bool EXACT>
static hipError_t launch_rows(MatmulArgs A, hipStream_t s) {
  A.otiles = (A.N + 16 * MT - 1) / (16 * MT);
  hipLaunchKernelGGL((rows_kernel<MT, TT, EXACT>), dim3((unsigned)((long)A.otiles * A.experts)), dim3(kRwThreads), 0, s, A);
  return hipGetLastError();
}

template <int WO, int WT, int MO, int TT, bool EXACT>
static hipError_t launch_tiles(MatmulArgs A, hipStream_t s) {
  constexpr int BO = WO * MO * 16, BT = WT * TT * 16;
  A.otiles = (A.N + BO - 1) / BO;
  // every expert's last tile may be short
  A.rtiles = A.offsets ? A.rows / BT + std::min(A.experts, A.rows) : (A.rows + BT - 1) / BT;
  const long total = (long)A.rtiles * A.otiles;
  hipLaunchKernelGGL((tile_kernel<WO, WT, MO, TT, EXACT>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(WO * WT * kWave), 0, s,
                     A);
  return hipGetLastError();
}

template <bool EXACT>
static hipError_t launch_matmul(const MatmulArgs& A, hipStream_t s) {
  const long per = ((long)A.rows + A.experts - 1) / A.experts;
  if (per <= 16) return launch_rows<1, 1, EXACT>(A, s);
  if (per <= 32) return launch_rows<2, 2, EXACT>(A, s);
  if (per <= 64) return launch_rows<2, 4, EXACT>(A, s);
  return launch_tiles<2, 2, 4, 4, EXACT>(A, s);
}

hipError_t launch_fp8_matmul(MatmulArgs A, hipStream_t s) {
  A.kblocks = (A.K + 127) / 128;
  A.nblocks = (A.N + 127) / 128;
  // 4 outputs are one store where every row begins on its boundary
  A.wide_out = A.N % 4 == 0 && ((uintptr_t)A.out & (A.out_dtype == kF32 ? 15 : 7)) == 0;
  return A.out_dtype == kF32 ? launch_matmul<true>(A, s) : launch_matmul<false>(A, s);
}

}  // namespace dsa
