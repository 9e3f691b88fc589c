// Matrix products of e4m3 rows with e4m3 weights (gfx950), scales by block:
//
//   out[t, o] = sum_b sa[t, b] sw[o / 128, b] sum_{k in block b} a[t, k] w[o, k]
//
// over the blocks b of 128 values of k (the last one may be short), for the
// tokens t and outputs o; sa is one scale a token instead, if the rows were
// quantised whole.  With offsets, token t's weights are those of the expert e
// with offsets[e] <= t < offsets[e + 1].  Reference:
// inference/modeling/kernels.py:120-221.
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
// Two kernels.  Up to 32 rows (of an expert, by the average) the weights are
// read once and are the cost: rows_kernel, whose waves divide k and stream the
// weights from memory into registers, four blocks ahead.  More rows:
// tile_kernel, tiles of 128 outputs x 128 tokens through LDS.  (33 to 64 rows of
// 7168 x 7168: 100-145 us by rows_kernel, whose registers run out, 43-45 by tiles.)
// Tiles divide outputs and rows, and K between two groups of waves at most, so
// few outputs leave most of the chip idle: 33 to 512 rows of 7168 x 7168 take
// 43-49 us (floor 11-19), of 2112 x 7168 37-42 (3.3-5.7), and of 128 x 16384
// 76-87 where 32 rows take 30.  The choice goes by the average over the experts:
// with 32 at most, an expert of many rows takes them 32 at a time, its weights
// read again for each (1031 rows of which one of 32 experts has 1000, 4096 x 7168:
// 174 us, floor 22; 64 experts with 1000 rows in one and 15 in the others 733 us,
// with 31 each 590, with 70 each 500).
//
// Measured, from memory: one token, 2112 x 7168, 8 us (1.9 TB/s: a launch and
// one wait for memory); 32 rows, 24576 x 1536, 15 us (2.7 TB/s); 128 rows over 32
// experts of 4096 x 7168, 736 MB of the weights of those that have any, 154 us
// (4.8 TB/s, a large copy's rate); 4097 rows, 18432 x 7168, 635 us (1.7 PFLOP/s), fp32
// outputs 996; 8191 rows over 32 experts 264 us (0.9 PFLOP/s: 487 MB to move in 97
// us, and a last tile of every expert that is part empty).  In the large one the
// matrix unit is busy 38% of the clocks and LDS 48%, more than half of those bank
// conflicts of the operand reads; waves wait for a third of their time.
#include <algorithm>

#include "dsa_kernels.h"
#include "quant_core.h"

namespace dsa {

typedef __attribute__((address_space(3))) void* mm_lds_ptr;
typedef const __attribute__((address_space(4))) float* const_float_ptr;  // (scalar loads)

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

// One workgroup: 16 MT outputs of one expert, 16 TT of its rows at a time.
// Wave w of W takes the blocks w, w + W, ... of k: it reads its operands from
// memory straight in the product's layout (lane (r, c) holds bytes [32 c, + 32)
// of row r: whole 128-byte lines), the weights kAhead blocks ahead, the rows,
// which the L2 holds, two; the waves' sums meet in LDS, in the order of the
// waves.
template <int MT, int TT, int W, bool EXACT>
__global__ __launch_bounds__(W* kWave, W >= 16 ? 4 : 3) void rows_kernel(const MatmulArgs A) {
  constexpr int kAhead = EXACT ? 2 : 4;  // (as many as find registers)
  __shared__ v4f part[W][MT * TT][kWave];
  const int lane = threadIdx.x & (kWave - 1), wv = wave_id();
  const int r = lane & 15, c = lane >> 4;
  const int ot = (int)(blockIdx.x % (unsigned)A.otiles), e = (int)(blockIdx.x / (unsigned)A.otiles);
  const int2 range = expert_rows(A, e);
  const int o0 = ot * 16 * MT;
  // Operands through buffer resources: what lies behind a row's end or the last
  // row is out of range and reads as zero, without a branch among the loads.
  constexpr uint32_t kNowhere = 0x80000000u;
  const __amdgpu_buffer_rsrc_t wr = dev_rsrc(A.w + ((long)e * A.N + o0) * A.K, (uint32_t)min(16 * MT, A.N - o0) * (uint32_t)A.K);
  const auto* sw = (const_float_ptr)(A.w_scale + ((long)e * A.nblocks + o0 / 128) * A.kblocks);  // (16 MT outputs share a block)
  // the wave's i-th block; behind its last, the last again (read, not used)
  const int count = A.kblocks > wv ? (A.kblocks - 1 - wv) / W + 1 : 0;
  const auto block_of = [&](int i) { return wv + W * max(min(i, count - 1), 0); };
  const auto load32 = [&](const __amdgpu_buffer_rsrc_t& res, uint32_t row, int b) DSA_INLINE {
    const int left = A.K - b * 128 - 32 * c;
    const uint32_t at = row * (uint32_t)A.K + (uint32_t)(b * 128 + 32 * c);
    return two16(__builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(res, left > 0 ? at : kNowhere, 0, 0)),
                 __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(res, left > 16 ? at + 16 : kNowhere, 0, 0)));
  };
  for (int t0 = range.x; t0 < range.y; t0 += 16 * TT) {
    const int here = min(16 * TT, range.y - t0);
    const __amdgpu_buffer_rsrc_t ar = dev_rsrc(A.a + (long)t0 * A.K, (uint32_t)here * (uint32_t)A.K);
    const __amdgpu_buffer_rsrc_t sr = dev_rsrc(A.a_scale + (long)t0 * A.a_groups, (uint32_t)here * (uint32_t)A.a_groups * 4u);
    v8i wq[kAhead][MT], aq[2][TT];
    float sq[2][TT], swq[2];
    const auto load_w = [&](int i, int u) DSA_INLINE {
      const int b = block_of(i);
#pragma unroll
      for (int m = 0; m < MT; ++m) wq[u][m] = load32(wr, (uint32_t)(16 * m + r), b);
    };
    const auto load_a = [&](int i, int u) DSA_INLINE {
      const int b = min(block_of(i), A.kblocks - 1);
      swq[u] = sw[b];
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        aq[u][t] = load32(ar, (uint32_t)(16 * t + r), b);
        const uint32_t at = 4u * ((uint32_t)(16 * t + r) * (uint32_t)A.a_groups + (uint32_t)(A.a_groups == 1 ? 0 : b));
        sq[u][t] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(sr, at, 0, 0));
      }
    };
    v4f acc[MT][TT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < TT; ++t) acc[m][t] = v4f{0.f, 0.f, 0.f, 0.f};
    if (count > 0) {
#pragma unroll
      for (int u = 0; u < kAhead; ++u) load_w(u, u);
      load_a(0, 0);
      load_a(1, 1);
      const auto blocks = [&](int i0, auto more) DSA_INLINE {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          Operand<EXACT> wf[MT], af[TT];
          float s[TT];
#pragma unroll
          for (int m = 0; m < MT; ++m) wf[m].set(wq[u][m]);
#pragma unroll
          for (int t = 0; t < TT; ++t) {
            af[t].set(aq[u & 1][t]);
            s[t] = sq[u & 1][t] * swq[u & 1];
          }
          if (i0 + u < count) {  // uniform
#pragma unroll
            for (int t = 0; t < TT; ++t)
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                const v4f d = block_product(wf[m], af[t]);
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[m][t][q] = __builtin_fmaf(s[t], d[q], acc[m][t][q]);
              }
          }
          if (decltype(more)::value) load_w(i0 + u + kAhead, u);
          if (decltype(more)::value || u + 2 < kAhead) load_a(i0 + u + 2, u & 1);
        }
      };
      int i0 = 0;
      for (; i0 + kAhead < count; i0 += kAhead) blocks(i0, std::true_type{});
      blocks(i0, std::false_type{});  // the last ones, with nothing behind them to load
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int t = 0; t < TT; ++t) part[wv][m * TT + t][lane] = acc[m][t];
    __syncthreads();
    // tile i of 64 lanes' sums to wave i (mod W)
    for (int i = wv; i < MT * TT; i += W) {
      v4f s = part[0][i][lane];
#pragma unroll
      for (int w = 1; w < W; ++w) s += part[w][i][lane];
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
// lie with their number xored with the row's, which halves the conflicts of the
// operand reads and leaves 4.9 clocks of an LDS instruction's 8.9 (a lane's chunks
// 2c and 2c + 1 keep the row's parity, so a read meets half of the banks; rows r
// and r + 8 of ss share one).  The rows' scales come 8 blocks
// at a time (loaded a block at a time into registers they cost a quarter of the
// time: as many lines as the operands, and a wait).
constexpr int kMmScales = 8;  // blocks' scales brought at a time
template <int WO, int WT, int MO, int TT, int KG, bool EXACT>
__global__ __launch_bounds__(KG* WO* WT* kWave, 2) void tile_kernel(const MatmulArgs A) {
  constexpr int BO = WO * MO * 16, BT = WT * TT * 16, kThreads = WO * WT * kWave;
  constexpr uint32_t kStage = (BO + BT) * 128;
  constexpr int kLoads = (BO + BT) * 8 / kThreads;
  static_assert(kLoads * kThreads == (BO + BT) * 8, "whole loads");
  static_assert((BO * 8) % kThreads == 0, "a load is of weights or of rows");
  __shared__ __align__(16) uint8_t lds[KG * 2 * kStage];
  __shared__ float ss[KG][2][BT][kMmScales];
  // (thread and wave of a group)
  const int kg = wave_id() / (WO * WT), t = (int)threadIdx.x - kg * kThreads, lane = t & (kWave - 1), wv = wave_id() - kg * (WO * WT);
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
  const uint32_t lds0 = (uint32_t)(uintptr_t)(mm_lds_ptr)lds + (uint32_t)kg * (2 * kStage);
  uint8_t* const mine = lds + kg * (2 * kStage);
  const auto issue = [&](int b, uint32_t buf) {
    // in the last, short block a chunk behind the row's end reads the row's
    // last instead; zeros take its place before the product
    const int jmax = min(8, (A.K - b * 128) / 16) - 1;
    const int row0 = t >> 3, j = min((t & 7) ^ (row0 & 7), jmax);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      constexpr int kRows = kThreads / 8;  // rows a load; (a multiple of 8: the swizzle is the thread's)
      static_assert(kRows % 8 == 0, "the swizzle");
      const bool weights = i * kRows < BO;
      const int last = weights ? A.N - 1 - o0 : rows.y - 1 - rows.x, first = weights ? i * kRows : i * kRows - BO;
      const uint8_t* base = (weights ? wbase + (long)o0 * A.K : abase) + (long)b * 128;
      const uint32_t o = (uint32_t)min(first + row0, last) * (uint32_t)A.K + 16u * j;
      const uint32_t dst = __builtin_amdgcn_readfirstlane(lds0 + buf + (uint32_t)(i * kThreads + wv * kWave) * 16u);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                   :
                   : "s"(dst), "v"(o), "s"(base)
                   : "memory", "m0");
    }
  };
  // the scales of the wave's outputs' block, by scalar loads
  const auto* sw = (const_float_ptr)(A.w_scale + ((long)e * A.nblocks + min(o0 + wo * MO * 16, A.N - 1) / 128) * A.kblocks);
  static_assert(MO * 16 <= 128 && 128 % (MO * 16) == 0, "a wave's outputs share a block");
  // those of the rows, for the group's kMmScales blocks from the i-th on
  const float* sbase = A.a_scale + (long)rows.x * A.a_groups;
  const uint32_t ss0 = (uint32_t)(uintptr_t)(mm_lds_ptr)ss[kg];
  const auto issue_scales = [&](int i0, int place) {
    constexpr int kEach = BT * kMmScales / kThreads;
    static_assert(kEach * kThreads == BT * kMmScales, "whole loads");
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int p = i * kThreads + t;
      const uint32_t row = (uint32_t)min(p / kMmScales, rows.y - 1 - rows.x), k = (uint32_t)min((i0 + p % kMmScales) * KG + kg, A.a_groups - 1);
      const uint32_t dst = __builtin_amdgcn_readfirstlane(ss0 + (uint32_t)(place * (BT * kMmScales) + i * kThreads + wv * kWave) * 4u);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                   :
                   : "s"(dst), "v"(4u * (row * (uint32_t)A.a_groups + k)), "s"(sbase)
                   : "memory", "m0");
    }
  };

  const uint32_t swz0 = (uint32_t)(((2 * c) ^ (r & 7)) * 16), swz1 = (uint32_t)(((2 * c + 1) ^ (r & 7)) * 16);
  const uint32_t wofs = (uint32_t)(wo * MO * 16 + r) * 128u, aofs = (uint32_t)(BO + wt * TT * 16 + r) * 128u;
  v4f acc[MO][TT];
#pragma unroll
  for (int m = 0; m < MO; ++m)
#pragma unroll
    for (int i = 0; i < TT; ++i) acc[m][i] = v4f{0.f, 0.f, 0.f, 0.f};
  const bool idle = rows.x + wt * TT * 16 >= rows.y || o0 + wo * MO * 16 >= A.N;  // none of the wave's tiles is needed

  const auto compute = [&](const uint8_t* buf, const float* s) {
    const auto frag = [&](uint32_t at) {
      Operand<EXACT> f;
      f.set(two16(*reinterpret_cast<const uint4*>(buf + at + swz0), *reinterpret_cast<const uint4*>(buf + at + swz1)));
      return f;
    };
    // A tile's results enter the sums one row of tiles later, beside its products.
    Operand<EXACT> a[TT], w = frag(wofs);
#pragma unroll
    for (int i = 0; i < TT; ++i) a[i] = frag(aofs + (uint32_t)i * (16 * 128));
    v4f d[TT];
#pragma unroll
    for (int m = 0; m <= MO; ++m) {
      Operand<EXACT> wn = w;
      if (m + 1 < MO) wn = frag(wofs + (uint32_t)(m + 1) * (16 * 128));
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        v4f x = d[i];
        if (m < MO) x = block_product(w, a[i]);
        if (m > 0)
#pragma unroll
          for (int q = 0; q < 4; ++q) acc[m - 1][i][q] = __builtin_fmaf(s[i], d[i][q], acc[m - 1][i][q]);
        d[i] = x;
      }
      w = wn;
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  issue_scales(0, 0);
  if (kg < A.kblocks) issue(kg, 0u);
  float nw = sw[min(kg, A.kblocks - 1)];
  uint32_t cur = 0;
  const int steps = (A.kblocks + KG - 1) / KG;
  for (int i = 0; i < steps; ++i) {
    const int b = i * KG + kg, nb = b + KG;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // block b has landed (every wave's loads), the other place is free
    const float w = nw;
    if (nb < A.kblocks) {
      nw = sw[nb];
      if ((i + 1) % kMmScales == 0) issue_scales(i + 1, (i + 1) / kMmScales & 1);
      issue(nb, kStage - cur);
    }
    if (i + 1 == steps && A.K % 128) {  // uniform, the last block is short: zeros behind the rows' ends
      const int left = A.K - b * 128;
#pragma unroll
      for (int j0 = 0; j0 < kLoads; ++j0) {
        const int p = j0 * kThreads + t, j = (p & 7) ^ ((p >> 3) & 7);
        if (16 * j >= left) *reinterpret_cast<uint4*>(mine + cur + 16 * p) = make_uint4(0, 0, 0, 0);
      }
      __syncthreads();
    }
    if (!idle && b < A.kblocks) {
      float s[TT];
#pragma unroll
      for (int q = 0; q < TT; ++q) s[q] = ss[kg][i / kMmScales & 1][(wt * TT + q) * 16 + r][i % kMmScales] * w;
      compute(mine + cur, s);
    }
    cur = kStage - cur;
  }
  if constexpr (KG > 1) {  // the other groups' sums, in their order
    static_assert(KG == 2 && WO * WT * MO * TT * kWave * sizeof(v4f) <= sizeof(lds), "the second group's sums fit");
    v4f* const sums = reinterpret_cast<v4f*>(lds) + wv * (MO * TT * kWave) + lane;
    __syncthreads();
    if (kg)
#pragma unroll
      for (int m = 0; m < MO; ++m)
#pragma unroll
        for (int i = 0; i < TT; ++i) sums[(m * TT + i) * kWave] = acc[m][i];
    __syncthreads();
    if (kg) return;
#pragma unroll
    for (int m = 0; m < MO; ++m)
#pragma unroll
      for (int i = 0; i < TT; ++i) acc[m][i] += sums[(m * TT + i) * kWave];
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

template <int MT, int TT, int W, bool EXACT>
static hipError_t launch_rows(MatmulArgs A, hipStream_t s) {
  A.otiles = (A.N + 16 * MT - 1) / (16 * MT);
  hipLaunchKernelGGL((rows_kernel<MT, TT, W, EXACT>), dim3((unsigned)((long)A.otiles * A.experts)), dim3(W * kWave), 0, s, A);
  return hipGetLastError();
}

template <int KG, bool EXACT>
static hipError_t launch_tiles(const MatmulArgs& A, hipStream_t s) {
  const long total = (long)A.rtiles * A.otiles;
  hipLaunchKernelGGL((tile_kernel<2, 2, 4, 4, KG, EXACT>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(KG * 4 * kWave), 0, s, A);
  return hipGetLastError();
}

template <bool EXACT>
static hipError_t launch_matmul(MatmulArgs A, hipStream_t s) {
  const long per = ((long)A.rows + A.experts - 1) / A.experts;
  if (per <= 32) {
    // few outputs of long rows: a workgroup's waves are all the loads its CU has under way
    const bool narrow = (long)A.experts * ((A.N + 15) / 16) <= 2L * device_cu_count() && A.kblocks >= 32;
    if (per <= 16 && A.experts == 1) return narrow ? launch_rows<1, 1, 16, EXACT>(A, s) : launch_rows<2, 1, 4, EXACT>(A, s);
    return narrow ? launch_rows<1, 2, 16, EXACT>(A, s) : launch_rows<2, 2, 4, EXACT>(A, s);
  }
  A.otiles = (A.N + 127) / 128;
  // every expert's last tile may be short
  A.rtiles = A.offsets ? A.rows / 128 + std::min(A.experts, A.rows) : (A.rows + 127) / 128;
  // no more tiles than CUs: two groups of waves share a tile's blocks
  return (long)A.rtiles * A.otiles <= device_cu_count() ? launch_tiles<2, EXACT>(A, s) : launch_tiles<1, EXACT>(A, s);
}

hipError_t launch_fp8_matmul(MatmulArgs A, hipStream_t s) {
  A.kblocks = (A.K + 127) / 128;
  A.nblocks = (A.N + 127) / 128;
  // 4 outputs are one store where every row begins on its boundary
  A.wide_out = A.N % 4 == 0 && ((uintptr_t)A.out & (A.out_dtype == kF32 ? 15 : 7)) == 0;
  return A.out_dtype == kF32 ? launch_matmul<true>(A, s) : launch_matmul<false>(A, s);
}

}  // namespace dsa
