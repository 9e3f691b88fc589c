// Sparse / dense MLA decode over a latent cache held in 4 bits (gfx950):
//   out[b,h,:] = sum_j softmax_j(sm * q[b,h,:] . kv_j) * kv_j[:512],
//   kv_j = e2m1 * 2^(scale byte[d/32] - 127) | bf16 rope, from a 400-byte row
//   [256 B: value 2i in the low half of byte i][16 e8m0][64 bf16].
// One value of a row is a 2-bit significand times a power of two, so its bf16
// form is exact.
//
// A workgroup (4 waves) takes a chunk of a row's keys for 32 heads, 128 keys a
// tile, two workgroups a CU.  The rows go from memory straight to LDS, as they
// are.  Each wave multiplies its 32 keys with the queries (S^T = K Q^T, the rows
// dequantised in registers by v_cvt_scalef32_pk_bf16_fp4) and leaves the
// probabilities in LDS; after a barrier each adds up 128 of the 512 dims over
// all 128 keys (O^T = V^T P^T).  V^T comes out of the matrix unit too: a
// 32x32x64 fp4 product of the rows as they lie in LDS, with their scales, and a
// matrix of ones and zeros that picks 32 dims gives their values with a dim in
// each lane and the keys in its registers, which rounds to the next product's A
// operand (exactly) without moving.  So a tile passes through LDS once in 4
// bits: a transpose of the bf16 values there cost 16 clocks a KB written, and
// sums of whole heads a wave 3-4 us at a chunk's end, where the waves' met.
//
// Chunks of the same row meet in a second, small launch: no workgroup waits
// for another, so the call needs no co-residency and keeps no state in its
// workspace.

#include <algorithm>
#include <type_traits>

#include "dsa_common.h"
#include "dsa_kernels.h"
#include "quant_core.h"

namespace dsa {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef int v8i_m4 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(1))) const void* m4_gvoid_ptr;
typedef __attribute__((address_space(3))) void* m4_lvoid_ptr;

constexpr int kM4Waves = 4;
constexpr int kM4Threads = kM4Waves * kWave;
constexpr int kM4Heads = 32;                        // heads a workgroup
constexpr int kM4Keys = 32;                         // keys a wave
constexpr int kM4Unit = kM4Waves * kM4Keys;         // keys a tile: chunks are multiples
constexpr int kM4QLd = DSA_QK_DIM + 8;              // query row stride while they are staged (bf16)
constexpr int kM4QReg = 16;                         // of the 36 query operands, those kept in registers
constexpr int kM4MergeThreads = 256;
constexpr int kM4MergeMax = 512;                    // chunks of a row
constexpr int kM4Ahead = 8;
constexpr float kM4Rise = 16.f;                     // log2 growth of the maximum that rescales the sums
constexpr size_t kM4WaveLds = (size_t)kM4Keys * DSA_FP4_ROW_BYTES;
constexpr size_t kM4RowLds = kM4Waves * kM4WaveLds;
constexpr size_t kM4ProbLds = (size_t)kM4Waves * 2 * kWave * 16;
constexpr size_t kM4QLds = (size_t)(36 - kM4QReg) * kWave * 16;
constexpr size_t kM4Lds = kM4RowLds + kM4ProbLds + kM4QLds;
static_assert((size_t)kM4Heads * kM4QLd * 2 <= kM4RowLds, "the queries are staged where the rows go");
static_assert(kM4Lds + 2048 <= 80 * 1024, "two workgroups a CU");

__device__ __forceinline__ v8bf m4_bf8(const uint4& a) {
  v8bf v;
  __builtin_memcpy(&v, &a, 16);
  return v;
}
__device__ __forceinline__ v8i_m4 m4_fp4(const uint4& a) { return v8i_m4{(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}; }
// A wave's 32 rows in LDS (fetch, below): where row r's pieces begin, and the
// order of its four pieces of a 64-byte line.
constexpr int kM4Last = 24 * kM4Keys * 16;
__device__ __forceinline__ int m4_piece(int r) { return (r >> 4) * 6144 + (r & 15) * 64; }
__device__ __forceinline__ int m4_swz(int r) { return r >> 2 & 3; }
// op over the two half-waves (lane l and l ^ 32)
template <class F>
__device__ __forceinline__ float m4_halves(float v, F op) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// heads of a block that there is room for in the partials
__device__ __host__ __forceinline__ int m4_heads(int H) { return H < kM4Heads ? H : kM4Heads; }

// The chunks of the rows, the same in every wave that asks.  Row b's keys are
// cut into chunks of `units` * kM4Unit; their partials lie behind those of
// the rows before it.
struct M4Plan {
  int units;  // of kM4Unit keys, a chunk
  int first;  // chunk number of the row's first
  int count;  // chunks of the row
};

__device__ __forceinline__ int m4_row_keys(const Mla4Args& A, int b) {
  return A.dense_pt ? max(0, min(A.dense_lens[b], A.keys)) : A.keys;
}

// Ragged rows share A.chunks chunks: the smallest chunk with which all rows'
// chunks fit, or one chunk a row.  Returns the keys' units a chunk.
__device__ __forceinline__ int m4_ragged_units(const Mla4Args& A, int lane) {
  uint32_t total = 0, longest = 0;
  for (int b0 = 0; b0 < A.B; b0 += kWave) {
    const int b = b0 + lane;
    const uint32_t u = b < A.B ? (uint32_t)(m4_row_keys(A, b) + kM4Unit - 1) / kM4Unit : 0u;
    total += wave_reduce<0>(u);
    longest = max(longest, wave_reduce<2>(u));
  }
  uint32_t cu = max(1u, (total + A.chunks - 1) / A.chunks);
  while (cu < longest) {
    uint32_t n = 0;
    for (int b0 = 0; b0 < A.B; b0 += kWave) {
      const int b = b0 + lane;
      const uint32_t u = b < A.B ? (uint32_t)(m4_row_keys(A, b) + kM4Unit - 1) / kM4Unit : 0u;
      n += wave_reduce<0>((u + cu - 1) / cu);
    }
    if (n <= (uint32_t)A.chunks) break;
    cu += max(1u, cu / 16);
  }
  return (int)cu;
}

// Row b's chunks.
__device__ __forceinline__ M4Plan m4_plan_row(const Mla4Args& A, int b, int lane) {
  M4Plan p;
  if (A.units) {  // rows of one length (selections), or a chunk a row
    p.units = A.units;
    p.count = A.per_row;
    p.first = b * A.per_row;
    return p;
  }
  p.units = m4_ragged_units(A, lane);
  p.first = 0;
  for (int b0 = 0; b0 <= b; b0 += kWave) {
    const int r = b0 + lane;
    const uint32_t u = r < A.B ? (uint32_t)(m4_row_keys(A, r) + kM4Unit - 1) / kM4Unit : 0u;
    const uint32_t c = (u + p.units - 1) / p.units;
    p.first += (int)wave_reduce<0>(r < b ? c : 0u);
    const uint32_t mine = wave_reduce<0>(r == b ? c : 0u);
    if (b < b0 + kWave) p.count = (int)mine;
  }
  return p;
}

// The row of chunk `id` (-1: none) and its plan.
__device__ __forceinline__ int m4_plan_chunk(const Mla4Args& A, int id, int lane, M4Plan& p) {
  if (A.units) {
    p.units = A.units;
    p.count = A.per_row;
    const int b = id / A.per_row;
    p.first = b * A.per_row;
    return b < A.B ? b : -1;
  }
  p.units = m4_ragged_units(A, lane);
  int before = 0;
  for (int b0 = 0; b0 < A.B; b0 += kWave) {
    const int r = b0 + lane;
    const uint32_t u = r < A.B ? (uint32_t)(m4_row_keys(A, r) + kM4Unit - 1) / kM4Unit : 0u;
    const uint32_t c = (u + p.units - 1) / p.units;
    const int end = before + (int)wave_scan_incl<0>(c);
    const uint64_t hit = __ballot(id < end && id >= end - (int)c);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      p.count = __builtin_amdgcn_readlane((int)c, src);
      p.first = __builtin_amdgcn_readlane(end, src) - p.count;
      return b0 + src;
    }
    before = __builtin_amdgcn_readlane(end, kWave - 1);
  }
  return -1;
}

template <bool DENSE>
__global__ __launch_bounds__(kM4Threads, 2) void mla_fp4_kernel(const Mla4Args A) {
  extern __shared__ __align__(16) unsigned char smem[];  // rows | probabilities | queries
  __shared__ __align__(16) float ref[kM4Heads][kM4Waves], wl[kM4Waves][kM4Heads];
  __shared__ __align__(16) uint32_t there[2][kM4Waves];  // a bit a key
  const int t = threadIdx.x, lane = t & (kWave - 1), wv = wave_id();
  const int n = lane & 31, h = lane >> 5;
  // a chunk's head blocks on one XCD (workgroup number modulo 8), whose L2
  // then serves all but the first's reads of its rows
  const int nhb = (A.H + kM4Heads - 1) / kM4Heads;
  const int hb = (blockIdx.x / 8) % nhb, id = (blockIdx.x / (8 * nhb)) * 8 + blockIdx.x % 8;
  M4Plan plan;
  const int b = m4_plan_chunk(A, id, lane, plan);
  if (b < 0) return;  // (the same in the whole workgroup)
  const int total = m4_row_keys(A, b);
  const long j0 = (long)(id - plan.first) * plan.units * kM4Unit;
  const int jend = (int)min((long)total, j0 + (long)plan.units * kM4Unit);
  const int tiles = (int)((max((long)jend, j0) - j0 + kM4Unit - 1) / kM4Unit);
  const int* idx_row = DENSE ? A.dense_pt + (long)b * A.dense_pt_stride : A.idx + (long)b * A.keys;
  // Key n of this wave's 32 in a tile: its index entry (read a tile ahead) and
  // its slot; -1: not there (row 0 is read then, and its probability is 0).
  const auto entry = [&](int tl) {
    const long j = max(min(j0 + (long)tl * kM4Unit + kM4Keys * wv + n, (long)jend - 1), 0L);
    return idx_row[DENSE ? j >> 6 : j];
  };
  const auto slot = [&](int tl, int e) {
    const long j = j0 + (long)tl * kM4Unit + kM4Keys * wv + n;
    const long sl = DENSE ? (long)e * DSA_PAGE_TOKENS + (j & (DSA_PAGE_TOKENS - 1)) : (long)e;
    return j < jend && e >= 0 && sl < A.kv_rows ? (int)sl : -1;
  };
  // This wave's rows to LDS, 16-byte piece by piece: pieces 4k .. 4k + 3 of 16
  // rows a load (64 bytes a row together), then the last pieces of all 32.
  // Piece q < 24 of row r lies at m4_piece(r) + 1024 (q / 4) + 16 ((q % 4) ^ m4_swz(r)),
  // piece 24 at kM4Last + 16 r: 8 rows' reads of one piece fall on 8 bank
  // groups, and a load needs no more than its lane's pointer.
  const auto fetch = [&](int sl) {
    const int from = sl < 0 ? 0 : sl;
    const uint8_t* src[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int r = 16 * k + (lane >> 2);
      src[k] = A.pool + (long)__builtin_amdgcn_ds_bpermute(r << 2, from) * DSA_FP4_ROW_BYTES + 16 * ((lane & 3) ^ m4_swz(r));
    }
    unsigned char* dst = smem + wv * kM4WaveLds;
#pragma unroll
    for (int k = 0; k < 12; ++k)
      __builtin_amdgcn_global_load_lds((m4_gvoid_ptr)(src[k / 6] + 64 * (k % 6)), (m4_lvoid_ptr)(dst + 1024 * k), 16, 0, 0);
    if (lane < kM4Keys)
      __builtin_amdgcn_global_load_lds((m4_gvoid_ptr)(A.pool + (long)from * DSA_FP4_ROW_BYTES + 384), (m4_lvoid_ptr)(dst + kM4Last), 16,
                                       0, 0);
  };

  // The queries, the B operand of QK (n = head): staged where the rows will go,
  // then to registers and a piece of LDS.  Operand 4i + u: dims 64i + 32h + 8u
  // .. + 7; 32 + u: rope dims 32h + 8u .. + 7.
  uint4* const qlds = reinterpret_cast<uint4*>(smem + kM4RowLds + kM4ProbLds) + lane;
  uint4 qf[kM4QReg];
  int sl = -1, e1 = 0;
  {
    constexpr int kRowVec = DSA_QK_DIM / 8, kPer = kM4Heads * kRowVec / kM4Threads;
    static_assert(kPer * kM4Threads == kM4Heads * kRowVec, "whole loads");
    int e = 0;
    if (tiles) e = entry(0), e1 = entry(1);
    const uint4* src = reinterpret_cast<const uint4*>(A.q + (long)b * A.H * DSA_QK_DIM);
    uint16_t* qs = reinterpret_cast<uint16_t*>(smem);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int i = t + k * kM4Threads;
      *reinterpret_cast<uint4*>(qs + (i / kRowVec) * kM4QLd + (i % kRowVec) * 8) =
          src[(long)min(hb * kM4Heads + i / kRowVec, A.H - 1) * kRowVec + i % kRowVec];
    }
    __syncthreads();
    const auto at = [&](int kk) {
      return *reinterpret_cast<const uint4*>(
          qs + n * kM4QLd + (kk < 32 ? 64 * (kk >> 2) + 32 * h + 8 * (kk & 3) : DSA_LATENT_DIM + 32 * h + 8 * (kk - 32)));
    };
#pragma unroll
    for (int kk = 0; kk < kM4QReg; ++kk) qf[kk] = at(kk);
    for (int kk = kM4QReg + wv; kk < 36; kk += kM4Waves) qlds[(kk - kM4QReg) * kWave] = at(kk);
    __syncthreads();
    if (tiles) fetch(sl = slot(0, e));
  }

  // Where this lane reads row n of a wave's 32: pieces 2i + h (dims 64i + 32h ..)
  // at code[i & 1] + 1024 (i / 2), the scales (piece 16) at scales, rope pieces
  // 17 + 4h + u at rope[u]; of all waves', dims 128 wv + 64 g + 32 h .. at
  // dims[g], their scales at dscales
  uint32_t code_at[2], dims_at[2], rope_at[4];
  const uint32_t row0 = m4_piece(n), swz = m4_swz(n), base = wv * kM4WaveLds;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    code_at[g] = base + row0 + 16 * ((2 * g + h) ^ swz);
    dims_at[g] = row0 + 1024 * wv + 16 * ((2 * g + h) ^ swz);
  }
  const uint32_t scales_at = base + row0 + 4096 + 16 * swz, dscales_at = row0 + 4096 + 16 * swz + 4 * wv;
#pragma unroll
  for (int u = 0; u < 3; ++u) rope_at[u] = base + row0 + 4096 + 1024 * h + 16 * ((u + 1) ^ swz);
  rope_at[3] = base + (h ? kM4Last + 16 * n : row0 + 5120 + 16 * swz);
  // [wave][16 keys][lane]: the lane's 8 probabilities of its head
  uint4* const probs = reinterpret_cast<uint4*>(smem + kM4RowLds) + lane;
  v16f o[4];  // O^T: dims 128 wv + 32 d + 8 (e / 4) + 4h + e % 4 of head n
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  // All sums are relative to `top`, the same in every wave, which trails the
  // maximum by at most kM4Rise.  It is a whole number, so that what is brought
  // down to a new one is scaled by a power of two, without another rounding.
  float top = -INFINITY, l = 0.f;
  const auto row_max = [&] {
    const v4f a = *reinterpret_cast<const v4f*>(&ref[n][0]);
    return fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3]));
  };

#pragma unroll 1
  for (int tl = 0; tl < tiles; ++tl) {
    // S^T: this wave's 32 keys, when their rows are there (the others' are
    // waited for with the probabilities)
    const uint32_t ok = (uint32_t)__ballot(sl >= 0);
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    asm volatile("" ::: "memory");
    uint4 code[kM4Ahead];
    const uint4 scv = *reinterpret_cast<const uint4*>(smem + scales_at);
    const auto codes = [&](int i) { code[i % kM4Ahead] = *reinterpret_cast<const uint4*>(smem + code_at[i & 1] + 1024 * (i >> 1)); };
#pragma unroll
    for (int i = 0; i < kM4Ahead; ++i) codes(i);
    if (lane == 0) there[tl & 1][wv] = ok;
    v16f s[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) s[0][e] = s[1][e] = 0.f;
    const auto product = [&](int kk, const uint4& k) {
      s[kk & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
          m4_bf8(k), m4_bf8(kk < kM4QReg ? qf[kk < kM4QReg ? kk : 0] : qlds[(kk - kM4QReg) * kWave]), s[kk & 1], 0, 0, 0);
    };
    const uint32_t scw[4] = {scv.x, scv.y, scv.z, scv.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float sc = __uint_as_float(((scw[i >> 1] >> (16 * (i & 1) + 8 * h)) & 0xffu) << 23);
      const uint4 c = code[i % kM4Ahead];
      product(4 * i, dequant8_fp4(c.x, sc));
      product(4 * i + 1, dequant8_fp4(c.y, sc));
      product(4 * i + 2, dequant8_fp4(c.z, sc));
      product(4 * i + 3, dequant8_fp4(c.w, sc));
      if (i + kM4Ahead < 8) codes(i + kM4Ahead);
      __builtin_amdgcn_sched_barrier(0x7ff);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      product(32 + u, *reinterpret_cast<const uint4*>(smem + rope_at[u]));
    // element e is key 8 (e / 4) + 4h + e % 4 of head n
    float tmax = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) s[0][e] = (s[0][e] + s[1][e]) * A.sm_log2;
    if (ok != ~0u) {  // keys that are not there
#pragma unroll
      for (int e = 0; e < 16; ++e) s[0][e] = (ok >> (4 * h)) & (1u << (8 * (e >> 2) + (e & 3))) ? s[0][e] : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) tmax = fmaxf(tmax, s[0][e]);
    tmax = m4_halves(tmax, [](float x, float y) { return fmaxf(x, y); });
    if (tl == 0) {  // the first tile's maximum is agreed on; later ones are seldom above it
      if (h == 0) ref[n][wv] = tmax;
      __syncthreads();
      top = ceilf(row_max());
      __syncthreads();
    }
    const float own = tmax > top + kM4Rise || top == -INFINITY ? ceilf(fmaxf(tmax, top)) : top;
    const float at = own == -INFINITY ? 0.f : own;
    uint32_t pk[8];
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      pk[e >> 1] = pack_bf16x2(__builtin_amdgcn_exp2f(s[0][e] - at), __builtin_amdgcn_exp2f(s[0][e + 1] - at));
      // the sum of the rounded probabilities, the ones PV multiplies: the
      // weights then add up to one
      sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, pk[e >> 1]), __builtin_bit_cast(v2bf, 0x3f803f80u), sum,
                                            false);
    }
    probs[(2 * wv) * kWave] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
    probs[(2 * wv + 1) * kWave] = make_uint4(pk[4], pk[5], pk[6], pk[7]);
    if (h == 0) ref[n][wv] = own;
    __syncthreads();  // the tile's probabilities and rows are there
    const float now = row_max();
    const bool uneven = __ballot(now != top) != 0;  // (the same in every wave)
    if (uneven) {  // a wave went above `top`: what is there comes down to the new one
      const float down = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now);
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= down;
      l *= down;
      const float f = own == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(own - now);
      sum *= f;
#pragma unroll
      for (int e = 0; e < 8; ++e) pk[e] = pack_bf16x2(bf16_lo(pk[e]) * f, bf16_hi(pk[e]) * f);
      probs[(2 * wv) * kWave] = make_uint4(pk[0], pk[1], pk[2], pk[3]);
      probs[(2 * wv + 1) * kWave] = make_uint4(pk[4], pk[5], pk[6], pk[7]);
      top = now;
      __syncthreads();
    }
    l += sum;

    const int e2 = entry(tl + 2);
    // O^T: this wave's 128 dims over blocks of 32 keys x 32 dims.  Block i: keys
    // 32 (i / 4) .., dims 128 wv + 32 (i % 4) ..; its values (V^T by the fp4
    // product) are two blocks ahead of their use.
    const uint4 there4 = *reinterpret_cast<const uint4*>(there[tl & 1]);
    const uint32_t th[4] = {there4.x, there4.y, there4.z, there4.w};
    uint32_t sc[kM4Waves];
#pragma unroll
    for (int kb = 0; kb < kM4Waves; ++kb) {
      // scale bytes of dims 128 wv + 64 g + 32 h: byte 2g after the shift; a
      // row that is not there at scale 1 (finite values)
      sc[kb] = *reinterpret_cast<const uint32_t*>(smem + dscales_at + kb * kM4WaveLds) >> (8 * h);
      sc[kb] = th[kb] >> n & 1 ? sc[kb] : 0x7f7f7f7fu;
    }
    // piece k: keys 32 (k / 2) .., dims 128 wv + 64 (k % 2) + 32 h ..
    const auto piece = [&](int k) {
      return *reinterpret_cast<const uint4*>(smem + dims_at[k & 1] + (k >> 1) * kM4WaveLds);
    };
    uint4 c[3] = {piece(0), piece(1), piece(2)};
    // The B operand that picks dims 32 half .. + 31 of 64: a one (code 2) at
    // k = 32 half + n (made here again each tile: its registers serve QK too)
    int ln = lane;
    asm volatile("" : "+v"(ln));
    uint4 pick[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t one = ln >> 5 == half ? 2u << (4 * (ln & 7)) : 0u;
      const int w = ln >> 3 & 3;
      pick[half] = make_uint4(w == 0 ? one : 0u, w == 1 ? one : 0u, w == 2 ? one : 0u, w == 3 ? one : 0u);
    }
    uint4 pr[2][2];
    const auto take = [&](int kb) {
#pragma unroll
      for (int k = 0; k < 2; ++k) pr[kb & 1][k] = probs[(2 * kb + k) * kWave];
    };
    take(0);
    const auto values = [&](int i) {
      const int kb = i >> 2, g = i >> 1 & 1, half = i & 1;
      v16f v;
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = 0.f;
      const v8i_m4 a = m4_fp4(c[(2 * kb + g) % 3]), p = m4_fp4(pick[half]);
      return g ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, p, v, 4, 4, 2, (int)sc[kb], 0, 0x7f7f7f7f)
               : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, p, v, 4, 4, 0, (int)sc[kb], 0, 0x7f7f7f7f);
    };
    v16f v[2] = {values(0), values(1)};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i % 4 == 0 && i < 12) take(i / 4 + 1);
      uint32_t w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = pack_bf16x2(v[i & 1][2 * e], v[i & 1][2 * e + 1]);
      __builtin_amdgcn_sched_barrier(0);  // (the next values go where these were)
      v16f& acc = o[i & 3];
      if (i + 2 < 16) v[i & 1] = values(i + 2);
      if (i % 2 == 1 && i / 2 + 3 < 8) c[(i / 2 + 3) % 3] = piece(i / 2 + 3);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(m4_bf8(make_uint4(w[0], w[1], w[2], w[3])), m4_bf8(pr[i >> 2 & 1][0]), acc, 0, 0, 0);
      acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(m4_bf8(make_uint4(w[4], w[5], w[6], w[7])), m4_bf8(pr[i >> 2 & 1][1]), acc, 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();  // the rows have been used
    if (tl + 1 < tiles) fetch(sl = slot(tl + 1, e1));
    e1 = e2;
  }

  l = m4_halves(l, [](float x, float y) { return x + y; });
  if (h == 0) wl[wv][n] = l;
  __syncthreads();
  float L = 0.f;
#pragma unroll
  for (int w = 0; w < kM4Waves; ++w) L += wl[w][n];
  const int head = hb * kM4Heads + n;
  if (head >= A.H) return;
  if (plan.count > 1) {
    // quad q (dims 8q + 4h .. + 3) of the lane's head, a lane after the other
    const long at = (long)id * nhb + hb;
    const int heads = m4_heads(A.H);
    v4f* part = reinterpret_cast<v4f*>(A.part_o) + at * (heads * DSA_LATENT_DIM / 4) + h * heads + n;
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const v16f& a = o[q >> 2];
      part[(16 * wv + q) * 2 * heads] = v4f{a[4 * (q & 3)], a[4 * (q & 3) + 1], a[4 * (q & 3) + 2], a[4 * (q & 3) + 3]};
    }
    if (t < kM4Heads) {
      A.part_ml[2 * (at * heads + n)] = top;
      A.part_ml[2 * (at * heads + n) + 1] = L;
    }
    return;
  }
  const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);  // no key: 0; NaN stays
  uint16_t* out = A.out + ((long)b * A.H + head) * DSA_LATENT_DIM + 128 * wv + 4 * h;
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const v16f& a = o[q >> 2];
    v2u_t w;
    w[0] = pack_bf16x2(a[4 * (q & 3)] * inv, a[4 * (q & 3) + 1] * inv);
    w[1] = pack_bf16x2(a[4 * (q & 3) + 2] * inv, a[4 * (q & 3) + 3] * inv);
    *reinterpret_cast<v2u_t*>(out + 8 * q) = w;
  }
}

// The chunks of a row meet: a workgroup takes kM4Quads of the 64 quads of a
// (row, head block), its waves every fourth chunk each; then the waves' sums
// meet in LDS.  Always in the same order.
constexpr int kM4Quads = 2;
constexpr int kM4MergeWaves = kM4MergeThreads / kWave;

__global__ __launch_bounds__(kM4MergeThreads) void mla_fp4_merge_kernel(const Mla4Args A) {
  __shared__ float sm[kM4MergeWaves][kM4Heads], sl[kM4MergeWaves][kM4Heads];
  __shared__ v4f so[kM4MergeWaves][kM4Quads][kWave];
  const int lane = threadIdx.x & (kWave - 1), wv = wave_id(), n = lane & 31, h = lane >> 5;
  const int nhb = (A.H + kM4Heads - 1) / kM4Heads;
  constexpr int kPer = 64 / kM4Quads;  // workgroups a (row, head block)
  const int q0 = (int)(blockIdx.x % kPer) * kM4Quads, hb = (int)(blockIdx.x / kPer % nhb), b = (int)(blockIdx.x / kPer / nhb);
  const M4Plan p = m4_plan_row(A, b, lane);
  if (p.count == 1) return;  // (the same in the whole workgroup)
  const int head = hb * kM4Heads + n;
  const bool in = head < A.H;
  const int heads = m4_heads(A.H);
  const v4f* part = reinterpret_cast<const v4f*>(A.part_o);
  const auto at = [&](int c) { return (long)(p.first + c) * nhb + hb; };
  float mx = -INFINITY;
  if (in)
    for (int c = 2 * wv + h; c < p.count; c += 2 * kM4MergeWaves) mx = fmaxf(mx, A.part_ml[2 * (at(c) * heads + n)]);
  mx = m4_halves(mx, [](float x, float y) { return fmaxf(x, y); });
  if (h == 0) sm[wv][n] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kM4MergeWaves; ++w) mx = fmaxf(mx, sm[w][n]);
  v4f acc[kM4Quads];
#pragma unroll
  for (int k = 0; k < kM4Quads; ++k) acc[k] = v4f{0.f, 0.f, 0.f, 0.f};
  float L = 0.f;
  if (in) {
#pragma unroll 4
    for (int c = wv; c < p.count; c += kM4MergeWaves) {
      const float m = A.part_ml[2 * (at(c) * heads + n)], lc = A.part_ml[2 * (at(c) * heads + n) + 1];
      const float f = m == -INFINITY ? 0.f : exp2f(m - mx);
      L += lc * f;
#pragma unroll
      for (int k = 0; k < kM4Quads; ++k) acc[k] += part[(at(c) * 128 + 2 * (q0 + k) + h) * heads + n] * f;
    }
  }
  if (h == 0) sl[wv][n] = L;
#pragma unroll
  for (int k = 0; k < kM4Quads; ++k) so[wv][k][lane] = acc[k];
  __syncthreads();
  if (wv >= kM4Quads || !in) return;
  L = 0.f;
  v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < kM4MergeWaves; ++w) {
    L += sl[w][n];
    x += so[w][wv][lane];
  }
  const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
  v2u_t w;
  w[0] = pack_bf16x2(x[0] * inv, x[1] * inv);
  w[1] = pack_bf16x2(x[2] * inv, x[3] * inv);
  *reinterpret_cast<v2u_t*>(A.out + ((long)b * A.H + head) * DSA_LATENT_DIM + 8 * (q0 + wv) + 4 * h) = w;
}

// Head blocks of a call, each a workgroup a chunk.
static int m4_blocks(int H) { return (H + kM4Heads - 1) / kM4Heads; }

// Chunks the rows share: nsplit a row, or (0) what fills the chip once, two a
// CU; at most kM4MergeMax where one row may take them all (kM4Ragged rows and
// fewer).
constexpr int kM4Ragged = 256;
static int m4_chunks(int B, int H, int nsplit) {
  const long want = nsplit > 0 ? (long)B * nsplit : 2L * device_cu_count() / m4_blocks(H);
  return (int)std::max((long)B, B <= kM4Ragged ? std::min(want, (long)kM4MergeMax) : want);
}

// The partials lie behind the barriers that the 8-bit decode keeps in a
// workspace, so calls over both formats may take turns with one.
size_t mla_fp4_workspace_bytes(int B, int H, int nsplit) {
  const int chunks = m4_chunks(B, H, nsplit);
  if (chunks / B <= 1) return 16;  // unsplit rows: none is read
  return attn_workspace_bytes(B, H, 0) + (size_t)chunks * m4_blocks(H) * m4_heads(H) * (DSA_LATENT_DIM + 2) * sizeof(float);
}

hipError_t launch_mla_fp4(Mla4Args A, int nsplit, void* workspace, hipStream_t s) {
  static PerDeviceOnce attr;
  const hipError_t e = attr.run([] {
    for (const void* f : {(const void*)mla_fp4_kernel<false>, (const void*)mla_fp4_kernel<true>})
      if (hipError_t r = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)kM4Lds)) return r;
    return hipSuccess;
  });
  if (e != hipSuccess) return e;
  const int blocks = m4_blocks(A.H);
  const int row_units = (A.keys + kM4Unit - 1) / kM4Unit;
  A.chunks = m4_chunks(A.B, A.H, nsplit);
  A.part_o = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + attn_workspace_bytes(A.B, A.H, 0));
  A.part_ml = A.part_o + (size_t)A.chunks * blocks * m4_heads(A.H) * DSA_LATENT_DIM;
  const int per_row = A.chunks / A.B;
  int grid_chunks = A.chunks;
  if (per_row <= 1 || !A.dense_pt || A.B > kM4Ragged) {  // the same split for every row
    A.units = (row_units + per_row - 1) / per_row;
    A.per_row = (row_units + A.units - 1) / A.units;
    grid_chunks = A.B * A.per_row;
  }
  const dim3 grid((unsigned)((grid_chunks + 7) / 8 * 8 * blocks));
  const auto kernel = A.dense_pt ? mla_fp4_kernel<true> : mla_fp4_kernel<false>;
  hipLaunchKernelGGL(kernel, grid, dim3(kM4Threads), kM4Lds, s, A);
  if (hipError_t r = hipGetLastError()) return r;
  if (A.units && A.per_row == 1) return hipSuccess;
  hipLaunchKernelGGL(mla_fp4_merge_kernel, dim3((unsigned)(A.B * blocks * (64 / kM4Quads))), dim3(kM4MergeThreads), 0, s, A);
  return hipGetLastError();
}

}  // namespace dsa
