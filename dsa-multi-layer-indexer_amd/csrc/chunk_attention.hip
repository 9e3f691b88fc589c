// Attention of new tokens over the paged latent cache (gfx950): the last tokens
// of several requests at once, each over its request's keys up to its own.
//
//   out[r, :] = sum_j softmax_j(sm * q[r, :] . k_j) * k_j[:512]
//
// over the keys j <= pos(i), where row r = (token i, head h).  All heads share
// the keys, so a request's rows, tokens times heads, are one tall matrix against
// them: the tile of prefill.hip, 128 rows against 32 keys, whose softmax and
// operand layout this kernel has too.  What differs is where the keys come from
// and how the work is cut.
//
// Keys: a tile is half a page, one contiguous piece of the pool.  It goes from
// memory straight to LDS as it is (656 or 400 bytes a row), two places, and the
// workgroup dequantises it once, into a bf16 tile for its 128 rows: tile t + 2
// while t is summed and t + 1 scored, with t + 3 on its way.  (Rows unpacked to bf16 in
// memory first, as prefill.hip has them, cost 2.75 times a row's bytes besides,
// which is more than the attention of up to a few hundred rows.)
//
// Work: the (row tile, key tile) pairs of all requests lie on one line, and each
// workgroup, one a CU, takes an equal share of it, whatever the requests'
// lengths: the tiles in the middle of its share whole, at most one tile that
// began before it and one that ends behind it in part.  Parts leave their sums
// and reference points in the workspace, where a second launch joins them in the
// order of the keys.
//
// 1999 tokens of 16 heads after 16001 keys take 1.25 ms (945 TFLOP/s; a library
// product of 8192 x 8192 x 8192 reaches 1435), 9 ragged chunks of 64 heads over
// 4-bit rows 1.05 ms (877).  Their matrix units are busy 42% and 37% of the clocks
// (1.85 and 2.0 GHz under this load), LDS 30% and 26% with no conflicts, and a wave,
// the only one of its SIMD, waits for a fifth of its time: what is left is where
// products, softmax, unpacking and a tile's first operand reads do not overlap.
// With few rows a key tile's latency shows: 16 requests of 4 tokens and 16 heads,
// 64 of a tile's 128 rows, in 102 us (1 TB/s; over 4-bit rows 97), matrix units busy
// 20%, 3.4 us a key tile against 2.2 for keys in the L2.  Every row tile and part
// of one begins cold besides: the first loads' offsets are spilled (180 and 192
// bytes a lane), and 16 of 18 (10 of 12 over 4-bit rows) wait for the load before
// them when theirs is read back; the steady loop has none of it.
//
// The probabilities are one bf16 term: error 0.0016 of the output's norm where fp32
// ones in torch have 0.0015, nearly all of either the output's rounding.  A second
// term gives 0.0015 for 15 to 25% of the time (the decode kernels, which wait for
// memory, take it for large probabilities).  Also tried and not kept: tiles brought
// into the L2 ahead (none, or 5% slower); waves without rows that dequantise for the
// others (139 us for 113, and the large case 1.5 times as slow: a second path takes
// registers from the first).
#include <algorithm>

#include "dsa_kernels.h"
#include "prefill_core.h"
#include "quant_core.h"

namespace dsa {

constexpr int kCaTileCost = 64;   // keys' worth of a row tile's start and end
constexpr int kCaShare = 128;     // the least share of a workgroup, in keys of a row tile
// A row's reference point lies this far above its first tile's maximum (in
// log2), and a score may rise this far above the reference: any point gives the
// same sums (bf16 and fp32 have 8 bits of exponent, and a probability's error is
// relative) while no probability overflows, and one that underflows is below
// 2^-46 of the row's largest (2^-80 / 2^-126).  Its products with the values lie as
// much lower: a value below 2^-46 makes subnormal sums, which the matrix unit
// keeps (errors as ever at 2^-56, 0.01 at 2^-64, nothing left at 2^-74; rows that
// this library packs have no value but 0 below 2^-38).  A share with a row whose scores
// rise by more, 144 in log2, is summed again from the rows' true maxima
// (a span of 96 redid whole shares for one key of 11 times the others' size, 187 in
// log2: 2.8 ms where 1.3 do).
constexpr float kCaAbove = 80.f, kCaRise = 64.f;
constexpr int kCaDepthK = 8, kCaDepthV = 6;  // operand fragments read ahead of their MFMA

// A workgroup's place on the line of work: request, row tile, key tile of it.
struct ChunkPos {
  int b, tile, kt;
};
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// A request's part of the batch: its rows, tiles and the position of its first
// token (negative: tokens before the first key).
struct ChunkReq {
  int first, T, tiles, P;
};
__device__ __forceinline__ ChunkReq chunk_req(const ChunkAttnArgs& A, int b) {
  ChunkReq r;
  r.first = min(max(A.q_start[b], 0), A.n);
  r.T = min(max(A.q_start[b + 1], r.first), A.n) - r.first;
  r.tiles = (int)(((uint32_t)r.T * (uint32_t)A.H + kPfRows - 1u) / kPfRows);  // (T * H below 2^31)
  r.P = max(A.seq_lens[b], 0) - r.T;
  return r;
}
// Cost of a request's first `t` row tiles, H times keys: 128 rows further down
// are 128 / H tokens, and as many keys, further, from none (tokens before the
// first key) up to what the page table holds.  Within a tile it is at most 64 +
// 8 keys and 1 above the keys that the tile sees, so two places kCaShare apart
// are in different key tiles: no share lies inside a tile without a part of it.
__device__ __forceinline__ long chunk_cost(const ChunkAttnArgs& A, const ChunkReq& r, long t) {
  const long HP = (long)A.H * r.P, most = (long)A.H * A.pt_stride * DSA_PAGE_TOKENS;
  const long none = HP < 0 ? min(t, -HP / kPfRows) : 0;  // tiles without a key
  const long from = max(0L, min(HP, most));
  const long grow = min(t - none, max(0L, (most - from) / kPfRows));
  return t * A.H * kCaTileCost + grow * from + kPfRows / 2 * grow * (grow + 1) + (t - none - grow) * most;
}
// Keys that any row of a tile sees.
__device__ __forceinline__ int chunk_keys(const ChunkAttnArgs& A, const ChunkReq& r, int tile) {
  const uint32_t R = (uint32_t)r.T * (uint32_t)A.H;  // (below 2^31)
  const int s_hi = (int)((min((tile + 1u) * (uint32_t)kPfRows, R) - 1u) / (uint32_t)A.H);
  return max(0, min(r.P + s_hi + 1, A.pt_stride * DSA_PAGE_TOKENS));
}

__device__ __forceinline__ long wave_prefix(long v) {
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const long u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ long lane_value(long v, int l) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)v, l), hi = (uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l);
  return (long)((uint64_t)hi << 32 | lo);
}

// The place at x of the line; every wave finds it for itself.
__device__ __forceinline__ ChunkPos chunk_find(const ChunkAttnArgs& A, long x) {
  const int lane = threadIdx.x & (kWave - 1);
  for (int b0 = 0; b0 < A.B; b0 += kWave) {
    long mine = 0;
    if (b0 + lane < A.B) {
      const ChunkReq r = chunk_req(A, b0 + lane);
      mine = chunk_cost(A, r, r.tiles);
    }
    const long incl = wave_prefix(mine);
    const uint64_t at = __ballot(x < incl);
    if (!at) {
      x -= lane_value(incl, kWave - 1);
      continue;
    }
    const int l = __builtin_ctzll(at), b = b0 + l;
    x -= lane_value(incl - mine, l);
    const ChunkReq r = chunk_req(A, b);
    // the last tile whose start is not behind x, 64 candidates at a time
    long lo = 0, step = 1;
    while (step * kWave < r.tiles) step *= kWave;
    for (;; step /= kWave) {
      const long t = lo + lane * step;
      const uint64_t ok = __ballot(t < r.tiles && chunk_cost(A, r, t) <= x);
      lo += (__builtin_popcountll(ok) - 1) * step;
      if (step == 1) break;
    }
    const int tile = uniform((int)lo);
    const long c0 = chunk_cost(A, r, tile), c1 = chunk_cost(A, r, tile + 1);
    const int kts = (chunk_keys(A, r, tile) + kPfKeys - 1) / kPfKeys;
    // (in fp64: its divisions are short; any rounding of both ends of a share is
    // the same for the share that ends there and the one that begins)
    const int kt = (int)((double)(x - c0) * kts / (double)(c1 - c0));
    return {uniform(b), tile, uniform(max(0, min(kt, kts - 1)))};
  }
  return {A.B, 0, 0};
}

// Workgroups that take a share: as many as there are, or fewer shares that are
// worth their join.
__device__ __forceinline__ long chunk_total(const ChunkAttnArgs& A) {
  const int lane = threadIdx.x & (kWave - 1);
  long sum = 0;
  for (int b0 = 0; b0 < A.B; b0 += kWave) {
    long mine = 0;
    if (b0 + lane < A.B) {
      const ChunkReq r = chunk_req(A, b0 + lane);
      mine = chunk_cost(A, r, r.tiles);
    }
    sum += lane_value(wave_prefix(mine), kWave - 1);
  }
  return sum;
}

// 8 values of a row in LDS, the codes at 8 lane and their scale, to bf16 in
// three steps that take their place between products.
template <int ROW>
struct Latent8 {
  static constexpr bool kE4m3 = ROW == DSA_LATENT_ROW_BYTES;
  v2u_t c;
  float s, f[8];
  __device__ __forceinline__ void load_codes(const uint8_t* row, int lane) {
    if constexpr (kE4m3) c = *reinterpret_cast<const v2u_t*>(row + 8 * lane);
    else c[0] = *reinterpret_cast<const uint32_t*>(row + 4 * lane);
  }
  __device__ __forceinline__ void load_scale(const uint8_t* row, int lane) {
    if constexpr (kE4m3) s = *reinterpret_cast<const float*>(row + DSA_LATENT_DIM + 4 * (lane >> 4));
    else s = __uint_as_float((uint32_t)row[DSA_LATENT_DIM / 2 + (lane >> 2)] << 23);
  }
  __device__ __forceinline__ void unpack() {
    if constexpr (kE4m3) {
      e4m3x4_to_f32(c[0], f);
      e4m3x4_to_f32(c[1], f + 4);
    } else {
      f[0] = __uint_as_float(c[0]);
    }
  }
  __device__ __forceinline__ void scale() {
    if constexpr (kE4m3) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= s;
    } else {
      const uint4 v = dequant8_fp4(__float_as_uint(f[0]), s);
      f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
    }
  }
  __device__ __forceinline__ uint4 bf16() const {
    if constexpr (kE4m3)
      return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
__device__ __forceinline__ bool any_nonfinite(const uint4& v) {
  const auto bad = [](uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; };
  return bad(v.x) || bad(v.y) || bad(v.z) || bad(v.w);
}

typedef const __attribute__((address_space(4))) int* const_int_ptr;

template <int ROW>
__global__ __launch_bounds__(kPfThreads, 1) void chunk_attention_kernel(const ChunkAttnArgs A) {
  constexpr int kRaw = kPfKeys * ROW;       // bytes of a tile in the pool
  constexpr int kRawChunks = kRaw / 16;     // 1312 or 800
  constexpr int kRawLoads = (kRawChunks + kPfThreads - 1) / kPfThreads;
  static_assert(kRaw % 16 == 0, "whole chunks");
  constexpr uint32_t kRawFlip = kRaw;  // (the two places: 0 and kRaw)
  __shared__ __align__(16) uint8_t kb[3 * kPfTileBytes];
  __shared__ __align__(16) uint8_t raw[2 * kRaw];
  __shared__ int redo;
  const int t = threadIdx.x, lane = t & (kWave - 1), wv = wave_id();
  const int n = lane & 31, h = lane >> 5;

  // this workgroup's share; neighbours on the line run on one XCD, whose L2
  // then holds the keys they have in common
  const int G = (int)gridDim.x;
  const int g = (int)(blockIdx.x % 8u) * (G / 8) + (int)(blockIdx.x / 8u);  // (G is a multiple of 8)
  const long total = chunk_total(A);
  const int shares = (int)min((double)G, max(1.0, (double)total / ((double)A.H * kCaShare)));
  if (t == 0) A.part[g] = int4{-1, 0, 0, 0};
  if (g >= shares || total == 0) return;
  const double share = (double)total / shares;
  ChunkPos at = chunk_find(A, (long)(share * g));
  const ChunkPos end = g + 1 == shares ? ChunkPos{A.B, 0, 0} : chunk_find(A, (long)(share * (g + 1)));

  // K operand: row n (+32), chunk 2kk + h
  uint32_t koff[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) koff[i] = (uint32_t)(n * (DSA_QK_DIM * 2) + ((2 * i + h) ^ pf_swz(n)) * 16);
  // V operand (transposed read): lane a of a 16-lane group addresses key 4h +
  // (a >> 2) (+8), dims 16 * (group & 1) + 4 (a & 3)
  const int a16 = lane & 15, g1 = (lane >> 4) & 1;
  uint32_t voff[2][2];
#pragma unroll
  for (int par = 0; par < 2; ++par)
#pragma unroll
    for (int e8 = 0; e8 < 2; ++e8) {
      const int r = 4 * h + (a16 >> 2) + 8 * e8;
      const int j = 4 * par + 2 * g1 + ((a16 >> 1) & 1);
      voff[par][e8] = (uint32_t)(r * (DSA_QK_DIM * 2) + (j ^ pf_swz(r)) * 16 + 8 * (a16 & 1));
    }
  const uint32_t raw0 = (uint32_t)(uintptr_t)(lvoid_ptr)raw;
  const long pool_bytes = A.kv_rows * ROW;

  while (at.b < end.b || (at.b == end.b && (at.tile < end.tile || (at.tile == end.tile && at.kt < end.kt)))) {
    ChunkReq rq = chunk_req(A, at.b);
    rq = {uniform(rq.first), uniform(rq.T), uniform(rq.tiles), uniform(rq.P)};
    if (at.tile >= rq.tiles) {  // the next request
      at = {at.b + 1, 0, 0};
      continue;
    }
    const int R = rq.T * A.H, r0 = at.tile * kPfRows;
    const int kend = uniform(chunk_keys(A, rq, at.tile)), ktiles = (kend + kPfKeys - 1) / kPfKeys;
    const int kfull = uniform(rq.P + r0 / A.H + 1);  // keys every row sees
    const int t0 = at.kt;
    const int t1 = at.b == end.b && at.tile == end.tile ? end.kt : ktiles;
    const bool whole = t0 == 0 && t1 == ktiles;
    // (in the constant address space: scalar loads, which do not wait in line
    // with the keys'; nothing writes the table meanwhile)
    const auto* pages = (const_int_ptr)(A.page_table + (long)at.b * A.pt_stride);

    const int row = min(r0 + kPfRowsPerWave * wv + n, R - 1);
    const int limit = min(rq.P + row / A.H + 1, kend);
    const uint16_t* qrow = A.q + ((long)rq.first * A.H + row) * DSA_QK_DIM + 8 * h;

    // rows of tile tl that hold keys (0: its page is none of the cache's), and
    // where its bytes are
    const auto rows_of = [&](int page, int tl) DSA_INLINE {
      const long slot = (long)page * DSA_PAGE_TOKENS + (tl & 1) * kPfKeys;
      if (page < 0 || slot >= A.kv_rows) return 0;
      return (int)min((long)min(kPfKeys, kend - tl * kPfKeys), A.kv_rows - slot);
    };
    const auto page_of = [&](int tl) DSA_INLINE { return pages[max(min(tl, t1 - 1), 0) >> 1]; };
    // Direct-to-LDS loads, written out because the compiler, which cannot tell
    // the buffers apart, would wait for them before the next LDS read: the
    // wait is the barrier's, one tile later.  m0 holds the wave's LDS base, to
    // which the hardware adds 16 bytes a lane.
    const auto issue = [&](int page, int tl, uint32_t buf) DSA_INLINE {
      if (!rows_of(page, tl)) return;  // uniform
      const long base = ((long)page * DSA_PAGE_TOKENS + (tl & 1) * kPfKeys) * ROW;
      const uint32_t last = (uint32_t)min((long)kRaw, pool_bytes - base) - 16u;  // rows behind the pool's end: read its last
      const uint8_t* src = A.pool + base;
#pragma unroll
      for (int it = 0; it < kRawLoads; ++it) {
        const int c = it * kPfThreads + t;
        if (c < kRawChunks) {
          const uint32_t off = min(16u * (uint32_t)c, last);
          const uint32_t dst = __builtin_amdgcn_readfirstlane(raw0 + buf + (uint32_t)(it * kPfThreads + wv * kWave) * 16u);
          asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                       :
                       : "s"(dst), "v"(off), "s"(src)
                       : "memory", "m0");
        }
      }
    };
    // Wave w dequantises rows w, w + 4, ... of the next tile, 8 values a lane,
    // between its products of this one: `from` its bytes, `to` its bf16 place.
    constexpr int kSteps = kPfKeys / kPfWaves;
    Latent8<ROW> lat;
    uint4 rope;
    int ln = lane;
    const auto conv_begin = [&](const uint8_t* from) DSA_INLINE {
      ln = lane;
      asm volatile("" : "+v"(ln));  // (addresses formed here: kept over the loop they would be spilled)
      lat.load_codes(from + wv * ROW, ln);
      lat.load_scale(from + wv * ROW, ln);
    };
    const auto conv_slice = [&](int i, const uint8_t* from, uint8_t* to) DSA_INLINE {
      const int st = i / 4, r = wv + kPfWaves * st;  // slices 4 st .. 4 st + 3: row st
      const uint8_t* const nextrow = from + (r + kPfWaves) * ROW;
      if (i % 4 == 0) {
        lat.unpack();
        if (st + 1 < kSteps) lat.load_codes(nextrow, ln);
      } else if (i % 4 == 1) {
        lat.scale();
        if (st + 1 < kSteps) lat.load_scale(nextrow, ln);
      } else if (i % 4 == 2) {
        *reinterpret_cast<uint4*>(to + r * (DSA_QK_DIM * 2) + 16 * (ln ^ pf_swz(r))) = lat.bf16();
      } else if (st == kSteps - 2) {  // the rope of the wave's 8 rows, 8 lanes a row
        rope = *reinterpret_cast<const uint4*>(from + (wv + kPfWaves * (ln >> 3)) * ROW + ROW - 128 + 16 * (ln & 7));
      } else if (st == kSteps - 1) {
        const int rr = wv + kPfWaves * (ln >> 3);
        *reinterpret_cast<uint4*>(to + rr * (DSA_QK_DIM * 2) + 64 * 16 + ((ln & 7) ^ pf_swz(rr)) * 16) = rope;
      }
    };
    // In a tile that some rows do not see to its end, 0 * NaN would reach those
    // rows' outputs: a key with a non-finite latent value (its score is NaN or
    // an infinity whatever the query) keeps a NaN in its rope, which only the
    // scores read, and zeros where the values are read; rows without a key are
    // zeros.  (A wave's own rows: no barrier.)
    const auto conv_end = [&](int tl, int page, uint8_t* to) DSA_INLINE {
      const int rows = rows_of(page, tl);
      if (tl * kPfKeys + kPfKeys <= kfull && rows == kPfKeys) return;  // uniform
#pragma nounroll
      for (int i = 0; i < kSteps; ++i) {
        const int r = wv + kPfWaves * i;
        uint8_t* dst = to + r * (DSA_QK_DIM * 2);
        const bool nan = __ballot(any_nonfinite(reinterpret_cast<const uint4*>(dst)[lane])) != 0;
        if (nan || r >= rows) reinterpret_cast<uint4*>(dst)[lane] = make_uint4(0, 0, 0, 0);
        if ((nan || r >= rows) && lane < 8) {
          const uint32_t x = r < rows ? 0x7fc07fc0u : 0u;
          reinterpret_cast<uint4*>(dst)[kWave + lane] = make_uint4(x, x, x, x);
        }
      }
    };

    v16f o[16];
    float m = -INFINITY, l = 0.f;
    uint4 qf[36];
    v16f s;       // scores of a tile, then its probabilities
    v16f sn;      // the next tile's scores

    const auto k_frag = [&](const uint8_t* kp, int kk) DSA_INLINE {
      return *reinterpret_cast<const uint4*>(kp + koff[kk & 3] + (kk >> 2) * 128);
    };
    // K Q^T of a tile, a slice of other work after each product (the compiler
    // would gather either)
    const auto scores = [&](const uint8_t* kp, auto slice) DSA_INLINE {
      uint4 kf[kCaDepthK];
#pragma unroll
      for (int i = 0; i < kCaDepthK; ++i) kf[i] = k_frag(kp, i);
#pragma unroll
      for (int kk = 0; kk < 36; ++kk) {
        const v4i ka = as_v4i(kf[kk % kCaDepthK]), qb = as_v4i(qf[kk]);
        if (kk == 0)
          asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(sn) : "v"(ka), "v"(qb));
        else
          asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(sn) : "v"(ka), "v"(qb));
        if (kk + kCaDepthK < 36) kf[kk % kCaDepthK] = k_frag(kp, kk + kCaDepthK);
        slice(kk);
        __builtin_amdgcn_sched_barrier(0);
      }
      // the matrix unit's results may be read 19 wait states after the last issue
      asm volatile("s_nop 15\n\ts_nop 7" : "+v"(sn));
    };
    // The next tile's scores become this one's: in the log2 domain, keys at or
    // past the row's limit -inf.  Element i is the tile's key 8 (i / 4) + 4h + (i % 4).
    const auto take_scores = [&](int tl, int rows) DSA_INLINE {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = sn[e] * A.sm_log2;
      const int k0 = tl * kPfKeys;
      if (k0 + kPfKeys > kfull || rows < kPfKeys) {  // uniform
        const int seen = min(limit - k0, rows) - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = 8 * (i >> 2) + (i & 3) < seen ? s[i] : -INFINITY;
      }
    };

    // A tile's softmax, in slices: 0-7 its maximum, 8 the reference point, 9-24
    // the probabilities, 25-32 their bf16 pairs and sum.
    float tmax = -INFINITY, top = -INFINITY, mr = 0.f;  // (top: of all tiles)
    uint32_t pk[8];
    const auto softmax_slice = [&](int i) DSA_INLINE {
      if (i < 8) {
        tmax = i ? fmaxf(tmax, fmaxf(s[2 * i], s[2 * i + 1])) : fmaxf(s[0], s[1]);
      } else if (i == 8) {
        tmax = half_swap_max(tmax);
        m = m == -INFINITY ? tmax + kCaAbove : m;
        top = fmaxf(top, tmax);
        mr = m == -INFINITY ? 0.f : m;
      } else if (i < 25) {
        s[i - 9] = __builtin_amdgcn_exp2f(s[i - 9] - mr);
      } else if (i < 33) {
        const int e = i - 25;
        pk[e] = pack_bf16x2(s[2 * e], s[2 * e + 1]);
        // the sum of the rounded probabilities, the ones PV multiplies: the
        // weights then add up to one
        l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, pk[e]), __builtin_bit_cast(v2bf, 0x3f803f80u), l, false);
      }
    };
    // O^T += V^T P^T of a tile, the tile after next's dequantisation between
    const auto values = [&](const uint8_t* kp, const uint8_t* from, uint8_t* to) DSA_INLINE {
      const auto v_frag = [&](int i) DSA_INLINE {
        const int ks = i >> 4, dt = i & 15;
        const uint32_t imm = (dt >> 1) * 128 + ks * (16 * DSA_QK_DIM * 2);
        const v4s_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_ptr)(kp + voff[dt & 1][0] + imm));
        const v4s_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_ptr)(kp + voff[dt & 1][1] + imm));
        uint4 vf;
        __builtin_memcpy(&vf.x, &lo, 8);
        __builtin_memcpy(&vf.z, &hi, 8);
        return vf;
      };
      uint4 vf[kCaDepthV];
      conv_begin(from);
#pragma unroll
      for (int i = 0; i < kCaDepthV; ++i) vf[i] = v_frag(i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const uint32_t* pr = pk + 4 * (i >> 4);
        o[i & 15] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            as_bf8(vf[i % kCaDepthV]), as_bf8(make_uint4(pr[0], pr[1], pr[2], pr[3])), o[i & 15], 0, 0, 0);
        if (i + kCaDepthV < 32) vf[i % kCaDepthV] = v_frag(i + kCaDepthV);
        conv_slice(i, from, to);
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    // A tile passes through: bytes (two places), bf16 (three), scores, values.
    // While tile tl is summed, tl + 1 is scored, tl + 2 dequantised, and tl + 3 on
    // its way.
    const auto pass = [&]() DSA_INLINE {
      int p0 = page_of(t0), p1 = page_of(t0 + 1), p2 = page_of(t0 + 2);
      issue(p0, t0, 0u);
      if (t0 + 1 < t1) issue(p1, t0 + 1, kRaw);
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        conv_begin(raw + j * kRaw);
#pragma unroll
        for (int i = 0; i < 32; ++i) conv_slice(i, raw + j * kRaw, kb + j * kPfTileBytes);
        conv_end(t0 + j, j ? p1 : p0, kb + j * kPfTileBytes);
      }
      __syncthreads();  // two tiles in bf16, their bytes' places free
      if (t0 + 2 < t1) issue(p2, t0 + 2, 0u);
      scores(kb, [](int) {});
      take_scores(t0, rows_of(p0, t0));
      const uint8_t* here = kb;
      uint8_t *next = kb + kPfTileBytes, *after = kb + 2 * kPfTileBytes;
      uint32_t at_raw = 0;  // tile tl + 2's bytes
      for (int tl = t0; tl < t1; ++tl) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // tile tl + 1 is in bf16, tl + 2 has landed; what held tl - 1 and tl + 1's bytes is free
        const int p3 = page_of(tl + 3);
        if (tl + 3 < t1) issue(p3, tl + 3, at_raw ^ kRawFlip);
        // (always, also where there is no next tile: a branch around the
        // products takes the accumulators through the vector file)
        scores(next, softmax_slice);
        values(here, raw + at_raw, after);
        take_scores(tl + 1, rows_of(p1, tl + 1));
        if (tl + 2 < t1) conv_end(tl + 2, p2, after);
        p1 = p2;
        p2 = p3;
        at_raw ^= kRawFlip;
        uint8_t* const old = const_cast<uint8_t*>(here);
        here = next;
        next = after;
        after = old;
      }
      __syncthreads();
    };
#pragma unroll
    for (int kk = 0; kk < 36; ++kk) qf[kk] = *reinterpret_cast<const uint4*>(qrow + 16 * kk);
    // waited for here: later the wait would count the key loads in flight too
#pragma unroll
    for (int kk = 0; kk < 36; ++kk) asm volatile("" : : "v"(as_v4i(qf[kk])));
    if (t == 0) redo = 0;
    for (int round = 0;; ++round) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
      l = 0.f;
      pass();
      if (round) break;
      if (__ballot(top > m + kCaRise) && lane == 0) redo = 1;
      __syncthreads();
      if (!uniform(redo)) break;
      m = top;
    }
    __syncthreads();  // (everyone has read redo)

    l = half_swap_sum(l);
    if (r0 + kPfRowsPerWave * wv + n < R) {
      // lane (n, h) holds dims 32 dt + 8 (i / 4) + 4h + (i % 4) of its row
      if (whole) {
        const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);  // a row without a key gives 0, NaN stays
        uint16_t* orow = A.out + ((long)rq.first * A.H + row) * DSA_LATENT_DIM + 4 * h;
#pragma unroll
        for (int dt = 0; dt < 16; ++dt)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            v2u_t w;
            w[0] = pack_bf16x2(o[dt][i] * inv, o[dt][i + 1] * inv);
            w[1] = pack_bf16x2(o[dt][i + 2] * inv, o[dt][i + 3] * inv);
            *reinterpret_cast<v2u_t*>(orow + 32 * dt + 2 * i) = w;
          }
      } else {
        // the part of a tile that began before this share, or of the one that ends behind it
        const long pr = (long)(2 * g + (t0 == 0)) * A.part_rows + (row - r0);
        float* po = A.part_o + pr * DSA_LATENT_DIM + 4 * h;
#pragma unroll
        for (int dt = 0; dt < 16; ++dt)
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            v4f w = {o[dt][i], o[dt][i + 1], o[dt][i + 2], o[dt][i + 3]};
            *reinterpret_cast<v4f*>(po + 32 * dt + 2 * i) = w;
          }
        if (h == 0) {
          A.part_ml[2 * pr] = m;
          A.part_ml[2 * pr + 1] = l;
        }
      }
    }
    if (t == 0 && !whole) {
      int4 d = A.part[g];
      if (t0 == 0) d.x = at.b, d.y = at.tile;       // began here, goes on in the next share
      else d.z = t1 == ktiles ? 2 : 1;              // began before: ends here, or not
      A.part[g] = d;
    }
    if (at.b == end.b && at.tile == end.tile) break;
    at = {at.b, at.tile + 1, 0};
  }
}

// Joins a row's parts: out = sum_s O_s 2^(m_s - m) / sum_s l_s 2^(m_s - m), m =
// max (m_s + log2 l_s): the reference points m_s alone can lie 144 apart from
// where their parts' weight is.  A workgroup: `per` rows of the i-th row tile that more than one
// share has part of.  With few parts a wave takes a row; with many the four
// waves take the parts of one row in turn (w, w + 4, ...; 8 dims a lane) and
// meet in LDS, always in the same order.
constexpr int kCaFewParts = 8;
__global__ __launch_bounds__(kPfThreads) void chunk_merge_kernel(const ChunkAttnArgs A, int G, int per) {
  __shared__ float sl[kPfWaves];
  __shared__ v4f so[kPfWaves][2 * kWave];
  const int lane = threadIdx.x & (kWave - 1), wv = wave_id();
  const int blocks = (A.part_rows + per - 1) / per;
  const int r_lo = (int)(blockIdx.x % (unsigned)blocks) * per;
  int left = (int)(blockIdx.x / (unsigned)blocks), first = -1;
  for (int g0 = 0; g0 < G && first < 0; g0 += kWave) {
    uint64_t has = __ballot(g0 + lane < G && A.part[min(g0 + lane, G - 1)].x >= 0);
    const int here = __builtin_popcountll(has);
    if (left >= here) {
      left -= here;
      continue;
    }
    for (; left > 0; --left) has &= has - 1;
    first = g0 + __builtin_ctzll(has);
  }
  if (first < 0) return;
  const int4 d = A.part[first];
  const ChunkReq rq = chunk_req(A, d.x);
  const long row0 = (long)d.y * kPfRows, R = (long)rq.T * A.H;
  int parts = 1;  // the first share's, then those up to the one where the tile ends
  for (int g0 = first + 1; g0 < G; g0 += kWave) {
    const uint64_t ends = __ballot(g0 + lane < G && A.part[min(g0 + lane, G - 1)].z == 2);
    if (ends) {
      parts += __builtin_ctzll(ends) + 1;
      break;
    }
    parts += kWave;
  }
  const bool few = parts <= kCaFewParts;
  const int step = few ? 1 : kPfWaves, mine = few ? 0 : wv;
  for (int r = r_lo + (few ? wv : 0); r < min(r_lo + per, A.part_rows) && row0 + r < R; r += few ? kPfWaves : 1) {
    const auto slot = [&](int s) { return (long)(s ? 2 * (first + s) : 2 * first + 1) * A.part_rows + r; };
    float m = -INFINITY;
    for (int s = lane; s < parts; s += kWave) m = fmaxf(m, A.part_ml[2 * slot(s)] + log2f(A.part_ml[2 * slot(s) + 1]));
    m = wave_max(m);
    const float mr = m == -INFINITY ? 0.f : m;
    float L = 0.f;
    v4f x0 = {0.f, 0.f, 0.f, 0.f}, x1 = x0;
    constexpr int kU = 4;
    for (int s0 = mine; s0 < parts; s0 += kU * step) {
      v4f a[kU], c[kU];
      float ms[kU], ls[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int s = s0 + u * step;
        const long pr = slot(s < parts ? s : mine);  // past the last: read again, weight 0
        const v4f* po = reinterpret_cast<const v4f*>(A.part_o + pr * DSA_LATENT_DIM) + 2 * lane;
        a[u] = po[0];
        c[u] = po[1];
        ms[u] = A.part_ml[2 * pr];
        ls[u] = A.part_ml[2 * pr + 1];
      }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (s0 + u * step >= parts) break;  // uniform
        const float w = exp2f(ms[u] - mr);
        L += ls[u] * w;
        x0 += a[u] * w;
        x1 += c[u] * w;
      }
    }
    uint16_t* const out = A.out + ((long)rq.first * A.H + row0 + r) * DSA_LATENT_DIM;
    if (few) {
      const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
      x0 *= inv;
      x1 *= inv;
      v2u_t* const o = reinterpret_cast<v2u_t*>(out) + 2 * lane;  // (out need begin on 8 bytes only)
      o[0] = v2u_t{pack_bf16x2(x0[0], x0[1]), pack_bf16x2(x0[2], x0[3])};
      o[1] = v2u_t{pack_bf16x2(x1[0], x1[1]), pack_bf16x2(x1[2], x1[3])};
      continue;
    }
    so[wv][2 * lane] = x0;
    so[wv][2 * lane + 1] = x1;
    if (lane == 0) sl[wv] = L;
    __syncthreads();
    const float tot = (sl[0] + sl[1]) + (sl[2] + sl[3]);
    const float inv = tot > 0.f ? 1.f / tot : (tot == tot ? 0.f : tot);
    if (threadIdx.x < 2 * kWave) {
      const int i = threadIdx.x;
      const v4f o = (so[0][i] + so[1][i]) + (so[2][i] + so[3][i]);
      v2u_t w;
      w[0] = pack_bf16x2(o[0] * inv, o[1] * inv);
      w[1] = pack_bf16x2(o[2] * inv, o[3] * inv);
      *reinterpret_cast<v2u_t*>(out + 4 * i) = w;
    }
    __syncthreads();
  }
}

static int chunk_shares() { return std::max(8, device_cu_count() / 8 * 8); }
static int chunk_part_rows(int n, int H) { return (int)std::min<long>(kPfRows, (long)n * H); }

// [a workgroup's two parts | (reference point, sum) of their rows | what they are parts of]
size_t chunk_workspace_bytes(int n, int H) {
  const size_t G = (size_t)chunk_shares();
  return 2 * G * chunk_part_rows(n, H) * (DSA_LATENT_DIM + 2) * sizeof(float) + G * sizeof(int4);
}

hipError_t launch_chunk_attention(ChunkAttnArgs A, int row_bytes, void* workspace, hipStream_t s) {
  const int G = chunk_shares();
  A.part_rows = chunk_part_rows(A.n, A.H);
  A.part_o = static_cast<float*>(workspace);
  A.part_ml = A.part_o + (size_t)2 * G * A.part_rows * DSA_LATENT_DIM;
  A.part = reinterpret_cast<int4*>(A.part_ml + (size_t)2 * G * A.part_rows * 2);
  const dim3 block(kPfThreads);
  if (row_bytes == DSA_LATENT_ROW_BYTES)
    hipLaunchKernelGGL(chunk_attention_kernel<DSA_LATENT_ROW_BYTES>, dim3(G), block, 0, s, A);
  else
    hipLaunchKernelGGL(chunk_attention_kernel<DSA_FP4_ROW_BYTES>, dim3(G), block, 0, s, A);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // row tiles there may be, and those that two shares can have part of
  const long tiles = (long)A.n * A.H / kPfRows + std::min(A.B, A.n);
  const long split = std::min<long>(tiles, G - 1);
  // rows a workgroup: about 8 workgroups a CU
  const int per = (int)std::min(16L, std::max(1L, split * A.part_rows / (8L * G)));
  const long blocks = split * ((A.part_rows + per - 1) / per);
  hipLaunchKernelGGL(chunk_merge_kernel, dim3((unsigned)blocks), block, 0, s, A, G, per);
  return hipGetLastError();
}

}  // namespace dsa
