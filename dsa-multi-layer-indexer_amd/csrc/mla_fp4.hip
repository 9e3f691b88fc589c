// Sparse / dense MLA decode over a latent cache held in 4 bits (gfx950):
//   out[b,h,:] = sum_j softmax_j(sm * q[b,h,:] . kv_j) * kv_j[:512],
//   kv_j = e2m1 * 2^(scale byte[d/32] - 127) | bf16 rope, from a 400-byte row
//   [256 B: value 2i in the low half of byte i][16 e8m0][64 bf16].
// One value of a row is a 2-bit significand times a power of two, so its bf16
// form is exact.
//
// A workgroup (8 waves, one a CU) takes a chunk of a row's keys for 32 heads,
// 128 keys a tile.  The rows go from memory straight to LDS, as they are, into
// one of three tiles' places.  Waves 0-3 multiply 32 keys each with the
// queries, which stay in their registers (S^T = K Q^T, the rows dequantised by
// v_cvt_scalef32_pk_bf16_fp4), and leave the probabilities in LDS, where the
// rows' rope part was; a barrier later waves 4-7 add up 128 of the 512 dims
// each over all 128 keys (O^T = V^T P^T), while the first four are at the next
// tile and the one after it is on its way.  So each SIMD holds one wave of each
// kind, and the softmax of one goes on beside the products of the other.
// V^T comes out of the matrix unit too: a 32x32x64 fp4 product of the rows as
// they lie in LDS, with their scales, and a matrix of ones and zeros that picks
// 32 dims gives their values with a dim in each lane and the keys in its
// registers, which rounds to the next product's A operand (exactly) without
// moving.  So a tile passes through LDS once in 4 bits: a transpose of the bf16
// values there cost 16 clocks a KB written.
//
// Measured: 8 rows of 16K keys, 128 heads: 50 us in a graph, merge included.  A
// tile takes 4.4K clocks, 2.7K of them the matrix unit's, with all CUs at it
// (which then run at 1.9 GHz: 0.98 PFLOP/s of scores and sums, four fifths of
// what a large bf16 product reaches, besides V^T); the start of a chunk 4 us
// (entries, then rows and queries), its end and the launch 4.  The same work in workgroups of 4 waves that each score and
// then sum, two a CU: 58 us (2.9 us a tile on an idle CU, 1.8 here).  64 heads a
// workgroup: a tenth fewer matrix operations, but twice the partial sums of as
// many workgroups: 70 us.
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

constexpr int kM4Threads = 512;      // waves 0-3: scores and probabilities, 4-7: sums
constexpr int kM4Heads = 32;         // heads a workgroup
constexpr int kM4Group = 32;         // keys a wave scores
constexpr int kM4Groups = 4;         // of a tile
constexpr int kM4Unit = kM4Groups * kM4Group;  // keys a tile: chunks are multiples
constexpr int kM4MergeMax = 512;     // chunks of up to kM4Ragged rows together
constexpr int kM4Ragged = 256;       // most rows that share chunks by their lengths
constexpr float kM4Rise = 16.f;      // log2 growth of the maximum that rescales the sums
constexpr int kM4Buffers = 3;        // tiles of rows: summed, scored, on their way
constexpr int kM4GroupLds = kM4Group * DSA_FP4_ROW_BYTES;
constexpr int kM4Tile = kM4Groups * kM4GroupLds;
constexpr int kM4Lds = kM4Buffers * kM4Tile;
constexpr int kM4QLines = DSA_QK_DIM * 2 / 64;  // 64-byte lines of a head's query
constexpr int kM4QueriesAt = 2 * kM4Tile;       // the queries on their way to registers, where tile 2 will be
static_assert(kM4QueriesAt + 2 * kM4QLines * 1024 <= kM4Lds && kM4Lds + 4096 <= 160 * 1024, "one workgroup a CU");
__host__ __device__ constexpr int m4_blocks(int H) { return (H + kM4Heads - 1) / kM4Heads; }
// heads of a block that there is room for in the partials
__host__ __device__ constexpr int m4_heads(int H) { return H < kM4Heads ? H : kM4Heads; }

__device__ __forceinline__ v8bf m4_bf8(const uint4& a) {
  v8bf v;
  __builtin_memcpy(&v, &a, 16);
  return v;
}
__device__ __forceinline__ v8i_m4 m4_fp4(const uint4& a) { return v8i_m4{(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}; }
// A wave's 32 rows in LDS (fetch, below): where row r's pieces begin, and the
// order of its four pieces of a 64-byte line.
constexpr int kM4Last = 24 * kM4Group * 16;
__device__ __forceinline__ int m4_piece(int r) { return (r >> 4) * 6144 + (r & 15) * 64; }
__device__ __forceinline__ int m4_swz(int r) { return r >> 2 & 3; }
// Every wave is here and sees the others' writes to LDS.  (__syncthreads()
// would also wait for loads that are on their way from memory to LDS.)
__device__ __forceinline__ void m4_meet() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// op over the two half-waves (lane l and l ^ 32)
template <class F>
__device__ __forceinline__ float m4_halves(float v, F op) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Row b's keys are cut into chunks of `units` * kM4Unit; their partials lie
// behind those of the rows before it.
struct M4Plan {
  int units;  // of kM4Unit keys, a chunk
  int first;  // chunk number of the row's first
  int count;  // chunks of the row, at least one
};

__device__ __forceinline__ int m4_row_keys(const Mla4Args& A, int b) {
  return A.dense_pt ? max(0, min(A.dense_lens[b], A.keys)) : A.keys;
}

// The row of chunk `id` (-1: none) and its plan, the same in every wave.
// Selections, and dense rows where there is no chunk to spare, are cut alike.
// Other dense rows (at most kM4Ragged) share A.chunks chunks: the smallest chunk
// with which all rows' fit.  Lane l holds rows 64k + l.
__device__ __forceinline__ int m4_plan_chunk(const Mla4Args& A, int id, int lane, M4Plan& p) {
  if (A.units) {
    const int b = id / A.per_row;
    p = {A.units, b * A.per_row, A.per_row};
    return b < A.B ? b : -1;
  }
  constexpr int kPer = kM4Ragged / 64;
  uint32_t u[kPer], c[kPer], total = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int b = 64 * k + lane;
    u[k] = b < A.B ? (uint32_t)(m4_row_keys(A, b) + kM4Unit - 1) / kM4Unit : 0u;
  }
#pragma unroll
  for (int k = 0; k < kPer; ++k)
    if (64 * k < A.B) total += wave_reduce<0>(u[k]);
  const auto chunks = [&](uint32_t cu) {  // of all rows (an empty one has one too)
    uint32_t n = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      c[k] = 64 * k + lane < A.B ? max(1u, (u[k] + cu - 1) / cu) : 0u;
      if (64 * k < A.B) n += wave_reduce<0>(c[k]);
    }
    return n;
  };
  // the search ends at a size that fits in any case: a row's last chunk may be short
  uint32_t lo = max(1u, (total + A.chunks - 1) / A.chunks);
  uint32_t hi = max(lo, (total + (uint32_t)(A.chunks - A.B) - 1) / (uint32_t)(A.chunks - A.B));
  uint32_t n = chunks(lo);
  if (n > (uint32_t)A.chunks) {
    while (hi - lo > 1) {  // lo does not fit, hi does
      const uint32_t mid = (lo + hi) / 2;
      (chunks(mid) > (uint32_t)A.chunks ? lo : hi) = mid;
    }
    lo = hi;
    n = chunks(lo);
  }
  p.units = (int)lo;
  int before = 0;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    if (64 * k >= A.B) break;
    const int end = before + (int)wave_scan_incl<0>(c[k]);
    const uint64_t hit = __ballot(id < end && id >= end - (int)c[k]);
    if (hit) {
      const int src = __builtin_ctzll(hit);
      p.count = __builtin_amdgcn_readlane((int)c[k], src);
      p.first = __builtin_amdgcn_readlane(end, src) - p.count;
      return 64 * k + src;
    }
    before = __builtin_amdgcn_readlane(end, kWave - 1);
  }
  return -1;
}

template <bool DENSE>
__global__ __launch_bounds__(kM4Threads, 2) void mla_fp4_kernel(const Mla4Args A) {
  extern __shared__ __align__(16) unsigned char smem[];  // three tiles' rows
  __shared__ __align__(16) float ref[2][kM4Heads][kM4Groups], wl[kM4Heads][kM4Groups];
  __shared__ __align__(16) uint32_t there[4][kM4Groups];  // a bit a key, of a tile and the three around it
  const int t = threadIdx.x, lane = t & (kWave - 1), wave = wave_id();
  const int n = lane & 31, h = lane >> 5;
  // a chunk's head blocks on one XCD (workgroup number modulo 8), whose L2
  // then serves all but the first's reads of its rows
  const int nhb = m4_blocks(A.H);
  const int hb = (blockIdx.x / 8) % nhb, id = (blockIdx.x / (8 * nhb)) * 8 + blockIdx.x % 8;
  M4Plan plan;
  const int b = m4_plan_chunk(A, id, lane, plan);
  if (b < 0) return;  // (the same in the whole workgroup)
  if (!A.units && id == plan.first && hb == 0 && t == 0) A.plan[b] = make_int2(plan.first, plan.count);  // for the merge
  const int total = m4_row_keys(A, b);
  const long j0 = (long)(id - plan.first) * plan.units * kM4Unit;
  const uint32_t keys = (uint32_t)max(min((long)total - j0, (long)plan.units * kM4Unit), 0L);
  const int tiles = (int)((keys + kM4Unit - 1) / kM4Unit);
  const uint32_t row0 = m4_piece(n), swz = m4_swz(n);
  // rows and heads of one LDS line's load: 16, four lanes each
  const int r16 = lane >> 2, p16 = 16 * ((lane & 3) ^ m4_swz(r16));

  // the rows' way in begins with their entries (waves 4-7)
  const int wv = wave & 3;
  const int jl = kM4Group * wv + n;
  const int* idx_row = DENSE ? A.dense_pt + (long)b * A.dense_pt_stride + (j0 >> 6) : A.idx + (long)b * A.keys + j0;
  const auto entry = [&](int tl) {
    const uint32_t j = min((uint32_t)tl * kM4Unit + jl, keys - 1);
    return idx_row[DENSE ? j >> 6 : j];
  };
  int e0 = 0, e1 = 0, e2 = 0, e3 = 0;  // of the next tiles
  if (wave >= 4 && tiles) e0 = entry(0), e1 = entry(1), e2 = entry(2), e3 = entry(3);
  // the queries' way in: lines of 64 bytes of 16 heads
  const uint8_t* qsrc = reinterpret_cast<const uint8_t*>(A.q) + (long)b * A.H * (DSA_QK_DIM * 2) + p16;
#pragma unroll
  for (int k = 0; k < (2 * kM4QLines + 7) / 8; ++k) {
    const int x = wave + 8 * k;
    if (x >= 2 * kM4QLines) break;
    const int head = min(hb * kM4Heads + x / kM4QLines * 16 + r16, A.H - 1);
    __builtin_amdgcn_global_load_lds((m4_gvoid_ptr)(qsrc + head * (DSA_QK_DIM * 2) + 64 * (x % kM4QLines)),
                                     (m4_lvoid_ptr)(smem + kM4QueriesAt + 1024 * x), 16, 0, 0);
  }

  if (wave < 4) {
    // Scores and probabilities: 32 keys and 32 heads of each tile.
    const int kg = wave;
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    __syncthreads();
    // Operand 4i + u: dims 64i + 32h + 8u .. + 7; 32 + u: rope dims 32h + 8u .. + 7.
    uint4 qf[36];
#pragma unroll
    for (int kk = 0; kk < 36; ++kk) {
      const int line = kk < 32 ? 2 * (kk >> 2) + h : 16 + h;
      qf[kk] = *reinterpret_cast<const uint4*>(smem + kM4QueriesAt + ((n >> 4) * kM4QLines + line) * 1024 + (n & 15) * 64 +
                                               16 * ((kk & 3) ^ swz));
    }
    // Where this lane reads row n of the wave's 32: pieces 2i + h (dims 64i + 32h ..)
    // at code_at[i & 1] + 1024 (i / 2), the scales (piece 16), rope pieces 17 + 4h + u
    const uint32_t base = kg * kM4GroupLds + row0;
    uint32_t code_at[2], rope_at[4];
#pragma unroll
    for (int g = 0; g < 2; ++g) code_at[g] = base + 16 * ((2 * g + h) ^ swz);
    const uint32_t scales_at = base + 4096 + 16 * swz;
#pragma unroll
    for (int u = 0; u < 3; ++u) rope_at[u] = base + 4096 + 1024 * h + 16 * ((u + 1) ^ swz);
    rope_at[3] = h ? kg * kM4GroupLds + kM4Last + 16 * n : base + 5120 + 16 * swz;
    const auto row_max = [&](int k) {
      const v4f a = *reinterpret_cast<const v4f*>(&ref[k][n][0]);
      return fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3]));
    };
    // All sums are relative to `top`, the same in every wave, which trails the
    // maximum by at most kM4Rise.  It is a whole number, so that what is brought
    // down to a new one is scaled by a power of two, without another rounding.
    float top = -INFINITY, l = 0.f;
    __syncthreads();  // tile 0 is there
    uint32_t buf = 0;
#pragma unroll 1
    for (int tl = 0; tl < tiles; ++tl) {
      const unsigned char* const rows = smem + buf;
      uint4 code[8];
      const uint4 scv = *reinterpret_cast<const uint4*>(rows + scales_at);
#pragma unroll
      for (int i = 0; i < 8; ++i) code[i] = *reinterpret_cast<const uint4*>(rows + code_at[i & 1] + 1024 * (i >> 1));
      const uint32_t ok = there[tl & 3][kg];
      v16f s;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.f;
      const auto product = [&](int kk, const uint4& k) {
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(m4_bf8(k), m4_bf8(qf[kk]), s, 0, 0, 0);
      };
      const uint32_t scw[4] = {scv.x, scv.y, scv.z, scv.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float sc = __uint_as_float(((scw[i >> 1] >> (16 * (i & 1) + 8 * h)) & 0xffu) << 23);
        product(4 * i, dequant8_fp4(code[i].x, sc));
        product(4 * i + 1, dequant8_fp4(code[i].y, sc));
        product(4 * i + 2, dequant8_fp4(code[i].z, sc));
        product(4 * i + 3, dequant8_fp4(code[i].w, sc));
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) product(32 + u, *reinterpret_cast<const uint4*>(rows + rope_at[u]));
      // element e is key 8 (e / 4) + 4h + e % 4 of head n; the scale waits for
      // the exponent's fma, unless it turns the order of the scores round
      float tmax = -INFINITY, scale = A.sm_log2;
      if (!(scale > 0.f)) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] *= scale;
        scale = 1.f;
      }
      if (ok != ~0u) {  // keys that are not there
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = (ok >> (4 * h)) & (1u << (8 * (e >> 2) + (e & 3))) ? s[e] : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) tmax = fmaxf(tmax, s[e]);
      tmax = m4_halves(tmax, [](float x, float y) { return fmaxf(x, y); }) * scale;
      if (tl == 0) {  // the first tile's maximum is agreed on; later ones are seldom above it
        if (h == 0) ref[1][n][kg] = tmax;
        __syncthreads();
        top = ceilf(row_max(1));
      }
      const float own = tmax > top + kM4Rise || top == -INFINITY ? ceilf(fmaxf(tmax, top)) : top;
      const float at = own == -INFINITY ? 0.f : own;
      uint32_t pk[8];
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        pk[e >> 1] = pack_bf16x2(__builtin_amdgcn_exp2f(__builtin_fmaf(s[e], scale, -at)),
                                 __builtin_amdgcn_exp2f(__builtin_fmaf(s[e + 1], scale, -at)));
        // the sum of the rounded probabilities, the ones that are multiplied
        // with the values: the weights then add up to one
        sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, pk[e >> 1]), __builtin_bit_cast(v2bf, 0x3f803f80u), sum,
                                              false);
      }
      // (where its rows' rope pieces 20-23 were, which have been used)
      unsigned char* const probs = smem + buf + kg * kM4GroupLds + 5120;
      *reinterpret_cast<uint4*>(probs + 16 * lane) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
      *reinterpret_cast<uint4*>(probs + 6144 + 16 * lane) = make_uint4(pk[4], pk[5], pk[6], pk[7]);
      if (h == 0) ref[tl & 1][n][kg] = own;
      __syncthreads();  // the probabilities are there, and the next tile's rows
      const float now = row_max(tl & 1);
      if (__ballot(now != top)) {  // a wave went above `top`
        l *= top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now);
        sum *= own == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(own - now);
        top = now;
      }
      l += sum;
      buf = buf == (kM4Buffers - 1) * kM4Tile ? 0u : buf + kM4Tile;
    }
    l = m4_halves(l, [](float x, float y) { return x + y; });
    if (h == 0) wl[n][kg] = l;
    __syncthreads();
    return;
  }

  // Sums: 128 dims of all the tile's keys and heads, a tile behind the scores;
  // and the rows' way in, a tile before them.
  //
  // A key's slot; -1: not there (row 0 is read then, and its probability is 0).
  const auto slot = [&](int tl, int e) {
    const uint32_t j = (uint32_t)tl * kM4Unit + jl;
    const long sl = DENSE ? (long)e * DSA_PAGE_TOKENS + (j & (DSA_PAGE_TOKENS - 1)) : (long)e;
    return j < keys && e >= 0 && sl < A.kv_rows ? (int)sl : -1;
  };
  // A tile's rows to LDS, 32 a wave, 16-byte piece by piece: pieces 4k .. 4k + 3 of 16
  // rows a load (64 bytes a row together), then the last pieces.  Piece q < 24
  // of row r of a group lies at m4_piece(r) + 1024 (q / 4) + 16 ((q % 4) ^ m4_swz(r)),
  // piece 24 at kM4Last + 16 r: 8 rows' reads of one piece fall on 8 bank
  // groups, and a load needs no more than its lane's pointer.
  struct Way {
    const uint8_t* src[3];
    unsigned char* dst;
  };
  const auto way = [&](int tl, int sl, uint32_t buf) {
    const int from = sl < 0 ? 0 : sl;
    const uint32_t ok = (uint32_t)__ballot(sl >= 0);
    if (lane == 0) there[tl & 3][wv] = ok;
    Way w;
    w.dst = smem + buf + wv * kM4GroupLds;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      w.src[k] = A.pool + (long)__builtin_amdgcn_ds_bpermute((16 * k + r16) << 2, from) * DSA_FP4_ROW_BYTES + p16;
    w.src[2] = A.pool + (long)from * DSA_FP4_ROW_BYTES + 384;
    return w;
  };
  // load k of 13
  const auto load = [&](const Way& w, int k) {
    if (k < 12)
      __builtin_amdgcn_global_load_lds((m4_gvoid_ptr)(w.src[k / 6] + 64 * (k % 6)), (m4_lvoid_ptr)(w.dst + 1024 * k), 16, 0, 0);
    else if (lane < kM4Group)
      __builtin_amdgcn_global_load_lds((m4_gvoid_ptr)w.src[2], (m4_lvoid_ptr)(w.dst + kM4Last), 16, 0, 0);
  };
  const auto fetch = [&](const Way& w) {
#pragma unroll
    for (int k = 0; k < 13; ++k) load(w, k);
  };
  // s_waitcnt vmcnt(k): all but the last k loads; 13 are a tile's
  constexpr int kNone = 0x0f70, kOneTile = 0x0f7d;
  // (a write to LDS would wait for loads to it: both before the first)
  const Way w0 = way(0, slot(0, e0), 0), w1 = way(1, slot(1, e1), kM4Tile);
  int sl = slot(2, e2), e = e3;
  if (tiles) fetch(w0);
  __builtin_amdgcn_s_waitcnt(kOneTile);
  m4_meet();  // the queries are there
  if (tiles > 1) fetch(w1);
  v16f o[4];  // O^T: dims 128 wv + 32 d + 8 (e / 4) + 4h + e % 4 of head n
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  // the B operand that picks dims 32 half .. + 31 of 64: a one (code 2) at k = 32 half + n
  uint4 pick[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint32_t one = h == half ? 2u << (4 * (n & 7)) : 0u;
    pick[half] = make_uint4(n >> 3 == 0 ? one : 0u, n >> 3 == 1 ? one : 0u, n >> 3 == 2 ? one : 0u, n >> 3 == 3 ? one : 0u);
  }
  // dims 128 wv + 64 g + 32 h .. of row n of a group at dims_at[g], their scales at dscales_at
  uint32_t dims_at[2];
#pragma unroll
  for (int g = 0; g < 2; ++g) dims_at[g] = row0 + 1024 * wv + 16 * ((2 * g + h) ^ swz);
  const uint32_t dscales_at = row0 + 4096 + 16 * swz + 4 * wv;
  float top = -INFINITY;
  if (tiles > 1)
    __builtin_amdgcn_s_waitcnt(kOneTile);
  else
    __builtin_amdgcn_s_waitcnt(kNone);
  m4_meet();  // tile 0 is there
  if (tiles) {
    m4_meet();  // (the first maximum)
    __builtin_amdgcn_s_waitcnt(kNone);
    m4_meet();  // tile 0's probabilities and tile 1's rows
  }
  uint32_t buf = 0;
  // tile tl; MORE: tile tl + 2 comes to where tile tl - 1 was, in a loop of its own,
  // because with branches between them the products move down to their uses
  const auto sum_tile = [&](int tl, auto more) {
    constexpr bool MORE = decltype(more)::value;
    const unsigned char* const rows = smem + buf;
    const v4f own = *reinterpret_cast<const v4f*>(&ref[tl & 1][n][0]);
    const float now = fmaxf(fmaxf(own[0], own[1]), fmaxf(own[2], own[3]));
    const bool risen = __ballot(now != top) != 0;
    if (risen) {  // a wave went above `top`: what is there comes down to the new one
      const float down = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now);
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= down;
      top = now;
    }
    // all that is read from LDS comes first: the loads to it that follow are
    // waited for by any later read
    uint4 c[2 * kM4Groups], pr[2 * kM4Groups];
    uint32_t sc[kM4Groups];
    const uint4 there4 = *reinterpret_cast<const uint4*>(there[tl & 3]);
    const uint32_t th[4] = {there4.x, there4.y, there4.z, there4.w};
#pragma unroll
    for (int kb = 0; kb < kM4Groups; ++kb) {
      // scale bytes of dims 128 wv + 64 g + 32 h: byte 2g after the shift; a
      // row that is not there at scale 1 (finite values)
      sc[kb] = *reinterpret_cast<const uint32_t*>(rows + dscales_at + kb * kM4GroupLds) >> (8 * h);
      sc[kb] = th[kb] >> n & 1 ? sc[kb] : 0x7f7f7f7fu;
#pragma unroll
      for (int g = 0; g < 2; ++g) c[2 * kb + g] = *reinterpret_cast<const uint4*>(rows + dims_at[g] + kb * kM4GroupLds);
    }
    const auto probability = [&](int x) {
      return *reinterpret_cast<const uint4*>(rows + 5120 + (x >> 1) * kM4GroupLds + 6144 * (x & 1) + 16 * lane);
    };
    if (!risen || tl == 0) {  // (the first tile's are all relative to its maximum)
#pragma unroll
      for (int x = 0; x < 2 * kM4Groups; ++x) pr[x] = probability(x);
    } else {
#pragma unroll
      for (int x = 0; x < 2 * kM4Groups; ++x) {
        const float f = own[x >> 1] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(own[x >> 1] - now);
        const uint4 p = probability(x);
        pr[x] = make_uint4(pack_bf16x2(bf16_lo(p.x) * f, bf16_hi(p.x) * f), pack_bf16x2(bf16_lo(p.y) * f, bf16_hi(p.y) * f),
                           pack_bf16x2(bf16_lo(p.z) * f, bf16_hi(p.z) * f), pack_bf16x2(bf16_lo(p.w) * f, bf16_hi(p.w) * f));
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    Way next = {};
    if constexpr (MORE) {
      next = way(tl + 2, sl, buf == 0 ? (kM4Buffers - 1) * kM4Tile : buf - kM4Tile);
      sl = slot(tl + 3, e);
      e = entry(tl + 4);
    }
    __builtin_amdgcn_sched_barrier(0);
    // Block i: keys 32 (i / 4) .., dims 128 wv + 32 (i % 4) ..; its values (V^T
    // by the fp4 product) are two blocks ahead of their use, rounded one ahead.
    const auto values = [&](int i) {
      const int kb = i >> 2, g = i >> 1 & 1;
      v16f v;
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = 0.f;
      const v8i_m4 a = m4_fp4(c[2 * kb + g]), p = m4_fp4(pick[i & 1]);
      return g ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, p, v, 4, 4, 2, (int)sc[kb], 0, 0x7f7f7f7f)
               : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, p, v, 4, 4, 0, (int)sc[kb], 0, 0x7f7f7f7f);
    };
    v16f v[2] = {values(0), values(1)};
    uint32_t w[2][8];
    const auto round4 = [&](int i, int k) {  // half k of block i's values
#pragma unroll
      for (int e = 4 * k; e < 4 * k + 4; ++e) w[i & 1][e] = pack_bf16x2(v[i & 1][2 * e], v[i & 1][2 * e + 1]);
    };
    round4(0, 0);
    round4(0, 1);
#pragma unroll
    for (int i = 0; i < 4 * kM4Groups; ++i) {
      // three products, the next block's roundings between them
      __builtin_amdgcn_sched_barrier(0);
      if (i + 2 < 4 * kM4Groups) v[i & 1] = values(i + 2);
      v16f& acc = o[i & 3];
      const uint32_t* a = w[i & 1];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        __builtin_amdgcn_sched_barrier(0);
        if (i + 1 < 4 * kM4Groups) round4(i + 1, k);
        if constexpr (MORE)
          if (2 * i + k < 13) load(next, 2 * i + k);
        __builtin_amdgcn_sched_barrier(0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(m4_bf8(make_uint4(a[4 * k], a[4 * k + 1], a[4 * k + 2], a[4 * k + 3])),
                                                      m4_bf8(pr[i / 4 * 2 + k]), acc, 0, 0, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(kNone);  // the rows of tile tl + 2
    if (MORE || tl + 1 < tiles) m4_meet();
    buf = buf == (kM4Buffers - 1) * kM4Tile ? 0u : buf + kM4Tile;
  };
  int tl = 0;
#pragma unroll 1
  for (; tl + 2 < tiles; ++tl) sum_tile(tl, std::true_type{});
#pragma unroll 1
  for (; tl < tiles; ++tl) sum_tile(tl, std::false_type{});
  __syncthreads();

  const v4f ls = *reinterpret_cast<const v4f*>(&wl[n][0]);
  const float L = (ls[0] + ls[1]) + (ls[2] + ls[3]);
  const int head = hb * kM4Heads + n;
  if (head >= A.H) return;
  if (plan.count > 1) {
    // quad q (dims 8q + 4h .. + 3): a head after the other
    const int heads = m4_heads(A.H);
    const long at = (long)id * nhb + hb;
    v4f* part = reinterpret_cast<v4f*>(A.part_o) + at * (heads * (DSA_LATENT_DIM / 4)) + h * heads + n;
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const v16f& a = o[q >> 2];
      part[(16 * wv + q) * 2 * heads] = v4f{a[4 * (q & 3)], a[4 * (q & 3) + 1], a[4 * (q & 3) + 2], a[4 * (q & 3) + 3]};
    }
    if (wv == 0 && h == 0) {
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

// The chunks of a row meet: a workgroup takes 8 heads x 8 of the 128 pieces of
// four dims (64 bytes of each head's output), a lane each; its waves take the
// chunks in turn, and their sums meet in LDS.  Always in the same order.
//
// Bound by the partial sums it reads, 64 KB a chunk and 32 heads: 16.8 MB in
// 5.2 us after 64 chunks of 128 heads, 2.5 us for 16 chunks of 16 heads.  16
// waves a workgroup where a row has many chunks (42 each: 6.3 us), else 4 (16
// waves took 4.2 us for 16 chunks).  Workgroups that go on to further pieces:
// 1-2 us more for split rows, 2 less for 100 rows that are not.
constexpr int kM4Quads = DSA_LATENT_DIM / 8;  // of eight dims, two pieces each
constexpr int kM4MergeAhead = 4;
constexpr int kM4MergeFew = 16;  // chunks of a row, on average, that 4 waves take

template <int W>
__global__ __launch_bounds__(W* kWave) void mla_fp4_merge_kernel(const Mla4Args A) {
  __shared__ float sm[W][kWave], sl[W][kWave];
  __shared__ v4f so[W][kWave];
  const int lane = threadIdx.x & (kWave - 1), wv = wave_id();
  const int nhb = m4_blocks(A.H), heads = m4_heads(A.H), per = kM4Quads * 2 * heads / kWave;
  const int hb = (int)(blockIdx.x / per), b = (int)blockIdx.y;
  const int2 plan = A.units ? make_int2(b * A.per_row, A.per_row) : A.plan[b];
  const int first = plan.x, count = plan.y;
  if (count == 1) return;  // (the same in the whole workgroup)
  const int eights = heads / 8, at8 = (int)(blockIdx.x % per);
  const int x = at8 % eights * 8 + (lane & 7), q = at8 / eights * 8 + (lane >> 3), head = hb * kM4Heads + x;
  const v4f* part = reinterpret_cast<const v4f*>(A.part_o);
  float mx = -INFINITY, L = 0.f;
  v4f acc = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = wv; c0 < count; c0 += W * kM4MergeAhead) {
    float m[kM4MergeAhead], l[kM4MergeAhead], next = mx;
    v4f a[kM4MergeAhead];
#pragma unroll
    for (int k = 0; k < kM4MergeAhead; ++k) {  // (past the last: chunk c0 again, for nothing)
      const bool have = c0 + k * W < count;
      const long at = (long)(first + (have ? c0 + k * W : c0)) * nhb + hb;
      const float2 ml = reinterpret_cast<const float2*>(A.part_ml)[at * heads + x];
      const v4f v = part[(at * (kM4Quads * 2) + q) * heads + x];
      m[k] = have ? ml.x : -INFINITY;
      l[k] = have ? ml.y : 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) a[k][e] = have ? v[e] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < kM4MergeAhead; ++k) next = fmaxf(next, m[k]);
    const float down = mx == -INFINITY ? 0.f : exp2f(mx - next);
    L *= down;
    acc *= down;
#pragma unroll
    for (int k = 0; k < kM4MergeAhead; ++k) {
      const float f = m[k] == -INFINITY ? 0.f : exp2f(m[k] - next);
      L += l[k] * f;
      acc += a[k] * f;
    }
    mx = next;
  }
  sm[wv][lane] = mx;
  sl[wv][lane] = L;
  so[wv][lane] = acc;
  __syncthreads();
  if (wv || head >= A.H) return;
  for (int w = 1; w < W; ++w) mx = fmaxf(mx, sm[w][lane]);
  L = 0.f;
  acc = v4f{0.f, 0.f, 0.f, 0.f};
  for (int w = 0; w < W; ++w) {
    const float f = sm[w][lane] == -INFINITY ? 0.f : exp2f(sm[w][lane] - mx);
    L += sl[w][lane] * f;
    acc += so[w][lane] * f;
  }
  const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
  v2u_t w;
  w[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  w[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
  *reinterpret_cast<v2u_t*>(A.out + ((long)b * A.H + head) * DSA_LATENT_DIM + 4 * q) = w;
}

// Chunks the rows share: nsplit a row, or (0) what fills the chip once, one
// workgroup a CU; at most kM4MergeMax for kM4Ragged rows and fewer, dense or
// selected (one dense row may take them all; the partials then stay within 17 MB
// for 16 heads, and twice the chip's CUs are there already).  Measured around 0's choice: 32 rows of 2048
// selected keys, 16 heads: 23.9 us at 2 a row, 18.7 at 4, 17.6 at 8 (0's), 23.4
// at 16; 8 rows of 16K keys, 128 heads: 66.5 at 4, 47.2 at 8 (0's), 52.7 at 16.
// Dense rows share by length wherever there are more chunks than rows: 100 rows
// of 64 heads, one of 16K keys and 99 of 500, take 23.7 us (a chunk each: 219);
// 100 of 2000 keys 43.8 (37.0).  At the chip's fill a chunk a row is the default:
// 64 rows of 128 heads and 1024 to 2048 keys 37.8 us, 61.7 with two a row.  So a
// long row among short ones is not cut there: 128 rows of 64 heads, one of 16K
// keys and 127 of 500, take 219 us, with two a row asked for 36.
static int m4_chunks(int B, int H, int nsplit) {
  const long want = nsplit > 0 ? (long)B * nsplit : (long)(device_cu_count() / m4_blocks(H));
  return (int)std::max((long)B, B <= kM4Ragged ? std::min(want, (long)kM4MergeMax) : want);
}

// Partial sums and plan of a call; 0: unsplit rows, none is read.
static size_t mla_fp4_partial_bytes(int B, int H, int nsplit) {
  const int chunks = m4_chunks(B, H, nsplit);
  if (chunks <= B) return 0;
  return (size_t)chunks * m4_blocks(H) * m4_heads(H) * (DSA_LATENT_DIM + 2) * sizeof(float) + (size_t)B * sizeof(int2);
}

// The partials lie behind as many barriers as an 8-bit call of the same rows and
// heads keeps at a workspace's start.  A call of more rows keeps more of them:
// mla_fp4_workspace_in() below moves this call's workspace behind those.
size_t mla_fp4_workspace_bytes(int B, int H, int nsplit) {
  const size_t partials = mla_fp4_partial_bytes(B, H, nsplit);
  return partials ? attn_workspace_bytes(B, H, 0) + partials : 16;
}

// The bytes at the start of a workspace of `bytes` that may hold barriers: an
// 8-bit call that fits has a barrier and one split's partials at least for each
// of its (row, head group)s.
static size_t mla_barrier_room(size_t bytes) { return bytes / attn_workspace_bytes(1, 16, 1) * attn_workspace_bytes(1, 16, 0); }

// Where in a workspace that 8-bit calls of any rows and heads share a 4-bit call
// has its own, so that its partials begin behind every barrier; -1: too small.
long mla_fp4_workspace_in(size_t bytes, int B, int H, int nsplit) {
  const size_t partials = mla_fp4_partial_bytes(B, H, nsplit), room = mla_barrier_room(bytes);
  if (!partials) return bytes >= 16 ? 0 : -1;
  const size_t own = attn_workspace_bytes(B, H, 0), from = std::max(room, own);
  return bytes >= from + partials ? (long)(from - own) : -1;
}

// Bytes for calls over both formats; nsplit 0: of every split count.
size_t mla_shared_workspace_bytes(int B, int H, int nsplit) {
  const size_t partials = std::max(mla_fp4_partial_bytes(B, H, nsplit), mla_fp4_partial_bytes(B, H, nsplit ? nsplit : 128));
  size_t bytes = attn_workspace_bytes(B, H, nsplit ? nsplit : 128);
  for (size_t need; (need = partials + std::max(mla_barrier_room(bytes), attn_workspace_bytes(B, H, 0))) > bytes;) bytes = need;
  return (bytes + 15) / 16 * 16;
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
  const int row_units = (A.keys - 1) / kM4Unit + 1;
  A.chunks = m4_chunks(A.B, A.H, nsplit);
  A.part_o = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + attn_workspace_bytes(A.B, A.H, 0));
  A.part_ml = A.part_o + (size_t)A.chunks * blocks * m4_heads(A.H) * DSA_LATENT_DIM;
  A.plan = reinterpret_cast<int2*>(A.part_ml + (size_t)A.chunks * blocks * m4_heads(A.H) * 2);
  const int per_row = A.chunks / A.B;
  int grid_chunks = A.chunks;
  if (A.chunks <= A.B || !A.dense_pt || A.B > kM4Ragged) {  // the same split for every row
    A.units = (row_units + per_row - 1) / per_row;
    A.per_row = (row_units + A.units - 1) / A.units;
    grid_chunks = A.B * A.per_row;
  }
  const dim3 grid((unsigned)((grid_chunks + 7) / 8 * 8 * blocks));
  const auto kernel = A.dense_pt ? mla_fp4_kernel<true> : mla_fp4_kernel<false>;
  hipLaunchKernelGGL(kernel, grid, dim3(kM4Threads), kM4Lds, s, A);
  if (hipError_t r = hipGetLastError()) return r;
  if (A.units && A.per_row == 1) return hipSuccess;
  const dim3 merge_grid((unsigned)(blocks * kM4Quads * 2 * m4_heads(A.H) / kWave), (unsigned)A.B);
  const bool many = (A.units ? A.per_row : A.chunks / A.B) > kM4MergeFew;
  hipLaunchKernelGGL(many ? mla_fp4_merge_kernel<16> : mla_fp4_merge_kernel<4>, merge_grid, dim3(kWave * (many ? 16 : 4)), 0, s, A);
  return hipGetLastError();
}

}  // namespace dsa
