// Sparse / dense MLA decode over a latent cache held in 4 bits (gfx950):
//   out[b,h,:] = sum_j softmax_j(sm * q[b,h,:] . kv_j) * kv_j[:512],
//   kv_j = e2m1 * 2^(scale byte[d/32] - 127) | bf16 rope, from a 400-byte row
//   [256 B: value 2i in the low half of byte i][16 e8m0][64 bf16].
// One value of a row is a 2-bit significand times a power of two, so its bf16
// form is exact: v_cvt_scalef32_pk_bf16_fp4 gives two a instruction.
//
// Every wave works alone on 16 keys a step: rows gathered to registers,
// dequantised, S^T = K Q^T with the rows as the A operand, the probabilities
// used where they come out (O^T = V^T P^T), the values transposed through a
// piece of LDS only this wave uses.  The next rows are in flight from the end
// of QK on.  A workgroup (8 waves) takes a chunk of a row's keys for 16
// heads; its waves' sums meet once, at the end.  Chunks of the same row meet
// in a second, small launch: no workgroup waits for another, so the call
// needs no co-residency and keeps no state in its workspace.
//
// Each probability enters PV as two bf16 terms, hi + lo, in the two halves of
// a k = 32 MFMA whose A operand repeats the 16 values.

#include "dsa_common.h"
#include "dsa_kernels.h"
#include "quant_core.h"

namespace dsa {

constexpr int kM4Waves = 8;
constexpr int kM4Threads = kM4Waves * kWave;
constexpr int kM4Keys = 16;                         // keys a wave's step
constexpr int kM4Unit = kM4Waves * kM4Keys;         // keys a workgroup's step: chunks are multiples
constexpr int kM4QLd = DSA_QK_DIM + 8;              // query row stride (bf16)
constexpr int kM4VLd = DSA_LATENT_DIM + 16;         // value row stride (bf16)
constexpr int kM4OLd = DSA_LATENT_DIM + 4;          // merge row stride (fp32)
constexpr int kM4Slots = kM4Waves / 2;              // waves' sums held at once by the merge
constexpr float kM4Rise = 16.f;                     // log2 growth of the maximum that rescales the sums
constexpr size_t kM4QLds = (size_t)kHeadGroup * kM4QLd * 2;
constexpr size_t kM4WaveLds = (size_t)kM4Keys * kM4VLd * 2;
constexpr size_t kM4SlotLds = (size_t)kHeadGroup * kM4OLd * 4;
constexpr size_t kM4Lds = kM4Waves * kM4WaveLds + kM4QLds;
static_assert(kM4Slots * kM4SlotLds <= kM4Waves * kM4WaveLds, "the merge's sums fit the value pieces");
static_assert(kM4Lds + 2048 <= 160 * 1024, "one CU's LDS");

typedef short v4s_m4 __attribute__((ext_vector_type(4)));
typedef v4s_m4 __attribute__((address_space(3)))* m4_lds_ptr;

__device__ __forceinline__ v8bf m4_bf8(const uint4& a) {
  v8bf v;
  __builtin_memcpy(&v, &a, 16);
  return v;
}
// op over the four 16-lane groups of a wave, the result in every lane
template <class F>
__device__ __forceinline__ float m4_groups(float v, F op) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

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
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float wm[kM4Waves][kHeadGroup], wl[kM4Waves][kHeadGroup];
  const int t = threadIdx.x, lane = t & (kWave - 1), wv = wave_id();
  const int kr = lane & 15, kc = lane >> 4;
  // a chunk's head groups on one XCD (workgroup number modulo 8), whose L2
  // then serves all but the first's reads of its rows
  const int nhg = A.H / kHeadGroup;
  const int hg = (blockIdx.x / 8) % nhg, id = (blockIdx.x / (8 * nhg)) * 8 + blockIdx.x % 8;
  M4Plan plan;
  const int b = m4_plan_chunk(A, id, lane, plan);
  if (b < 0) return;  // (the same in the whole workgroup)
  const int total = m4_row_keys(A, b);
  const long j0 = (long)(id - plan.first) * plan.units * kM4Unit;
  const int jend = (int)min((long)total, j0 + (long)plan.units * kM4Unit);
  const int steps = (int)((max((long)jend, j0) - j0 + kM4Keys - 1) / kM4Keys);
  const int* idx_row = DENSE ? A.dense_pt + (long)b * A.dense_pt_stride : A.idx + (long)b * A.keys;
  const auto slot = [&](int st) {
    const long j = j0 + (long)st * kM4Keys + kr;
    if (j >= jend) return -1L;
    if constexpr (!DENSE) return (long)idx_row[j];
    const long page = idx_row[j >> 6];
    return page < 0 ? -1L : page * DSA_PAGE_TOKENS + (j & (DSA_PAGE_TOKENS - 1));
  };

  // the query block, staged once: the B operand (n = head kr), read in the
  // keys' dim order: step 4i + u -> dims 128i + 32kc + 8u .. + 7;
  // 16 + s -> rope dims 32s + 8kc .. + 7
  uint16_t* qs = reinterpret_cast<uint16_t*>(smem + kM4Waves * kM4WaveLds);
  {
    constexpr int kVec = kHeadGroup * DSA_QK_DIM / 8, kRowVec = DSA_QK_DIM / 8;
    const uint4* src = reinterpret_cast<const uint4*>(A.q + ((long)b * A.H + hg * kHeadGroup) * DSA_QK_DIM);
    for (int i = t; i < kVec; i += kM4Threads)
      *reinterpret_cast<uint4*>(qs + (i / kRowVec) * kM4QLd + (i % kRowVec) * 8) = src[i];
  }
  __syncthreads();
  const uint16_t* qrow = qs + kr * kM4QLd;
  const auto q_op = [&](int s) {
    return m4_bf8(*reinterpret_cast<const uint4*>(
        qrow + (s < 16 ? 128 * (s >> 2) + 32 * kc + 8 * (s & 3) : DSA_LATENT_DIM + 32 * (s - 16) + 8 * kc)));
  };

  // One step's rows: lane (kr, kc) holds key kr's dims 128i + 32kc .. + 31 of
  // each 128 (16 bytes, one scale), rope dims 32s + 8kc .. + 7.
  struct Rows {
    uint4 nope[4], rope[2], sc;
    bool ok;
  };
  const auto load = [&](long sl, Rows& r) {
    r.ok = sl >= 0 && sl < A.kv_rows;
    const uint8_t* p = A.pool + (r.ok ? sl : 0) * DSA_FP4_ROW_BYTES;
    r.sc = make_uint4(0, 0, 0, 0);
    r.rope[0] = r.rope[1] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.nope[i] = make_uint4(0, 0, 0, 0);
    if (r.ok) {
      r.sc = *reinterpret_cast<const uint4*>(p + DSA_LATENT_DIM / 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) r.nope[i] = *reinterpret_cast<const uint4*>(p + 64 * i + 16 * kc);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        r.rope[s] = *reinterpret_cast<const uint4*>(p + DSA_LATENT_DIM / 2 + 16 + 64 * s + 16 * kc);
    }
  };

  uint16_t* vt = reinterpret_cast<uint16_t*>(smem + wv * kM4WaveLds);  // [16 keys][dims], this wave's
  const uint16_t* vsrc = vt + (4 * kc + (kr >> 2)) * kM4VLd + 4 * (kr & 3);
  v4f o[32];  // O^T: dims 16 dt + 4 kc + i of head kr
#pragma unroll
  for (int dt = 0; dt < 32; ++dt) o[dt] = v4f{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;  // sums are relative to m, which trails the maximum by at most kM4Rise

  Rows r;
  int st = wv;
  long sl1 = slot(st + kM4Waves);
  if (st < steps) load(slot(st), r);
  for (; st < steps; st += kM4Waves) {
    asm volatile("" ::: "memory");  // the query operands' reads stay here (hoisted, they spill)
    const long sl2 = slot(st + 2 * kM4Waves);
    v4f s = {0.f, 0.f, 0.f, 0.f};
    const uint32_t scw[4] = {r.sc.x, r.sc.y, r.sc.z, r.sc.w};
    uint4* vrow = reinterpret_cast<uint4*>(vt + kr * kM4VLd + 32 * kc);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float sc = __uint_as_float(((scw[i] >> (8 * kc)) & 0xffu) << 23);
      const uint32_t cw[4] = {r.nope[i].x, r.nope[i].y, r.nope[i].z, r.nope[i].w};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint4 k = dequant8_fp4(cw[u], sc);
        s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(m4_bf8(k), q_op(4 * i + u), s, 0, 0, 0);
        vrow[16 * i + u] = k;
      }
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
      s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(m4_bf8(r.rope[x]), q_op(16 + x), s, 0, 0, 0);
    // element i is key 4kc + i of head kr; its validity is the gathering
    // lane's (kr = 4kc + i of any group)
    const uint64_t okm = __ballot(r.ok);
    const uint32_t mine = (uint32_t)(okm >> (4 * kc));
    if (st + kM4Waves < steps) load(sl1, r);
    sl1 = sl2;
    if (okm == 0) continue;
    float tmax = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = mine & (1u << i) ? s[i] * A.sm_log2 : -INFINITY;
      tmax = fmaxf(tmax, s[i]);
    }
    tmax = m4_groups(tmax, [](float x, float y) { return fmaxf(x, y); });
    if (__ballot(tmax > m + kM4Rise || m == -INFINITY) != 0) {
      const float mn = fmaxf(m, tmax);
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
      for (int dt = 0; dt < 32; ++dt) o[dt] *= f;
      l *= f;
      m = mn;
    }
    const float mr = m == -INFINITY ? 0.f : m;
    uint32_t ph[2], pl[2];
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const float p0 = __builtin_amdgcn_exp2f(s[i] - mr), p1 = __builtin_amdgcn_exp2f(s[i + 1] - mr);
      const uint32_t w = pack_bf16x2(p0, p1);
      ph[i >> 1] = w;
      pl[i >> 1] = pack_bf16x2(p0 - __uint_as_float(w << 16), p1 - __uint_as_float(w & 0xffff0000u));
      l += p0 + p1;
    }
    const v8bf pb = m4_bf8(make_uint4(ph[0], ph[1], pl[0], pl[1]));
#pragma unroll
    for (int dt = 0; dt < 32; ++dt) {
      const v2u_t x = __builtin_bit_cast(v2u_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((m4_lds_ptr)(vsrc + 16 * dt)));
      o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(m4_bf8(make_uint4(x[0], x[1], x[0], x[1])), pb, o[dt], 0, 0, 0);
    }
  }

  // the waves' sums meet: wave w takes in wave w + 4's (same lanes, same
  // elements), then the four are added relative to the largest maximum
  l = m4_groups(l, [](float x, float y) { return x + y; });
  if (kc == 0) {
    wm[wv][kr] = m;
    wl[wv][kr] = l;
  }
  __syncthreads();
  float* os = reinterpret_cast<float*>(smem + (wv % kM4Slots) * kM4SlotLds) + kr * kM4OLd + 4 * kc;  // [head][dim]
  if (wv >= kM4Slots)
#pragma unroll
    for (int dt = 0; dt < 32; ++dt) *reinterpret_cast<v4f*>(os + 16 * dt) = o[dt];
  __syncthreads();
  if (wv < kM4Slots) {
    const float m2 = wm[wv + kM4Slots][kr], l2 = wl[wv + kM4Slots][kr];
    const float mm = fmaxf(m, m2);
    const float f1 = m == -INFINITY ? 0.f : exp2f(m - mm), f2 = m2 == -INFINITY ? 0.f : exp2f(m2 - mm);
#pragma unroll
    for (int dt = 0; dt < 32; ++dt) {
      v4f* p = reinterpret_cast<v4f*>(os + 16 * dt);
      *p = o[dt] * f1 + *p * f2;
    }
    if (kc == 0) {
      wm[wv][kr] = mm;
      wl[wv][kr] = l * f1 + l2 * f2;
    }
  }
  __syncthreads();
  const int h = t >> 5, d0 = 4 * (t & 31);
  float mx = -INFINITY, L = 0.f, f[kM4Slots];
#pragma unroll
  for (int w = 0; w < kM4Slots; ++w) mx = fmaxf(mx, wm[w][h]);
#pragma unroll
  for (int w = 0; w < kM4Slots; ++w) {
    f[w] = wm[w][h] == -INFINITY ? 0.f : exp2f(wm[w][h] - mx);
    L += wl[w][h] * f[w];
  }
  const auto sum = [&](int d) {
    v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kM4Slots; ++w)
      acc += *reinterpret_cast<const v4f*>(reinterpret_cast<const float*>(smem + w * kM4SlotLds) + h * kM4OLd + d) * f[w];
    return acc;
  };
  if (plan.count > 1) {
    const long at = ((long)id * nhg + hg) * kHeadGroup + h;
    float* part = A.part_o + at * DSA_LATENT_DIM;
#pragma unroll
    for (int j = 0; j < DSA_LATENT_DIM / 128; ++j) *reinterpret_cast<v4f*>(part + d0 + 128 * j) = sum(d0 + 128 * j);
    if (d0 == 0) {
      A.part_ml[2 * at] = mx;
      A.part_ml[2 * at + 1] = L;
    }
    return;
  }
  const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);  // no key: 0; NaN stays
  uint16_t* out = A.out + ((long)b * A.H + hg * kHeadGroup + h) * DSA_LATENT_DIM + d0;
#pragma unroll
  for (int j = 0; j < DSA_LATENT_DIM / 128; ++j) {
    const v4f acc = sum(d0 + 128 * j);
    v2u_t w;
    w[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    w[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<v2u_t*>(out + 128 * j) = w;
  }
}

// The chunks of a row meet: a wave takes 256 dims of a head, in the chunks'
// order.  Rows of one chunk are done; one without a key becomes 0.
constexpr int kM4MergeThreads = 256;
constexpr int kM4MergeMax = 512;  // chunks of a row

__global__ __launch_bounds__(kM4MergeThreads) void mla_fp4_merge_kernel(const Mla4Args A) {
  __shared__ float fs[kM4MergeThreads / kWave][kM4MergeMax];
  const int lane = threadIdx.x & (kWave - 1), wv = wave_id();
  const int unit = blockIdx.x * (kM4MergeThreads / kWave) + wv;  // (row, head, half)
  const int half = unit & 1, h = (unit >> 1) % A.H, b = (unit >> 1) / A.H;
  if (b >= A.B) return;
  const M4Plan p = m4_plan_row(A, b, lane);
  if (p.count == 1) return;
  const int nhg = A.H / kHeadGroup;
  const auto at = [&](int c) { return ((long)(p.first + c) * nhg + h / kHeadGroup) * kHeadGroup + h % kHeadGroup; };
  float mx = -INFINITY, L = 0.f;
  for (int c = lane; c < p.count; c += kWave) mx = fmaxf(mx, A.part_ml[2 * at(c)]);
  mx = wave_max(mx);
  for (int c = lane; c < p.count; c += kWave) {
    const float m = A.part_ml[2 * at(c)];
    const float f = m == -INFINITY ? 0.f : exp2f(m - mx);
    fs[wv][c] = f;
    L += A.part_ml[2 * at(c) + 1] * f;
  }
  for (int o = 32; o >= 1; o >>= 1) L += __shfl_xor(L, o);
  __builtin_amdgcn_wave_barrier();
  v4f acc = {0.f, 0.f, 0.f, 0.f};
  const int d = 256 * half + 4 * lane;
#pragma unroll 8
  for (int c = 0; c < p.count; ++c) acc += *reinterpret_cast<const v4f*>(A.part_o + at(c) * DSA_LATENT_DIM + d) * fs[wv][c];
  const float inv = L > 0.f ? 1.f / L : (L == L ? 0.f : L);
  v2u_t w;
  w[0] = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  w[1] = pack_bf16x2(acc[2] * inv, acc[3] * inv);
  *reinterpret_cast<v2u_t*>(A.out + ((long)b * A.H + h) * DSA_LATENT_DIM + d) = w;
}

// Chunks the rows share: nsplit a row, or (0) what fills the chip once; at
// most kM4MergeMax where one row may take them all (kM4Ragged rows and fewer).
constexpr int kM4Ragged = 256;
static int m4_chunks(int B, int H, int nsplit) {
  const long want = nsplit > 0 ? (long)B * nsplit : device_cu_count() / (H / kHeadGroup);
  return (int)max((long)B, B <= kM4Ragged ? min(want, (long)kM4MergeMax) : want);
}

// The partials lie behind the barriers that the 8-bit decode keeps in a
// workspace, so calls over both formats may take turns with one.
size_t mla_fp4_workspace_bytes(int B, int H, int nsplit) {
  const int chunks = m4_chunks(B, H, nsplit);
  if (chunks / B <= 1) return 16;  // unsplit rows: none is read
  return attn_workspace_bytes(B, H, 0) + (size_t)chunks * H * (DSA_LATENT_DIM + 2) * sizeof(float);
}

hipError_t launch_mla_fp4(Mla4Args A, int nsplit, void* workspace, hipStream_t s) {
  static PerDeviceOnce attr;
  const hipError_t e = attr.run([] {
    for (const void* f : {(const void*)mla_fp4_kernel<false>, (const void*)mla_fp4_kernel<true>})
      if (hipError_t r = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)kM4Lds)) return r;
    return hipSuccess;
  });
  if (e != hipSuccess) return e;
  const int nhg = A.H / kHeadGroup;
  const int row_units = (A.keys + kM4Unit - 1) / kM4Unit;
  A.chunks = m4_chunks(A.B, A.H, nsplit);
  A.part_o = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + attn_workspace_bytes(A.B, A.H, 0));
  A.part_ml = A.part_o + (size_t)A.chunks * A.H * DSA_LATENT_DIM;
  const int per_row = A.chunks / A.B;
  int grid_chunks = A.chunks;
  if (per_row <= 1 || !A.dense_pt || A.B > kM4Ragged) {  // the same split for every row
    A.units = (row_units + per_row - 1) / per_row;
    A.per_row = (row_units + A.units - 1) / A.units;
    grid_chunks = A.B * A.per_row;
  }
  const dim3 grid((unsigned)((grid_chunks + 7) / 8 * 8 * nhg));
  if (A.dense_pt) hipLaunchKernelGGL(mla_fp4_kernel<true>, grid, dim3(kM4Threads), kM4Lds, s, A);
  else hipLaunchKernelGGL(mla_fp4_kernel<false>, grid, dim3(kM4Threads), kM4Lds, s, A);
  if (hipError_t r = hipGetLastError()) return r;
  if (A.units && A.per_row == 1) return hipSuccess;
  const int waves = 2 * A.B * A.H, per = kM4MergeThreads / kWave;
  hipLaunchKernelGGL(mla_fp4_merge_kernel, dim3((unsigned)((waves + per - 1) / per)), dim3(kM4MergeThreads), 0, s, A);
  return hipGetLastError();
}

}  // namespace dsa
