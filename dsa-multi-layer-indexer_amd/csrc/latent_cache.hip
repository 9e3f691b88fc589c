// Appending a layer's new tokens to the paged caches, with the norm and the
// rotation on the way, and reading latent rows back (gfx950).
//
// Append, per token (request rows[i], position pos[i], the caches' slot from
// the page table):
//   latent row: c = latent[:512], normed when a weight is given
//     (c / sqrt(mean(c^2) + eps) * w), quantised by quant_core.h's rules to
//     656 bytes (e4m3, 4 fp32 scales) or 400 (e2m1, 16 e8m0 scales); the 64
//     rope values rotated by the position and rounded to bf16;
//   index key: the first 64 of 128 rotated, quantised into its page.
// One wave a latent row, 16 lanes an index key, both in one launch.
//
// The norm is computed in 64 bits: the value it gives decides the code, and
// a value next to a code's border would otherwise be stored a whole step
// off, depending on the order of the sum.  (In 64 bits a lane's 8 values cost
// 0.8 of the 9 us below; a division and a root in place of the reciprocal root 3
// more.)
//
// 8191 tokens, latent to 400 bytes and index key: 8.7 us for 18 MB, bound by the
// arithmetic of the norm and the two quantisers (half of it) and the chain from
// the position over the page to the store; to 656 bytes 9.2 (20 MB), without the
// norm 7.4.  One token: 2.3 us.
#include "dsa_kernels.h"
#include "quant_core.h"

namespace dsa {

constexpr int kAppendThreads = 256;
constexpr int kAppendUnits = kAppendThreads / kWave;  // waves a workgroup

// sum over the wave, the same value in every lane
__device__ __forceinline__ double wave_sum64(double v) {
  const auto sh = [](auto ctrl, auto rows, double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = dpp_u32<decltype(ctrl)::value, decltype(rows)::value>((uint32_t)b, 0u);
    const uint32_t hi = dpp_u32<decltype(ctrl)::value, decltype(rows)::value>((uint32_t)(b >> 32), 0u);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  };
  using All = std::integral_constant<int, 0xf>;
  v += sh(std::integral_constant<int, 0x111>{}, All{}, v);
  v += sh(std::integral_constant<int, 0x112>{}, All{}, v);
  v += sh(std::integral_constant<int, 0x114>{}, All{}, v);
  v += sh(std::integral_constant<int, 0x118>{}, All{}, v);
  v += sh(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{}, v);
  v += sh(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{}, v);
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 63);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), 63);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Where a token goes, in both caches.  slot < 0: nowhere (no request, page or
// table row, or a place that one of the caches that are given does not have: a
// key whose latent row is not there could be selected).
struct Place {
  int pos;
  long page, slot;
};
__device__ __forceinline__ Place place_of(const AppendArgs& A, int t) {
  Place p{A.pos[t], -1, -1};
  const int r = A.rows[t];
  if (r < 0 || r >= A.B || p.pos < 0 || p.pos / DSA_PAGE_TOKENS >= A.pt_stride || (A.table && p.pos >= A.table_rows))
    return p;
  p.page = A.page_table[(long)r * A.pt_stride + p.pos / DSA_PAGE_TOKENS];
  p.slot = p.page * DSA_PAGE_TOKENS + p.pos % DSA_PAGE_TOKENS;
  if (p.page < 0 || (A.latent && p.slot >= A.kv_rows) || (A.keys && p.page >= A.num_pages)) p.slot = -1;
  return p;
}

// A wave's latent row: 8 values of the latent part a lane, a pair of the
// rope part for lanes 0-31.  All inputs are on their way before the place is
// known.
template <int DT, bool WIDE, int BYTES>
__device__ __forceinline__ void append_latent_row(const AppendArgs& A, int t) {
  constexpr int kHalf = DSA_ROPE_DIM / 2;
  const int lane = threadIdx.x & (kWave - 1), pair = lane & (kHalf - 1);
  const long src = (long)t * A.latent_stride;
  float x[8], w[8];
  load8<DT, WIDE>(A.latent, src + 8 * lane, x);
  const int ia = A.interleaved ? 2 * pair : pair, ib = A.interleaved ? 2 * pair + 1 : pair + kHalf;
  const float a = load_elem<DT>(A.latent, src + DSA_LATENT_DIM + ia);
  const float b = load_elem<DT>(A.latent, src + DSA_LATENT_DIM + ib);
  if (A.norm_w) {
    if (A.norm_w_f32) load8<kF32, WIDE>(A.norm_w, 8 * lane, w);
    else load8<DT, WIDE>(A.norm_w, 8 * lane, w);
  }
  const Place p = place_of(A, t);
  if (p.slot < 0) return;
  float c = 1.f, s = 0.f;
  if (A.table) {
    c = A.table[(long)p.pos * DSA_ROPE_DIM + pair];
    s = A.table[(long)p.pos * DSA_ROPE_DIM + kHalf + pair];
  }
  if (A.norm_w) {
    double ss = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = __builtin_fma((double)x[e], (double)x[e], ss);
    const double rs = rsqrt(wave_sum64(ss) * (1.0 / DSA_LATENT_DIM) + A.eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)((double)x[e] * rs * (double)w[e]);
  }
  uint8_t* dst = A.pool + p.slot * BYTES;
  if constexpr (BYTES == DSA_LATENT_ROW_BYTES) {
    const float scale = row_scale<true>(x);
    *reinterpret_cast<v2u_t*>(dst + 8 * lane) = quant8<true>(x, scale);
    if ((lane & 15) == 0) reinterpret_cast<float*>(dst + DSA_LATENT_DIM)[lane >> 4] = scale;
  } else {
    const uint32_t sb = fp4_scale_byte(x);
    reinterpret_cast<uint32_t*>(dst)[lane] = quant8_fp4(x, sb);
    if ((lane & 3) == 0) dst[DSA_LATENT_DIM / 2 + (lane >> 2)] = (uint8_t)sb;
  }
  if (lane < kHalf) {
    uint16_t* rope = reinterpret_cast<uint16_t*>(dst + BYTES - 2 * DSA_ROPE_DIM);
    float ya = a, yb = b;
    if (A.table) turn(a, b, c, s, ya, yb);
    const uint32_t v = pack_bf16x2(ya, yb);
    if (A.interleaved) {
      reinterpret_cast<uint32_t*>(rope)[lane] = v;
    } else {
      rope[lane] = (uint16_t)v;
      rope[lane + kHalf] = (uint16_t)(v >> 16);
    }
  }
}

// 16 lanes' index key, 8 values each; lanes 0-7 hold the turned half.
template <int DT, bool WIDE>
__device__ __forceinline__ void append_key(const AppendArgs& A, int t) {
  const int i = threadIdx.x & 15;
  const long src = (long)t * A.keys_stride;
  float x[8], o[8];  // o: lane i ^ 4's, the partners of the half layout
  load8<DT, WIDE>(A.keys, src + 8 * i, x);
  const bool turned = A.table && i < DSA_ROPE_DIM / 8;
  if (turned && !A.index_interleaved) load8<DT, WIDE>(A.keys, src + 8 * (i ^ 4), o);
  const Place p = place_of(A, t);
  if (p.slot < 0) return;
  if (turned) {
    constexpr int kHalf = DSA_ROPE_DIM / 2;
    const float* cs = A.table + (long)p.pos * DSA_ROPE_DIM;
    if (A.index_interleaved) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        turn(x[2 * k], x[2 * k + 1], cs[4 * i + k], cs[kHalf + 4 * i + k], x[2 * k], x[2 * k + 1]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float c = cs[8 * (i & 3) + e], s = cs[kHalf + 8 * (i & 3) + e];
        x[e] = __builtin_fmaf(o[e], i < 4 ? -s : s, x[e] * c);  // (turn, this lane's side)
      }
    }
  }
  const float scale = row_scale<true>(x);
  uint8_t* base = A.index_k + p.page * DSA_INDEX_PAGE_BYTES;
  const int slot = p.pos % DSA_PAGE_TOKENS;
  *reinterpret_cast<v2u_t*>(base + slot * DSA_INDEX_DIM + 8 * i) = quant8<true>(x, scale);
  if (i == 0) reinterpret_cast<float*>(base + DSA_PAGE_TOKENS * DSA_INDEX_DIM)[slot] = scale;
}

// Waves 0 .. n - 1: a latent row each (when there is a latent); those behind:
// four index keys each.
template <int DT, bool WIDE, int BYTES>
__global__ __launch_bounds__(kAppendThreads) void append_tokens_kernel(const AppendArgs A) {
  const long unit = (long)blockIdx.x * kAppendUnits + wave_id();
  const long n_lat = A.latent ? A.n : 0;
  if (unit < n_lat) {
    append_latent_row<DT, WIDE, BYTES>(A, (int)unit);
    return;
  }
  const long t = 4 * (unit - n_lat) + ((threadIdx.x & (kWave - 1)) >> 4);
  if (A.keys && t < A.n) append_key<DT, WIDE>(A, (int)t);
}

template <int DT>
static hipError_t launch_append_dt(const AppendArgs& A, int row_bytes, hipStream_t s) {
  constexpr int es = DT == kF32 ? 4 : 2;
  const auto on16 = [](const void* p, long stride) { return (((uintptr_t)p | (uintptr_t)(stride * es)) & 15) == 0; };
  const bool wide = (!A.latent || on16(A.latent, A.latent_stride)) && (!A.keys || on16(A.keys, A.keys_stride)) &&
                    on16(A.norm_w, 0);
  const auto go = [&](auto kernel) {
    // (a token has up to a wave and a quarter)
    return in_launches(A.n, 1L << 25, [&](long at, long n) {
      AppendArgs P = A;
      P.rows += at, P.pos += at, P.n = (int)n;
      if (A.latent) P.latent = static_cast<const uint8_t*>(A.latent) + at * A.latent_stride * es;
      if (A.keys) P.keys = static_cast<const uint8_t*>(A.keys) + at * A.keys_stride * es;
      const long units = (A.latent ? n : 0) + (A.keys ? (n + 3) / 4 : 0);
      hipLaunchKernelGGL(kernel, dim3((unsigned)((units + kAppendUnits - 1) / kAppendUnits)), dim3(kAppendThreads), 0, s, P);
      return hipGetLastError();
    });
  };
  if (row_bytes == DSA_LATENT_ROW_BYTES)
    return wide ? go(append_tokens_kernel<DT, true, DSA_LATENT_ROW_BYTES>)
                : go(append_tokens_kernel<DT, false, DSA_LATENT_ROW_BYTES>);
  return wide ? go(append_tokens_kernel<DT, true, DSA_FP4_ROW_BYTES>) : go(append_tokens_kernel<DT, false, DSA_FP4_ROW_BYTES>);
}

hipError_t launch_append_tokens(const AppendArgs& A, int dtype, int row_bytes, hipStream_t s) {
  if (A.n <= 0) return hipSuccess;
  if (dtype == kF32) return launch_append_dt<kF32>(A, row_bytes, s);
  if (dtype == kBF16) return launch_append_dt<kBF16>(A, row_bytes, s);
  return launch_append_dt<kF16>(A, row_bytes, s);
}

// ---- reading rows back: a wave takes kReadRows rows, both in flight ----
//
// Bound by its bytes: 65536 rows of 400 bytes to 1152: 102 MB in 20.5 us (5.0
// TB/s, what a large copy reaches); 1, 4 and 8 rows a wave: 21.2, 21.5, 20.1.
// 777 rows of 656 bytes: 2.9 us, a launch and two trips to memory; 8 a wave: 3.8.
constexpr int kReadRows = 2;

template <int BYTES>
__global__ __launch_bounds__(kAppendThreads) void read_latent_kernel(const uint8_t* pool, long kv_rows, const int* slots,
                                                                      int n, uint16_t* out) {
  constexpr bool kFp8 = BYTES == DSA_LATENT_ROW_BYTES;
  const int lane = threadIdx.x & (kWave - 1);
  const long t0 = ((long)blockIdx.x * kAppendUnits + wave_id()) * kReadRows;
  uint2 code[kReadRows];
  float sc[kReadRows];
  uint4 rope[kReadRows];
#pragma unroll
  for (int k = 0; k < kReadRows; ++k) {
    code[k] = make_uint2(0, 0);
    sc[k] = 0.f;
    rope[k] = make_uint4(0, 0, 0, 0);
    const long slot = t0 + k < n ? slots[t0 + k] : -1;
    if (slot < 0 || slot >= kv_rows) continue;
    const uint8_t* src = pool + slot * BYTES;
    if constexpr (kFp8) {
      code[k] = *reinterpret_cast<const uint2*>(src + 8 * lane);
      sc[k] = reinterpret_cast<const float*>(src + DSA_LATENT_DIM)[lane >> 4];
    } else {
      code[k].x = reinterpret_cast<const uint32_t*>(src)[lane];
      sc[k] = __uint_as_float((uint32_t)src[DSA_LATENT_DIM / 2 + (lane >> 2)] << 23);
    }
    if (lane < DSA_ROPE_DIM / 8) rope[k] = *reinterpret_cast<const uint4*>(src + BYTES - 2 * DSA_ROPE_DIM + 16 * lane);
  }
#pragma unroll
  for (int k = 0; k < kReadRows; ++k) {
    if (t0 + k >= n) return;
    uint4 v;
    if constexpr (kFp8) {
      float f[8];
      e4m3x4_to_f32(code[k].x, f);
      e4m3x4_to_f32(code[k].y, f + 4);
      v = make_uint4(pack_bf16x2(f[0] * sc[k], f[1] * sc[k]), pack_bf16x2(f[2] * sc[k], f[3] * sc[k]),
                     pack_bf16x2(f[4] * sc[k], f[5] * sc[k]), pack_bf16x2(f[6] * sc[k], f[7] * sc[k]));
    } else {
      v = dequant8_fp4(code[k].x, sc[k]);
    }
    uint4* dst = reinterpret_cast<uint4*>(out + (t0 + k) * DSA_QK_DIM);
    dst[lane] = v;
    if (lane < DSA_ROPE_DIM / 8) dst[kWave + lane] = rope[k];
  }
}

hipError_t launch_read_latent(const void* pool, long kv_rows, int row_bytes, const int* slots, int n, void* out,
                              hipStream_t s) {
  if (n <= 0) return hipSuccess;
  constexpr int per = kAppendUnits * kReadRows;
  const auto kernel = row_bytes == DSA_LATENT_ROW_BYTES ? read_latent_kernel<DSA_LATENT_ROW_BYTES>
                                                        : read_latent_kernel<DSA_FP4_ROW_BYTES>;
  return in_launches(n, 1L << 26, [&](long at, long rows) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)((rows + per - 1) / per)), dim3(kAppendThreads), 0, s,
                       static_cast<const uint8_t*>(pool), kv_rows, slots + at, (int)rows,
                       static_cast<uint16_t*>(out) + at * DSA_QK_DIM);
    return hipGetLastError();
  });
}

}  // namespace dsa
