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
// off, depending on the order of the sum.
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

template <int DT, bool WIDE, int BYTES>
__device__ __forceinline__ void append_latent_row(const AppendArgs& A, int t, int pos, long slot) {
  const int lane = threadIdx.x & (kWave - 1);
  const long src = (long)t * A.latent_stride;
  float x[8];
  load8<DT, WIDE>(A.latent, src + 8 * lane, x);
  if (A.norm_w) {
    double ss = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = __builtin_fma((double)x[e], (double)x[e], ss);
    const double rs = 1.0 / sqrt(wave_sum64(ss) / DSA_LATENT_DIM + A.eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float w = A.norm_w_f32 ? load_elem<kF32>(A.norm_w, 8 * lane + e) : load_elem<DT>(A.norm_w, 8 * lane + e);
      x[e] = (float)((double)x[e] * rs * (double)w);
    }
  }
  uint8_t* dst = A.pool + slot * BYTES;
  if constexpr (BYTES == DSA_LATENT_ROW_BYTES) {
    const float scale = row_scale<true>(x);
    *reinterpret_cast<v2u_t*>(dst + 8 * lane) = quant8<true>(x, scale);
    if ((lane & 15) == 0) reinterpret_cast<float*>(dst + DSA_LATENT_DIM)[lane >> 4] = scale;
  } else {
    const uint32_t sb = fp4_scale_byte(x);
    reinterpret_cast<uint32_t*>(dst)[lane] = quant8_fp4(x, sb);
    if ((lane & 3) == 0) dst[DSA_LATENT_DIM / 2 + (lane >> 2)] = (uint8_t)sb;
  }
  if (lane < DSA_ROPE_DIM / 2) {
    constexpr int kHalf = DSA_ROPE_DIM / 2;
    uint16_t* rope = reinterpret_cast<uint16_t*>(dst + BYTES - 2 * DSA_ROPE_DIM);
    const int ia = A.interleaved ? 2 * lane : lane, ib = A.interleaved ? 2 * lane + 1 : lane + kHalf;
    const float a = load_elem<DT>(A.latent, src + DSA_LATENT_DIM + ia);
    const float b = load_elem<DT>(A.latent, src + DSA_LATENT_DIM + ib);
    float ya = a, yb = b;
    if (A.table) {
      const float c = A.table[(long)pos * DSA_ROPE_DIM + lane], s = A.table[(long)pos * DSA_ROPE_DIM + kHalf + lane];
      turn(a, b, c, s, ya, yb);
    }
    const uint32_t w = pack_bf16x2(ya, yb);
    if (A.interleaved) {
      reinterpret_cast<uint32_t*>(rope)[lane] = w;
    } else {
      rope[lane] = (uint16_t)w;
      rope[lane + kHalf] = (uint16_t)(w >> 16);
    }
  }
}

template <int DT, bool WIDE>
__device__ __forceinline__ void append_key(const AppendArgs& A, int t, int pos, long page) {
  const int i = threadIdx.x & 15;
  const long src = (long)t * A.keys_stride;
  float x[8];
  load8<DT, WIDE>(A.keys, src + 8 * i, x);
  if (A.table && i < DSA_ROPE_DIM / 8) {  // lanes 0-7 hold the rotated half
    constexpr int kHalf = DSA_ROPE_DIM / 2;
    const float* cs = A.table + (long)pos * DSA_ROPE_DIM;
    if (A.index_interleaved) {
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float c = cs[4 * i + p], s = cs[kHalf + 4 * i + p], a = x[2 * p], b = x[2 * p + 1];
        turn(a, b, c, s, x[2 * p], x[2 * p + 1]);
      }
    } else {  // the partner's 8 are lane i ^ 4's
      float o[8];
      load8<DT, WIDE>(A.keys, src + 8 * (i ^ 4), o);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float c = cs[8 * (i & 3) + e], s = cs[kHalf + 8 * (i & 3) + e];
        x[e] = __builtin_fmaf(o[e], i < 4 ? -s : s, x[e] * c);  // (turn, this lane's side)
      }
    }
  }
  const float scale = row_scale<true>(x);
  uint8_t* base = A.index_k + page * DSA_INDEX_PAGE_BYTES;
  const int slot = pos % DSA_PAGE_TOKENS;
  *reinterpret_cast<v2u_t*>(base + slot * DSA_INDEX_DIM + 8 * i) = quant8<true>(x, scale);
  if (i == 0) reinterpret_cast<float*>(base + DSA_PAGE_TOKENS * DSA_INDEX_DIM)[slot] = scale;
}

// Waves 0 .. n - 1: a latent row each (when there is a latent); those behind:
// four index keys each.
template <int DT, bool WIDE, int BYTES>
__global__ __launch_bounds__(kAppendThreads) void append_tokens_kernel(const AppendArgs A) {
  const long unit = (long)blockIdx.x * kAppendUnits + wave_id();
  const long n_lat = A.latent ? A.n : 0;
  const int lane = threadIdx.x & (kWave - 1);
  const long at = unit < n_lat ? unit : 4 * (unit - n_lat) + (lane >> 4);
  if (at >= A.n) return;
  const int t = (int)at, r = A.rows[t], pos = A.pos[t];
  // a token without a request, a page or a table row is skipped
  if (r < 0 || r >= A.B || pos < 0 || pos / DSA_PAGE_TOKENS >= A.pt_stride || (A.table && pos >= A.table_rows)) return;
  const long page = A.page_table[(long)r * A.pt_stride + pos / DSA_PAGE_TOKENS];
  if (page < 0) return;
  if (unit < n_lat) {
    const long slot = page * DSA_PAGE_TOKENS + pos % DSA_PAGE_TOKENS;
    if (slot < A.kv_rows) append_latent_row<DT, WIDE, BYTES>(A, t, pos, slot);
  } else if (page < A.num_pages) {
    append_key<DT, WIDE>(A, t, pos, page);
  }
}

template <int DT>
static hipError_t launch_append_dt(const AppendArgs& A, int row_bytes, hipStream_t s) {
  constexpr int es = DT == kF32 ? 4 : 2;
  const auto on16 = [](const void* p, long stride) { return (((uintptr_t)p | (uintptr_t)(stride * es)) & 15) == 0; };
  const bool wide = (!A.latent || on16(A.latent, A.latent_stride)) && (!A.keys || on16(A.keys, A.keys_stride));
  const long units = (A.latent ? A.n : 0) + (A.keys ? (A.n + 3L) / 4 : 0);
  const dim3 grid((unsigned)((units + kAppendUnits - 1) / kAppendUnits));
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kAppendThreads), 0, s, A);
    return hipGetLastError();
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

// ---- reading rows back: one wave a row ----

template <int BYTES>
__global__ __launch_bounds__(kAppendThreads) void read_latent_kernel(const uint8_t* pool, long kv_rows, const int* slots,
                                                                      int n, uint16_t* out) {
  const int t = blockIdx.x * kAppendUnits + wave_id(), lane = threadIdx.x & (kWave - 1);
  if (t >= n) return;
  const long slot = slots[t];
  uint4* dst = reinterpret_cast<uint4*>(out + (long)t * DSA_QK_DIM);
  const bool ok = slot >= 0 && slot < kv_rows;
  const uint8_t* src = pool + (ok ? slot : 0) * BYTES;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (ok) {
    if constexpr (BYTES == DSA_LATENT_ROW_BYTES) {
      const v2u_t c = *reinterpret_cast<const v2u_t*>(src + 8 * lane);
      const float sc = reinterpret_cast<const float*>(src + DSA_LATENT_DIM)[lane >> 4];
      float f[8];
      e4m3x4_to_f32(c[0], f);
      e4m3x4_to_f32(c[1], f + 4);
      v = make_uint4(pack_bf16x2(f[0] * sc, f[1] * sc), pack_bf16x2(f[2] * sc, f[3] * sc),
                     pack_bf16x2(f[4] * sc, f[5] * sc), pack_bf16x2(f[6] * sc, f[7] * sc));
    } else {
      v = dequant8_fp4(reinterpret_cast<const uint32_t*>(src)[lane],
                       __uint_as_float((uint32_t)src[DSA_LATENT_DIM / 2 + (lane >> 2)] << 23));
    }
  }
  dst[lane] = v;
  if (lane < DSA_ROPE_DIM / 8)
    dst[kWave + lane] = ok ? *reinterpret_cast<const uint4*>(src + BYTES - 2 * DSA_ROPE_DIM + 16 * lane) : make_uint4(0, 0, 0, 0);
}

hipError_t launch_read_latent(const void* pool, long kv_rows, int row_bytes, const int* slots, int n, void* out,
                              hipStream_t s) {
  if (n <= 0) return hipSuccess;
  const dim3 grid((unsigned)((n + kAppendUnits - 1) / kAppendUnits));
  const uint8_t* p = static_cast<const uint8_t*>(pool);
  uint16_t* o = static_cast<uint16_t*>(out);
  if (row_bytes == DSA_LATENT_ROW_BYTES)
    hipLaunchKernelGGL(read_latent_kernel<DSA_LATENT_ROW_BYTES>, grid, dim3(kAppendThreads), 0, s, p, kv_rows, slots, n, o);
  else
    hipLaunchKernelGGL(read_latent_kernel<DSA_FP4_ROW_BYTES>, grid, dim3(kAppendThreads), 0, s, p, kv_rows, slots, n, o);
  return hipGetLastError();
}

}  // namespace dsa
