// RMS norm with the residual's addition, and rotary positions (gfx950).
//
//   h = x + r,  y = h / sqrt(mean(h^2) + eps) * w        (all in fp32)
//
// h is stored rounded to the input's type; the norm reads the unrounded sum.
// y leaves in the input's type, or as e4m3 by quant_core.h's rule with one
// scale per 128 values or per row (a NaN in a group makes its scale and its
// codes NaN).
//
//   rotary: (a, b) -> (a c - b s, b c + a s) with c, s of the token's position;
//   a, b = elements i, i + R/2 (half) or 2i, 2i + 1 (interleaved); the
//   inverse turns by -s, which is also the operation's adjoint.
#include <algorithm>

#include "dsa_kernels.h"
#include "quant_core.h"

namespace dsa {

// sum over the wave, the same value in every lane
__device__ __forceinline__ float wave_sum(float v) {
  const auto sh = [](auto ctrl, auto rows, float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, decltype(rows)::value,
                                                      0xf, false));
  };
  using All = std::integral_constant<int, 0xf>;
  v += sh(std::integral_constant<int, 0x111>{}, All{}, v);
  v += sh(std::integral_constant<int, 0x112>{}, All{}, v);
  v += sh(std::integral_constant<int, 0x114>{}, All{}, v);
  v += sh(std::integral_constant<int, 0x118>{}, All{}, v);
  v += sh(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{}, v);
  v += sh(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{}, v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// sum over 16 lanes, the same value in each
__device__ __forceinline__ float sum16(float v) {
  const auto sh = [](auto ctrl, float x) { return __uint_as_float(dpp_u32<decltype(ctrl)::value, 0xf>(__float_as_uint(x), 0u)); };
  v += sh(std::integral_constant<int, 0x121>{}, v);
  v += sh(std::integral_constant<int, 0x122>{}, v);
  v += sh(std::integral_constant<int, 0x124>{}, v);
  return v + sh(std::integral_constant<int, 0x128>{}, v);
}

// V vectors of 8 elements a lane, as they come from memory.
template <int DT, int V>
struct RawRow {
  uint4 v[V][DT == kF32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ void unpack8(const uint4* v, float* x) {
  if constexpr (DT == kF32) {
    const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(w[e]);
  } else {
    const uint32_t w[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == kBF16) {
        x[2 * e] = bf16_lo(w[e]);
        x[2 * e + 1] = bf16_hi(w[e]);
      } else {
        x[2 * e] = (float)__builtin_bit_cast(_Float16, (uint16_t)w[e]);
        x[2 * e + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e] >> 16));
      }
    }
  }
}
// Row `p`'s vectors of thread t of T (zeros past D).  WIDE: on 16-byte
// boundaries and whole; otherwise the loads are as wide, but may lie across a
// boundary (global memory allows that), and the last vector comes one by one.
template <int DT, int V, bool WIDE>
__device__ __forceinline__ void load_raw(const void* p, int t, int T, int D, RawRow<DT, V>& r) {
  constexpr int es = DT == kF32 ? 4 : 2, k = DT == kF32 ? 2 : 1;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = 8 * (v * T + t);
    const uint8_t* at = static_cast<const uint8_t*>(p) + (long)i * es;
    if (WIDE ? i < D : i + 8 <= D) {
      if constexpr (WIDE) {
#pragma unroll
        for (int c = 0; c < k; ++c) r.v[v][c] = reinterpret_cast<const uint4*>(at)[c];
      } else {
        __builtin_memcpy(r.v[v], __builtin_assume_aligned(at, es), 16 * k);
      }
      continue;
    }
#pragma unroll
    for (int c = 0; c < k; ++c) r.v[v][c] = make_uint4(0, 0, 0, 0);
    if constexpr (!WIDE) {
      uint32_t w[4 * k] = {};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i + e < D) {
          if constexpr (DT == kF32) w[e] = reinterpret_cast<const uint32_t*>(at)[e];
          else w[e >> 1] |= (uint32_t)reinterpret_cast<const uint16_t*>(at)[e] << (16 * (e & 1));
        }
#pragma unroll
      for (int c = 0; c < k; ++c) r.v[v][c] = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
    }
  }
}
// Elements i .. i + 7, all there; and those of a row of D that are to be stored.
template <int DT, bool WIDE>
__device__ __forceinline__ void load_row8(const void* p, int i, float* x) {
  constexpr int es = DT == kF32 ? 4 : 2;
  if constexpr (WIDE) {
    load8<DT>(p, i, x);
  } else {
    uint4 w[DT == kF32 ? 2 : 1];
    __builtin_memcpy(w, __builtin_assume_aligned(static_cast<const uint8_t*>(p) + (long)i * es, es), sizeof(w));
    load8<DT>(w, 0, x);
  }
}
template <int DT, bool WIDE>
__device__ __forceinline__ void store_row8(void* p, long row, int i, const float* x, int D) {
  if (WIDE || i + 8 > D) {
    store8<DT, WIDE>(p, row + i, x, row + D);
    return;
  }
  constexpr int es = DT == kF32 ? 4 : 2;
  uint4 w[DT == kF32 ? 2 : 1];
  store8<DT, true>(w, 0, x, 0);
  __builtin_memcpy(__builtin_assume_aligned(static_cast<uint8_t*>(p) + (row + i) * es, es), w, sizeof(w));
}

// A workgroup of T threads holds a row, V vectors of 8 elements each (vector v
// of thread t: elements 8 (v T + t) ..); the 16 lanes of a DPP row hold 128
// consecutive elements, one quantisation group.  WIDE: D a multiple of 8 and
// every row on 16-byte boundaries.  Workgroups go on to further rows, with the
// weight in registers and the next row in flight from before the reduction on.
//
// Bound by its bytes: 8191 rows of 7168 bf16 with a residual, to e4m3 with a
// scale per 128 values, move 412 MB in 79 us, 5.2 TB/s (as a large copy).  A row
// a workgroup, the weight read again for each: 195 us.  Without the residual the
// quantiser's arithmetic is next (42 us for 176 MB).  With a scale
// per row: 79 and 44.  Rows of 3001 values, which begin between boundaries: 4096
// of bf16 with a residual 25 us, of 3000 16 us: the same bytes from memory (both
// ways within 1 %), but 2.5 times the accesses to the L1 by loads and stores that
// lie across a boundary; value by value they took 62.  One token: 2.7 us, a launch
// and two trips to memory.
constexpr int kNormWaves = 16;  // most waves a row

template <int DT, int V, bool WIDE>
__global__ __launch_bounds__(kNormWaves* kWave) void rms_norm_kernel(const NormArgs A) {
  constexpr int es = DT == kF32 ? 4 : 2;
  __shared__ float red[2][kNormWaves];
  __shared__ uint32_t redm[2][kNormWaves];
  const int T = (int)blockDim.x, waves = T / kWave, t = (int)threadIdx.x, D = A.D, wv = wave_id();
  const float inv_d = 1.f / (float)D;
  if (t >= waves && t < kNormWaves) red[0][t] = red[1][t] = 0.f, redm[0][t] = redm[1][t] = 0;
  long row = blockIdx.x;
  const auto at = [&](const void* p, long r, long rs) { return static_cast<const uint8_t*>(p) + r * rs * es; };
  // four vectors of the next row do not fit beside this one's: 2000 x 18432 bf16
  // with a residual took 66 us with them (spilled), 52 without, fp32 176 and 118
  constexpr bool kAhead = V < 4;
  RawRow<DT, V> x, r;
  const auto load = [&](long row) {
    load_raw<DT, V, WIDE>(at(A.x, row, A.xs), t, T, D, x);
    if (A.r) load_raw<DT, V, WIDE>(at(A.r, row, A.rs), t, T, D, r);
  };
  if (kAhead) load(row);
  float w[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = 8 * (v * T + t);
    if (i + 8 <= D) {
      if (A.w_f32) load_row8<kF32, WIDE>(A.w, i, w[v]);
      else load_row8<DT, WIDE>(A.w, i, w[v]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        w[v][e] = i + e >= D ? 0.f : A.w_f32 ? load_elem<kF32>(A.w, i + e) : load_elem<DT>(A.w, i + e);
    }
  }
  for (int par = 0; row < A.n; row += gridDim.x, par ^= 1) {
    if (!kAhead) load(row);
    float h[V][8];
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = 8 * (v * T + t);
      unpack8<DT>(x.v[v], h[v]);
      if (A.r) {
        float f[8];
        unpack8<DT>(r.v[v], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[v][e] += f[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(h[v][e], h[v][e], ss);
      if (A.h && i < D) store_row8<DT, WIDE>(A.h, row * A.hs, i, h[v], D);
    }
    if (kAhead && row + gridDim.x < A.n) load(row + gridDim.x);
    ss = wave_sum(ss);
    if (waves > 1) {
      if ((t & (kWave - 1)) == 0) red[par][wv] = ss;
      __syncthreads();
      ss = sum16(red[par][t & (kNormWaves - 1)]);
    }
    const float rs = rsqrtf(ss * inv_d + A.eps);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[v][e] = h[v][e] * rs * w[v][e];
    if (A.y) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = 8 * (v * T + t);
        if (i < D) store_row8<DT, WIDE>(A.y, row * D, i, h[v], D);
      }
      continue;
    }
    uint32_t am = 0;
    if (A.group == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) am = max(am, amax_bits<true>(h[v]));
      am = wave_reduce<2>(am);
      if (waves > 1) {
        if ((t & (kWave - 1)) == 0) redm[par][wv] = am;
        __syncthreads();
        am = row16_max(redm[par][t & (kNormWaves - 1)]);
      }
    }
    const int groups = A.group ? (D + 127) / 128 : 1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = 8 * (v * T + t);
      const float sc = A.group ? row_scale<true>(h[v]) : scale_of_amax(am);
      const v2u_t c = quant8<true>(h[v], sc);
      if (i >= D) continue;
      uint8_t* dst = A.codes + row * D + i;
      if constexpr (WIDE) {
        *reinterpret_cast<v2u_t*>(dst) = c;
      } else if (i + 8 <= D) {
        __builtin_memcpy(dst, &c, 8);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < D) dst[e] = (uint8_t)(c[e >> 2] >> (8 * (e & 3)));
      }
      if (A.group ? (i & 127) == 0 : i == 0) A.scales[row * groups + (A.group ? i / 128 : 0)] = sc;
    }
  }
}

template <int DT, int V>
static hipError_t launch_norm(const NormArgs& A, bool wide, hipStream_t s) {
  const int vecs = (A.D + 7) / 8;
  const int threads = ((vecs + V - 1) / V + kWave - 1) / kWave * kWave;
  const long most = (long)device_cu_count() * (2048 / threads);  // what is resident at once
  const auto kernel = wide ? rms_norm_kernel<DT, V, true> : rms_norm_kernel<DT, V, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)std::min((long)A.n, most)), dim3(threads), 0, s, A);
  return hipGetLastError();
}

template <int DT>
static hipError_t launch_norm_dim(const NormArgs& A, hipStream_t s) {
  constexpr int es = DT == kF32 ? 4 : 2;
  const auto on16 = [](const void* p, long stride) { return (((uintptr_t)p | (uintptr_t)(stride * es)) & 15) == 0; };
  const bool wide = A.D % 8 == 0 && on16(A.x, A.xs) && (!A.r || on16(A.r, A.rs)) && (!A.h || on16(A.h, A.hs)) &&
                    (!A.y || on16(A.y, 0)) && ((uintptr_t)A.codes & 7) == 0 && on16(A.w, 0);
  // the fewest vectors a thread that 1024 threads allow, but two where the
  // quantiser's arithmetic bounds the row (8191 x 7168 bf16: 42.5 us, in one
  // vector 47.7; 4096 x 3000: 12.7 and 13.1; 8191 x 1536: 13.8 and 12.4; not
  // quantised: 40.1 and 37.6).  In four, without the next row: 42.2 and 39.1.
  if (A.D <= 8192 && (!A.codes || DT == kF32 || A.D <= 2048)) return launch_norm<DT, 1>(A, wide, s);
  if (A.D <= 16384) return launch_norm<DT, 2>(A, wide, s);
  return launch_norm<DT, 4>(A, wide, s);
}

hipError_t launch_rms_norm(const NormArgs& A, int dtype, hipStream_t s) {
  if (A.n <= 0) return hipSuccess;
  if (dtype == kF32) return launch_norm_dim<kF32>(A, s);
  if (dtype == kBF16) return launch_norm_dim<kBF16>(A, s);
  return launch_norm_dim<kF16>(A, s);
}

// ---- rotary positions ----

// One item of a head: WIDE a vector of 8 elements of the rotated part (half:
// and its partners R/2 on), otherwise a pair; behind them, where the output
// is another tensor, the elements outside the rotated part (vectors of 8, or
// one by one).  A thread keeps its item and goes through heads, kRopeBatch at
// a time, so that the table is read once for all of them and several loads
// are in flight.
//
// Bound by its bytes: 64 values of each of 128 heads of 4097 tokens, 384 bytes
// apart on the way in, take 32 us for 134 MB (4.2 TB/s); in place 27, with the
// other 128 values copied 79 (403 MB, 5.1 TB/s); halves as pairs 30 and 86.  One item a thread,
// the table read again for every head: 44 us; batches of 1, 2 and 8 heads:
// 33.0, 32.4 and 32.6.  32 tokens of 16 heads: 3.1 us, a launch and its latency.
constexpr int kRopeThreads = 256, kRopeBatch = 4;

template <int DT, bool WIDE, bool INTER>
__global__ __launch_bounds__(kRopeThreads) void rotary_kernel(const RopeArgs A) {
  const int rot_items = WIDE ? A.R / (INTER ? 8 : 16) : A.R / 2;
  const int items = rot_items + (A.copy ? (A.D - A.R) / (WIDE ? 8 : 1) : 0);
  const int per = items * A.heads;  // threads a token (items of as many heads)
  const int lt = per < kRopeThreads ? (int)threadIdx.x / per : 0;
  const int tid = (int)threadIdx.x - lt * per;
  const long token = (long)blockIdx.x * A.tokens + lt;
  if (lt >= A.tokens || token >= A.n) return;
  const long pos = A.pos64 ? static_cast<const int64_t*>(A.pos)[token] : (long)static_cast<const int32_t*>(A.pos)[token];
  const bool in = pos >= 0 && pos < A.max_pos;
  if (!in && !A.copy) return;
  const float* cs = A.table + (in ? pos : 0) * A.R;
  const float sign = A.inverse ? -1.f : 1.f;
  const int hr = A.R / 2, h0 = tid / items + (int)blockIdx.y * A.heads, hstep = (int)gridDim.y * A.heads;
  for (int it = tid % items; it < items; it += kRopeThreads) {  // (one pass unless a head has more items)
    const bool turned = it < rot_items;
    constexpr int kC = WIDE ? (INTER ? 4 : 8) : 1, kE = WIDE ? 8 : 1, kPart = (INTER && WIDE) ? 1 : 2;
    int d = WIDE ? 8 * it : INTER ? 2 * it : it;
    if (turned) {
      d += A.start;
    } else {
      d = (it - rot_items) * kE;
      d += d >= A.start ? A.R : 0;
    }
    const int d2 = d + (WIDE || !INTER ? hr : 1);  // the partners (kPart == 2)
    float c[kC], sn[kC];
#pragma unroll
    for (int k = 0; k < kC; ++k) c[k] = 1.f, sn[k] = 0.f;
    if (turned && in) {
      if constexpr (WIDE) {
#pragma unroll
        for (int k = 0; k < kC; k += 4) {
          const v4f a = *reinterpret_cast<const v4f*>(cs + kC * it + k);
          const v4f b = *reinterpret_cast<const v4f*>(cs + hr + kC * it + k);
#pragma unroll
          for (int e = 0; e < 4; ++e) c[k + e] = a[e], sn[k + e] = sign * b[e];
        }
      } else {
        c[0] = cs[it], sn[0] = sign * cs[hr + it];
      }
    }
    for (int hb = h0; hb < A.H; hb += hstep * kRopeBatch) {
      float x[kRopeBatch][kPart][kE];
#pragma unroll
      for (int k = 0; k < kRopeBatch; ++k) {
        const int h = hb + k * hstep;
        if (h >= A.H) break;
        const long xi = token * A.xn + h * A.xh;
        if constexpr (WIDE) {
          load8<DT>(A.x, xi + d, x[k][0]);
          if constexpr (kPart == 2)
            if (turned) load8<DT>(A.x, xi + d2, x[k][1]);
        } else {
          x[k][0][0] = load_elem<DT>(A.x, xi + d);
          if (turned) x[k][1][0] = load_elem<DT>(A.x, xi + d2);
        }
      }
#pragma unroll
      for (int k = 0; k < kRopeBatch; ++k) {
        const int h = hb + k * hstep;
        if (h >= A.H) break;
        const long oi = token * A.on + h * A.oh;
        if (turned && in) {
          if constexpr (kPart == 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) turn(x[k][0][2 * e], x[k][0][2 * e + 1], c[e], sn[e], x[k][0][2 * e], x[k][0][2 * e + 1]);
          } else {
#pragma unroll
            for (int e = 0; e < kE; ++e) turn(x[k][0][e], x[k][1][e], c[e], sn[e], x[k][0][e], x[k][1][e]);
          }
        }
        if constexpr (WIDE) {
          store8<DT, true>(A.out, oi + d, x[k][0], 0);
          if constexpr (kPart == 2)
            if (turned) store8<DT, true>(A.out, oi + d2, x[k][1], 0);
        } else {
          store8<DT, false>(A.out, oi + d, x[k][0], oi + d + 1);
          if (turned) store8<DT, false>(A.out, oi + d2, x[k][1], oi + d2 + 1);
        }
      }
    }
  }
}

template <int DT>
static hipError_t launch_rotary_dt(RopeArgs A, hipStream_t s) {
  constexpr int es = DT == kF32 ? 4 : 2;
  const uintptr_t strides = (uintptr_t)((A.xn | A.xh | A.on | A.oh) * es);
  const bool wide = A.R % (A.interleaved ? 8 : 16) == 0 && A.start % 8 == 0 && (!A.copy || A.D % 8 == 0) &&
                    (((uintptr_t)A.x | (uintptr_t)A.out | (uintptr_t)A.table | strides) & 15) == 0;
  const int items = (wide ? A.R / (A.interleaved ? 8 : 16) : A.R / 2) + (A.copy ? (A.D - A.R) / (wide ? 8 : 1) : 0);
  // a workgroup: as many heads of a token as fit, then as many tokens
  A.heads = items >= kRopeThreads ? 1 : std::min(A.H, kRopeThreads / items);
  A.tokens = std::max(1, kRopeThreads / (A.heads * items));
  const auto blocks = [&](long n) { return (n + A.tokens - 1) / A.tokens; };
  // few tokens: their heads over several workgroups (a token of 128 heads of
  // 192 values: 3.4 us; in one workgroup 6.3)
  const int turns = (A.H + A.heads - 1) / A.heads;
  const int y = (int)std::max(1L, std::min({(long)turns, 65535L, 2L * device_cu_count() / blocks(A.n)}));
  const auto kernel = A.interleaved ? (wide ? rotary_kernel<DT, true, true> : rotary_kernel<DT, false, true>)
                                    : (wide ? rotary_kernel<DT, true, false> : rotary_kernel<DT, false, false>);
  constexpr long kMostBlocks = (1L << 31) / kRopeThreads;
  return in_launches(A.n, kMostBlocks * A.tokens, [&](long at, long n) {
    RopeArgs P = A;
    P.x = static_cast<const uint8_t*>(A.x) + at * A.xn * es;
    P.out = static_cast<uint8_t*>(A.out) + at * A.on * es;
    P.pos = static_cast<const uint8_t*>(A.pos) + at * (A.pos64 ? 8 : 4);
    P.n = (int)n;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks(n), (unsigned)y), dim3(kRopeThreads), 0, s, P);
    return hipGetLastError();
  });
}

hipError_t launch_rotary(const RopeArgs& A, int dtype, hipStream_t s) {
  if (A.n <= 0 || A.H <= 0) return hipSuccess;
  if (dtype == kF32) return launch_rotary_dt<kF32>(A, s);
  if (dtype == kBF16) return launch_rotary_dt<kBF16>(A, s);
  return launch_rotary_dt<kF16>(A, s);
}

}  // namespace dsa
