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

// A row is held by T threads, V vectors of 8 elements each (vector v of
// thread t: elements 8 (v T + t) ..); the 16 lanes of a DPP row hold 128
// consecutive elements, one quantisation group.  WIDE: D a multiple of 8 and
// every row on 16-byte boundaries.
template <int DT, int T, int V, bool WIDE>
__global__ __launch_bounds__(T < 256 ? 256 : T) void rms_norm_kernel(const NormArgs A) {
  constexpr int kBlock = T < 256 ? 256 : T, kRows = kBlock / T, kWaves = T / kWave;
  __shared__ float red[2][kWaves];
  __shared__ uint32_t redm[2][kWaves];
  const int t = threadIdx.x % T, D = A.D, wv = t / kWave;
  float w[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = 8 * (v * T + t) + e;
      w[v][e] = i >= D ? 0.f : A.w_f32 ? load_elem<kF32>(A.w, i) : load_elem<DT>(A.w, i);
    }
  int par = 0;
  for (long row = (long)blockIdx.x * kRows + threadIdx.x / T; row < A.n; row += (long)gridDim.x * kRows, par ^= 1) {
    float h[V][8];
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = 8 * (v * T + t);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[v][e] = 0.f;
      if constexpr (WIDE) {
        if (i < D) {
          load8<DT>(A.x, row * A.xs + i, h[v]);
          if (A.r) {
            float r[8];
            load8<DT>(A.r, row * A.rs + i, r);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[v][e] += r[e];
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < D) {
            h[v][e] = load_elem<DT>(A.x, row * A.xs + i + e);
            if (A.r) h[v][e] += load_elem<DT>(A.r, row * A.rs + i + e);
          }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(h[v][e], h[v][e], ss);
      if (A.h && (!WIDE || i < D)) store8<DT, WIDE>(A.h, row * A.hs + i, h[v], row * A.hs + D);
    }
    ss = wave_sum(ss);
    if constexpr (kWaves > 1) {
      if ((t & (kWave - 1)) == 0) red[par][wv] = ss;
      __syncthreads();
      ss = 0.f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) ss += red[par][k];
    }
    const float rs = 1.f / sqrtf(ss / (float)D + A.eps);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[v][e] = h[v][e] * rs * w[v][e];
    if (A.y) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int i = 8 * (v * T + t);
        if (!WIDE || i < D) store8<DT, WIDE>(A.y, row * D + i, h[v], row * D + D);
      }
      continue;
    }
    uint32_t am = 0;
    if (A.group == 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) am = max(am, amax_bits<true>(h[v]));
      am = wave_reduce<2>(am);
      if constexpr (kWaves > 1) {
        if ((t & (kWave - 1)) == 0) redm[par][wv] = am;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kWaves; ++k) am = max(am, redm[par][k]);
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
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (i + e < D) dst[e] = (uint8_t)(c[e >> 2] >> (8 * (e & 3)));
      }
      if (A.group ? (i & 127) == 0 : i == 0) A.scales[row * groups + (A.group ? i / 128 : 0)] = sc;
    }
  }
}

template <int DT, int T, int V>
static hipError_t launch_norm(const NormArgs& A, bool wide, hipStream_t s) {
  constexpr int kBlock = T < 256 ? 256 : T, kRows = kBlock / T;
  const long blocks = ((long)A.n + kRows - 1) / kRows;
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
  const auto kernel = wide ? rms_norm_kernel<DT, T, V, true> : rms_norm_kernel<DT, T, V, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(kBlock), 0, s, A);
  return hipGetLastError();
}

template <int DT>
static hipError_t launch_norm_dim(const NormArgs& A, hipStream_t s) {
  constexpr int es = DT == kF32 ? 4 : 2;
  const auto on16 = [](const void* p, long stride) { return (((uintptr_t)p | (uintptr_t)(stride * es)) & 15) == 0; };
  const bool wide = A.D % 8 == 0 && on16(A.x, A.xs) && (!A.r || on16(A.r, A.rs)) && (!A.h || on16(A.h, A.hs)) &&
                    (!A.y || on16(A.y, 0)) && ((uintptr_t)A.codes & 7) == 0;
  if (A.D <= 512) return launch_norm<DT, 64, 1>(A, wide, s);
  if (A.D <= 1024) return launch_norm<DT, 64, 2>(A, wide, s);
  if (A.D <= 2048) return launch_norm<DT, 256, 1>(A, wide, s);
  if (A.D <= 4096) return launch_norm<DT, 256, 2>(A, wide, s);
  if (A.D <= 8192) return launch_norm<DT, 256, 4>(A, wide, s);
  if (A.D <= 16384) return launch_norm<DT, 1024, 2>(A, wide, s);
  return launch_norm<DT, 1024, 4>(A, wide, s);
}

hipError_t launch_rms_norm(const NormArgs& A, int dtype, hipStream_t s) {
  if (A.n <= 0) return hipSuccess;
  if (dtype == kF32) return launch_norm_dim<kF32>(A, s);
  if (dtype == kBF16) return launch_norm_dim<kBF16>(A, s);
  return launch_norm_dim<kF16>(A, s);
}

// ---- rotary positions ----

// One item: WIDE a vector of 8 elements (of a half: and its partners R/2
// on), otherwise a pair; behind them, where the output is another tensor,
// the elements outside the rotated part (vectors of 8, or one by one).
// A workgroup takes whole tokens, so that a thread's table entries serve all
// its heads (kRopeThreads is a multiple of the items of every width that is
// a power of two).
constexpr int kRopeThreads = 256;

template <int DT, bool WIDE, bool INTER>
__global__ __launch_bounds__(kRopeThreads) void rotary_kernel(const RopeArgs A) {
  const int rot_items = WIDE ? A.R / (INTER ? 8 : 16) : A.R / 2;
  const int items = rot_items + (A.copy ? (A.D - A.R) / (WIDE ? 8 : 1) : 0);
  const int per = A.H * items;                                  // items a token
  const int tok = per < kRopeThreads ? kRopeThreads / per : 1;  // tokens a workgroup
  const int lt = per < kRopeThreads ? (int)threadIdx.x / per : 0;
  const long token = (long)blockIdx.x * tok + lt;
  if (lt >= tok || token >= A.n) return;
  const long pos = A.pos64 ? static_cast<const int64_t*>(A.pos)[token] : (long)static_cast<const int32_t*>(A.pos)[token];
  const bool in = pos >= 0 && pos < A.max_pos;
  const float* cs = A.table + (in ? pos : 0) * A.R;
  const float sign = A.inverse ? -1.f : 1.f;
  const int hr = A.R / 2;
  for (int j = (int)threadIdx.x - lt * per; j < per; j += kRopeThreads) {
    const int head = j / items, it = j - head * items;
    const long xi = token * A.xn + head * A.xh, oi = token * A.on + head * A.oh;
    if (it >= rot_items) {  // outside the rotated part
      int d = (it - rot_items) * (WIDE ? 8 : 1);
      d += d >= A.start ? A.R : 0;
      if constexpr (WIDE) {
        float x[8];
        load8<DT>(A.x, xi + d, x);
        store8<DT, true>(A.out, oi + d, x, 0);
      } else {
        if constexpr (DT == kF32) static_cast<float*>(A.out)[oi + d] = static_cast<const float*>(A.x)[xi + d];
        else static_cast<uint16_t*>(A.out)[oi + d] = static_cast<const uint16_t*>(A.x)[xi + d];
      }
      continue;
    }
    if (!in && !A.copy) return;
    if constexpr (WIDE && INTER) {
      const int d = A.start + 8 * it;
      float x[8], y[8];
      load8<DT>(A.x, xi + d, x);
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float c = in ? cs[4 * it + p] : 1.f, sn = in ? sign * cs[hr + 4 * it + p] : 0.f;
        turn(x[2 * p], x[2 * p + 1], c, sn, y[2 * p], y[2 * p + 1]);
      }
      store8<DT, true>(A.out, oi + d, in ? y : x, 0);
    } else if constexpr (WIDE) {
      const int d = A.start + 8 * it;
      float a[8], b[8], ya[8], yb[8];
      load8<DT>(A.x, xi + d, a);
      load8<DT>(A.x, xi + d + hr, b);
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float c = in ? cs[8 * it + p] : 1.f, sn = in ? sign * cs[hr + 8 * it + p] : 0.f;
        turn(a[p], b[p], c, sn, ya[p], yb[p]);
      }
      store8<DT, true>(A.out, oi + d, in ? ya : a, 0);
      store8<DT, true>(A.out, oi + d + hr, in ? yb : b, 0);
    } else {
      const int da = A.start + (INTER ? 2 * it : it), db = INTER ? da + 1 : da + hr;
      const float a = load_elem<DT>(A.x, xi + da), b = load_elem<DT>(A.x, xi + db);
      const float c = in ? cs[it] : 1.f, sn = in ? sign * cs[hr + it] : 0.f;
      float ya[8], yb[8];
      turn(a, b, c, sn, ya[0], yb[0]);
      if (!in) ya[0] = a, yb[0] = b;
      store8<DT, false>(A.out, oi + da, ya, oi + da + 1);
      store8<DT, false>(A.out, oi + db, yb, oi + db + 1);
    }
  }
}

template <int DT>
static hipError_t launch_rotary_dt(const RopeArgs& A, hipStream_t s) {
  constexpr int es = DT == kF32 ? 4 : 2;
  const uintptr_t strides = (uintptr_t)((A.xn | A.xh | A.on | A.oh) * es);
  const bool wide = A.R % (A.interleaved ? 8 : 16) == 0 && A.start % 8 == 0 && (!A.copy || A.D % 8 == 0) &&
                    (((uintptr_t)A.x | (uintptr_t)A.out | strides) & 15) == 0;
  const int items = (wide ? A.R / (A.interleaved ? 8 : 16) : A.R / 2) + (A.copy ? (A.D - A.R) / (wide ? 8 : 1) : 0);
  const long per = (long)A.H * items;
  const int tok = per < kRopeThreads ? (int)(kRopeThreads / per) : 1;
  const dim3 grid((unsigned)(((long)A.n + tok - 1) / tok));
  const auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(kRopeThreads), 0, s, A);
    return hipGetLastError();
  };
  if (A.interleaved) return wide ? go(rotary_kernel<DT, true, true>) : go(rotary_kernel<DT, false, true>);
  return wide ? go(rotary_kernel<DT, true, false>) : go(rotary_kernel<DT, false, false>);
}

hipError_t launch_rotary(const RopeArgs& A, int dtype, hipStream_t s) {
  if (A.n <= 0 || A.H <= 0) return hipSuccess;
  if (dtype == kF32) return launch_rotary_dt<kF32>(A, s);
  if (dtype == kBF16) return launch_rotary_dt<kBF16>(A, s);
  return launch_rotary_dt<kF16>(A, s);
}

}  // namespace dsa
