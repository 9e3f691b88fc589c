// Rows to e4m3 with a scale per 128 values or per row (gfx950): the operands
// of an 8-bit product that no norm makes.
//
//   y = x, or x * g / (1 + e^-g)          (in fp32)
//   scale = max(amax |y|, 1e-6) / 448,  code = e4m3_rne(y / scale)
//
// quant_core.h's rule: a NaN among a group's values makes its scale and its
// codes NaN.  Reference: inference/modeling/kernels.py:35-117.
//
// Bound by memory: 16 lanes hold a group of 128 (8 values each, one load), whose
// maximum is four steps across the lanes, and a workgroup's 16 groups are one
// contiguous piece.  Gated rows, 380 MB read and written, take 79 us (4.8 TB/s, a
// large copy's rate; 74 with one scale a row); a token 9 us, a launch and its wait
// for memory.
#include "dsa_kernels.h"
#include "quant_core.h"

namespace dsa {

constexpr int kQrThreads = 256;

// x * g * sigmoid(g).  e^-g by 2^n 2^f with f from two terms of log2 e, so
// that the argument's rounding does not grow with |g|; the quotient corrected
// once by its exact remainder.  Of 75 million codes 141 to 145 are on the wrong
// side of a border, 130 to 150 where y is a 64-bit silu rounded to fp32; two
// floats up to the product, with the exponential by its series, make that 117 to
// 132 and take a fifth longer.
constexpr float kHi = 1.44269502f, kLo = 1.92596299e-8f;  // log2 e in two floats
__device__ __forceinline__ float silu_times(float g, float x) {
  const float n = fminf(fmaxf(rintf(-g * kHi), -200.f), 200.f);
  const float f = __builtin_fmaf(-g, kLo, __builtin_fmaf(-g, kHi, -n));
  const float d = 1.f + __builtin_ldexpf(__builtin_amdgcn_exp2f(f), (int)n);
  const float r = __builtin_amdgcn_rcpf(d);
  float q = g * r;
  // (an infinite g or d has no remainder; a NaN passes through either way)
  if (__builtin_fabsf(g) < INFINITY && d < INFINITY) q = __builtin_fmaf(__builtin_fmaf(-q, d, g), r, q);
  return q * x;
}

// The same for gates from -150 to -86, where the quotient is not a normal number
// (the reciprocal is flushed to 0 from d = 2^126 on) though an x of 1e30 and more
// makes the product an ordinary one: x g e^g, its power of two last.  Below, no x
// brings it to the least scale.
constexpr float kSmallSilu = -86.f;
__device__ __forceinline__ bool silu_is_small(float g) { return g < kSmallSilu && g > -150.f; }
__device__ __forceinline__ float small_silu_times(float g, float x) {
  const float n = rintf(g * kHi);
  const float f = __builtin_fmaf(g, kLo, __builtin_fmaf(g, kHi, -n));
  return __builtin_ldexpf(g * __builtin_amdgcn_exp2f(f) * (x * 0x1p-16f), (int)n + 16);
}

// Elements i .. i + 7 of a row of D (zeros past its end), gated if GATE; `least`:
// of the gates seen.
template <int DT, bool GATE, bool WIDE>
__device__ __forceinline__ void load_y8(const QuantRowsArgs& A, long row, int i, float* y, float& least) {
  float g[8];
  if (!WIDE && i + 8 > A.D) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool in = i + e < A.D;
      y[e] = in ? load_elem<DT>(A.x, row * A.xs + i + e) : 0.f;
      if constexpr (GATE) g[e] = in ? load_elem<DT>(A.gate, row * A.gs + i + e) : 0.f;
    }
  } else {
    load8<DT, WIDE>(A.x, row * A.xs + i, y);
    if constexpr (GATE) load8<DT, WIDE>(A.gate, row * A.gs + i, g);
  }
  if constexpr (GATE) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      least = fminf(least, g[e]);
      y[e] = silu_times(g[e], y[e]);
    }
  }
}

// Puts in those of elements i .. i + 7 whose gate is small, read once more: a
// branch behind all loads that hardly any call takes (selected element by element
// it cost 5%, branched to between the loads of a whole row 17%).
template <int DT>
__device__ __forceinline__ void put_small(const QuantRowsArgs& A, long row, int i, float* y) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (i + e >= A.D) break;
    const float g = load_elem<DT>(A.gate, row * A.gs + i + e);
    if (silu_is_small(g)) y[e] = small_silu_times(g, load_elem<DT>(A.x, row * A.xs + i + e));
    __builtin_amdgcn_sched_barrier(0);  // (gathered, the loads take registers from the other path)
  }
}

template <bool WIDE>
__device__ __forceinline__ void store_codes(const QuantRowsArgs& A, long row, int i, v2u_t c) {
  uint8_t* p = A.codes + row * A.D + i;
  if constexpr (WIDE) {
    *reinterpret_cast<v2u_t*>(p) = c;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (i + e < A.D) p[e] = (uint8_t)(c[e >> 2] >> (8 * (e & 3)));
  }
}

// A scale per 128 values: 16 lanes a group, 16 groups a workgroup, `segs`
// workgroups a row.
template <int DT, bool GATE, bool WIDE>
__global__ __launch_bounds__(kQrThreads) void quant_groups_kernel(const QuantRowsArgs A) {
  const long row = blockIdx.x / (unsigned)A.segs;
  const int i = 8 * ((int)(blockIdx.x % (unsigned)A.segs) * kQrThreads + (int)threadIdx.x);
  if ((i & ~127) >= A.D) return;  // whole groups leave together
  float y[8];
  if (WIDE && i >= A.D) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = 0.f;
  } else {
    float least = 0.f;
    load_y8<DT, GATE, WIDE>(A, row, i, y, least);
    if (GATE && __builtin_expect(least < kSmallSilu, 0)) put_small<DT>(A, row, i, y);
  }
  const float scale = row_scale<true>(y);
  const v2u_t c = quant8<true>(y, scale);
  if (!WIDE || i < A.D) store_codes<WIDE>(A, row, i, c);
  if ((threadIdx.x & 15) == 0) A.scales[row * ((A.D + 127) / 128) + (i >> 7)] = scale;
}

// One scale a row: a workgroup of T threads a row, up to V vectors of 8 a
// thread, kept in registers between the maximum and the codes.  (64 registers at
// most: two workgroups of 1024 a CU, 73 us for gated rows, 86 with one.)
template <int DT, bool GATE, bool WIDE, int T, int V>
__global__ __launch_bounds__(T, WIDE ? 8 : 1) void quant_whole_rows_kernel(const QuantRowsArgs A) {
  __shared__ uint32_t top[T / kWave];
  const long row = blockIdx.x;
  float y[V][8], least = 0.f;
  uint32_t am = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = 8 * (v * T + (int)threadIdx.x);
    if (i < A.D) {
      load_y8<DT, GATE, WIDE>(A, row, i, y[v], least);
      am = max(am, amax_bits<true>(y[v]));
    }
  }
  if (GATE && __builtin_expect(least < kSmallSilu, 0)) {  // (what they were before is 0 or about the same)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int i = 8 * (v * T + (int)threadIdx.x);
      if (i < A.D) {
        put_small<DT>(A, row, i, y[v]);
        am = max(am, amax_bits<true>(y[v]));
      }
    }
  }
  am = wave_reduce<2>(am);
  if ((threadIdx.x & (kWave - 1)) == 0) top[threadIdx.x / kWave] = am;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < T / kWave; ++w) am = max(am, top[w]);
  const float scale = scale_of_amax(am);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = 8 * (v * T + (int)threadIdx.x);
    if (i < A.D) store_codes<WIDE>(A, row, i, quant8<true>(y[v], scale));
  }
  if (threadIdx.x == 0) A.scales[row] = scale;
}

template <int DT, bool GATE, bool WIDE>
static hipError_t launch_quant_rows_of(QuantRowsArgs A, hipStream_t s) {
  const long n = A.n;
  const auto at = [&](long first) {
    QuantRowsArgs B = A;
    constexpr int es = DT == kF32 ? 4 : 2;
    B.x = static_cast<const uint8_t*>(A.x) + first * A.xs * es;
    if (GATE) B.gate = static_cast<const uint8_t*>(A.gate) + first * A.gs * es;
    B.codes += first * A.D;
    B.scales += first * (A.group ? (A.D + 127) / 128 : 1);
    return B;
  };
  constexpr long kMost = 1L << 31;  // threads a launch
  if (A.group) {
    A.segs = (A.D + 8 * kQrThreads - 1) / (8 * kQrThreads);
    return in_launches(n, kMost / kQrThreads / A.segs, [&](long first, long count) {
      hipLaunchKernelGGL((quant_groups_kernel<DT, GATE, WIDE>), dim3((unsigned)(count * A.segs)), dim3(kQrThreads), 0, s,
                         at(first));
      return hipGetLastError();
    });
  }
  const auto go = [&](auto kernel, int threads) {
    return in_launches(n, kMost / threads, [&](long first, long count) {
      hipLaunchKernelGGL(kernel, dim3((unsigned)count), dim3(threads), 0, s, at(first));
      return hipGetLastError();
    });
  };
  static_assert(DSA_NORM_MAX_DIM == 8 * 1024 * 4, "the widest form holds the longest row");
  if (A.D <= 8 * 256) return go(quant_whole_rows_kernel<DT, GATE, WIDE, 256, 1>, 256);
  if (A.D <= 8 * 256 * 4) return go(quant_whole_rows_kernel<DT, GATE, WIDE, 256, 4>, 256);
  return go(quant_whole_rows_kernel<DT, GATE, WIDE, 1024, 4>, 1024);
}

template <int DT>
static hipError_t launch_quant_rows_typed(const QuantRowsArgs& A, hipStream_t s) {
  constexpr int es = DT == kF32 ? 4 : 2;
  const auto even = [](const void* p, long stride) { return (((uintptr_t)p | (uintptr_t)(stride * es)) & 15) == 0; };
  // whole 16-byte vectors in every row, and 8 codes on an 8-byte boundary
  const bool wide = A.D % 8 == 0 && even(A.x, A.n > 1 ? A.xs : 0) && (!A.gate || even(A.gate, A.n > 1 ? A.gs : 0)) &&
                    ((uintptr_t)A.codes & 7) == 0;
  if (A.gate) return wide ? launch_quant_rows_of<DT, true, true>(A, s) : launch_quant_rows_of<DT, true, false>(A, s);
  return wide ? launch_quant_rows_of<DT, false, true>(A, s) : launch_quant_rows_of<DT, false, false>(A, s);
}

hipError_t launch_quantize_rows(const QuantRowsArgs& A, int dtype, hipStream_t s) {
  switch (dtype) {
    case kF32: return launch_quant_rows_typed<kF32>(A, s);
    case kBF16: return launch_quant_rows_typed<kBF16>(A, s);
    default: return launch_quant_rows_typed<kF16>(A, s);
  }
}

}  // namespace dsa
