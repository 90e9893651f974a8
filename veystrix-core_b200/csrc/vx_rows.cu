// Row kernels that end in 8 bits: RMSNorm with the residual's addition, and
// SwiGLU, each row written as e4m3 with one float32 scale.
//
//   norm    s = x + residual                 (float32; the norm sees the sum
//                                             before its rounding to the
//                                             residual's type)
//           v_i = s_i * (1/sqrt(mean(s^2) + eps)) * gain_i
//   swiglu  v_i = g_i / (1 + exp(-g_i)) * u_i
//   8 bits  scale = max(max_i |v_i| / 448, 2^-126),  q_i = e4m3(v_i / scale)
//
// The norm's factor r = 1/sqrt(...) is common to a row, so max |v| is
// r * max |s_i * gain_i|: sum and maximum come from the same pass, and one
// block reduction serves both.  Rows whose squares or products s * gain leave
// the float32 range take a second one over scaled values, or the values
// themselves.  Rows are bound by memory: a row's elements
// are read once, stay in the registers of its threads (as float32) until the
// reduction is done, and every output is written once.  The maximum is taken
// over the bit patterns of |v|, an order in which NaN is above infinity, so a
// NaN anywhere makes the row's scale NaN as the formula does.
//
// A row belongs to one warp (four rows a CTA) while its elements fit one
// warp's registers, else to one CTA.  V is the elements a load brings: 8
// where every row starts on a 16-byte boundary and the width is a multiple
// of 8, else 1.  Rows too wide for the registers of 1,024 threads are read
// twice (LOOP).
#include <cuda_fp8.h>

#include <type_traits>

#include "vx_common.cuh"
#include "vx_launch.h"

namespace vx {

constexpr float kE4m3Max = 448.0f;
constexpr float kScaleMin = 0x1p-126f;
constexpr float kFloatMax = 0x1.fffffep127f;

VX_DEVICE uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// {scale, 1/scale} of a row whose largest |v| is amax (NaN stays NaN).
VX_DEVICE float2 row_scale(float amax) {
  float s = __fdiv_rn(amax, kE4m3Max);
  s = s < kScaleMin ? kScaleMin : s;
  return make_float2(s, __fdiv_rn(1.0f, s));
}

VX_DEVICE uint32_t e4m3x2(float lo, float hi) {   // lo in the low byte
  return uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3));
}
VX_DEVICE uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// 1/(1 + exp(-g)) within a few float32 ulp: with e = exp(-|g|) <= 1 the
// denominator stays in [1, 2], where the approximate division is exact to 2
// ulp, and nothing overflows.
VX_DEVICE float sigmoid_f32(float g) {
  const float e = expf(-fabsf(g));
  return __fdividef(g < 0.f ? e : 1.0f, 1.0f + e);
}

template <int V>
VX_DEVICE void load_row(const uint16_t* p, float (&f)[V]) {
  if constexpr (V == 8) {
    const uint4 v = ldg_nc(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else {
    f[0] = bf16_to_f32(__ldg(p));
  }
}
template <int V>
VX_DEVICE void load_row(const float* p, float (&f)[V]) {
  if constexpr (V == 8) {
    const uint4 a = ldg_nc(p), b = ldg_nc(p + 4);
    f[0] = __uint_as_float(a.x), f[1] = __uint_as_float(a.y), f[2] = __uint_as_float(a.z),
    f[3] = __uint_as_float(a.w), f[4] = __uint_as_float(b.x), f[5] = __uint_as_float(b.y),
    f[6] = __uint_as_float(b.z), f[7] = __uint_as_float(b.w);
  } else {
    f[0] = __ldg(p);
  }
}
template <int V>
VX_DEVICE void store_row(uint16_t* p, const float (&f)[V]) {
  if constexpr (V == 8)
    *reinterpret_cast<uint4*>(p) =
        make_uint4(bf16x2(f[0], f[1]), bf16x2(f[2], f[3]), bf16x2(f[4], f[5]), bf16x2(f[6], f[7]));
  else
    *p = uint16_t(bf16x2(f[0], 0.f));
}
template <int V>
VX_DEVICE void store_row(float* p, const float (&f)[V]) {
  if constexpr (V == 8) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *p = f[0];
  }
}
template <int V>
VX_DEVICE void store_row(uint8_t* p, const float (&f)[V]) {
  if constexpr (V == 8)
    *reinterpret_cast<uint2*>(p) = make_uint2(e4m3x2(f[0], f[1]) | (e4m3x2(f[2], f[3]) << 16),
                                              e4m3x2(f[4], f[5]) | (e4m3x2(f[6], f[7]) << 16));
  else
    *p = uint8_t(e4m3x2(f[0], 0.f));
}

// Sum (SUM) and largest bit pattern over the threads of a row: its warp, or
// the CTA (ONE_WARP false).  Every thread adds the warps' sums in the same order.
template <bool ONE_WARP, bool SUM>
VX_DEVICE void row_reduce(float& sum, uint32_t& top) {
  if (SUM) sum = warp_sum<32>(sum);
  top = __reduce_max_sync(0xFFFFFFFFu, top);
  if (ONE_WARP) return;
  __shared__ float sums[32];
  __shared__ uint32_t tops[32];
  const int warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum, tops[threadIdx.x >> 5] = top;
  __syncthreads();
  sum = 0.f, top = 0;
  for (int w = 0; w < warps; ++w) {
    if (SUM) sum += sums[w];
    top = max(top, tops[w]);
  }
}

// The place of this thread's row and its stride in it: ONE_WARP puts four
// rows into a CTA.  Returns the first element's index / V.
template <bool ONE_WARP>
VX_DEVICE int row_place(int64_t* row, int* lanes) {
  if (ONE_WARP) {
    *row = int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    *lanes = 32;
    return threadIdx.x & 31;
  }
  *row = blockIdx.x;
  *lanes = blockDim.x;
  return threadIdx.x;
}

template <int V, int NV, bool ONE_WARP, typename RES, bool LOOP>
__global__ void __launch_bounds__(1024) add_rmsnorm_kernel(
    const uint16_t* __restrict__ x, int64_t ldx, const RES* __restrict__ residual, int64_t ldr,
    const uint16_t* __restrict__ gain, int64_t T, int d, float eps, RES* __restrict__ residual_out,
    uint16_t* __restrict__ y, uint8_t* __restrict__ q, float* __restrict__ scales) {
  chain_begin();
  int64_t t;
  int lanes;
  const int i0 = row_place<ONE_WARP>(&t, &lanes) * V, step = lanes * V;
  if (ONE_WARP && t >= T) return;   // whole warps
  const uint16_t* xr = x + t * ldx;
  const RES* rr = residual ? residual + t * ldr : nullptr;

  // s of this thread's elements; kept in registers unless LOOP
  float s[NV][V], g[NV][V];
  float sum = 0.f;
  uint32_t top = 0;
  auto load = [&](int i, float (&sv)[V], float (&gv)[V]) {
    load_row<V>(xr + i, sv);
    if (rr) {
      float r[V];
      load_row<V>(rr + i, r);
#pragma unroll
      for (int j = 0; j < V; ++j) sv[j] += r[j];
    }
    load_row<V>(gain + i, gv);
  };
  auto gather = [&](const float (&sv)[V], const float (&gv)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      sum = fmaf(sv[j], sv[j], sum);
      top = max(top, abs_bits(sv[j] * gv[j]));
    }
  };
  if constexpr (LOOP) {
    for (int i = i0; i < d; i += step) {
      load(i, s[0], g[0]);
      gather(s[0], g[0]);
    }
  } else {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int i = i0 + n * step;
      if (i < d) {
        load(i, s[n], g[n]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) s[n][j] = g[n][j] = 0.f;
      }
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) gather(s[n], g[n]);
  }
  row_reduce<ONE_WARP, true>(sum, top);
  // f(s, gain) over the thread's elements once more: the two rare cases below
  auto again = [&](auto&& f) {
    if constexpr (LOOP) {
      for (int i = i0; i < d; i += step) {
        load(i, s[0], g[0]);
#pragma unroll
        for (int j = 0; j < V; ++j) f(s[0][j], g[0][j]);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int j = 0; j < V; ++j) f(s[n][j], g[n][j]);
    }
    if (!ONE_WARP) __syncthreads();   // row_reduce's shared memory is read by now
  };
  float r;
  if (sum > kFloatMax) {
    // the squares left the float32 range: the same on s / 2^70 (both
    // branches are taken by whole rows)
    sum = 0.f;
    uint32_t unused = 0;
    again([&](float sv, float) {
      sv *= 0x1p-70f;
      sum = fmaf(sv, sv, sum);
    });
    row_reduce<ONE_WARP, true>(sum, unused);
    r = __fdiv_rn(0x1p-70f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum, float(d)), eps * 0x1p-140f)));
  } else {
    r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum, float(d)), eps)));
  }
  if (scales && (top >= 0x7F800000u || top < 0x0D800000u)) {
    // some |s g| is no finite number, or all are below 2^-100 and lose bits:
    // the maximum of the values themselves
    top = 0;
    again([&](float sv, float gv) { top = max(top, abs_bits(sv * r * gv)); });
    row_reduce<ONE_WARP, false>(sum, top);
  } else {
    top = __float_as_uint(r * __uint_as_float(top));   // max|v| up to the rounding of one product
  }
  const float2 sc = row_scale(__uint_as_float(top));
  if (scales && i0 == 0) scales[t] = sc.x;

  auto write = [&](int i, float (&sv)[V], const float (&gv)[V]) {
    if (residual_out) store_row<V>(residual_out + t * d + i, sv);
#pragma unroll
    for (int j = 0; j < V; ++j) sv[j] = sv[j] * r * gv[j];
    if (y) store_row<V>(y + t * d + i, sv);
    if (q) {
#pragma unroll
      for (int j = 0; j < V; ++j) sv[j] *= sc.y;
      store_row<V>(q + t * d + i, sv);
    }
  };
  if constexpr (LOOP) {
    for (int i = i0; i < d; i += step) {
      load(i, s[0], g[0]);
      write(i, s[0], g[0]);
    }
  } else {
#pragma unroll
    for (int n = 0; n < NV; ++n)
      if (i0 + n * step < d) write(i0 + n * step, s[n], g[n]);
  }
}

template <int V, int NV, bool ONE_WARP, bool LOOP>
__global__ void __launch_bounds__(1024) swiglu_e4m3_kernel(const uint16_t* __restrict__ gate, int64_t ldg,
                                                           const uint16_t* __restrict__ up, int64_t ldu,
                                                           int64_t rows, int width, uint8_t* __restrict__ q,
                                                           float* __restrict__ scales) {
  chain_begin();
  int64_t t;
  int lanes;
  const int i0 = row_place<ONE_WARP>(&t, &lanes) * V, step = lanes * V;
  if (ONE_WARP && t >= rows) return;
  const uint16_t *gr = gate + t * ldg, *ur = up + t * ldu;
  float v[NV][V], unused = 0.f;
  uint32_t top = 0;
  auto load = [&](int i, float (&o)[V]) {
    float g[V], u[V];
    load_row<V>(gr + i, g);
    load_row<V>(ur + i, u);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = g[j] * sigmoid_f32(g[j]) * u[j];
  };
  if constexpr (LOOP) {
    for (int i = i0; i < width; i += step) {
      load(i, v[0]);
#pragma unroll
      for (int j = 0; j < V; ++j) top = max(top, abs_bits(v[0][j]));
    }
  } else {
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      if (i0 + n * step < width) {
        load(i0 + n * step, v[n]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[n][j] = 0.f;
      }
    }
#pragma unroll
    for (int n = 0; n < NV; ++n)
#pragma unroll
      for (int j = 0; j < V; ++j) top = max(top, abs_bits(v[n][j]));
  }
  row_reduce<ONE_WARP, false>(unused, top);
  const float2 sc = row_scale(__uint_as_float(top));
  if (i0 == 0) scales[t] = sc.x;
  auto write = [&](int i, float (&o)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] *= sc.y;
    store_row<V>(q + t * width + i, o);
  };
  if constexpr (LOOP) {
    for (int i = i0; i < width; i += step) {
      load(i, v[0]);
      write(i, v[0]);
    }
  } else {
#pragma unroll
    for (int n = 0; n < NV; ++n)
      if (i0 + n * step < width) write(i0 + n * step, v[n]);
  }
}

// ---- host side --------------------------------------------------------------

static bool starts_on(const void* p, int64_t ld, int64_t size, int64_t bytes) {
  return !p || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && ld * size % bytes == 0);
}

// Calls f(V, NV, one_warp, loop as integral constants, grid, threads) for
// rows of `width` elements.
template <typename F>
static cudaError_t per_row_shape(bool wide, int64_t rows, int width, F&& f) {
  using std::integral_constant;
  if (rows > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const int v = wide ? 8 : 1;
  const int vecs = (width + v - 1) / v;
  auto warps = [](int n) { return (n + 31) / 32 * 32; };
  const dim3 four(unsigned((rows + 3) / 4)), one((unsigned(rows)));
#define VX_ROWS(V, NV, W, L, grid, threads)                                                              \
  f(integral_constant<int, V>(), integral_constant<int, NV>(), integral_constant<bool, W>(),             \
    integral_constant<bool, L>(), grid, threads)
  if (wide) {
    if (vecs <= 32) return VX_ROWS(8, 1, true, false, four, 128);
    if (vecs <= 1024) return VX_ROWS(8, 1, false, false, one, warps(vecs));
    if (vecs <= 2048) return VX_ROWS(8, 2, false, false, one, warps((vecs + 1) / 2));
    return VX_ROWS(8, 1, false, true, one, 1024);
  }
  if (vecs <= 128) return VX_ROWS(1, 4, true, false, four, 128);
  if (vecs <= 4096) return VX_ROWS(1, 4, false, false, one, warps((vecs + 3) / 4));
  return VX_ROWS(1, 1, false, true, one, 1024);
#undef VX_ROWS
}

template <typename RES>
static cudaError_t add_rmsnorm_as(const uint16_t* x, int64_t ldx, const RES* residual, int64_t ldr,
                                  const uint16_t* gain, int64_t T, int d, float eps, RES* residual_out,
                                  uint16_t* y, uint8_t* q, float* scales, cudaStream_t st) {
  const bool wide = d % 8 == 0 && starts_on(x, ldx, 2, 16) && starts_on(residual, ldr, sizeof(RES), 16) &&
                    starts_on(gain, 0, 2, 16) && starts_on(residual_out, d, sizeof(RES), 16) &&
                    starts_on(y, d, 2, 16) && starts_on(q, d, 1, 8);
  return per_row_shape(wide, T, d, [&](auto v, auto nv, auto w, auto l, dim3 grid, int threads) {
    return launch_chained(add_rmsnorm_kernel<decltype(v)::value, decltype(nv)::value, decltype(w)::value, RES,
                                             decltype(l)::value>,
                          grid, dim3(threads), 0, st, x, ldx, residual, ldr, gain, T, d, eps, residual_out, y, q,
                          scales);
  });
}

cudaError_t launch_add_rmsnorm(const uint16_t* x, int64_t ldx, const void* residual, bool residual_f32, int64_t ldr,
                               const uint16_t* gain, int64_t T, int d, float eps, void* residual_out, uint16_t* y,
                               uint8_t* q, float* scales, cudaStream_t st) {
  if (T == 0) return cudaSuccess;
  if (residual_f32)
    return add_rmsnorm_as(x, ldx, static_cast<const float*>(residual), ldr, gain, T, d, eps,
                          static_cast<float*>(residual_out), y, q, scales, st);
  return add_rmsnorm_as(x, ldx, static_cast<const uint16_t*>(residual), ldr, gain, T, d, eps,
                        static_cast<uint16_t*>(residual_out), y, q, scales, st);
}

cudaError_t launch_swiglu_e4m3(const uint16_t* gate, int64_t ldg, const uint16_t* up, int64_t ldu, int64_t rows,
                               int width, uint8_t* q, float* scales, cudaStream_t st) {
  if (rows == 0) return cudaSuccess;
  const bool wide = width % 8 == 0 && starts_on(gate, ldg, 2, 16) && starts_on(up, ldu, 2, 16) &&
                    starts_on(q, width, 1, 8);
  return per_row_shape(wide, rows, width, [&](auto v, auto nv, auto w, auto l, dim3 grid, int threads) {
    return launch_chained(swiglu_e4m3_kernel<decltype(v)::value, decltype(nv)::value, decltype(w)::value,
                                             decltype(l)::value>,
                          grid, dim3(threads), 0, st, gate, ldg, up, ldu, rows, width, q, scales);
  });
}

}  // namespace vx
