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
// block reduction serves both.  Rows whose squares leave the float32 range at
// either end take a second one over scaled values, rows whose products s *
// gain leave it one over the values themselves.  Rows are bound by memory: a
// row's elements are read once, stay in the registers of its threads (as
// float32) until the reduction is done, and every output is written once.  The
// maximum keeps NaN, so a NaN anywhere makes the row's scale NaN as the formula
// does.
//
// Rows are dealt round robin to groups of threads, a warp (four groups a CTA)
// or a CTA; a group has its next row's loads in flight while it reduces and
// writes the present one.  V is the elements an access takes: the largest of 8,
// 4, 2 and 1 that divides the width and on whose boundary every row starts.
// Rows too wide for the registers of 1,024 threads are read twice (LOOP).
#include <cuda_fp8.h>

#include <initializer_list>
#include <type_traits>

#include "vx_common.cuh"
#include "vx_launch.h"

namespace vx {

constexpr float kE4m3Max = 448.0f;
constexpr float kScaleMin = 0x1p-126f;
constexpr float kFloatMax = 0x1.fffffep127f;

// {scale, 1/scale} of a row whose largest |v| is amax (NaN stays NaN).  Values
// are multiplied by the rounded inverse (2^-24 off) rather than divided: one
// that lies so close to a border between two e4m3 values (whose half step is
// 2^-4) may go to either.
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

// g / (1 + exp(-g)) * u.  With e = exp(-|g|) <= 1 the denominator stays in
// [1, 2] and nothing overflows.  e is the square of h = 2^(-|g| log2(e) / 2); a
// negative g's factor e goes in as two factors h, one at g and one at u: e alone
// leaves the normal range at g = -87, h at -174, where the product is below
// 2^-115 whatever u is (and counts as zero).  So the flush-to-zero exponential
// serves (half the instructions of the one that keeps subnormals).  Off by a
// few 2^-22, and by |g| 2^-23 of e.
VX_DEVICE float swiglu_f32(float g, float u) {
  float h, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(h) : "f"(fabsf(g) * -0.72134752f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(h, h, 1.0f)));
  if (g < 0.f) g *= h, u *= h;
  return g * r * u;
}
// The larger of top and |v|, NaN if one of them is.
VX_DEVICE float max_abs(float top, float v) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(v)));
  return top;
}

// V elements of a row as they lie in memory, and as float32.
template <int V, typename E>
struct Raw {
  static constexpr int kWords = V * int(sizeof(E)) / 4;   // 32-bit words
  uint32_t w[kWords];
  template <bool AGAIN>
  VX_DEVICE void read(const E* p) {
    if constexpr (kWords % 4 == 0) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4* q = reinterpret_cast<const uint4*>(p) + i / 4;
        const uint4 v = AGAIN ? __ldg(q) : ldg_nc(q);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    } else if constexpr (kWords == 2) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = v.x, w[1] = v.y;
    } else {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    }
  }
  VX_DEVICE void load(const E* p) { read<false>(p); }
  VX_DEVICE void load_again(const E* p) { read<true>(p); }   // what every row reads: kept in L1
  VX_DEVICE void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  VX_DEVICE void get(float (&f)[V]) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if (sizeof(E) == 2) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      } else {
        f[i] = __uint_as_float(w[i]);
      }
    }
  }
};
template <typename E>
struct Raw<1, E> {
  E v;
  VX_DEVICE void load(const E* p) { v = __ldg(p); }
  VX_DEVICE void load_again(const E* p) { v = __ldg(p); }
  VX_DEVICE void zero() { v = 0; }
  VX_DEVICE void get(float (&f)[1]) const { f[0] = sizeof(E) == 2 ? bf16_to_f32(uint16_t(v)) : float(v); }
};

template <int V>
VX_DEVICE void store_row(uint16_t* p, const float (&f)[V]) {
  if constexpr (V == 8)
    *reinterpret_cast<uint4*>(p) =
        make_uint4(bf16x2(f[0], f[1]), bf16x2(f[2], f[3]), bf16x2(f[4], f[5]), bf16x2(f[6], f[7]));
  else if constexpr (V == 4)
    *reinterpret_cast<uint2*>(p) = make_uint2(bf16x2(f[0], f[1]), bf16x2(f[2], f[3]));
  else if constexpr (V == 2)
    *reinterpret_cast<uint32_t*>(p) = bf16x2(f[0], f[1]);
  else
    *p = uint16_t(bf16x2(f[0], 0.f));
}
template <int V>
VX_DEVICE void store_row(float* p, const float (&f)[V]) {
  if constexpr (V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4)
      *reinterpret_cast<float4*>(p + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
  } else if constexpr (V == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(f[0], f[1]);
  } else {
    *p = f[0];
  }
}
template <int V>
VX_DEVICE void store_row(uint8_t* p, const float (&f)[V]) {
  if constexpr (V == 8)
    *reinterpret_cast<uint2*>(p) = make_uint2(e4m3x2(f[0], f[1]) | (e4m3x2(f[2], f[3]) << 16),
                                              e4m3x2(f[4], f[5]) | (e4m3x2(f[6], f[7]) << 16));
  else if constexpr (V == 4)
    *reinterpret_cast<uint32_t*>(p) = e4m3x2(f[0], f[1]) | (e4m3x2(f[2], f[3]) << 16);
  else if constexpr (V == 2)
    *reinterpret_cast<uint16_t*>(p) = uint16_t(e4m3x2(f[0], f[1]));
  else
    *p = uint8_t(e4m3x2(f[0], 0.f));
}

// Sum (SUM) and largest value over the threads of a row: its warp, or
// the CTA (ONE_WARP false).  Every thread adds the warps' sums in the same
// order.  Successive calls alternate `turn` between two sets of shared
// memory, so one barrier a call is enough.
template <bool ONE_WARP, bool SUM>
VX_DEVICE void row_reduce(float& sum, float& largest, int& turn) {
  if (SUM) sum = warp_sum<32>(sum);
  // not negative: ordered like their bit patterns, NaN on top
  uint32_t top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(largest));
  largest = __uint_as_float(top);
  if (ONE_WARP) return;
  __shared__ float sums[2][32];
  __shared__ uint32_t tops[2][32];
  const int warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) sums[turn][threadIdx.x >> 5] = sum, tops[turn][threadIdx.x >> 5] = top;
  __syncthreads();
  sum = 0.f, top = 0;
  for (int w = 0; w < warps; ++w) {
    if (SUM) sum += sums[turn][w];
    top = max(top, tops[turn][w]);
  }
  largest = __uint_as_float(top);
  turn ^= 1;
}

// This thread's group of rows: the first row, the stride, and the thread's
// place in the row and number of threads in it.
template <bool ONE_WARP>
struct Group {
  int64_t row, stride;
  int place, threads;
  VX_DEVICE Group() {
    if (ONE_WARP) {
      row = int64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
      stride = int64_t(gridDim.x) * (blockDim.x >> 5);
      place = threadIdx.x & 31, threads = 32;
    } else {
      row = blockIdx.x, stride = gridDim.x;
      place = threadIdx.x, threads = blockDim.x;
    }
  }
};

template <int V, int NV, bool ONE_WARP, typename RES, bool LOOP>
__global__ void __launch_bounds__(ONE_WARP ? 128 : 1024) add_rmsnorm_kernel(
    const uint16_t* __restrict__ x, int64_t ldx, const RES* __restrict__ residual, int64_t ldr,
    const uint16_t* __restrict__ gain, int64_t T, int d, float eps, RES* __restrict__ residual_out,
    uint16_t* __restrict__ y, uint8_t* __restrict__ q, float* __restrict__ scales) {
  chain_begin();
  const Group<ONE_WARP> grp;
  const int i0 = grp.place * V, step = grp.threads * V;
  int turn = 0;
  Raw<V, uint16_t> xw[NV];
  Raw<V, RES> rw[NV];
  auto fetch = [&](int64_t t, int i, int n) {
    if (i < d) {
      xw[n].load(x + t * ldx + i);
      if (residual) rw[n].load(residual + t * ldr + i);
    } else {
      xw[n].zero();
      rw[n].zero();
    }
  };
  auto sum_of = [&](int n, float (&sv)[V]) {
    xw[n].get(sv);
    if (residual) {
      float r[V];
      rw[n].get(r);
#pragma unroll
      for (int j = 0; j < V; ++j) sv[j] += r[j];
    }
  };
  // The gains are the same for every row: from L1, or held where they take few
  // registers (odd rows, whose accesses bring one or two elements).
  constexpr bool kHeld = V <= 2 && !LOOP;
  float held[kHeld ? NV : 1][V];
  auto read_gains = [&](int i, float (&gv)[V]) {
    Raw<V, uint16_t> w;
    if (i < d) w.load_again(gain + i); else w.zero();
    w.get(gv);
  };
  auto gains = [&](int i, int n, float (&gv)[V]) {
    if constexpr (kHeld) {
#pragma unroll
      for (int j = 0; j < V; ++j) gv[j] = held[n][j];
    } else {
      read_gains(i, gv);
    }
  };
  if constexpr (kHeld) {
#pragma unroll
    for (int n = 0; n < NV; ++n) read_gains(i0 + n * step, held[n]);
  }
  if (!LOOP && grp.row < T) {
#pragma unroll
    for (int n = 0; n < NV; ++n) fetch(grp.row, i0 + n * step, n);
  }
  for (int64_t t = grp.row; t < T; t += grp.stride) {   // whole groups
    float s[NV][V];
    float sum = 0.f, top = 0.f;   // top: max |s gain|, then max |v|
    // f(s, gain) over the thread's elements
    auto each = [&](auto&& f) {
      if constexpr (LOOP) {
        for (int i = i0; i < d; i += step) {
          float gv[V];
          fetch(t, i, 0);
          sum_of(0, s[0]);
          gains(i, 0, gv);
#pragma unroll
          for (int j = 0; j < V; ++j) f(s[0][j], gv[j]);
        }
      } else {
#pragma unroll
        for (int n = 0; n < NV; ++n) {
          float gv[V];
          gains(i0 + n * step, n, gv);
#pragma unroll
          for (int j = 0; j < V; ++j) f(s[n][j], gv[j]);
        }
      }
    };
    if constexpr (!LOOP) {
#pragma unroll
      for (int n = 0; n < NV; ++n) sum_of(n, s[n]);
      if (t + grp.stride < T) {
#pragma unroll
        for (int n = 0; n < NV; ++n) fetch(t + grp.stride, i0 + n * step, n);
      }
    }
    each([&](float sv, float gv) {
      sum = fmaf(sv, sv, sum);
      top = max_abs(top, sv * gv);
    });
    row_reduce<ONE_WARP, true>(sum, top, turn);
    // The norm's factor is pre * r; pre is 1 but for the rows below (all
    // branches here are taken by whole rows).
    float pre = 1.f;
    if (sum > kFloatMax) {
      // The squares left the range upwards: the same on s / 2^80.  s < 2^128, so
      // its squares are below 2^96 and 2^29 of them below 2^125; the largest is
      // at least 2^(128 - 29 - 160), so what drops below the range is nothing
      // beside it.
      pre = 0x1p-80f;
    } else if (sum < 0x1p-100f && eps < 0x1p-100f) {
      // Squares may have lost bits or become zero (2^-150 each, which is nothing
      // beside a sum of 2^-100, nor their mean's error beside such an eps): on
      // 2^100 s, below 2^50, the least of them 2^-49.
      pre = 0x1p100f;
    }
    if (pre != 1.f) {
      sum = 0.f;
      float unused = 0.f;
      each([&](float sv, float) {
        sv *= pre;
        sum = fmaf(sv, sv, sum);
      });
      row_reduce<ONE_WARP, true>(sum, unused, turn);
    }
    // eps pre^2 in two steps: pre^2 alone is no float32
    const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sum, float(d)), eps * pre * pre)));
    if (scales && !(pre == 1.f && top <= kFloatMax && top >= 0x1p-100f)) {
      // some |s g| is no finite number, or all are below 2^-100 and lose bits, or
      // s is scaled: the maximum of the values themselves
      top = 0.f;
      each([&](float sv, float gv) { top = max_abs(top, sv * pre * r * gv); });
      row_reduce<ONE_WARP, false>(sum, top, turn);
    } else {
      top *= r;   // max|v| up to the rounding of one product
    }
    const float2 sc = row_scale(top);
    if (scales && i0 == 0) scales[t] = sc.x;

    auto write = [&](int i, int n, float (&sv)[V]) {
      float gv[V];
      gains(i, n, gv);
      if (residual_out) store_row<V>(residual_out + t * d + i, sv);
      if (pre != 1.f) {
#pragma unroll
        for (int j = 0; j < V; ++j) sv[j] *= pre;
      }
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
        fetch(t, i, 0);
        sum_of(0, s[0]);
        write(i, 0, s[0]);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NV; ++n)
        if (i0 + n * step < d) write(i0 + n * step, n, s[n]);
    }
  }
}

template <int V, int NV, bool ONE_WARP, bool LOOP>
__global__ void __launch_bounds__(ONE_WARP ? 128 : 1024) swiglu_e4m3_kernel(
    const uint16_t* __restrict__ gate, int64_t ldg, const uint16_t* __restrict__ up, int64_t ldu, int64_t rows,
    int width, uint8_t* __restrict__ q, float* __restrict__ scales) {
  chain_begin();
  const Group<ONE_WARP> grp;
  const int i0 = grp.place * V, step = grp.threads * V;
  int turn = 0;
  Raw<V, uint16_t> gw[NV], uw[NV];
  auto fetch = [&](int64_t t, int i, int n) {
    if (i < width) {
      gw[n].load(gate + t * ldg + i);
      uw[n].load(up + t * ldu + i);
    } else {
      gw[n].zero();
      uw[n].zero();
    }
  };
  auto value = [&](int n, float (&o)[V]) {
    float u[V];
    gw[n].get(o);
    uw[n].get(u);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = swiglu_f32(o[j], u[j]);
  };
  if (!LOOP && grp.row < rows) {
#pragma unroll
    for (int n = 0; n < NV; ++n) fetch(grp.row, i0 + n * step, n);
  }
  for (int64_t t = grp.row; t < rows; t += grp.stride) {   // whole groups
    float v[NV][V], unused = 0.f, top = 0.f;
    if constexpr (LOOP) {
      for (int i = i0; i < width; i += step) {
        fetch(t, i, 0);
        value(0, v[0]);
#pragma unroll
        for (int j = 0; j < V; ++j) top = max_abs(top, v[0][j]);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NV; ++n) value(n, v[n]);
      if (t + grp.stride < rows) {
#pragma unroll
        for (int n = 0; n < NV; ++n) fetch(t + grp.stride, i0 + n * step, n);
      }
#pragma unroll
      for (int n = 0; n < NV; ++n)
#pragma unroll
        for (int j = 0; j < V; ++j) top = max_abs(top, v[n][j]);
    }
    row_reduce<ONE_WARP, false>(unused, top, turn);
    const float2 sc = row_scale(top);
    if (i0 == 0) scales[t] = sc.x;
    auto write = [&](int i, float (&o)[V]) {
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] *= sc.y;
      store_row<V>(q + t * width + i, o);
    };
    if constexpr (LOOP) {
      for (int i = i0; i < width; i += step) {
        fetch(t, i, 0);
        value(0, v[0]);
        write(i, v[0]);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NV; ++n)
        if (i0 + n * step < width) write(i0 + n * step, v[n]);
    }
  }
}

// ---- host side --------------------------------------------------------------

// Rows p + i * ld of elements of `size` bytes (null: none).
struct RowsAt {
  const void* p;
  int64_t ld, size;
};
// Elements an access may take: the largest of 8, 4, 2, 1 that divides the width
// and on whose boundary every row starts.
static int access_width(int width, std::initializer_list<RowsAt> all) {
  int v = 8;
  while (width % v) v /= 2;
  for (const RowsAt& r : all) {
    auto fits = [&] {
      const int64_t bytes = v * r.size < 16 ? v * r.size : 16;
      return !r.p || (reinterpret_cast<uintptr_t>(r.p) % bytes == 0 && r.ld * r.size % bytes == 0);
    };
    while (v > 1 && !fits()) v /= 2;
  }
  return v;
}

// Registers a thread of `kernel` uses (a property of the code: looked up once).
template <typename K>
static int registers_of(K* kernel) {
  cudaFuncAttributes attr;
  if (cudaFuncGetAttributes(&attr, reinterpret_cast<const void*>(kernel)) != cudaSuccess) return 64;
  return attr.numRegs > 0 ? attr.numRegs : 64;
}

// CTAs for `groups` groups: four rounds of what is resident at once.  A group
// goes on to its next row with the loads in flight, and the rounds fill the
// gaps that groups ending early leave: norm 16,384 x 2,560 68 us with one
// round, 67 with two, 63 with four, 61 with eight, 65 with a row a group; swiglu
// 81,920 x 640 46, 45, 44, 44, 50.
static unsigned row_ctas(int64_t groups, int threads, int registers) {
  const int by_regs = 65536 / (((registers + 7) & ~7) * threads), by_threads = 2048 / threads;
  int per_sm = by_regs < by_threads ? by_regs : by_threads;
  per_sm = per_sm < 1 ? 1 : per_sm > 32 ? 32 : per_sm;
  const int64_t most = 4 * int64_t(sm_count()) * per_sm;
  return unsigned(groups < most ? groups : most);
}

// Calls f with the variant for rows of `width` elements (V, NV, one warp,
// loop as integral constants), the groups and the threads of a CTA.
template <typename F>
static cudaError_t per_row_shape(int v, int64_t rows, int width, F&& f) {
  using std::integral_constant;
  const int vecs = (width + v - 1) / v;
  auto run = [&](auto V, auto NV, auto W, auto L) {
    const int threads = W ? 128 : L ? 1024 : ((vecs + NV - 1) / NV + 31) / 32 * 32;
    return f(V, NV, W, L, W ? (rows + 3) / 4 : rows, threads);
  };
#define VX_ROWS(V, NV, W, L)                                                                 \
  run(integral_constant<int, V>(), integral_constant<int, NV>(), integral_constant<bool, W>(), \
      integral_constant<bool, L>())
  const bool many = rows >= 4 * int64_t(sm_count());
  if (v == 8) {
    if (vecs <= 32) return VX_ROWS(8, 1, true, false);
    // A batch that fills the GPU gives each row fewer threads with more loads
    // each, one warp where the registers allow (no CTA barrier): norm 65,536 x
    // 512 52 against 60 us, swiglu 20,480 x 1,024 18.8 against 21.6 us; a
    // smaller batch spreads its rows: norm 64 x 2,048 2.1 us either way.
    if (many && vecs <= 64) return VX_ROWS(8, 2, true, false);
    if (many && vecs <= 96) return VX_ROWS(8, 3, true, false);
    if (many && vecs <= 128) return VX_ROWS(8, 4, true, false);
    if (vecs <= 1024 && !many) return VX_ROWS(8, 1, false, false);
    if (vecs <= 2048) return VX_ROWS(8, 2, false, false);
    return VX_ROWS(8, 1, false, true);
  }
  // The same with narrower accesses: a warp up to 32 of them a lane, then more
  // a thread.  Norm 20,000 x 555 36 against 50 us, 13,012 x 1,187 54 / 68, 8,192 x
  // 1,004 15.2 / 14.7; swiglu 47,605 x 413 25 / 52, 20,000 x 777 21 / 42, 20,000 x
  // 996 17 / 21, 4,000 x 4,002 21 / 25.
  if (v == 4 && many && vecs > 128 && vecs <= 256) return VX_ROWS(4, 8, true, false);
  if (v <= 2 && many && vecs > 128 && vecs <= 8192) {
    if (vecs <= 256) return v == 2 ? VX_ROWS(2, 8, true, false) : VX_ROWS(1, 8, true, false);
    if (vecs <= 512) return v == 2 ? VX_ROWS(2, 16, true, false) : VX_ROWS(1, 16, true, false);
    if (vecs <= 1024) return v == 2 ? VX_ROWS(2, 32, true, false) : VX_ROWS(1, 32, true, false);
    return v == 2 ? VX_ROWS(2, 8, false, false) : VX_ROWS(1, 8, false, false);
  }
#define VX_NARROW(V)                                                                            \
  (vecs <= 128 ? VX_ROWS(V, 4, true, false) : vecs <= 4096 ? VX_ROWS(V, 4, false, false) : VX_ROWS(V, 1, false, true))
  return v == 4 ? VX_NARROW(4) : v == 2 ? VX_NARROW(2) : VX_NARROW(1);
#undef VX_NARROW
#undef VX_ROWS
}

template <typename RES>
static cudaError_t add_rmsnorm_as(const uint16_t* x, int64_t ldx, const RES* residual, int64_t ldr,
                                  const uint16_t* gain, int64_t T, int d, float eps, RES* residual_out,
                                  uint16_t* y, uint8_t* q, float* scales, cudaStream_t st) {
  const int access = access_width(d, {{x, ldx, 2}, {residual, ldr, sizeof(RES)}, {gain, 0, 2},
                                      {residual_out, d, sizeof(RES)}, {y, d, 2}, {q, d, 1}});
  return per_row_shape(access, T, d, [&](auto v, auto nv, auto w, auto l, int64_t groups, int threads) {
    auto k = add_rmsnorm_kernel<decltype(v)::value, decltype(nv)::value, decltype(w)::value, RES, decltype(l)::value>;
    static const int registers = registers_of(k);
    return launch_chained(k, dim3(row_ctas(groups, threads, registers)), dim3(threads), 0, st, x, ldx, residual, ldr,
                          gain, T, d, eps, residual_out, y, q, scales);
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
  const int access = access_width(width, {{gate, ldg, 2}, {up, ldu, 2}, {q, width, 1}});
  return per_row_shape(access, rows, width, [&](auto v, auto nv, auto w, auto l, int64_t groups, int threads) {
    auto k = swiglu_e4m3_kernel<decltype(v)::value, decltype(nv)::value, decltype(w)::value, decltype(l)::value>;
    static const int registers = registers_of(k);
    return launch_chained(k, dim3(row_ctas(groups, threads, registers)), dim3(threads), 0, st, gate, ldg, up, ldu, rows,
                          width, q, scales);
  });
}

}  // namespace vx
