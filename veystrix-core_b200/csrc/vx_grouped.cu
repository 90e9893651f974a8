// Products grouped by expert over unquantised (bf16) or 8-bit (e4m3) banks:
//
//   out[p, n] = bf16( sx[row p] * sw[e, n] * sum_k x[row p, k] * w[e, n, k] )
//
// for the positions p in [offsets[e], offsets[e+1]) of expert e, row p =
// rows[p] / slots, or p itself; the scales only with e4m3.  Sums in float32,
// one rounding.  Positions from offsets[E] on are left as they were.
#include <cuda_fp8.h>

#include "vx_common.cuh"
#include "vx_launch.h"

namespace vx {

VX_DEVICE float elem_f32(const uint16_t* p) { return bf16_to_f32(__ldg(p)); }
VX_DEVICE float elem_f32(const uint8_t* p) {
  __nv_fp8_e4m3 v;
  v.__x = __ldg(p);
  return float(v);
}

// The row of x that position p reads; -1 where it lies outside x.
VX_DEVICE int64_t row_of(const GroupedArgs& a, int64_t p) {
  if (!a.rows) return p;
  const int r = a.rows[p];
  return r >= 0 && r / a.slots < a.x_rows ? r / a.slots : -1;
}

// One CTA = one expert x 64 outputs: 64 x 64 tiles, 4 x 4 outputs a thread,
// 16 inputs of both operands at a time in shared memory.
template <typename E>
__global__ void __launch_bounds__(256) grouped_kernel(const GroupedArgs a) {
  chain_begin();
  __shared__ float xs[16][65], ws[16][65];
  const E* x = static_cast<const E*>(a.x);
  const E* w = static_cast<const E*>(a.w) + int64_t(blockIdx.x) * a.N * a.K;
  const int64_t first = min(max(int64_t(a.offsets[blockIdx.x]), int64_t(0)), a.P);
  const int64_t last = min(max(int64_t(a.offsets[blockIdx.x + 1]), first), a.P);
  const int n0 = blockIdx.y * 64, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  for (int64_t p0 = first; p0 < last; p0 += 64) {
    float acc[4][4] = {};
    for (int k0 = 0; k0 < a.K; k0 += 16) {
      for (int i = threadIdx.x; i < 64 * 16; i += 256) {
        const int r = i >> 4, k = i & 15;
        float xv = 0.f, wv = 0.f;
        if (p0 + r < last && k0 + k < a.K) {
          const int64_t row = row_of(a, p0 + r);
          if (row >= 0) xv = elem_f32(x + row * a.ldx + k0 + k);
        }
        if (n0 + r < a.N && k0 + k < a.K) wv = elem_f32(w + int64_t(n0 + r) * a.K + k0 + k);
        xs[k][r] = xv;
        ws[k][r] = wv;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 16; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[k][ty * 4 + i], ws[k][tx + 16 * j], acc[i][j]);
      __syncthreads();
    }
    for (int i = 0; i < 4; ++i) {
      const int64_t p = p0 + ty * 4 + i;
      if (p >= last) continue;
      float sx = 1.f;
      if (a.x_scales) {
        const int64_t row = row_of(a, p);
        sx = row >= 0 ? a.x_scales[row] : 0.f;
      }
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + tx + 16 * j;
        if (n >= a.N) continue;
        const float sw = a.w_scales ? a.w_scales[int64_t(blockIdx.x) * a.N + n] : 1.f;
        a.out[p * a.ldo + n] = f32_to_bf16(acc[i][j] * sx * sw);
      }
    }
  }
}

cudaError_t launch_grouped(const GroupedArgs& a, bool e4m3, cudaStream_t st) {
  if (a.P == 0 || a.N == 0) return cudaSuccess;
  const dim3 grid(unsigned(a.experts), unsigned((a.N + 63) / 64));
  return e4m3 ? launch_chained(grouped_kernel<uint8_t>, grid, dim3(256), 0, st, a)
              : launch_chained(grouped_kernel<uint16_t>, grid, dim3(256), 0, st, a);
}

}  // namespace vx
