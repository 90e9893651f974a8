// Low-rank adapters of many requests beside one shared projection:
//
//   out[t] = bf16( y[t] + scale_a * B_a (A_a x_t) ),  a = adapters[t]
//
// with A [L][R][K], B [L][N][R] bf16 and only the first ranks[a] of the R
// components.  A token whose adapter is outside [0, L) gets out = y.  The R
// inner values stay in float32; the sum is rounded once.
#include "vx_common.cuh"
#include "vx_launch.h"

namespace vx {

// One CTA = one token: a warp per inner value, then a thread per output.
__global__ void __launch_bounds__(256) lora_kernel(const LoraArgs a) {
  chain_begin();
  __shared__ float h[kLoraMaxRank];
  const int64_t t = blockIdx.x;
  const int e = a.adapters[t];
  const bool live = e >= 0 && e < a.L;
  const int rank = !live ? 0 : a.ranks ? min(max(a.ranks[e], 0), a.R) : a.R;
  const uint16_t* x = a.x + t * a.ldx;
  for (int r = threadIdx.x >> 5; r < rank; r += 8) {
    const uint16_t* ar = a.a + (int64_t(e) * a.R + r) * a.K;
    float s = 0.f;
    for (int k = threadIdx.x & 31; k < a.K; k += 32) s = fmaf(bf16_to_f32(x[k]), bf16_to_f32(ar[k]), s);
    s = warp_sum<32>(s);
    if ((threadIdx.x & 31) == 0) h[r] = s * (a.scales ? a.scales[e] : 1.0f);
  }
  __syncthreads();
  for (int n = threadIdx.x; n < a.N; n += blockDim.x) {
    float s = 0.f;
    for (int r = 0; r < rank; ++r) s = fmaf(h[r], bf16_to_f32(a.b[(int64_t(e) * a.N + n) * a.R + r]), s);
    a.out[t * a.ldo + n] = f32_to_bf16(bf16_to_f32(a.y[t * a.ldy + n]) + s);
  }
}

cudaError_t launch_lora(const LoraArgs& a, cudaStream_t st) {
  if (a.T == 0 || a.N == 0) return cudaSuccess;
  return launch_chained(lora_kernel, dim3(unsigned(a.T)), dim3(256), 0, st, a);
}

}  // namespace vx
