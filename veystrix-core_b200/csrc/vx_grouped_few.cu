// Products grouped by expert where there are few rows (decode): the formula of
// vx_grouped.cu, bound by the bank's bytes alone.  64 tokens over 512 bf16
// experts: 226 us for 1.54 GB, 1.04 of the measured copy rate; one token e4m3
// 9.9 us for 21 MB, most of it the launch, the table of groups and the
// latency of the first reads.
//
// A work item is an expert and up to 8 of its positions, a unit an item and
// 16 of the bank's outputs.  One warp multiplies a unit (S = 1), or S warps of
// a CTA share it over K, with mma.sync m16n8:
//
//   D[16 outputs][8 positions] += W[16][K] . X[8][K]^T
//
// The operands go from global memory straight into the fragments: a lane
// reads 16 bytes of its row at once, and as both operands are read alike, the
// order of the inputs inside a fragment does not matter.  A warp has
// few_ahead() such reads of each of its two bank rows a lane in flight.
//
// Why not the tensor tiles of vx_grouped.cu: those have 256 outputs a CTA pair,
// so a few tokens leave SMs idle (ten experts of 1,024 outputs are 40 tiles
// for 74 pairs), their prologue is longer, and their MMAs spend power on
// columns of padding.
#include "vx_async.cuh"
#include "vx_common.cuh"
#include "vx_grouped.cuh"
#include "vx_launch.h"

namespace vx {

constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewPos = 8;        // positions of an item: the MMA's N
constexpr int kFewRows = 16;      // outputs of a unit: its M
// 64-byte steps of K in flight a warp, and CTAs an SM.  Many units: the longest
// reads (64 tokens bf16: 8 steps and 2 CTAs 223 us, 4 and 3 230, 6 and 3 238);
// few: more CTAs that start at once (4 tokens: 36 against 31 us).
constexpr int few_ahead(int S) { return S == 1 ? 8 : 4; }
constexpr int few_ctas(int S) { return S == 1 ? 2 : 3; }

template <bool FP8>
VX_DEVICE void few_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (FP8)
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    mma16816(d, a0, a1, a2, a3, b0, b1);
}

template <bool FP8, int S>
__global__ void __launch_bounds__(kFewThreads, few_ctas(S)) grouped_few_kernel(const GroupedArgs a) {
  constexpr int kAhead = few_ahead(S);
  extern __shared__ int smem_int[];
  __shared__ float part[S > 1 ? kFewWarps : 1][kFewRows][kFewPos + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  chain_wait();
  const GroupTable<kFewThreads> groups(a, smem_int, kFewPos);
  const int64_t row_bytes = int64_t(a.K) * (FP8 ? 1 : 2), ld_bytes = a.ldx * (FP8 ? 1 : 2);
  const int steps = int((row_bytes + 63) / 64), each = ((steps + S - 1) / S + 1) & ~1;   // whole 128-byte lines
  const int step0 = (warp % S) * each, step1 = min(steps, step0 + each);
  const int tiles = (a.N + kFewRows - 1) / kFewRows, per = kFewWarps / S;
  const int stacks = (tiles + per - 1) / per;   // CTA units of an item
  const char* W = static_cast<const char*>(a.w);

  for (int64_t u = blockIdx.x; u < int64_t(groups.items()) * stacks; u += gridDim.x) {
    const int item = int(u / stacks), tile = int(u - int64_t(item) * stacks) * per + warp / S, n0 = tile * kFewRows;
    int p0;
    int e;
    const int count = groups.item(item, &e, &p0);   // positions p0 .. p0 + count - 1
    float acc[4] = {};
    if (tile < tiles) {
      int row = -1;
      if (g < count) row = a.rows ? row_of(a, p0 + g) : p0 + g;
      const char* x = row >= 0 ? static_cast<const char*>(a.x) + row * ld_bytes : nullptr;
      const char* w0 = W + (int64_t(e) * a.N + n0 + g) * row_bytes;
      const char* w1 = w0 + 8 * row_bytes;
      const bool in0 = n0 + g < a.N, in1 = n0 + 8 + g < a.N;
      for (int s = step0; s < step1; s += kAhead) {
        uint4 v0[kAhead], v1[kAhead], xv[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int64_t off = int64_t(s + i) * 64 + c * 16;
          const bool in = s + i < step1 && off < row_bytes;
          v0[i] = in && in0 ? ldg_nc(w0 + off) : make_uint4(0, 0, 0, 0);
          v1[i] = in && in1 ? ldg_nc(w1 + off) : make_uint4(0, 0, 0, 0);
          xv[i] = in && x ? __ldg(reinterpret_cast<const uint4*>(x + off)) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          few_mma<FP8>(acc, v0[i].x, v1[i].x, v0[i].y, v1[i].y, xv[i].x, xv[i].y);
          few_mma<FP8>(acc, v0[i].z, v1[i].z, v0[i].w, v1[i].w, xv[i].z, xv[i].w);
        }
      }
    }
    // acc: outputs g and g + 8, positions 2 c and 2 c + 1
    auto finish = [&](float v, int n, int pos) {
      const int p = p0 + pos, row = a.rows ? row_of(a, p) : p;
      if (row < 0)
        v = 0.f;   // names no row: zeros whatever the bank holds
      else if (FP8)
        v = scaled(v, __ldg(a.x_scales + row), __ldg(a.w_scales + int64_t(e) * a.N + n));
      a.out[int64_t(p0 + pos) * a.ldo + n] = f32_to_bf16(v);
    };
    if (S == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int n = n0 + g + 8 * (i >> 1), pos = 2 * c + (i & 1);
        if (pos < count && n < a.N && tile < tiles) finish(acc[i], n, pos);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) part[warp][g + 8 * (i >> 1)][2 * c + (i & 1)] = acc[i];
      __syncthreads();
      // a thread an output and position: rows of 16 per tile of the stack
      for (int i = tid; i < per * kFewRows * count; i += kFewThreads) {
        const int pos = i / (per * kFewRows), r = i - pos * (per * kFewRows), t = r / kFewRows;
        const int n = (int(u - int64_t(item) * stacks) * per + t) * kFewRows + r % kFewRows;
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < S; ++q) v += part[t * S + q][r % kFewRows][pos];
        if (n < a.N) finish(v, n, pos);
      }
      __syncthreads();
    }
  }
}

// ---- host side --------------------------------------------------------------

template <bool FP8, int S>
static cudaError_t launch_few_as(const GroupedArgs& a, int64_t ctas, cudaStream_t st) {
  return launch_chained(grouped_few_kernel<FP8, S>, dim3(unsigned(ctas)), dim3(kFewThreads),
                        size_t(2 * (a.experts + 1)) * sizeof(int), st, a);
}

cudaError_t launch_grouped_few(const GroupedArgs& a, bool e4m3, cudaStream_t st) {
  const int64_t full = (a.P + kFewPos - 1) / kFewPos + a.experts, items = full < a.P ? full : a.P;
  const int64_t tiles = (a.N + kFewRows - 1) / kFewRows, sms = sm_count();
  if (items * tiles > 0x7FFFFFFF) return cudaErrorInvalidValue;
  // warps to a unit: one if the CTAs' stacks of units keep the SMs busy for
  // several rounds, else as many as give every resident CTA a stack
  auto ctas = [&](int s) { return items * ((tiles + kFewWarps / s - 1) / (kFewWarps / s)); };
  int S = 1;
  if (ctas(1) < 8 * sms)
    for (S = 2; S < 8 && ctas(S) < few_ctas(S) * sms;) S *= 2;
  const int64_t resident = few_ctas(S) * sms, n = ctas(S) < resident ? ctas(S) : resident;
  if (e4m3)
    return S == 1   ? launch_few_as<true, 1>(a, n, st)
           : S == 2 ? launch_few_as<true, 2>(a, n, st)
           : S == 4 ? launch_few_as<true, 4>(a, n, st)
                    : launch_few_as<true, 8>(a, n, st);
  return S == 1   ? launch_few_as<false, 1>(a, n, st)
         : S == 2 ? launch_few_as<false, 2>(a, n, st)
         : S == 4 ? launch_few_as<false, 4>(a, n, st)
                  : launch_few_as<false, 8>(a, n, st);
}

}  // namespace vx
