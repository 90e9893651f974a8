// Low-rank adapters of many requests beside one shared projection:
//
//   out[t] = bf16( y[t] + B_e (scale_e * A_e x_t) ),  e = adapters[t]
//
// with A [L][R][K], B [L][N][R] bf16 and only the first ranks[e] of the R
// components.  A token whose adapter is outside [0, L) gets out = y.
//
// Work items are up to TM = 16 * MT tokens of one adapter, whichever places
// of the batch they stand at.  Both products are bound by memory (2 TM flops
// per byte of A and B), so the operands go from global memory into mma.sync
// fragments without a stop in shared memory: the order of the inputs inside a
// fragment is free as long as both operands share it, so a lane reads 8
// consecutive inputs at once.
//
// The inner values h = A_e x stay in float32 through their sums; for the
// second product they enter the MMA as two bf16 terms (h = hi + lo, 16 bits
// of mantissa), so what is lost is 2^-17 of h, and out is rounded once.
//
// Up to kLoraSmall tokens: one launch.  The batch is grouped inside the
// kernel; a cluster of C CTAs shares an item of 16 tokens: CTA i forms A_e x
// over its part of K, the cluster adds the parts (distributed shared memory,
// in CTA order), and CTA i writes its part of N.  B and y are on their way
// (L2 prefetches, then registers) while h is being summed.
//
// Above: lora_group_kernel sorts the batch into items of 32 tokens,
// lora_shrink_kernel (a CTA an item) writes h as bf16 pairs, and
// lora_expand_kernel (a CTA an item and kExpandCols outputs) streams y.
#include "vx_common.cuh"
#include "vx_launch.h"

namespace vx {

constexpr int kLoraThreads = 256;
constexpr int kLoraWarps = kLoraThreads / 32;
constexpr int kLoraRankChunk = 64;     // components whose sums a warp holds in registers
constexpr int kLoraSmall = kLoraThreads;

VX_DEVICE uint32_t lora_cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
VX_DEVICE uint32_t lora_cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
VX_DEVICE void lora_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
VX_DEVICE float peer_f32(const float* p, uint32_t rank) {   // the same place in CTA `rank`
  const uint32_t own = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  uint32_t addr;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(own), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

VX_DEVICE int lora_id(const LoraArgs& a, int64_t t) {
  const int e = __ldg(a.adapters + t);
  return e >= 0 && e < a.L ? e : -1;
}

// Eight neighbouring values of a row of y, from column n on.  WIDE: 16-byte
// aligned and n + 8 <= N.  y may be written in place, so no read-only path.
template <bool WIDE>
struct Eight {
  uint32_t w[WIDE ? 4 : 8];
  VX_DEVICE void load(const uint16_t* row, int n, int N) {
    if (WIDE) {
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                   : "l"(row + n)
                   : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = n + i < N ? uint32_t(row[n + i]) << 16 : 0u;
    }
  }
  VX_DEVICE float get(int i) const {
    if (WIDE) return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
    return __uint_as_float(w[i]);
  }
};
VX_DEVICE uint32_t lora_bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <bool WIDE>
VX_DEVICE void store8(uint16_t* row, int n, int N, const float (&v)[8]) {
  if (WIDE) {
    *reinterpret_cast<uint4*>(row + n) = make_uint4(lora_bf16x2(v[0], v[1]), lora_bf16x2(v[2], v[3]),
                                                    lora_bf16x2(v[4], v[5]), lora_bf16x2(v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < N) row[n + i] = uint16_t(lora_bf16x2(v[i], 0.f));
  }
}

__host__ __device__ constexpr int lora_part_floats(int tm, int R) {   // the warps' sums of a rank chunk
  return kLoraWarps * tm * (R < kLoraRankChunk ? R : kLoraRankChunk);
}
__host__ __device__ constexpr int lora_frag_bytes(int mt, int R) { return (R + 15) / 16 * mt * 1024; }

// Components of adapter e that count.
VX_DEVICE int lora_rank(const LoraArgs& a, int e) {
  return e < 0 ? 0 : a.ranks ? min(max(__ldg(a.ranks + e), 0), a.R) : a.R;
}

// sums[row][r] (TM x R floats) = A_e x over the 32-input blocks first, first
// + stride, ... of the CTA's warps; part: lora_part_floats.
template <int MT>
VX_DEVICE void lora_shrink(const LoraArgs& a, int e, int rank, const int* tok, int first, int stride, float* part,
                           float* sums) {
  constexpr int TM = 16 * MT;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const uint16_t* xrow[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    const int t = tok[8 * i + g];
    xrow[i] = t >= 0 ? a.x + t * a.ldx : nullptr;
  }
  const uint16_t* A = a.a + int64_t(e) * a.R * a.K;
  const int blocks = (a.K + 31) / 32;
  for (int r0 = 0; r0 < rank; r0 += kLoraRankChunk) {
    const int cols = min(kLoraRankChunk, rank - r0), tiles = (cols + 7) / 8;
    float acc[MT][8][4] = {};
    for (int kb = first; kb < blocks; kb += stride) {
      const int k = kb * 32 + c * 8;
      uint4 xf[2 * MT], af[8];
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i)
        xf[i] = xrow[i] && k < a.K ? ldg_nc(xrow[i] + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = r0 + 8 * j + g;
        af[j] = j < tiles && r < rank && k < a.K ? ldg_nc(A + int64_t(r) * a.K + k) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j >= tiles) break;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          mma16816(acc[m][j], xf[2 * m].x, xf[2 * m + 1].x, xf[2 * m].y, xf[2 * m + 1].y, af[j].x, af[j].y);
          mma16816(acc[m][j], xf[2 * m].z, xf[2 * m + 1].z, xf[2 * m].w, xf[2 * m + 1].w, af[j].z, af[j].w);
        }
      }
    }
    const int pitch = min(kLoraRankChunk, a.R);
    float* mine = part + warp * TM * pitch;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j >= tiles) break;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float* p = mine + (16 * m + g) * pitch + 8 * j + 2 * c;
        *reinterpret_cast<float2*>(p) = make_float2(acc[m][j][0], acc[m][j][1]);
        *reinterpret_cast<float2*>(p + 8 * pitch) = make_float2(acc[m][j][2], acc[m][j][3]);
      }
    }
    __syncthreads();
    for (int i = tid; i < TM * tiles * 8; i += kLoraThreads) {
      const int row = i / (tiles * 8), col = i - row * (tiles * 8);
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kLoraWarps; ++w) s += part[(w * TM + row) * pitch + col];
      sums[row * a.R + r0 + col] = s;
    }
    __syncthreads();
  }
}

// v = hi + lo in bf16 (lo zero where hi is no finite number).
VX_DEVICE void lora_split(float v, uint16_t* hi, uint16_t* lo) {
  *hi = f32_to_bf16(v);
  *lo = (*hi & 0x7F80u) != 0x7F80u ? f32_to_bf16(v - bf16_to_f32(*hi)) : uint16_t(0);
}
// Place of h's component r of item row `row` in the fragments [16 components]
// [MT][hi, lo][lane][8 halves]: component q of 16 belongs to the lanes q/4 of
// four, like their reads of B; the lo half lies 256 halves on.
template <int MT>
VX_DEVICE int lora_frag_at(int row, int r) {
  const int q = r & 15, reg = (q & 2) + ((row & 15) >> 3), lane = (row & 7) * 4 + (q >> 2);
  return (((r >> 4) * MT + (row >> 4)) * 64 + lane) * 8 + reg * 2 + (q & 1);
}

// B of one 32-output block: kExpandKb blocks of 16 components x 4 MMA tiles.
// Column q of MMA tile j is output 8 (q/2) + 2 j + q%2 of the 32, so a lane
// ends up with 8 neighbours.  Components from `rank` on count as zero.
constexpr int kExpandKb = 2;
VX_DEVICE void load_b(const LoraArgs& a, const uint16_t* B, int rank, int nb, int kb0, uint2 (&bf)[kExpandKb][4]) {
  const int g = (threadIdx.x & 31) >> 2, c = threadIdx.x & 3;
#pragma unroll
  for (int u = 0; u < kExpandKb; ++u) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = nb * 32 + 8 * (g >> 1) + 2 * j + (g & 1), r = (kb0 + u) * 16 + 4 * c;
      uint2 v = make_uint2(0, 0);
      if (r < rank && row < a.N) {
        v = __ldg(reinterpret_cast<const uint2*>(B + int64_t(row) * a.R + r));
        const int left = rank - r;
        if (left < 4) {
          if (left < 2) v.x &= 0xFFFFu;
          v.y = left < 3 ? 0u : v.y & 0xFFFFu;
        }
      }
      bf[u][j] = v;
    }
  }
}
template <int MT, bool WIDE>
VX_DEVICE void load_y(const LoraArgs& a, const int (&t)[2 * MT], int nb, Eight<WIDE> (&y)[2 * MT]) {
  const int n = nb * 32 + 8 * (threadIdx.x & 3);
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i)
    if (t[i] >= 0 && (!WIDE || n < a.N)) y[i].load(a.y + t[i] * a.ldy, n, a.N);
}
// out = y + B h for one block whose y and first B are loaded.
template <int MT, bool WIDE>
VX_DEVICE void lora_expand(const LoraArgs& a, const uint16_t* B, int rank, const uint4* frag, const int (&t)[2 * MT],
                           int nb, const Eight<WIDE> (&y)[2 * MT], uint2 (&bf)[kExpandKb][4]) {
  const int lane = threadIdx.x & 31, n = nb * 32 + 8 * (lane & 3), kbs = (rank + 15) / 16;
  float acc[MT][4][4] = {};
  for (int kb0 = 0; kb0 < kbs; kb0 += kExpandKb) {
    if (kb0 > 0) load_b(a, B, rank, nb, kb0, bf);
#pragma unroll
    for (int u = 0; u < kExpandKb; ++u) {
      if (kb0 + u >= kbs) break;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint4* h = frag + ((kb0 + u) * MT + m) * 64 + lane;
        const uint4 hi = h[0], lo = h[32];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mma16816(acc[m][j], hi.x, hi.y, hi.z, hi.w, bf[u][j].x, bf[u][j].y);
          mma16816(acc[m][j], lo.x, lo.y, lo.z, lo.w, bf[u][j].x, bf[u][j].y);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) {
    if (t[i] < 0 || (WIDE && n >= a.N)) continue;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = y[i].get(j);
      if (rank > 0) v[j] += acc[i >> 1][j >> 1][2 * (i & 1) + (j & 1)];
    }
    store8<WIDE>(a.out + t[i] * a.ldo, n, a.N, v);
  }
}

// ---- small batches: one launch ------------------------------------------------

static int lora_small_smem(int R) { return (lora_part_floats(16, R) + 16 * R) * 4 + lora_frag_bytes(1, R); }

template <bool WIDE>
__global__ void __launch_bounds__(kLoraThreads, 2) lora_small_kernel(const LoraArgs a) {
  chain_begin();
  constexpr int TM = 16;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ int tok[TM];          // the item's tokens, -1 behind the last
  __shared__ __align__(16) int s_ids[kLoraSmall];
  __shared__ int s_lead[kLoraWarps], s_item[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = int(lora_cluster_size()), cta = int(lora_cluster_rank());
  const int item = int(blockIdx.x) / C, T = int(a.T);

  // Thread t: how many earlier tokens share its adapter.  Every TM-th token
  // of an adapter leads an item; items are numbered by their leaders.
  const int mine = tid < T ? lora_id(a, tid) : -2;
  s_ids[tid] = mine;
  if (tid < TM) tok[tid] = -1;
  int before = __popc(__match_any_sync(0xFFFFFFFFu, mine) & ((1u << lane) - 1u));
  __syncthreads();
  if (tid < T) {
    for (int i = 0; i < warp * 8; ++i) {
      const int4 v = reinterpret_cast<const int4*>(s_ids)[i];
      before += (v.x == mine) + (v.y == mine) + (v.z == mine) + (v.w == mine);
    }
  }
  const bool leads = tid < T && before % TM == 0;
  const uint32_t b = __ballot_sync(0xFFFFFFFFu, leads);
  if (lane == 0) s_lead[warp] = __popc(b);
  __syncthreads();
  int number = __popc(b & ((1u << lane) - 1u)), all = 0;
#pragma unroll
  for (int w = 0; w < kLoraWarps; ++w) {
    if (w < warp) number += s_lead[w];
    all += s_lead[w];
  }
  if (item >= all) return;   // the whole cluster
  if (leads && number == item) s_item[0] = mine, s_item[1] = before / TM;
  __syncthreads();
  const int e = s_item[0];
  if (tid < T && mine == e && before / TM == s_item[1]) tok[before % TM] = tid;
  __syncthreads();
  const int rank = lora_rank(a, e);

  float* part = reinterpret_cast<float*>(smem_raw);
  float* sums = part + lora_part_floats(TM, a.R);
  uint4* frag = reinterpret_cast<uint4*>(sums + TM * a.R);
  const uint16_t* B = a.b + int64_t(e < 0 ? 0 : e) * a.N * a.R;
  const int nb0 = cta * kLoraWarps + warp, stride = C * kLoraWarps;
  // lane i: row i of the blocks of B that this warp reads later
  for (int nb = nb0; nb * 32 < a.N; nb += stride) {
    if (nb * 32 + lane < a.N)
      for (int r = 0; r < rank; r += 64)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(B + int64_t(nb * 32 + lane) * a.R + r));
  }
  if (rank > 0) lora_shrink<1>(a, e, rank, tok, nb0, stride, part, sums);

  int t[2];
  Eight<WIDE> y[2];
  uint2 bf[kExpandKb][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) t[i] = tok[8 * i + (lane >> 2)];
  if (nb0 * 32 < a.N) {
    load_y<1, WIDE>(a, t, nb0, y);
    load_b(a, B, rank, nb0, 0, bf);
  }
  // h of the whole item
  if (rank > 0) {
    if (C > 1) lora_cluster_sync();
    const int cols = (rank + 15) & ~15;
    const float scale = a.scales ? __ldg(a.scales + e) : 1.0f;
    uint16_t* f = reinterpret_cast<uint16_t*>(frag);
    for (int i = tid; i < TM * cols; i += kLoraThreads) {
      const int row = i / cols, r = i - row * cols;
      float v = 0.f;
      if (r < rank) {
        if (C == 8) {   // all parts on their way before the first is added
          float p[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) p[q] = peer_f32(sums + row * a.R + r, q);
#pragma unroll
          for (int q = 0; q < 8; ++q) v += p[q];
        } else {
          for (int q = 0; q < C; ++q) v += peer_f32(sums + row * a.R + r, q);
        }
      }
      uint16_t* at = f + lora_frag_at<1>(row, r);
      lora_split(v * scale, at, at + 256);
    }
    if (C > 1)
      lora_cluster_sync();   // nobody leaves while its sums are read
    else
      __syncthreads();
  }
  for (int nb = nb0; nb * 32 < a.N; nb += stride) {
    if (nb != nb0) {
      load_y<1, WIDE>(a, t, nb, y);
      load_b(a, B, rank, nb, 0, bf);
    }
    lora_expand<1, WIDE>(a, B, rank, frag, t, nb, y, bf);
  }
}

// ---- large batches ------------------------------------------------------------

constexpr int kLargeMt = 2, kLargeTm = 16 * kLargeMt;
constexpr int kExpandCols = 512;       // outputs of an expanding CTA

// An item of lora_group_kernel: {adapter or -1, first place of `order`, tokens}.
struct LoraItem {
  int e, begin, n;
};
VX_DEVICE LoraItem lora_item(const int32_t* items, int i) {
  const int32_t* p = items + 1 + 3 * i;
  return {__ldg(p), __ldg(p + 1), __ldg(p + 2)};
}

static int lora_shrink_smem(int R) { return (lora_part_floats(kLargeTm, R) + kLargeTm * R) * 4; }

// h [place of order][16 components][hi, lo][16] of every item.
__global__ void __launch_bounds__(kLoraThreads, 2) lora_shrink_kernel(const LoraArgs a,
                                                                      const int32_t* __restrict__ order,
                                                                      const int32_t* __restrict__ items,
                                                                      uint16_t* __restrict__ h) {
  chain_begin();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ int tok[kLargeTm];
  const int tid = threadIdx.x;
  if (int(blockIdx.x) >= __ldg(items)) return;
  const LoraItem it = lora_item(items, blockIdx.x);
  const int rank = lora_rank(a, it.e);
  if (rank == 0) return;
  if (tid < kLargeTm) tok[tid] = tid < it.n ? __ldg(order + it.begin + tid) : -1;
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem_raw);
  float* sums = part + lora_part_floats(kLargeTm, a.R);
  lora_shrink<kLargeMt>(a, it.e, rank, tok, tid >> 5, kLoraWarps, part, sums);
  const int cols = (rank + 15) & ~15, pitch = ((a.R + 15) & ~15) * 2;
  const float scale = a.scales ? __ldg(a.scales + it.e) : 1.0f;
  for (int i = tid; i < it.n * cols; i += kLoraThreads) {
    const int row = i / cols, r = i - row * cols;
    uint16_t* p = h + int64_t(it.begin + row) * pitch + (r >> 4) * 32 + (r & 15);
    lora_split(r < rank ? sums[row * a.R + r] * scale : 0.f, p, p + 16);
  }
}

template <bool WIDE>
__global__ void __launch_bounds__(kLoraThreads, 3) lora_expand_kernel(const LoraArgs a,
                                                                      const int32_t* __restrict__ order,
                                                                      const int32_t* __restrict__ items,
                                                                      const uint16_t* __restrict__ h) {
  chain_begin();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (int(blockIdx.x) >= __ldg(items)) return;
  const LoraItem it = lora_item(items, blockIdx.x);
  const int rank = lora_rank(a, it.e);
  int t[2 * kLargeMt];
#pragma unroll
  for (int i = 0; i < 2 * kLargeMt; ++i) {
    const int row = 8 * i + (lane >> 2);
    t[i] = row < it.n ? __ldg(order + it.begin + row) : -1;
  }
  // the fragments: thread = 4 components of a row, hi or lo
  uint4* frag = reinterpret_cast<uint4*>(smem_raw);
  const int kbs = (rank + 15) / 16, pitch = ((a.R + 15) & ~15) * 2;
  for (int i = tid; i < kLargeTm * kbs * 8; i += kLoraThreads) {
    const int row = i / (kbs * 8), piece = i - row * (kbs * 8), kb = piece >> 3, lo = (piece >> 2) & 1, q = piece & 3;
    uint2 v = make_uint2(0, 0);
    if (row < it.n)
      v = *reinterpret_cast<const uint2*>(h + int64_t(it.begin + row) * pitch + kb * 32 + lo * 16 + q * 4);
    uint32_t* p = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(frag) +
                                              lora_frag_at<kLargeMt>(row, kb * 16 + q * 4) + lo * 256);
    p[0] = v.x;   // components 0, 1 of the four
    p[2] = v.y;   // 2, 3: two registers on
  }
  __syncthreads();
  const uint16_t* B = a.b + int64_t(it.e < 0 ? 0 : it.e) * a.N * a.R;
  const int end = min(a.N, int(blockIdx.y + 1) * kExpandCols);
  for (int nb = int(blockIdx.y) * (kExpandCols / 32) + warp; nb * 32 < end; nb += kLoraWarps) {
    Eight<WIDE> y[2 * kLargeMt];
    uint2 bf[kExpandKb][4];
    load_y<kLargeMt, WIDE>(a, t, nb, y);
    load_b(a, B, rank, nb, 0, bf);
    lora_expand<kLargeMt, WIDE>(a, B, rank, frag, t, nb, y, bf);
  }
}

// One CTA: tokens counted per adapter (bucket L: none), buckets cut into
// items of TM tokens.  items: the count, then {adapter, first place of
// `order`, tokens} each.  The order inside a bucket does not matter: a
// token's sums are the same whichever row of an item it takes.
constexpr int kGroupThreads = 1024;

__global__ void __launch_bounds__(kGroupThreads) lora_group_kernel(const LoraArgs a, int tm, int32_t* __restrict__ place,
                                                                   int32_t* __restrict__ order,
                                                                   int32_t* __restrict__ items) {
  chain_begin();
  extern __shared__ int s_cnt[];                 // [L+1] tokens, then first place; [L+2] first item
  int* s_first = s_cnt + a.L + 1;
  __shared__ int2 s_warp[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int buckets = a.L + 1;
  const int64_t T = a.T;
  for (int i = tid; i < buckets; i += kGroupThreads) s_cnt[i] = 0;
  __syncthreads();
  for (int64_t t0 = 0; t0 < T; t0 += kGroupThreads) {
    const int64_t t = t0 + tid;
    const bool in = t < T;
    const int e = in ? lora_id(a, t) : -2, b = e == -1 ? a.L : e;
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, b);
    int base = 0;
    const int first = __ffs(same) - 1;
    if (in && lane == first) base = atomicAdd(&s_cnt[b], __popc(same));
    base = __shfl_sync(0xFFFFFFFFu, base, first);
    if (in) place[t] = base + __popc(same & ((1u << lane) - 1u));
  }
  __syncthreads();
  // exclusive scans of tokens and items over the buckets
  const int per = (buckets + kGroupThreads - 1) / kGroupThreads;
  int2 own = make_int2(0, 0);
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i, n = b < buckets ? s_cnt[b] : 0;
    own.x += n;
    own.y += (n + tm - 1) / tm;
  }
  int2 inc = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xFFFFFFFFu, inc.x, o), y = __shfl_up_sync(0xFFFFFFFFu, inc.y, o);
    if (lane >= o) inc.x += x, inc.y += y;
  }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  int2 at = make_int2(inc.x - own.x, inc.y - own.y);
  int total = 0;
  for (int w = 0; w < 32; ++w) {
    if (w < warp) at.x += s_warp[w].x, at.y += s_warp[w].y;
    total += s_warp[w].y;
  }
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i;
    if (b >= buckets) break;
    const int n = s_cnt[b];
    s_cnt[b] = at.x;
    s_first[b] = at.y;
    at.x += n;
    at.y += (n + tm - 1) / tm;
  }
  if (tid == 0) items[0] = total, s_first[buckets] = total;
  __syncthreads();
  for (int64_t t = tid; t < T; t += kGroupThreads) {
    const int e = lora_id(a, t);
    order[s_cnt[e < 0 ? a.L : e] + place[t]] = int32_t(t);
  }
  for (int i = tid; i < total; i += kGroupThreads) {
    int lo = 0, hi = buckets;   // the last bucket with s_first <= i: the one that holds item i
    while (hi - lo > 1) {
      const int m = (lo + hi) >> 1;
      if (s_first[m] <= i) lo = m; else hi = m;
    }
    const int begin = s_cnt[lo] + (i - s_first[lo]) * tm;
    const int end = lo + 1 < buckets ? s_cnt[lo + 1] : int(T);
    items[1 + 3 * i] = lo == a.L ? -1 : lo;
    items[2 + 3 * i] = begin;
    items[3 + 3 * i] = min(tm, end - begin);
  }
}

// ---- host side --------------------------------------------------------------

static int64_t lora_max_items(int64_t T, int L, int tm) {
  const int64_t full = (T + tm - 1) / tm + L + 1;
  return full < T ? full : T;
}

// Workspace of a large batch: order, place, items, h.
struct LoraSpace {
  int64_t place, items, h, bytes;   // offsets; order comes first
};
static LoraSpace lora_space(int64_t T, int L, int R) {
  auto up = [](int64_t n) { return (n + 255) & ~int64_t(255); };
  LoraSpace s;
  s.place = up(4 * T);
  s.items = s.place + up(4 * T);
  s.h = s.items + up(4 * (1 + 3 * lora_max_items(T, L, kLargeTm)));
  s.bytes = s.h + T * ((R + 15) / 16 * 64);
  return s;
}
int64_t lora_workspace_bytes(int64_t T, int L, int R) { return T <= kLoraSmall ? 0 : lora_space(T, L, R).bytes; }

template <bool WIDE>
static cudaError_t launch_lora_small(const LoraArgs& a, cudaStream_t st) {
  const int64_t n = lora_max_items(a.T, a.L, 16);
  // CTAs to an item: as many as keep the whole grid within two rounds of two
  // CTAs per SM
  int C = 8;
  while (C > 1 && n * C > 4 * int64_t(sm_count())) C /= 2;
  auto k = lora_small_kernel<WIDE>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(k), lora_small_smem(kLoraMaxRank), done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(n * C));
  cfg.blockDim = dim3(kLoraThreads);
  cfg.dynamicSmemBytes = size_t(lora_small_smem(a.R));
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(C);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = chain_enabled(false) ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, k, a);
}

template <bool WIDE>
static cudaError_t launch_lora_large(const LoraArgs& a, char* ws, cudaStream_t st) {
  const LoraSpace sp = lora_space(a.T, a.L, a.R);
  int32_t *order = reinterpret_cast<int32_t*>(ws), *place = reinterpret_cast<int32_t*>(ws + sp.place),
          *items = reinterpret_cast<int32_t*>(ws + sp.items);
  uint16_t* h = reinterpret_cast<uint16_t*>(ws + sp.h);
  const unsigned n = unsigned(lora_max_items(a.T, a.L, kLargeTm));
  static std::atomic<uint64_t> done1{0}, done2{0};
  auto expand = lora_expand_kernel<WIDE>;
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(lora_shrink_kernel), lora_shrink_smem(kLoraMaxRank), done1);
  if (e == cudaSuccess)
    e = allow_smem(reinterpret_cast<const void*>(expand), lora_frag_bytes(kLargeMt, kLoraMaxRank), done2);
  if (e == cudaSuccess)
    e = launch_chained(lora_group_kernel, dim3(1), dim3(kGroupThreads), size_t(2 * a.L + 3) * sizeof(int), st, a,
                       kLargeTm, place, order, items);
  if (e == cudaSuccess)
    e = launch_chained(lora_shrink_kernel, dim3(n), dim3(kLoraThreads), size_t(lora_shrink_smem(a.R)), st, a, order,
                       items, h);
  if (e == cudaSuccess)
    e = launch_chained(expand, dim3(n, unsigned((a.N + kExpandCols - 1) / kExpandCols)), dim3(kLoraThreads),
                       size_t(lora_frag_bytes(kLargeMt, a.R)), st, a, order, items, h);
  return e;
}

cudaError_t launch_lora(const LoraArgs& a, void* workspace, cudaStream_t st) {
  if (a.T == 0 || a.N == 0) return cudaSuccess;
  auto aligned = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; };
  const bool wide = a.N % 8 == 0 && aligned(a.y, a.T > 1 ? a.ldy : 0) && aligned(a.out, a.T > 1 ? a.ldo : 0);
  if (a.T <= kLoraSmall) return wide ? launch_lora_small<true>(a, st) : launch_lora_small<false>(a, st);
  if ((a.N + kExpandCols - 1) / kExpandCols > 65535) return cudaErrorInvalidValue;
  char* ws = static_cast<char*>(workspace);
  return wide ? launch_lora_large<true>(a, ws, st) : launch_lora_large<false>(a, ws, st);
}

}  // namespace vx
