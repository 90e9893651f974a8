// Low-rank adapters of many requests beside one shared projection:
//
//   out[t] = bf16( y[t] + B_e (scale_e * A_e x_t) ),  e = adapters[t]
//
// with A [L][R][K], B [L][N][R] bf16 and only the first ranks[e] of the R
// components.  A token whose adapter is outside [0, L) gets out = y.
//
// Work items are up to TM = 16 * MT tokens of one adapter, whichever places
// of the batch they stand at.  A cluster of C CTAs shares an item: CTA i
// forms A_e x over its part of K, the cluster adds the parts (distributed
// shared memory, in CTA order), and CTA i writes its part of N.  Both
// products are bound by memory (2 TM flops per byte of A and B), so the
// operands go from global memory into mma.sync fragments without a stop in
// shared memory: the order of the inputs inside a fragment is free as long
// as both operands share it, so a lane reads 8 consecutive inputs at once.
//
// The inner values h = A_e x stay in float32 through both sums; for the
// second product they enter the MMA as two bf16 terms (h = hi + lo, 16 bits
// of mantissa), so what is lost is 2^-17 of h, and out is rounded once.
//
// Batches of at most kLoraSmall tokens group themselves inside the kernel
// (one launch); larger ones take their items from lora_group_kernel.
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

// v[0..7] of a bf16 row from column n on (n + 8 <= N when wide).
template <bool WIDE>
VX_DEVICE void load8(const uint16_t* row, int n, int N, float (&v)[8]) {
  if (WIDE) {
    uint4 w;   // y may be written in place: no read-only path
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "l"(row + n));
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = n + i < N ? bf16_to_f32(row[n + i]) : 0.f;
  }
}
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

// Shared memory: the warps' partial sums of a chunk of components, the CTA's
// sums [TM][R], the fragments of h (hi and lo) per 16 components.
__host__ __device__ constexpr int lora_part_floats(int tm, int R) {
  return kLoraWarps * tm * (R < kLoraRankChunk ? R : kLoraRankChunk);
}
static int lora_smem(int mt, int R) {
  const int tm = 16 * mt;
  return (lora_part_floats(tm, R) + tm * R) * 4 + (R + 15) / 16 * mt * 1024;
}

template <int MT, bool WIDE>
__global__ void __launch_bounds__(kLoraThreads, 2) lora_kernel(const LoraArgs a, const int32_t* __restrict__ order,
                                                               const int32_t* __restrict__ items) {
  chain_begin();
  constexpr int TM = 16 * MT;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ int tok[TM];          // the item's tokens, -1 behind the last
  __shared__ int s_ids[kLoraSmall], s_lead[kLoraWarps], s_item[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int C = int(lora_cluster_size()), cta = int(lora_cluster_rank());
  const int item = int(blockIdx.x) / C;

  int e;
  if (items) {
    if (item >= __ldg(items)) return;   // the whole cluster
    const int32_t* it = items + 1 + 3 * item;
    e = __ldg(it);
    if (tid < TM) tok[tid] = tid < __ldg(it + 2) ? __ldg(order + __ldg(it + 1) + tid) : -1;
    __syncthreads();
  } else {
    // Thread t: how many earlier tokens share its adapter.  Every TM-th token
    // of an adapter leads an item; items are numbered by their leaders.
    const int T = int(a.T);
    const int mine = tid < T ? lora_id(a, tid) : -2;
    s_ids[tid] = mine;
    if (tid < TM) tok[tid] = -1;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < tid; ++i) before += s_ids[i] == mine;
    const bool leads = tid < T && before % TM == 0;
    const uint32_t b = __ballot_sync(0xFFFFFFFFu, leads);
    if (lane == 0) s_lead[warp] = __popc(b);
    __syncthreads();
    int number = __popc(b & ((1u << lane) - 1u)), all = 0;
    for (int w = 0; w < kLoraWarps; ++w) {
      if (w < warp) number += s_lead[w];
      all += s_lead[w];
    }
    if (item >= all) return;   // the whole cluster
    if (leads && number == item) s_item[0] = mine, s_item[1] = before / TM;
    __syncthreads();
    e = s_item[0];
    if (tid < T && mine == e && before / TM == s_item[1]) tok[before % TM] = tid;
    __syncthreads();
  }
  const int rank = e < 0 ? 0 : a.ranks ? min(max(__ldg(a.ranks + e), 0), a.R) : a.R;

  float* part = reinterpret_cast<float*>(smem_raw);
  float* sums = part + lora_part_floats(TM, a.R);
  uint4* frag = reinterpret_cast<uint4*>(sums + TM * a.R);   // [16 components][MT][hi, lo][lane]

  // ---- h = A x over this CTA's 32-input blocks, 64 components at a time
  if (rank > 0) {
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
      for (int kb = cta * kLoraWarps + warp; kb < blocks; kb += C * kLoraWarps) {
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
  // ---- h of the whole item, as fragments: component q of 16 is input q/4 of
  // lane group q%4's four, like the lanes' reads of B
  const int kbs = (rank + 15) / 16;
  if (rank > 0) {
    if (C > 1) lora_cluster_sync();
    const float scale = a.scales ? __ldg(a.scales + e) : 1.0f;
    uint16_t* f = reinterpret_cast<uint16_t*>(frag);
    for (int i = tid; i < TM * kbs * 16; i += kLoraThreads) {
      const int row = i / (kbs * 16), r = i - row * (kbs * 16);
      float v = 0.f;
      if (r < rank) {
        if (C > 1) {
          for (int p = 0; p < C; ++p) v += peer_f32(sums + row * a.R + r, p);
        } else {
          v = sums[row * a.R + r];
        }
        v *= scale;
      }
      const uint16_t hi = f32_to_bf16(v);
      const bool finite = (hi & 0x7F80u) != 0x7F80u;
      const uint16_t lo = finite ? f32_to_bf16(v - bf16_to_f32(hi)) : uint16_t(0);
      const int q = r & 15, reg = (q & 2) + ((row & 15) >> 3), fl = (row & 7) * 4 + (q >> 2);
      const int at = (((r >> 4) * MT + (row >> 4)) * 2 * 32 + fl) * 8 + reg * 2 + (q & 1);
      f[at] = hi;
      f[at + 32 * 8] = lo;
    }
    if (C > 1)
      lora_cluster_sync();   // nobody leaves while its sums are read
    else
      __syncthreads();
  }

  // ---- out = y + B h, 32 outputs a warp and step.  Column q of MMA tile j is
  // output 8 (q/2) + 2 j + q%2 of the 32, so a lane ends up with 8 neighbours.
  const uint16_t* B = a.b + int64_t(e < 0 ? 0 : e) * a.N * a.R;
  int t[2 * MT];
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i) t[i] = tok[8 * i + g];
  for (int nb = cta * kLoraWarps + warp; nb * 32 < a.N; nb += C * kLoraWarps) {
    const int n = nb * 32 + 8 * c;
    float yv[2 * MT][8];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i)
      if (t[i] >= 0 && (!WIDE || n < a.N)) load8<WIDE>(a.y + t[i] * a.ldy, n, a.N, yv[i]);
    float acc[MT][4][4] = {};
    for (int kb0 = 0; kb0 < kbs; kb0 += 4) {
      uint2 bf[4][4];   // [16 components][tile]
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = nb * 32 + 8 * (g >> 1) + 2 * j + (g & 1), r = (kb0 + u) * 16 + 4 * c;
          uint2 v = make_uint2(0, 0);
          if (r < rank && row < a.N) {
            v = __ldg(reinterpret_cast<const uint2*>(B + int64_t(row) * a.R + r));
            const int left = rank - r;   // components behind the adapter's rank count as zero
            if (left < 4) {
              if (left < 2) v.x &= 0xFFFFu;
              v.y = left < 3 ? 0u : v.y & 0xFFFFu;
            }
          }
          bf[u][j] = v;
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
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
      if (rank > 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          yv[i][2 * j] += acc[i >> 1][j][2 * (i & 1)];
          yv[i][2 * j + 1] += acc[i >> 1][j][2 * (i & 1) + 1];
        }
      }
      store8<WIDE>(a.out + t[i] * a.ldo, n, a.N, yv[i]);
    }
  }
}

// ---- items of a large batch ---------------------------------------------------

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

static int64_t lora_max_items(const LoraArgs& a, int tm) {
  const int64_t full = (a.T + tm - 1) / tm + a.L + 1;
  return full < a.T ? full : a.T;
}

constexpr int kLoraLargeTm = 32;

int64_t lora_workspace_bytes(int64_t T, int L) {
  if (T <= kLoraSmall) return 0;
  LoraArgs a = {};
  a.T = T;
  a.L = L;
  return (2 * T + 1 + 3 * lora_max_items(a, kLoraLargeTm)) * int64_t(sizeof(int32_t));
}

template <int MT, bool WIDE>
static cudaError_t launch_lora_as(const LoraArgs& a, const int32_t* order, const int32_t* items, cudaStream_t st) {
  const int64_t n = lora_max_items(a, 16 * MT);
  // CTAs to an item: as many as keep the whole grid within two rounds of two
  // CTAs per SM (a cluster's barriers cost more than idle SMs above that)
  int C = 8;
  while (C > 1 && n * C > 4 * int64_t(sm_count())) C /= 2;
  if (n * C > 0x7FFFFFFF) return cudaErrorInvalidValue;
  auto k = lora_kernel<MT, WIDE>;
  const int smem = lora_smem(MT, a.R);
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(k), lora_smem(MT, kLoraMaxRank), done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(n * C));
  cfg.blockDim = dim3(kLoraThreads);
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(C);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = chain_enabled(false) ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, k, a, order, items);
}

cudaError_t launch_lora(const LoraArgs& a, void* workspace, cudaStream_t st) {
  if (a.T == 0 || a.N == 0) return cudaSuccess;
  auto aligned = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; };
  const bool wide = a.N % 8 == 0 && aligned(a.y, a.T > 1 ? a.ldy : 0) && aligned(a.out, a.T > 1 ? a.ldo : 0);
  if (a.T <= kLoraSmall)
    return wide ? launch_lora_as<1, true>(a, nullptr, nullptr, st) : launch_lora_as<1, false>(a, nullptr, nullptr, st);
  int32_t* order = static_cast<int32_t*>(workspace);
  int32_t *place = order + a.T, *items = place + a.T;
  cudaError_t e = launch_chained(lora_group_kernel, dim3(1), dim3(kGroupThreads),
                                 size_t(2 * a.L + 3) * sizeof(int), st, a, kLoraLargeTm, place, order, items);
  if (e != cudaSuccess) return e;
  return wide ? launch_lora_as<kLoraLargeTm / 16, true>(a, order, items, st)
              : launch_lora_as<kLoraLargeTm / 16, false>(a, order, items, st);
}

}  // namespace vx
