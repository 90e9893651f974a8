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
// over its part of K and stores it into the shared memory of every CTA
// (st.async on the receiver's mbarrier: a cluster barrier costs 1,400 cycles,
// and two would stand here), each adds the parts in CTA order, and CTA i
// writes its part of N.  B and y are on their way while h is being summed.
//
// Above: lora_group_kernel sorts the batch into items of 32 tokens,
// lora_shrink_kernel (a CTA an item and 32 components) writes h as bf16 pairs, and
// lora_expand_kernel (a CTA an item and 512 to 4,096 outputs) streams y.
#include "vx_async.cuh"
#include "vx_common.cuh"
#include "vx_launch.h"

namespace vx {

constexpr int kLoraThreads = 256;
constexpr int kLoraWarps = kLoraThreads / 32;
constexpr int kLoraSmall = VX_LORA_SMALL;
static_assert(kLoraSmall <= kLoraThreads, "a thread a token");

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
VX_DEVICE void lora_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
VX_DEVICE void lora_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Four floats to the same place in CTA `rank`, counted on its barrier `bar`.
VX_DEVICE void push4(const float* p, uint64_t* bar, uint32_t rank, float4 v) {
  uint32_t to, on;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(p)), "r"(rank));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(on) : "r"(smem_u32(bar)), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to),
               "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(on)
               : "memory");
}
// Bounded wait for phase 0 of `bar` (false after a second).
VX_DEVICE bool lora_wait(uint64_t* bar) {
  const uint64_t t0 = global_ns();
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0; selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(smem_u32(bar))
        : "memory");
    if (ok) return true;
    if ((i & 255) == 255 && global_ns() - t0 > kWaitLimitNs) return false;
  }
  return false;
}

VX_DEVICE int lora_id(const LoraArgs& a, int64_t t) {
  const int e = __ldg(a.adapters + t);
  return e >= 0 && e < a.L ? e : -1;
}

// A lane's eight values of a row of y in a block of 32 outputs.  WIDE: eight
// neighbours, 16-byte aligned.  Else value i is output 8 (i / 2) + 4 (i % 2) + c
// for lane c of four, so that a load of four lanes is four neighbours (8,192
// tokens x 2,047 outputs 103 us, 128 with eight neighbours a lane).  y may be
// written in place, so no read-only path.
template <bool WIDE>
VX_DEVICE int first_of(int nb) {
  return nb * 32 + (WIDE ? 8 : 1) * int(threadIdx.x & 3);
}
VX_DEVICE int narrow_at(int n, int i) { return n + 8 * (i >> 1) + 4 * (i & 1); }
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
      for (int i = 0; i < 8; ++i) w[i] = narrow_at(n, i) < N ? uint32_t(row[narrow_at(n, i)]) << 16 : 0u;
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
      if (narrow_at(n, i) < N) row[narrow_at(n, i)] = uint16_t(lora_bf16x2(v[i], 0.f));
  }
}

__host__ __device__ constexpr int lora_frag_bytes(int mt, int R) { return (R + 31) / 32 * mt * 2048; }

// Components of adapter e that count.
VX_DEVICE int lora_rank(const LoraArgs& a, int e) {
  return e < 0 ? 0 : a.ranks ? min(max(__ldg(a.ranks + e), 0), a.R) : a.R;
}

// A_e x of the item's n tokens over the 32-input blocks first, first + stride,
// ... of the CTA's warps, 8 * NT components at a time, those from r_first,
// r_first + r_step, ...; out(row, r, v) gets four neighbouring sums of the CTA.
// part: the warps' sums, 128 MT NT floats each.  AHEAD: the next block's
// operands are loaded before the present one's MMAs.  ready() is called by
// every thread once, before the first out().
template <int MT, int NT, bool AHEAD, typename G, typename F>
VX_DEVICE void lora_shrink(const LoraArgs& a, int e, int rank, int r_first, int r_step, const int* tok, int n,
                           int first, int stride, float* part, G&& ready, F&& out) {
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
  for (int r0 = r_first; r0 < rank; r0 += r_step) {
    const int tiles = (min(8 * NT, rank - r0) + 7) / 8;
    float acc[MT][NT][4] = {};
    auto load = [&](int kb, uint4 (&xf)[2 * MT], uint4 (&af)[NT]) {
      const int k = kb * 32 + c * 8;
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i)
        xf[i] = xrow[i] && k < a.K ? ldg_nc(xrow[i] + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int r = r0 + 8 * j + g;
        af[j] = r < rank && k < a.K ? ldg_nc(A + int64_t(r) * a.K + k) : make_uint4(0, 0, 0, 0);
      }
    };
    auto multiply = [&](const uint4 (&xf)[2 * MT], const uint4 (&af)[NT]) {
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if (j >= tiles) break;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          mma16816(acc[m][j], xf[2 * m].x, xf[2 * m + 1].x, xf[2 * m].y, xf[2 * m + 1].y, af[j].x, af[j].y);
          mma16816(acc[m][j], xf[2 * m].z, xf[2 * m + 1].z, xf[2 * m].w, xf[2 * m + 1].w, af[j].z, af[j].w);
        }
      }
    };
    uint4 xf[2 * MT], af[NT];
    if constexpr (AHEAD) {
      uint4 xn[2 * MT], an[NT];
      int kb = first;
      if (kb < blocks) load(kb, xf, af);
      while (kb < blocks) {   // two blocks a turn, so that neither set is copied
        if (kb + stride < blocks) load(kb + stride, xn, an);
        multiply(xf, af);
        kb += stride;
        if (kb >= blocks) break;
        if (kb + stride < blocks) load(kb + stride, xf, af);
        multiply(xn, an);
        kb += stride;
      }
    } else {
      for (int kb = first; kb < blocks; kb += stride) {
        load(kb, xf, af);
        multiply(xf, af);
      }
    }
    constexpr int kPitch = 8 * NT;
    float* mine = part + warp * TM * kPitch;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      if (j >= tiles) break;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float* p = mine + (16 * m + g) * kPitch + 8 * j + 2 * c;
        *reinterpret_cast<float2*>(p) = make_float2(acc[m][j][0], acc[m][j][1]);
        *reinterpret_cast<float2*>(p + 8 * kPitch) = make_float2(acc[m][j][2], acc[m][j][3]);
      }
    }
    __syncthreads();
    if (r0 == r_first) ready();
    for (int i = tid; i < n * 2 * NT; i += kLoraThreads) {
      const int row = i / (2 * NT), col = i % (2 * NT) * 4;
      if (col >= tiles * 8) continue;
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kLoraWarps; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(part + (w * TM + row) * kPitch + col);
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      }
      out(row, r0 + col, s);
    }
    __syncthreads();
  }
}

// v = hi + lo in bf16 (lo zero where v is no finite number).  A finite v that
// would round to an infinity takes the largest bf16 as hi.
VX_DEVICE void lora_split(float v, uint16_t* hi, uint16_t* lo) {
  *hi = f32_to_bf16(v);
  if ((*hi & 0x7FFFu) == 0x7F80u && fabsf(v) <= 0x1.fffffep127f) *hi -= 1;
  *lo = (*hi & 0x7F80u) != 0x7F80u ? f32_to_bf16(v - bf16_to_f32(*hi)) : uint16_t(0);
}
// Place of h's component r of item row `row` in the fragments [16 components]
// [MT][hi, lo][lane][8 halves].  Of every 32 components the lanes c of four
// own 8 c .. 8 c + 7, as one 16-byte read of B brings them: the first four in
// the first MMA's 16, the others in the second's.  lo lies 256 halves on.
template <int MT>
VX_DEVICE int lora_frag_at(int row, int r) {
  const int kb = (r >> 5) * 2 + ((r >> 2) & 1), lane = (row & 7) * 4 + ((r >> 3) & 3);
  const int reg = (r & 2) + ((row & 15) >> 3);
  return ((kb * MT + (row >> 4)) * 64 + lane) * 8 + reg * 2 + (r & 1);
}

// B of one 32-output block: KB pairs of 16 components x 4 MMA tiles.  Column q
// of MMA tile j is output 8 (q/2) + 2 j + q%2 of the 32, so a lane ends up with
// 8 neighbours; not WIDE 8 j + 4 (q%2) + q/2 (Eight).
template <int KB, bool WIDE>
VX_DEVICE void load_b(const LoraArgs& a, const uint16_t* B, int rank, int nb, int kb0, uint4 (&bf)[KB][4]) {
  const int g = (threadIdx.x & 31) >> 2, c = threadIdx.x & 3;
#pragma unroll
  for (int u = 0; u < KB; ++u) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = nb * 32 + (WIDE ? 8 * (g >> 1) + 2 * j + (g & 1) : 8 * j + 4 * (g & 1) + (g >> 1));
      const int r = (kb0 + u) * 32 + 8 * c;
      bf[u][j] = r < rank && row < a.N ? __ldg(reinterpret_cast<const uint4*>(B + int64_t(row) * a.R + r))
                                       : make_uint4(0, 0, 0, 0);
    }
  }
}
template <int MT, bool WIDE>
VX_DEVICE void load_y(const LoraArgs& a, const int (&t)[2 * MT], int nb, Eight<WIDE> (&y)[2 * MT]) {
  const int n = first_of<WIDE>(nb);
#pragma unroll
  for (int i = 0; i < 2 * MT; ++i)
    if (t[i] >= 0 && (!WIDE || n < a.N)) y[i].load(a.y + t[i] * a.ldy, n, a.N);
}
// out = y + B h for one block whose y and first B are loaded.
template <int MT, int KB, bool WIDE>
VX_DEVICE void lora_expand(const LoraArgs& a, const uint16_t* B, int rank, const uint4* frag, const int (&t)[2 * MT],
                           int nb, const Eight<WIDE> (&y)[2 * MT], uint4 (&bf)[KB][4]) {
  const int lane = threadIdx.x & 31, c = lane & 3, n = first_of<WIDE>(nb), kbs = (rank + 31) / 32;
  float acc[MT][4][4] = {};
  for (int kb0 = 0; kb0 < kbs; kb0 += KB) {
    if (kb0 > 0) load_b<KB, WIDE>(a, B, rank, nb, kb0, bf);
#pragma unroll
    for (int u = 0; u < KB; ++u) {
      if (kb0 + u >= kbs) break;
      // components behind the adapter's rank count as zero, whatever they hold
      const int left = rank - ((kb0 + u) * 32 + 8 * c);
      if (left < 8) {
        auto keep = [&](int i) { return left > 2 * i + 1 ? ~0u : left > 2 * i ? 0xFFFFu : 0u; };
#pragma unroll
        for (int j = 0; j < 4; ++j)
          bf[u][j] = make_uint4(bf[u][j].x & keep(0), bf[u][j].y & keep(1), bf[u][j].z & keep(2), bf[u][j].w & keep(3));
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint4* h = frag + ((2 * (kb0 + u) + half) * MT + m) * 64 + lane;
          const uint4 hi = h[0], lo = h[32];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t b0 = half ? bf[u][j].z : bf[u][j].x, b1 = half ? bf[u][j].w : bf[u][j].y;
            mma16816(acc[m][j], hi.x, hi.y, hi.z, hi.w, b0, b1);
            mma16816(acc[m][j], lo.x, lo.y, lo.z, lo.w, b0, b1);
          }
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
// The 32-output blocks first, first + stride, ... below `end`, each one's y
// and B loaded before its predecessor is computed; the first block's are
// loaded by the caller.
template <int MT, int KB, bool WIDE>
VX_DEVICE void lora_expand_all(const LoraArgs& a, const uint16_t* B, int rank, const uint4* frag,
                               const int (&t)[2 * MT], int first, int stride, int end, Eight<WIDE> (&y)[2 * MT],
                               uint4 (&bf)[KB][4]) {
  Eight<WIDE> yn[2 * MT];
  uint4 bn[KB][4];
  int nb = first;
  while (nb * 32 < end) {   // two blocks a turn, so that neither set is copied
    int next = nb + stride;
    if (next * 32 < end) {
      load_y<MT, WIDE>(a, t, next, yn);
      load_b<KB, WIDE>(a, B, rank, next, 0, bn);
    }
    lora_expand<MT, KB, WIDE>(a, B, rank, frag, t, nb, y, bf);
    nb = next;
    if (nb * 32 >= end) break;
    next = nb + stride;
    if (next * 32 < end) {
      load_y<MT, WIDE>(a, t, next, y);
      load_b<KB, WIDE>(a, B, rank, next, 0, bf);
    }
    lora_expand<MT, KB, WIDE>(a, B, rank, frag, t, nb, yn, bn);
    nb = next;
  }
}

// ---- small batches: one launch ------------------------------------------------

constexpr int kSmallNt = 8, kSmallKb = 2;
constexpr int kSmallPart = kLoraWarps * 16 * 8 * kSmallNt;   // floats
// the warps' sums, the parts of C CTAs [C][16][R], the fragments
static int lora_small_smem(int R, int C) { return (kSmallPart + C * 16 * R) * 4 + lora_frag_bytes(1, R); }

template <bool WIDE>
__global__ void __launch_bounds__(kLoraThreads, 2) lora_small_kernel(const LoraArgs a) {
  chain_begin();
  constexpr int TM = 16;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __shared__ int tok[TM];          // the item's tokens, -1 behind the last
  __shared__ __align__(16) int s_ids[kLoraSmall];
  __shared__ int s_lead[kLoraWarps], s_item[2];
  __shared__ __align__(8) uint64_t arrived;   // bytes of the cluster's parts
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int C = int(lora_cluster_size()), cta = int(lora_cluster_rank());
  const int item = int(blockIdx.x) / C, T = int(a.T);

  // Thread t: how many earlier tokens share its adapter.  Every TM-th token
  // of an adapter leads an item; items are numbered by their leaders.
  const int mine = tid < T ? lora_id(a, tid) : -2;
  s_ids[tid] = mine;
  if (tid < TM) tok[tid] = -1;
  if (tid == 0) {
    mbar_init(smem_u32(&arrived));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
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
  const bool member = tid < T && mine == e && before / TM == s_item[1];
  if (member) tok[before % TM] = tid;
  const int n = __syncthreads_count(member);
  const int rank = lora_rank(a, e);
  __syncwarp();
  if (rank > 0) lora_cluster_arrive();   // the barrier above is initialised

  float* part = reinterpret_cast<float*>(smem_raw);
  float* parts = part + kSmallPart;
  uint4* frag = reinterpret_cast<uint4*>(parts + C * TM * a.R);
  const uint16_t* B = a.b + int64_t(e < 0 ? 0 : e) * a.N * a.R;
  const int nb0 = cta * kLoraWarps + warp, stride = C * kLoraWarps;
  int t[2];
  Eight<WIDE> y[2];
  uint4 bf[kSmallKb][4];
#pragma unroll
  for (int i = 0; i < 2; ++i) t[i] = tok[8 * i + (lane >> 2)];
  if (rank > 0) {
    if (tid == 0) mbar_expect(smem_u32(&arrived), uint32_t(C * n * ((rank + 7) / 8) * 32));
    // the cluster barrier is a warp's, not a thread's: whole warps wait at it
    lora_shrink<1, kSmallNt, false>(
        a, e, rank, 0, 8 * kSmallNt, tok, n, nb0, stride, part, [] { lora_cluster_wait(); },
        [&](int row, int r, float4 v) {
          for (int q = 0; q < C; ++q) push4(parts + (cta * TM + row) * a.R + r, &arrived, q, v);
        });
  }
  if (nb0 * 32 < a.N) {
    load_y<1, WIDE>(a, t, nb0, y);
    load_b<kSmallKb, WIDE>(a, B, rank, nb0, 0, bf);
  }
  if (rank > 0) {
    const bool ok = lora_wait(&arrived);
    if (!ok) lora_wait(&arrived);   // given up: let the parts on their way land (bounded)
    const int cols = (rank + 31) & ~31;
    const float scale = ok ? a.scales ? __ldg(a.scales + e) : 1.0f : __uint_as_float(0x7FC00000u);
    uint16_t* f = reinterpret_cast<uint16_t*>(frag);
    for (int i = tid; i < n * cols; i += kLoraThreads) {   // rows behind the last token are not stored
      const int row = i / cols, r = i - row * cols;
      float v = 0.f;
      if (r < rank)
        for (int q = 0; q < C; ++q) v += parts[(q * TM + row) * a.R + r];
      uint16_t* at = f + lora_frag_at<1>(row, r);
      lora_split(v * scale, at, at + 256);
    }
    __syncthreads();
  }
  lora_expand_all<1, kSmallKb, WIDE>(a, B, rank, frag, t, nb0, stride, a.N, y, bf);
}

// ---- large batches ------------------------------------------------------------

constexpr int kLargeMt = 2, kLargeTm = 16 * kLargeMt;
constexpr int kLargeNt = 4, kLargeKb = 1;
constexpr int kPassRank = 8 * kLargeNt;   // components a CTA forms at a time
constexpr int kLargePart = kLoraWarps * kLargeTm * 8 * kLargeNt;   // floats

// An item of lora_group_kernel: {adapter or -1, first place of `order`,
// tokens (0: no item), rank}.

// h [place of order][16 components][hi, lo][16] of every item.
// A CTA forms 32 components of an item (neighbouring CTAs the others, over the
// same x): 2,693 tokens of 51 adapters of rank 80, K = 3,352, 30 against 55 us
// with the passes in a row, 8,192 of rank 64 52.5 against 53.2.
__global__ void __launch_bounds__(kLoraThreads, 2) lora_shrink_kernel(const LoraArgs a,
                                                                      const int32_t* __restrict__ order,
                                                                      const int4* __restrict__ items,
                                                                      uint16_t* __restrict__ h,
                                                                      int passes) {
  chain_begin();
  __shared__ __align__(16) float part[kLargePart];
  __shared__ int tok[kLargeTm];
  const int tid = threadIdx.x;
  const int4 it = __ldg(items + blockIdx.x / passes);
  const int e = it.x, begin = it.y, n = it.z, rank = it.w, first = int(blockIdx.x % passes) * kPassRank;
  if (n == 0 || first >= rank) return;
  if (tid < kLargeTm) tok[tid] = tid < n ? __ldg(order + begin + tid) : -1;
  const float scale = a.scales ? __ldg(a.scales + e) : 1.0f;
  __syncthreads();
  const int pitch = ((a.R + 15) & ~15) * 2;
  lora_shrink<kLargeMt, kLargeNt, true>(
      a, e, rank, first, passes * kPassRank, tok, n, tid >> 5, kLoraWarps, part, [] {},
      [&](int row, int r, float4 v) {
        const float f[4] = {v.x, v.y, v.z, v.w};
        uint16_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) lora_split(r + i < rank ? f[i] * scale : 0.f, &hi[i], &lo[i]);
        uint16_t* p = h + int64_t(begin + row) * pitch + (r >> 4) * 32 + (r & 15);
        *reinterpret_cast<uint2*>(p) = make_uint2(hi[0] | uint32_t(hi[1]) << 16, hi[2] | uint32_t(hi[3]) << 16);
        *reinterpret_cast<uint2*>(p + 16) = make_uint2(lo[0] | uint32_t(lo[1]) << 16, lo[2] | uint32_t(lo[3]) << 16);
      });
}

// Not WIDE one CTA an SM: with two its registers spill (2,000 tokens x 1,001
// outputs 23 / 30 us, 8,192 x 2,047 103 / 99).
template <bool WIDE>
__global__ void __launch_bounds__(kLoraThreads, WIDE ? 2 : 1) lora_expand_kernel(const LoraArgs a,
                                                                      const int32_t* __restrict__ order,
                                                                      const int4* __restrict__ items,
                                                                      const uint16_t* __restrict__ h, int cols) {
  chain_begin();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int4 it = __ldg(items + blockIdx.x);
  const int e = it.x, begin = it.y, n = it.z, rank = it.w;
  if (n == 0) return;
  int t[2 * kLargeMt];
#pragma unroll
  for (int i = 0; i < 2 * kLargeMt; ++i) {
    const int row = 8 * i + (lane >> 2);
    t[i] = row < n ? __ldg(order + begin + row) : -1;
  }
  const uint16_t* B = a.b + int64_t(e < 0 ? 0 : e) * a.N * a.R;
  const int end = min(a.N, int(blockIdx.y + 1) * cols), nb0 = int(blockIdx.y) * (cols / 32) + warp;
  Eight<WIDE> y[2 * kLargeMt];
  uint4 bf[kLargeKb][4];
  if (nb0 * 32 < end) {
    load_b<kLargeKb, WIDE>(a, B, rank, nb0, 0, bf);
    load_y<kLargeMt, WIDE>(a, t, nb0, y);
  }
  // the fragments: a thread brings 4 components of a row, hi or lo.  What
  // shrink did not write (above the rank's last 8) counts as zero: its column
  // of B does, and h must be finite there.
  uint4* frag = reinterpret_cast<uint4*>(smem_raw);
  const int pieces = (rank + 31) / 32 * 16, pitch = ((a.R + 15) & ~15) * 2;   // 8 of hi, 8 of lo for 32 components
  for (int i = tid; i < kLargeTm * pieces; i += kLoraThreads) {
    const int row = i / pieces, piece = i - row * pieces, r = (piece >> 1) * 4, lo = piece & 1;
    uint2 v = make_uint2(0, 0);
    if (row < n && r < rank)
      v = *reinterpret_cast<const uint2*>(h + int64_t(begin + row) * pitch + (r >> 4) * 32 + lo * 16 + (r & 15));
    uint32_t* p = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(frag) + lora_frag_at<kLargeMt>(row, r) +
                                              lo * 256);
    p[0] = v.x;   // components 0, 1 of the four
    p[2] = v.y;   // 2, 3: two registers on
  }
  __syncthreads();
  lora_expand_all<kLargeMt, kLargeKb, WIDE>(a, B, rank, frag, t, nb0, kLoraWarps, end, y, bf);
}

// One CTA: tokens counted per adapter (bucket L: none), buckets cut into
// items of kLargeTm tokens; the items behind the last get no tokens.  The
// order inside a bucket does not matter: a token's sums are the same
// whichever row of an item it takes.
constexpr int kGroupThreads = 1024;

constexpr int kGroupBatch = 8;   // tokens of a thread whose loads are in flight together

__global__ void __launch_bounds__(kGroupThreads) lora_group_kernel(const LoraArgs a, int32_t* __restrict__ place,
                                                                   int32_t* __restrict__ order,
                                                                   int4* __restrict__ items, int max_items) {
  chain_begin();
  constexpr int tm = kLargeTm;
  extern __shared__ int s_cnt[];                 // [L+1] tokens, then first place; [L+1] first item
  int* s_first = s_cnt + a.L + 1;
  __shared__ int2 s_warp[32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int buckets = a.L + 1;
  const int64_t T = a.T, round = int64_t(kGroupBatch) * kGroupThreads;
  int b[kGroupBatch], at[kGroupBatch];           // buckets (-1: no token) and places of a round's tokens
  auto load = [&](int64_t t0) {
#pragma unroll
    for (int u = 0; u < kGroupBatch; ++u) {
      const int64_t t = t0 + u * kGroupThreads;
      b[u] = t < T ? lora_id(a, t) : -2;
    }
#pragma unroll
    for (int u = 0; u < kGroupBatch; ++u) b[u] = b[u] == -1 ? a.L : b[u] == -2 ? -1 : b[u];
  };
  load(tid);
  for (int i = tid; i < buckets; i += kGroupThreads) s_cnt[i] = 0;
  __syncthreads();
  for (int64_t r0 = 0; r0 < T; r0 += round) {
    if (r0 > 0) load(r0 + tid);
#pragma unroll
    for (int u = 0; u < kGroupBatch; ++u) {
      if (r0 + u * kGroupThreads >= T) break;   // the whole CTA
      // a warp of one bucket (packed prompts) adds once, others lane by lane
      if (__all_sync(0xFFFFFFFFu, b[u] == __shfl_sync(0xFFFFFFFFu, b[u], 0))) {
        int base = 0;
        if (lane == 0 && b[u] >= 0) base = atomicAdd(&s_cnt[b[u]], 32);
        at[u] = __shfl_sync(0xFFFFFFFFu, base, 0) + lane;
      } else if (b[u] >= 0) {
        at[u] = atomicAdd(&s_cnt[b[u]], 1);
      }
      if (T > round && b[u] >= 0) place[r0 + u * kGroupThreads + tid] = at[u];
    }
  }
  __syncthreads();
  // exclusive scans of tokens and items over the buckets
  const int per = (buckets + kGroupThreads - 1) / kGroupThreads;
  int2 own = make_int2(0, 0);
  for (int i = 0; i < per; ++i) {
    const int bucket = tid * per + i, n = bucket < buckets ? s_cnt[bucket] : 0;
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
  int2 next = make_int2(inc.x - own.x, inc.y - own.y);
  int total = 0;
  const int used = (buckets + 32 * per - 1) / (32 * per);   // warps that hold buckets
  for (int w = 0; w < used; ++w) {
    if (w < warp) next.x += s_warp[w].x, next.y += s_warp[w].y;
    total += s_warp[w].y;
  }
  for (int i = 0; i < per; ++i) {
    const int bucket = tid * per + i;
    if (bucket >= buckets) break;
    const int n = s_cnt[bucket];
    s_cnt[bucket] = next.x;
    s_first[bucket] = next.y;
    next.x += n;
    next.y += (n + tm - 1) / tm;
  }
  __syncthreads();
  for (int64_t r0 = 0; r0 < T; r0 += round) {
    if (T > round) {   // else still in registers
      load(r0 + tid);
#pragma unroll
      for (int u = 0; u < kGroupBatch; ++u) {
        const int64_t t = r0 + u * kGroupThreads + tid;
        at[u] = t < T ? place[t] : 0;
      }
    }
#pragma unroll
    for (int u = 0; u < kGroupBatch; ++u) {
      const int64_t t = r0 + u * kGroupThreads + tid;
      if (t < T) order[s_cnt[b[u]] + at[u]] = int32_t(t);
    }
  }
  for (int i = tid; i < max_items; i += kGroupThreads) {
    int4 it = make_int4(-1, 0, 0, 0);
    if (i < total) {
      int lo = 0, hi = buckets;   // the last bucket with s_first <= i: the one that holds item i
      while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (s_first[m] <= i) lo = m; else hi = m;
      }
      const int begin = s_cnt[lo] + (i - s_first[lo]) * tm;
      const int end = lo + 1 < buckets ? s_cnt[lo + 1] : int(T);
      it = make_int4(lo == a.L ? -1 : lo, begin, min(tm, end - begin), lora_rank(a, lo == a.L ? -1 : lo));
    }
    items[i] = it;
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
  s.h = s.items + up(16 * lora_max_items(T, L, kLargeTm));
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
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(k), lora_small_smem(kLoraMaxRank, 8), done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(n * C));
  cfg.blockDim = dim3(kLoraThreads);
  cfg.dynamicSmemBytes = size_t(lora_small_smem(a.R, C));
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
  int32_t *order = reinterpret_cast<int32_t*>(ws), *place = reinterpret_cast<int32_t*>(ws + sp.place);
  int4* items = reinterpret_cast<int4*>(ws + sp.items);
  uint16_t* h = reinterpret_cast<uint16_t*>(ws + sp.h);
  const unsigned n = unsigned(lora_max_items(a.T, a.L, kLargeTm));
  // Outputs of an expanding CTA: the number that costs least, a round of the
  // resident CTAs taken as its outputs and 160 for its start, as long as three
  // CTAs to two SMs are left.  8,192 tokens x 4,096 outputs take 52.2 us with
  // 4,096, 54.1 with 1,024; 5,000 x 8,192 take 62.5 with 1,024, 64.2 with 512
  // and with 2,048; 512 x 4,096 take 20.8 with 512, 23.1 with 1,024.
  const int64_t resident = 2 * int64_t(sm_count());
  int cols = 512;
  for (int64_t c = 512, best = 0; c <= 4096; c *= 2) {
    const int64_t ctas = int64_t(n) * ((a.N + c - 1) / c), cost = (ctas + resident - 1) / resident * (c + 160);
    if (c == 512 || (4 * ctas >= 3 * resident && cost < best)) best = cost, cols = int(c);
  }
  const unsigned passes = unsigned(a.R + kPassRank - 1) / kPassRank;
  static std::atomic<uint64_t> done{0};
  auto expand = lora_expand_kernel<WIDE>;
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(expand), lora_frag_bytes(kLargeMt, kLoraMaxRank), done);
  if (e == cudaSuccess)
    e = launch_chained(lora_group_kernel, dim3(1), dim3(kGroupThreads), size_t(2 * a.L + 2) * sizeof(int), st, a,
                       place, order, items, int(n));
  if (e == cudaSuccess)
    e = launch_chained(lora_shrink_kernel, dim3(n * passes), dim3(kLoraThreads), 0, st, a, order, items, h,
                       int(passes));
  if (e == cudaSuccess)
    e = launch_chained(expand, dim3(n, unsigned((a.N + cols - 1) / cols)), dim3(kLoraThreads),
                       size_t(lora_frag_bytes(kLargeMt, a.R)), st, a, order, items, h, cols);
  return e;
}

cudaError_t launch_lora(const LoraArgs& a, void* workspace, cudaStream_t st) {
  if (a.T == 0 || a.N == 0) return cudaSuccess;
  auto aligned = [](const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; };
  const bool wide = a.N % 8 == 0 && aligned(a.y, a.T > 1 ? a.ldy : 0) && aligned(a.out, a.T > 1 ? a.ldo : 0);
  if (a.T <= kLoraSmall) return wide ? launch_lora_small<true>(a, st) : launch_lora_small<false>(a, st);
  char* ws = static_cast<char*>(workspace);
  return wide ? launch_lora_large<true>(a, ws, st) : launch_lora_large<false>(a, ws, st);
}

}  // namespace vx
