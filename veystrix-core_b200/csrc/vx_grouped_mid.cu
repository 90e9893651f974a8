// Products grouped by expert where an expert has tens of rows (prefill): the
// formula of vx_grouped.cu, still bound by the bank's bytes.
//
// A CTA computes tiles of up to 128 positions x 256 outputs of one expert:
//
//   D[128 positions][256 outputs] += X[128][K] . W[256][K]^T   (or 64 positions)
//
// The positions are the MMA's M side here and the bank its N side, so a tile
// has 256 outputs on one SM (32 KB of the bank in flight a stage) where the
// tiles of vx_grouped.cu have 128, TMEM holds a position's outputs side by
// side, and a tile begins and ends without a word to another CTA: with short
// bank rows (K = 512 e4m3: four stages a tile) that is what counts, 98 against
// 146 us for 20,480 rows over 512 experts of 2,048 outputs.  From about a
// hundred positions an expert on the pairs' tiles are better: they fill up to
// 256 columns and share the bank's rows.  The padding rows of X are not
// copied; they hold what the ring held before, and their rows of D are not
// read.  A tile of at most 64 positions takes M = 64: less power, and with it
// higher clocks (2,048 tokens over 512 e4m3 experts in steady state 206 us,
// 219 with M = 128 throughout).  Those 2,048 tokens: 194 us at full clocks for
// 1.12 GB, 0.88 of the measured copy rate, the gathering of the rows included.
//
// Warp roles (384 threads, one CTA an SM, persistent):
//   warp 0      TMA: 256 bank rows (32 KB) and the real positions' rows (boxes
//               of 128, 64, 32 and 16) into a ring of kMidStages stages
//   warp 1      allocates TMEM (two accumulators of 256 columns) and issues
//               the MMAs
//   warps 4-11  epilogue: TMEM lane = position, column = output; a lane
//               stores 16 neighbouring outputs at once (32 bytes) where out's
//               rows allow it, else lanes share rows, 4 or 1 outputs each
// Rows are gathered by a launch of their own before (gather_rows_kernel).
// Every wait is bounded as in vx_grouped.cu.
#include <cudaTypedefs.h>

#include "vx_async.cuh"
#include "vx_common.cuh"
#include "vx_grouped.cuh"
#include "vx_launch.h"
#include "vx_tc.cuh"

namespace vx {

constexpr int kMidPos = 128, kMidOut = 256;
constexpr int kMidThreads = 384;
constexpr int kMidStages = 4;
constexpr int kMidBank = kMidOut * 128, kMidStage = kMidBank + kMidPos * 128;
constexpr int kMidEpiWarps = 8;
constexpr int kPiecePitch = 9;   // words of 16 outputs in shared memory, one more for the banks

struct GroupedMid {
  CUtensorMap tm_w, tm_x[4];   // x: boxes of 16, 32, 64 and 128 rows
  GroupedArgs a;               // rows null
  int row_tiles;
  int vec;                     // outputs a store may take: 16, 4 or 1
};

VX_DEVICE void load_3d(uint32_t dst, const void* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
template <bool FP8>
VX_DEVICE void mid_mma(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool acc) {
  if (FP8)
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(int(acc))
        : "memory");
  else
    mma_bf16(d, adesc, bdesc, idesc, acc);
}

// A tile: expert, first output, first position, number of positions.
struct MidTile {
  int e, n0, p0, count;
  VX_DEVICE int m() const { return count <= kMidPos / 2 ? kMidPos / 2 : kMidPos; }   // the MMA's M
};

template <bool FP8>
__global__ void __launch_bounds__(kMidThreads, 1) grouped_mid_kernel(const __grid_constant__ GroupedMid g) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[kMidStages], empty[kMidStages], acc_full[2], acc_empty[2];
  __shared__ __align__(16) float w_scale[FP8 ? kMidEpiWarps : 1][kMidOut / 2];   // an epilogue warp's outputs
  __shared__ uint32_t pieces[kMidEpiWarps][32 * kPiecePitch];
  __shared__ uint32_t tmem_slot;
  __shared__ int dead;
  const GroupedArgs& a = g.a;
  const int warp = int(uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  int* table = reinterpret_cast<int*>(smem_raw + (base - smem_u32(smem_raw)) + kMidStages * kMidStage);

  if (threadIdx.x == 0) {
    dead = 0;
    for (int s = 0; s < kMidStages; ++s) {
      mbar_init_n(smem_u32(&full[s]), 1);
      mbar_init_n(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init_n(smem_u32(&acc_full[b]), 1);
      mbar_init_n(smem_u32(&acc_empty[b]), kMidEpiWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_slot), 512);
  if (warp == 0 && lane < 5) prefetch_map(lane == 4 ? &g.tm_w : &g.tm_x[lane]);
  chain_wait();
  const GroupTable<kMidThreads> groups(a, table, kMidPos);
  const int tiles = groups.items() * g.row_tiles;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(tmem_slot);

  auto tile_at = [&](int t) {
    // an expert's tiles: full parts and a rest, each with all the row tiles
    const int part = t / g.row_tiles, rt = t - part * g.row_tiles;
    int e, p0;
    const int count = groups.item(part, &e, &p0);
    return MidTile{e, rt * kMidOut, p0, count};
  };
  const int steps = (a.K * (FP8 ? 1 : 2) + 127) >> 7;
  auto stage_w = [&](int s) { return base + s * kMidStage; };
  auto stage_x = [&](int s) { return base + s * kMidStage + kMidBank; };

  int stopped_at = 0;               // stage and phase after warp 0's last copies
  uint32_t stopped_phase = 1;
  if (warp == 0) {
    // ---- copies
    int s = 0;
    uint32_t ph = 1;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
      const MidTile c = tile_at(t);
      const int rows = (c.count + 15) & ~15;
      const uint32_t bytes = uint32_t(kMidBank + rows * 128);
      // lane i < 4 copies the box of 16 << i rows if `rows` has that bit, the
      // larger boxes first
      const bool box = lane < 4 && ((rows >> (4 + lane)) & 1);
      const int at = rows & ~((32 << lane) - 1);
      for (int k = 0; k < steps; ++k) {
        if (!role_wait(smem_u32(&empty[s]), ph, &dead)) {
          ok = false;
          break;
        }
        const uint32_t bar = smem_u32(&full[s]);
        const int x = k * (FP8 ? 128 : 64);
        if (lane == 0) {
          mbar_expect(bar, bytes);
          load_3d(stage_w(s), &g.tm_w, x, c.n0, c.e, bar);
        }
        __syncwarp();   // the expectation comes before any of the stage's copies
        if (box) tma_load_2d(stage_x(s) + at * 128, &g.tm_x[lane], x, c.p0 + at, bar);
        if (++s == kMidStages) s = 0, ph ^= 1;
      }
    }
    stopped_at = s, stopped_phase = ph;
  } else if (warp == 1) {
    // ---- MMAs: the whole warp waits, one lane issues
    int s = 0, b = 0;
    uint32_t ph = 0, aph = 1;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
      const MidTile c = tile_at(t);
      const int n = min(kMidOut, (a.N - c.n0 + 15) & ~15);
      const uint32_t d = tmem + b * kMidOut;
      // float32 accumulator, both operands K-major, M = 64 or 128; bf16 is
      // format 1, e4m3 format 0 of kind::f8f6f4
      const uint32_t f = FP8 ? 0u : 1u;
      const uint32_t idesc = uniform((1u << 4) | (f << 7) | (f << 10) | (uint32_t(n >> 3) << 17) | (uint32_t(c.m() >> 4) << 24));
      ok = role_wait(smem_u32(&acc_empty[b]), aph, &dead);
      tc_fence_after();
      for (int k = 0; ok && k < steps; ++k) {
        ok = role_wait(smem_u32(&full[s]), ph, &dead);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t xd = sw128_desc(stage_x(s)), wd = sw128_desc(stage_w(s));
#pragma unroll
          for (int i = 0; i < 4; ++i) mid_mma<FP8>(d, xd + 2 * i, wd + 2 * i, idesc, k > 0 || i > 0);
          mma_commit(smem_u32(&empty[s]));
          if (k + 1 == steps) mma_commit(smem_u32(&acc_full[b]));
        }
        __syncwarp();
        if (++s == kMidStages) s = 0, ph ^= 1;
      }
      if (++b == 2) b = 0, aph ^= 1;
    }
  } else if (warp >= 4) {
    // ---- epilogue: warp = a quarter of the positions, half h of the outputs
    const int quarter = warp & 3, h = (warp - 4) >> 2;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    float* scale = w_scale[FP8 ? warp - 4 : 0];
    int b = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
      const MidTile c = tile_at(t);
      // M = 128: lane = position; M = 64: each quarter's lower 16 lanes hold 16
      const int rows = c.m() / 4, pos = quarter * rows + lane, n0 = c.n0 + h * (kMidOut / 2);
      const bool real = lane < rows && pos < c.count;
      float sx = 1.f;
      if ((FP8 || a.gathered) && real) sx = __ldg(a.x_scales + c.p0 + pos);
      const bool none = names_none(a, sx);
      bool fit = true;
      if (FP8) {
        float sw[4];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = n0 + 32 * i + lane;
          sw[i] = n < a.N ? __ldg(a.w_scales + int64_t(c.e) * a.N + n) : 0.f;
          scale[32 * i + lane] = sw[i];
        }
        fit = products_fit(sw, sx);
        __syncwarp();
      }
      if (ok) ok = role_wait(smem_u32(&acc_full[b]), ph, &dead);
      tc_fence_after();
      if (quarter * rows < c.count) {   // else no real position in this warp's lanes
        uint16_t* out = a.out + int64_t(c.p0 + pos) * a.ldo + n0;
#pragma unroll
        for (int i = 0; i < kMidOut / 32; ++i) {
          const int left = a.N - n0 - 16 * i;   // outputs from here on
          if (left <= 0) break;
          float v[16];
          tmem_ld16(tmem + lanes + b * kMidOut + h * (kMidOut / 2) + 16 * i, v);
          if (FP8 && fit) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float4 f = *reinterpret_cast<const float4*>(scale + 16 * i + 4 * j);
              v[4 * j] *= f.x * sx, v[4 * j + 1] *= f.y * sx, v[4 * j + 2] *= f.z * sx, v[4 * j + 3] *= f.w * sx;
            }
          } else if (FP8) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = scaled(v[j], scale[16 * i + j], sx);
          }
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = !ok ? 0x7FFF7FFFu : none ? 0u : bf16_pair(v[2 * j], v[2 * j + 1]);   // NaN
          if (g.vec == 16 && left >= 16) {
            if (real)
              asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + 16 * i), "r"(w[0]),
                           "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                           : "memory");
          } else if (g.vec > 1 && rows < 32) {
            if (real) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (4 * j < left)
                  *reinterpret_cast<uint2*>(out + 16 * i + 4 * j) = make_uint2(w[2 * j], w[2 * j + 1]);
            }
          } else {
            // through shared memory, neighbouring lanes to neighbouring pieces
            // of a row: lanes that store their own rows are 32 sectors an
            // instruction (30,502 rows of 2,596 172 against 80 us, 2,008 of 766
            // 27 / 14).  Four outputs of 16 rows go out faster as they lie: 341
            // groups of 7 rows of 1,324 44 / 26, of 24 43 / 29; of 55 44 / 47.
            uint32_t* r = pieces[warp - 4] + lane * kPiecePitch;
#pragma unroll
            for (int j = 0; j < 8; ++j) r[j] = w[j];
            __syncwarp();
            const int last = min(rows, c.count - quarter * rows);   // the warp's real positions
            uint16_t* to = a.out + int64_t(c.p0 + quarter * rows) * a.ldo + n0 + 16 * i;
            if (g.vec > 1) {
              const int piece = 4 * (lane & 3);
              if (piece < left)
                for (int q = lane >> 2; q < last; q += 8) {
                  const uint32_t* from = pieces[warp - 4] + q * kPiecePitch + piece / 2;
                  *reinterpret_cast<uint2*>(to + q * a.ldo + piece) = make_uint2(from[0], from[1]);
                }
            } else if ((lane & 15) < left) {
              for (int q = lane >> 4; q < last; q += 2)
                to[q * a.ldo + (lane & 15)] =
                    reinterpret_cast<const uint16_t*>(pieces[warp - 4] + q * kPiecePitch)[lane & 15];
            }
            __syncwarp();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&acc_empty[b]));
      if (++b == 2) b = 0, ph ^= 1;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (dead && threadIdx.x == 0) {
    // given up: let the copies in flight land (bounded)
    const uint64_t t0 = global_ns();
    for (int i = 0; i < kMidStages; ++i)
      while (!mbar_try(smem_u32(&full[i]), i < stopped_at ? stopped_phase ^ 1 : stopped_phase) &&
             global_ns() - t0 < kWaitLimitNs) {
      }
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- host side --------------------------------------------------------------

template <bool FP8>
static cudaError_t launch_mid_as(const GroupedMid& g, int64_t ctas, cudaStream_t st) {
  auto k = grouped_mid_kernel<FP8>;
  constexpr int kRing = kMidStages * kMidStage + 1024;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(k), kRing + 2 * (kGroupedMaxExperts + 1) * int(sizeof(int)),
                             done);
  if (e != cudaSuccess) return e;
  return launch_chained(k, dim3(unsigned(ctas)), dim3(kMidThreads),
                        size_t(kRing + 2 * (g.a.experts + 1) * int(sizeof(int))), st, g);
}

cudaError_t launch_grouped_mid(const GroupedArgs& a, bool e4m3, cudaStream_t st) {
  GroupedMid g;
  g.a = a;
  g.row_tiles = (a.N + kMidOut - 1) / kMidOut;
  const uintptr_t out = reinterpret_cast<uintptr_t>(a.out);
  g.vec = a.N % 4 == 0 && a.ldo % 4 == 0 && out % 8 == 0 ? a.ldo % 16 == 0 && out % 32 == 0 ? 16 : 4 : 1;
  const int64_t parts = (a.P + kMidPos - 1) / kMidPos + (a.P < a.experts ? a.P : a.experts);
  if (parts * g.row_tiles > 0x7FFFFFFF) return cudaErrorInvalidValue;
  if (!encode_k_rows(&g.tm_w, a.w, e4m3, a.K, a.N, a.K, a.experts, kMidOut)) return cudaErrorInvalidValue;
  for (int i = 0; i < 4; ++i)
    if (!encode_k_rows(&g.tm_x[i], a.x, e4m3, a.K, a.x_rows, a.ldx, 0, 16 << i)) return cudaErrorInvalidValue;
  int64_t ctas = sm_count();
  if (parts * g.row_tiles < ctas) ctas = parts * g.row_tiles;
  return e4m3 ? launch_mid_as<true>(g, ctas, st) : launch_mid_as<false>(g, ctas, st);
}

}  // namespace vx
