// Products grouped by expert over unquantised (bf16) or 8-bit (e4m3) banks:
//
//   out[p, n] = bf16( sx[row p] * sw[e, n] * sum_k x[row p, k] * w[e, n, k] )
//
// for the positions p in [offsets[e], offsets[e+1]) of expert e, row p =
// rows[p] / slots, or p itself; the scales only with e4m3.  Sums in float32,
// one rounding.  Positions from offsets[E] on are left as they were.
//
// Three kernels, by the number of positions (few_rows, mid_rows): a few,
// vx_grouped_few.cu; some tens an expert or short bank rows,
// vx_grouped_mid.cu; else the tiles here.  With `rows`, the latter two have x
// gathered by a launch of its own first.
//
// A CTA pair (cluster of two, cta_group::2) computes tiles of 256 outputs x
// up to 256 positions of one expert with tcgen05.mma:
//
//   D[256 outputs][N positions] += W[256][K] . X[N][K]^T
//
// The bank's rows are the MMA's M side, so a group of any size fills it and
// only N follows the ragged group (a multiple of 32).  Each CTA of the pair
// stages its own 128 bank rows and half of the positions, 128 bytes of K at a
// time (64 bf16 or 128 e4m3 inputs), so a 256 x 256 tile moves 32 KB per CTA
// and step through L2 where two single CTAs would move 48.  K past the end
// and rows past a bank's outputs arrive as zeros.  With one group of 16,384
// rows, K = N = 4,096, it runs at 1.59 PFLOP/s, 0.98 of the library's product;
// what holds it in steady state is the power limit.
//
// Warp roles of a CTA (384 threads):
//   warp 0      TMA: the bank rows and the positions (boxes of 128, 64, 32 and
//               16 rows that add up to them) into a ring of kGtStages stages.
//               Both CTAs' copies complete on the leader's barrier.
//   warp 1      leader only: issues the MMAs of both CTAs and commits each
//               stage back to both producers.
//   warp 2      allocates TMEM: two accumulators of 256 columns, so that a
//               tile's epilogue runs beside the next tile's MMAs.
//   warps 4-11  epilogue: TMEM lane = output, column = position.  Four lanes
//               exchange 4 x 4 values so that a lane stores four neighbouring
//               outputs of one position (8 bytes; single outputs where out's
//               rows do not allow it): 2-byte stores kept the warps at a tile
//               for 13,800 cycles, of 16,000 that its MMAs take at K = 2,048.
//               The next tile's place and scales are on their way meanwhile.
// Only rows of real positions are copied; the columns of a tile's padding
// hold what the ring held before and are not stored.  The real positions are
// dealt evenly to the halves.
// The grid is persistent (a pair per two SMs); pair i takes tiles i, i + G,
// ...  Tiles are numbered expert by expert (prefix sums over the groups in
// shared memory), so pairs running side by side share one bank and its
// positions in L2.  A group of more than 256 positions is cut into equal
// tiles rather than full ones and a rest.
//
// Every wait is bounded: one that runs out ends the CTA's roles, and the
// tiles left over are filled with NaN.
#include <cudaTypedefs.h>

#include "vx_async.cuh"
#include "vx_common.cuh"
#include "vx_grouped.cuh"
#include "vx_launch.h"
#include "vx_tc.cuh"

namespace vx {

constexpr int kGtRows = 256;                        // outputs of a pair's tile
constexpr int kGtCols = 256;                        // positions of a tile, at most
constexpr int kGtThreads = 384;
constexpr int kGtStages = 6;
constexpr int kGtHalf = 128 * 128;                  // 128 rows x 128 bytes of K
constexpr int kGtStage = 2 * kGtHalf;               // bank rows, positions
constexpr int kGtEpiWarps = 8;

struct GroupedTc {
  CUtensorMap tm_w, tm_x[4];                        // x: boxes of 16, 32, 64 and 128 rows
  GroupedArgs a;                                    // rows null
  int row_tiles;                                    // 256-output tiles of a bank
  int by_four;                                      // out's rows take 8-byte stores
};

VX_DEVICE uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Address of the same shared-memory location in CTA `rank` of the cluster.
VX_DEVICE uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
VX_DEVICE void cluster_sync() {
  __syncwarp();   // whole warps arrive and wait
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
VX_DEVICE void arrive_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// TMA loads of a CTA pair: into the own shared memory, completing on a
// barrier of either CTA (no multicast).
VX_DEVICE void pair_load_3d(uint32_t dst, const void* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], "
      "[%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
VX_DEVICE void pair_load_2d(uint32_t dst, const void* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], "
      "[%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

// One MMA of the pair over 32 bytes of K (16 bf16 or 32 e4m3 inputs).
template <bool FP8>
VX_DEVICE void pair_mma(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool acc) {
  if (FP8)
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(int(acc))
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(int(acc))
        : "memory");
}
// Arrives on `bar` of both CTAs once the MMAs issued so far are done.
VX_DEVICE void pair_commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(uint16_t(3))
      : "memory");
}
// float32 accumulator, both operands K-major, M = 256: bf16 (format 1) or
// e4m3 (format 0 of kind::f8f6f4).
template <bool FP8>
VX_DEVICE uint32_t pair_idesc(int n) {
  const uint32_t f = FP8 ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | (uint32_t(n >> 3) << 17) | (uint32_t(kGtRows >> 4) << 24);
}

// A tile: expert, first output, first position and number of positions.  The
// MMA's N columns are two halves, one staged by each CTA: the first holds
// positions 0 .. split(), the second the others, both padded to half().
struct Tile {
  int e, row0, p0, n;
  VX_DEVICE int split() const { return (n + 1) >> 1; }
  VX_DEVICE int half() const { return (split() + 15) & ~15; }
  VX_DEVICE int first(int h) const { return h ? p0 + split() : p0; }      // position of half h's column 0
  VX_DEVICE int count(int h) const { return h ? n - split() : split(); }  // real columns of half h
};

template <bool FP8>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGtThreads, 1)
    grouped_kernel(const __grid_constant__ GroupedTc g) {
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[kGtStages], empty[kGtStages], acc_full[2], acc_empty[2];
  __shared__ __align__(16) float x_scale[kGtEpiWarps][kGtCols / 2];   // an epilogue warp's columns
  __shared__ uint32_t tmem_slot;
  __shared__ int dead;
  const GroupedArgs& a = g.a;
  const int warp = int(uniform(threadIdx.x >> 5)), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  int* table = reinterpret_cast<int*>(smem_raw + (base - smem_u32(smem_raw)) + kGtStages * kGtStage);
  if (threadIdx.x == 0) {
    dead = 0;
    for (int s = 0; s < kGtStages; ++s) {
      mbar_init_n(smem_u32(&full[s]), 1);
      mbar_init_n(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init_n(smem_u32(&acc_full[b]), 1);
      mbar_init_n(smem_u32(&acc_empty[b]), 2 * kGtEpiWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == 1 && lane < 5) prefetch_map(lane == 4 ? &g.tm_w : &g.tm_x[lane]);
  chain_wait();

  const GroupTable<kGtThreads> groups(a, table, kGtCols);
  const int tiles = groups.items() * g.row_tiles;
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = uniform(tmem_slot);
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  auto tile_at = [&](int t) {
    // an expert's tiles: its parts, each with all the row tiles
    const int part = t / g.row_tiles, rt = t - part * g.row_tiles;
    const int e = groups.expert(part), n = groups.size(e), parts = (n + kGtCols - 1) / kGtCols;
    const int each = ((n + parts - 1) / parts + 31) & ~31;   // whole MMA steps of 32 columns
    const int skip = (part - groups.first[e]) * each;
    return Tile{e, rt * kGtRows, groups.starts[e] + skip, min(each, n - skip)};
  };
  const int steps = (a.K * (FP8 ? 1 : 2) + 127) >> 7;
  auto stage_w = [&](int s) { return base + s * kGtStage; };
  auto stage_x = [&](int s) { return base + s * kGtStage + kGtHalf; };

  int stopped_at = 0;               // stage and phase after warp 0's last copies
  uint32_t stopped_phase = 1;
  if (warp == 0) {
    // ---- copies
    int s = 0;
    uint32_t ph = 1;
    bool ok = true;
    for (int t = pair; ok && t < tiles; t += pairs) {
      const Tile c = tile_at(t);
      const int p0 = c.first(rank), w0 = c.row0 + rank * 128;
      // rows copied by each CTA: its real positions, rounded up to the smallest box
      auto copied = [&](int r) { return (c.count(r) + 15) & ~15; };
      const int mine = copied(rank);
      const uint32_t bytes = 2 * kGtHalf + (copied(0) + copied(1)) * 128;
      // lane i < 4 copies the box of 16 << i rows if `mine` has that bit; the
      // larger boxes come first, so box i starts at the bits above it
      const bool box = lane < 4 && ((mine >> (4 + lane)) & 1);
      const int at = mine & ~((32 << lane) - 1);
      for (int k = 0; k < steps; ++k) {
        if (!role_wait(smem_u32(&empty[s]), ph, &dead)) {
          ok = false;
          break;
        }
        const uint32_t bar = in_cta(smem_u32(&full[s]), 0);
        const int x = k * (FP8 ? 128 : 64);
        if (lane == 0) {
          if (rank == 0) mbar_expect(smem_u32(&full[s]), bytes);
          pair_load_3d(stage_w(s), &g.tm_w, x, w0, c.e, bar);
        }
        if (box) pair_load_2d(stage_x(s) + at * 128, &g.tm_x[lane], x, p0 + at, bar);
        if (++s == kGtStages) s = 0, ph ^= 1;
      }
    }
    stopped_at = s, stopped_phase = ph;
  } else if (warp == 1 && rank == 0) {
    // ---- MMAs of the pair: the whole warp waits, one lane issues
    int s = 0, b = 0;
    uint32_t ph = 0, aph = 1;
    bool ok = true;
    int half = pair < tiles ? tile_at(pair).half() : 0;
    for (int t = pair; ok && t < tiles; t += pairs) {
      const uint32_t idesc = uniform(pair_idesc<FP8>(2 * half)), d = tmem + b * kGtCols;
      ok = role_wait(smem_u32(&acc_empty[b]), aph, &dead);
      tc_fence_after();
      for (int k = 0; ok && k < steps; ++k) {
        ok = role_wait(smem_u32(&full[s]), ph, &dead);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint64_t ad = sw128_desc(stage_w(s)), bd = sw128_desc(stage_x(s));
#pragma unroll
          for (int i = 0; i < 4; ++i) pair_mma<FP8>(d, ad + 2 * i, bd + 2 * i, idesc, k > 0 || i > 0);
          pair_commit(smem_u32(&empty[s]));
          if (k + 1 == steps) pair_commit(smem_u32(&acc_full[b]));
        }
        __syncwarp();
        if (++s == kGtStages) s = 0, ph ^= 1;
      }
      if (++b == 2) b = 0, aph ^= 1;
      if (t + pairs < tiles) half = tile_at(t + pairs).half();   // while the MMAs run
    }
  } else if (warp >= 4) {
    // ---- epilogue: warp = a quarter of the outputs, half h of the positions
    const int quarter = warp & 3, h = (warp - 4) >> 2;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    float* scale = x_scale[warp - 4];
    const uint32_t pick = lane & 1 ? 0x3276u : 0x5410u;
    int b = 0;
    uint32_t ph = 0;
    bool ok = true;
    // a tile and the scales that this lane brings for it, one tile ahead
    struct Next {
      Tile c;
      float sw, sx[kGtCols / 64];
    } next;
    auto fetch = [&](int t) {
      if (t >= tiles) return;
      next.c = tile_at(t);
      if (!FP8 && !a.gathered) return;
      const int n = next.c.row0 + int(rank) * 128 + quarter * 32 + lane;
      next.sw = FP8 && n < a.N ? __ldg(a.w_scales + int64_t(next.c.e) * a.N + n) : 0.f;
#pragma unroll
      for (int i = 0; i < kGtCols / 64; ++i)
        next.sx[i] = 32 * i + lane < next.c.count(h) ? __ldg(a.x_scales + next.c.first(h) + 32 * i + lane) : 0.f;
    };
    fetch(pair);
    for (int t = pair; t < tiles; t += pairs) {
      const Tile c = next.c;
      const int cols = c.count(h), p0 = c.first(h);
      const int n = c.row0 + int(rank) * 128 + quarter * 32 + lane;   // this lane's output
      const float sw = next.sw;
      bool fit = true;   // no column's or output's scale, and no column, out of the ordinary
      if (FP8 || a.gathered) {
        fit = products_fit(next.sx, sw);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kGtCols / 64; ++i) scale[32 * i + lane] = next.sx[i];
        __syncwarp();
      }
      fetch(t + pairs);
      if (ok) ok = role_wait(smem_u32(&acc_full[b]), ph, &dead);
      tc_fence_after();
      const uint32_t acc = tmem + lanes + b * kGtCols + h * c.half();
      // lane 4 i + q stores column c0 + 4 j + q of outputs 4 i .. 4 i + 3
      uint16_t* o4 = a.out + int64_t(p0 + (lane & 3)) * a.ldo + (n & ~3);
      uint16_t* o1 = a.out + int64_t(p0) * a.ldo + n;
#pragma unroll
      for (int i = 0; i < kGtCols / 32; ++i) {
        const int c0 = 16 * i;
        if (c0 >= cols) break;
        float v[16];
        tmem_ld16(acc + c0, v);
        if (FP8 && fit) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 f = *reinterpret_cast<const float4*>(scale + c0 + 4 * j);
            v[4 * j] *= f.x * sw, v[4 * j + 1] *= f.y * sw, v[4 * j + 2] *= f.z * sw, v[4 * j + 3] *= f.w * sw;
          }
        } else if (!fit) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float f = scale[c0 + j];
            v[j] = names_none(a, f) ? 0.f : FP8 ? scaled(v[j], f, sw) : v[j];
          }
        }
        if (!ok) {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(0x7FC00000u);
        }
        if (g.by_four) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t lo = bf16_pair(v[4 * j], v[4 * j + 1]), hi = bf16_pair(v[4 * j + 2], v[4 * j + 3]);
            // columns 0, 1 of lanes 2 i, 2 i + 1; columns 2, 3 of the same
            const uint32_t a01 = prmt(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, 1), pick);
            const uint32_t a23 = prmt(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, 1), pick);
            const bool up = lane & 2;
            const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, up ? a01 : a23, 2);
            if (c0 + 4 * j + (lane & 3) < cols && n < a.N)
              *reinterpret_cast<uint2*>(o4 + int64_t(c0 + 4 * j) * a.ldo) = make_uint2(up ? got : a01, up ? a23 : got);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c0 + j < cols && n < a.N) o1[int64_t(c0 + j) * a.ldo] = uint16_t(bf16_pair(v[j], 0.f));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_at(in_cta(smem_u32(&acc_empty[b]), 0));
      if (++b == 2) b = 0, ph ^= 1;
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (dead && rank == 0 && threadIdx.x == 0) {
    // given up: let the copies in flight land (bounded)
    const uint64_t t0 = global_ns();
    for (int i = 0; i < kGtStages; ++i)
      while (!mbar_try(smem_u32(&full[i]), i < stopped_at ? stopped_phase ^ 1 : stopped_phase) &&
             global_ns() - t0 < kWaitLimitNs) {
      }
  }
  cluster_sync();   // the peer's copies and MMAs touch this CTA no more
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ---- rows gathered first ------------------------------------------------------

// x row of every position (zeros where it lies outside x), and its scale (1 if
// x has none, kNoRow outside x).  A warp copies kGatherPiece bytes of a row,
// all of its loads at once: many short warps hide the row number's latency
// better than fewer with several rows each.  20,480 rows of 2,048 bytes take
// 10 us.
constexpr int kGatherThreads = 256, kGatherAhead = 4, kGatherPiece = kGatherAhead * 512;

__global__ void __launch_bounds__(kGatherThreads) gather_rows_kernel(const GroupedArgs a, int row_bytes,
                                                                     int64_t ld_bytes,
                                                                     unsigned char* __restrict__ rows_out,
                                                                     float* __restrict__ scales_out) {
  chain_begin();
  const int lane = threadIdx.x & 31, pieces = (row_bytes + kGatherPiece - 1) / kGatherPiece;
  const int64_t unit = int64_t(blockIdx.x) * (kGatherThreads / 32) + (threadIdx.x >> 5), p = unit / pieces;
  if (p >= a.P) return;
  const int from = int(unit - p * pieces) * kGatherPiece + lane * 16, row = row_of(a, int(p));
  if (from == 0) {
    const float s = row >= 0 && a.x_scales ? __ldg(a.x_scales + row) : 1.f;
    scales_out[p] = __uint_as_float(row < 0 ? kNoRow : s == s ? __float_as_uint(s) : 0x7FC00000u);
  }
  const unsigned char* src = static_cast<const unsigned char*>(a.x) + (row < 0 ? 0 : row * ld_bytes);
  unsigned char* dst = rows_out + p * row_bytes;
  uint4 v[kGatherAhead];
#pragma unroll
  for (int u = 0; u < kGatherAhead; ++u)
    v[u] = from + 512 * u < row_bytes && row >= 0 ? ldg_nc(src + from + 512 * u) : make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int u = 0; u < kGatherAhead; ++u)
    if (from + 512 * u < row_bytes) *reinterpret_cast<uint4*>(dst + from + 512 * u) = v[u];
}

// ---- host side --------------------------------------------------------------

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn_grouped() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p) : nullptr;
  }();
  return fn;
}

// 128 bytes of K (128-byte swizzle) x `box_rows` rows of [outer][rows][K].
bool encode_k_rows(CUtensorMap* m, const void* p, bool fp8, int64_t K, int64_t rows, int64_t ld, int64_t outer,
                          int box_rows) {
  auto fn = encode_fn_grouped();
  if (!fn) return false;
  const int size = fp8 ? 1 : 2;
  const cuuint64_t dims[3] = {cuuint64_t(K), cuuint64_t(rows), cuuint64_t(outer)};
  const cuuint64_t strides[2] = {cuuint64_t(ld) * size, cuuint64_t(ld) * size * cuuint64_t(rows)};
  const cuuint32_t box[3] = {cuuint32_t(128 / size), cuuint32_t(box_rows), 1};
  const cuuint32_t step[3] = {1, 1, 1};
  return fn(m, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, outer ? 3 : 2,
            const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Which kernel runs, by the positions P of E experts (times in us, K = 2,048).
//
// Few rows (vx_grouped_few.cu) / the tiles here: N = 1,024, E = 512: one token
// bf16 11.8 / 14.0, four 31 / 40, e4m3 19.6 / 24.8, 100 positions bf16 121 /
// 121, e4m3 75 / 66; N = 2,048: E = 1 and 32 positions 8.1 / 12.4, 64 11.7 /
// 12.8, 128 19 / 14, E = 8 and 64 15.8 / 18.6, 128 23 / 19.  64 tokens over 512
// bf16 experts cold 234 / 225, but in steady state, under the power limit, 231
// / 239 (1.50 / 1.34 GHz: memory-bound MMAs here cost more power); e4m3 cold
// 141 / 120.
static bool few_rows(int64_t P, int experts, bool e4m3) { return P <= 64 || (!e4m3 && P <= 2 * int64_t(experts)); }
// Tens of rows (vx_grouped_mid.cu) / the tiles here, E = 512, N = 1,024: 10
// rows an expert e4m3 176 / 177, 40 bf16 363 / 371, 80 e4m3 224 / 222; E = 64,
// 128 rows 69.3 / 69.0, 640 158 / 150.  Banks of short rows are stores first,
// which are wider there: K = 512 e4m3, N = 2,048 40 rows 98 / 146, 160 183 /
// 198, E = 1 and 20,000 rows 37 / 45; K = 256 bf16 E = 8 and 2,048 rows 27 /
// 36, E = 4 and 500 7.2 / 9.0; K = 512 bf16, N = 2,048 160 rows 270 / 267.  It
// cuts a bank into half as many tiles, so with long rows they have to be
// enough for the SMs: E = 8, 16 rows 21.7 / 18.9.
static bool mid_rows(const GroupedArgs& a, int64_t row_bytes) {
  const int64_t groups = a.P < a.experts ? a.P : a.experts, tiles = groups * ((a.N + 255) / 256);
  return row_bytes <= 512 || (a.P <= 64 * int64_t(a.experts) && tiles >= sm_count());
}

int64_t grouped_workspace_bytes(int64_t P, int experts, int K, bool e4m3, bool rows) {
  if (!rows || few_rows(P, experts, e4m3)) return 0;
  const int64_t row = int64_t(K) * (e4m3 ? 1 : 2);
  return ((P * row + 255) & ~int64_t(255)) + 4 * P;
}

// x and its scales in the order of the positions, in the workspace; a takes
// their place.
static cudaError_t gather_rows(GroupedArgs& a, bool e4m3, void* workspace, cudaStream_t st) {
  const int size = e4m3 ? 1 : 2, row_bytes = a.K * size;
  unsigned char* rows = static_cast<unsigned char*>(workspace);
  float* scales = reinterpret_cast<float*>(rows + ((a.P * row_bytes + 255) & ~int64_t(255)));
  const int64_t units = a.P * ((row_bytes + kGatherPiece - 1) / kGatherPiece);
  const int64_t ctas = (units + kGatherThreads / 32 - 1) / (kGatherThreads / 32);
  if (ctas > 0x7FFFFFFF) return cudaErrorInvalidValue;
  const cudaError_t e = launch_chained(gather_rows_kernel, dim3(unsigned(ctas)), dim3(kGatherThreads), 0, st, a,
                                       row_bytes, a.ldx * size, rows, scales);
  a.x = rows;
  a.x_rows = a.P;
  a.ldx = a.K;
  a.x_scales = scales;
  a.rows = nullptr;
  a.slots = 1;
  a.gathered = true;
  return e;
}

template <bool FP8>
static cudaError_t launch_pairs(const GroupedTc& g, int pairs, cudaStream_t st) {
  auto k = grouped_kernel<FP8>;
  constexpr int kRing = kGtStages * kGtStage + 1024;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(k), kRing + 2 * (kGroupedMaxExperts + 1) * int(sizeof(int)),
                             done);
  if (e != cudaSuccess) return e;
  return launch_chained(k, dim3(2 * pairs), dim3(kGtThreads),
                        size_t(kRing + 2 * (g.a.experts + 1) * int(sizeof(int))), st, g);
}

cudaError_t launch_grouped(GroupedArgs a, bool e4m3, void* workspace, cudaStream_t st) {
  if (a.P == 0 || a.N == 0) return cudaSuccess;
  if (few_rows(a.P, a.experts, e4m3)) return launch_grouped_few(a, e4m3, st);
  if (a.rows) {
    const cudaError_t e = gather_rows(a, e4m3, workspace, st);
    if (e != cudaSuccess) return e;
  }
  if (mid_rows(a, int64_t(a.K) * (e4m3 ? 1 : 2))) return launch_grouped_mid(a, e4m3, st);
  GroupedTc g;
  g.a = a;
  g.row_tiles = (a.N + kGtRows - 1) / kGtRows;
  g.by_four = a.N % 4 == 0 && a.ldo % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % 8 == 0;
  // no more pairs than the groups can have tiles
  const int64_t groups = (a.P + kGtCols - 1) / kGtCols + (a.P < a.experts ? a.P : a.experts);
  if (groups * g.row_tiles > 0x7FFFFFFF) return cudaErrorInvalidValue;
  int64_t pairs = sm_count() / 2;
  if (groups * g.row_tiles < pairs) pairs = groups * g.row_tiles;
  if (!encode_k_rows(&g.tm_w, a.w, e4m3, a.K, a.N, a.K, a.experts, 128)) return cudaErrorInvalidValue;
  for (int i = 0; i < 4; ++i)
    if (!encode_k_rows(&g.tm_x[i], a.x, e4m3, a.K, a.x_rows, a.ldx, 0, 16 << i)) return cudaErrorInvalidValue;
  return e4m3 ? launch_pairs<true>(g, int(pairs), st) : launch_pairs<false>(g, int(pairs), st);
}

}  // namespace vx
