// What the grouped products share: a position's row, the table of groups that
// each CTA builds in its shared memory, bounded waits, tensor maps.
#pragma once

#include "vx_async.cuh"
#include "vx_common.cuh"
#include "vx_launch.h"

namespace vx {

// The row of x that position p reads; -1 where it lies outside x.
VX_DEVICE int row_of(const GroupedArgs& a, int p) {
  const int r = __ldg(a.rows + p);
  return r >= 0 && r / a.slots < a.x_rows ? r / a.slots : -1;
}
// The scale that a gathered position has if it names no row (a NaN that no
// other position gets).  Its row is zeros, and so is its output, also where
// the bank or its scales are no finite numbers.
constexpr uint32_t kNoRow = 0xFFFFFFFFu;
VX_DEVICE bool names_none(const GroupedArgs& a, float scale) {
  return a.gathered && __float_as_uint(scale) == kNoRow;
}

// mbar_try that also acquires what the other CTA of the pair released.
VX_DEVICE bool pair_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
VX_DEVICE uint32_t bf16_pair(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Bounded wait of a role, by a whole warp: false, in every lane, once this CTA
// has given up.  (With an answer of its own a lane could leave a loop whose
// other lanes wait for it at a __syncwarp.)
VX_DEVICE bool role_wait(uint32_t bar, uint32_t parity, volatile int* dead) {
  bool done = pair_try(bar, parity);
  if (!done) {
    const uint64_t t0 = global_ns();
    for (uint32_t i = 0; i < kSpinLimit && !done; ++i) {
      done = pair_try(bar, parity);
      if ((i & 255) == 255 && (*dead || global_ns() - t0 > kWaitLimitNs)) break;
    }
  }
  done = __all_sync(0xFFFFFFFFu, done);
  if (!done) *dead = 1;
  return done;
}

// Starts of the groups, clamped to [0, P] and to ascend (group e is starts[e]
// .. starts[e + 1], so all of them have P positions at most), and the
// exclusive scan of the number of items that each is cut into (at most `most`
// positions an item).  Every thread of the CTA constructs it; memory: 2
// (experts + 1) ints.
template <int THREADS>
struct GroupTable {
  int* first;    // items before expert e
  int* starts;
  int experts, most;

  // Inclusive scan over the CTA's threads; *all: over all of them.
  template <typename F>
  VX_DEVICE static int scan(int v, F&& join, int* all) {
    __shared__ int warps[THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xFFFFFFFFu, v, o);
      if (lane >= o) v = join(u, v);
    }
    if (lane == 31) warps[warp] = v;
    __syncthreads();
    int before = 0, total = 0;   // 0: neutral for what is scanned here
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before = join(before, warps[w]);
      total = join(total, warps[w]);
    }
    *all = total;
    return join(before, v);
  }

  VX_DEVICE GroupTable(const GroupedArgs& a, int* memory, int most_) : experts(a.experts), most(most_) {
    first = memory;
    starts = memory + experts + 1;
    // a thread takes neighbouring entries, all its loads at once
    const int P = int(a.P), each = (experts + THREADS) / THREADS, e0 = threadIdx.x * each;
    const int e1 = min(e0 + each, experts + 1);
    int top = 0, all;
    for (int e = e0; e < e1; ++e) {
      top = max(top, min(__ldg(a.offsets + e), P));
      starts[e] = top;   // among the thread's own
    }
    const int upper = scan(top, [](int x, int y) { return max(x, y); }, &all);   // of the threads up to this one
    // what the threads before this one reach: entry e0 - 1 after their own pass
    if (e0 < e1) first[e1 - 1] = upper;
    __syncthreads();
    const int before = e0 > 0 && e0 < e1 ? first[e0 - 1] : 0;
    for (int e = e0; e < e1; ++e) starts[e] = max(starts[e], before);
    __syncthreads();
    int v = 0;
    for (int e = e0; e < min(e1, experts); ++e) {
      first[e] = v;   // inside the thread's range
      v += (starts[e + 1] - starts[e] + most - 1) / most;
    }
    const int upto = scan(v, [](int x, int y) { return x + y; }, &all);
    for (int e = e0; e < min(e1, experts); ++e) first[e] += upto - v;
    if (threadIdx.x == 0) first[experts] = all;
    __syncthreads();
  }

  VX_DEVICE int items() const { return first[experts]; }

  // The expert that item i belongs to: the last e with first[e] <= i.  Called
  // by whole warps: 32 samples, then the entries between two of them (two
  // reads of shared memory, where a binary search waits for nine).
  VX_DEVICE int expert(int i) const {
    const int lane = threadIdx.x & 31, stride = (experts + 31) / 32;
    auto last = [&](int from, int by, int end) {   // of from, from + by, ... below end
      const int e = from + lane * by;
      const uint32_t under = __ballot_sync(0xFFFFFFFFu, e < end && first[e] <= i);
      return under ? from + (31 - __clz(under)) * by : -1;
    };
    int e = last(0, stride, experts);
    const int end = min(e + stride, experts);
    for (int from = e; from < end; from += 32) e = max(e, last(from, 1, end));
    return e;
  }
  VX_DEVICE int size(int e) const { return starts[e + 1] - starts[e]; }   // of a group with items

  // Item i of full items and a rest: its expert, first position and number of positions.
  VX_DEVICE int item(int i, int* e, int* p0) const {
    *e = expert(i);
    const int skip = (i - first[*e]) * most;
    *p0 = starts[*e] + skip;
    return min(most, size(*e) - skip);
  }
};

// v * a * b for the two scales of a value.  Their product in one where that is a
// normal number; where it would overflow or lose bits below 2^-126 although
// the value does not, they enter one by one: below, the larger first (v is a
// sum of e4m3 products, 2^-18 to 2^48: v times it stays in range), above, the
// smaller.  A zero enters first.
VX_DEVICE bool is_normal(float p) { return fabsf(p) >= 0x1p-126f && fabsf(p) <= 0x1.fffffep127f; }
VX_DEVICE float scaled(float v, float a, float b) {
  const float p = a * b;
  if (is_normal(p)) return v * p;
  const bool first = fabsf(a) > fabsf(b);
  const float hi = first ? a : b, lo = first ? b : a;
  return fabsf(p) < 1.f && lo != 0.f ? v * hi * lo : v * lo * hi;
}
// Whether v * (a * b) does for every scale a of the warp (N a lane, in s) and
// every lane's b: no product of theirs that is neither zero nor normal, and no
// kNoRow.  One check a tile, so that the tiles' inner loops multiply by the
// product.
template <int N>
VX_DEVICE bool products_fit(const float (&s)[N], float b) {
  uint32_t hi = 0, lo = 0x7F800000u;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t m = __float_as_uint(fabsf(s[i]));   // ordered as their values, NaN on top
    hi = max(hi, m);
    if (m) lo = min(lo, m);
  }
  hi = __reduce_max_sync(0xFFFFFFFFu, hi), lo = __reduce_min_sync(0xFFFFFFFFu, lo);
  const float m = fabsf(b);
  return __all_sync(0xFFFFFFFFu, m * __uint_as_float(hi) <= 0x1.fffffep127f &&
                                     (m == 0.f || m * __uint_as_float(lo) >= 0x1p-126f));
}

// True in one lane, the same one in every call, of a converged warp.  MMAs
// issued under it in a loop that the whole warp runs keep their operands in
// uniform registers; under `lane == 0` the compiler moves them there one by
// one, and an MMA takes 120 cycles to issue however small it is (M = 256, N =
// 32: 57 this way, N = 144: 72).
VX_DEVICE bool elect_one() {
  uint32_t one;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xFFFFFFFF; selp.u32 %0, 1, 0, p; }" : "=r"(one));
  return one != 0;
}
// v of lane 0, which the compiler then knows to be the same in all lanes.
VX_DEVICE uint32_t uniform(uint32_t v) { return __shfl_sync(0xFFFFFFFFu, v, 0); }

VX_DEVICE void prefetch_map(const void* m) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(m)) : "memory");
}

// Tensor map of 128 bytes of K (128-byte swizzle) x `box_rows` rows of
// [outer][rows][K] (outer 0: [rows][K]); false if it cannot be encoded.
bool encode_k_rows(CUtensorMap* m, const void* p, bool fp8, int64_t K, int64_t rows, int64_t ld, int64_t outer,
                   int box_rows);

}  // namespace vx
