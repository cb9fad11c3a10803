// Window attention's gradients on tcgen05 tiles.  One pipeline, two forms:
//
//   form     owns (128 rows)  streams     accumulates
//   kKeys    K, V             Q, dO       dK += dS^T Q, dV += P^T dO
//   queries  Q, dO            K, V        dQ += dS K
//
// Each step forms S = own1 str1^T and dP = own2 str2^T (fp32, TMEM, the owned
// rows on the lanes), the elementwise warps turn them into P = exp2(S c - lse)
// and dS = P (dP - delta) as bf16 in TMEM, and those are the A operands of the
// accumulating products, whose B operands are the streamed tiles again (now
// read along their rows).  Every output element has one owner that adds in a
// fixed order: no atomics, equal bits from call to call.  (Where a key tile's
// steps would be the longest chain of the launch -- sinks are seen by all later
// queries, or there are few tiles -- they are divided among `parts` CTAs, whose
// fp32 sums part_sum_kernel adds in order.)
//
// TMEM (all 512 columns at D = 128): kSBufs buffers of S, one of dP, the
// accumulators.  P and dS overwrite their S.  A step is a chain of signals of
// about 300 cycles each (product -> barrier -> TMEM load -> barrier -> next
// product), longer than its products: with one buffer of S and dP the chain
// took 2,050 cycles a step where the products need 1,280 (kKeys).  So S runs
// steps ahead, and dP alone waits for its one buffer, which is free as soon as
// it is in the registers.  kKeys steps are 64 queries wide: at D = 128 two
// accumulators of D columns leave no room for 128 (at D = 64 they would; the
// kernel is the same there).
//
// Roles: elementwise and epilogue warps (warp w: lanes 32 (w % 4), the w / 4th
// share of the columns), then a TMA warp, one that issues S and dP and one that
// issues the accumulating products.  Waits are bounded as in the forward kernel.
#pragma once

#include "attention_kernel.cuh"
#include "ptx.cuh"
#include "view.cuh"

namespace b200 {
namespace bwd {

constexpr int kOwn = 128;  // owned rows
constexpr int kBarQuad = 1;  // named barriers 1-4: the warps of a lane quadrant

template <int D, bool kKeys>
struct TileCfg {
  static constexpr int kN = kKeys ? 64 : 128;  // streamed rows of a step
  static constexpr int kGroups = 4;                 // elementwise warpgroups
  static constexpr int kWarps = 4 * kGroups;     // elementwise warps
  static constexpr int kCols = kN / kGroups;     // columns of a step for each
  static constexpr int kThreads = 32 * (kWarps + 4);
  // Epilogue: warpgroups of an accumulator, columns for each.
  static constexpr int kAccGroups = kKeys ? kGroups / 2 : kGroups;
  static constexpr int kAccCols = D / kAccGroups;
  // Ring depths of the two streamed tensors.  Both of kKeys' live until the
  // accumulating products have read them, but V only until dP has: K gets the
  // odd stage.
  static constexpr int kStages1 = (kKeys ? 4 : 3) * (128 / D);
  static constexpr int kStages2 = (kKeys ? 4 : 2) * (128 / D);
  static constexpr int kBoxes = D / 64;
  static constexpr int kOwnBox = kOwn * 128;
  static constexpr int kOwnBytes = kBoxes * kOwnBox;
  static constexpr int kStrBox = kN * 128;
  static constexpr int kStrBytes = kBoxes * kStrBox;
  static constexpr int kStatBytes = kKeys ? 2 * kN * 4 : 0;  // -lse, -delta of the queries
  static constexpr int kRingOff = 2 * kOwnBytes;
  static constexpr int kRing2Off = kRingOff + kStages1 * kStrBytes;
  static constexpr int kStatOff = kRing2Off + kStages2 * kStrBytes;
  static constexpr int kBarOff = kStatOff + kStages2 * kStatBytes;
  // own_full own_empty p_free[3] sd_ready dp_free p_ready[3] acc_full acc_empty drain
  static constexpr int kNumBars = 13 + 2 * (kStages1 + kStages2);
  static constexpr int kSlotOff = kBarOff + kNumBars * 8;
  static constexpr int kSmemBytes = kSlotOff + 16 + 1024;  // + alignment slack
  static_assert(kSmemBytes <= 232448, "exceeds the 227 KiB of shared memory a CTA may use");
  static_assert(kSmemBytes > 116 * 1024, "one CTA per SM: each takes all of TMEM");
  static constexpr int kSBufs = kKeys ? 3 : 2;
  static constexpr uint32_t kColDp = kSBufs * kN;
  static constexpr uint32_t kDs = kKeys ? kN / 2 : 0;  // dS in its S buffer (P at 0)
  static constexpr uint32_t kColAcc1 = 512 - 2 * D, kColAcc2 = 512 - D;
  static_assert(kColDp + kN <= (kKeys ? kColAcc1 : kColAcc2), "TMEM columns");
  static constexpr uint32_t kIdescS = idesc_bf16_f32(kOwn, kN, false, false);
  static constexpr uint32_t kIdescAcc = idesc_bf16_f32(kOwn, D, false, true);
};

struct TileParams {
  View out1, out2;       // kKeys: dK, dV; queries: dQ
  const float* stats;    // [2][B * Hq][sq_pad]: -lse in log2 units, -delta
  int64_t stat_plane;    // B * Hq * sq_pad
  int sq_pad;            // Sq up to a multiple of 64
  const int32_t* kv_len;
  int B, Hq, Hkv, group, Sq, Skv;
  int tiles;             // owned tiles of a (batch, head)
  int n_items;
  // kKeys: the first part_tiles tiles are divided into parts units each
  // (0: none are), which write [B * Hkv][part_tiles][parts][dK, dV][128][D].
  int part_tiles, parts;
  float* part_sums;
  int window, sinks;
  float scale, scale_log2;
  // Coordinate factors of broadcast axes (own1, own2, str1, str2; batch, head).
  int o1_b, o1_h, o2_b, o2_h, s1_b, s1_h, s2_b, s2_h;
};

enum : uint32_t {
  kSiteBwdOwn = 0x20, kSiteBwdFull, kSiteBwdEmpty, kSiteBwdS, kSiteBwdP,
  kSiteBwdAcc
};

// -lse and -delta of every query row, padded with zeros.  D/8 lanes to a row
// (16 bytes each of dO and O); a block's rows lie in one (batch, head).
constexpr int kStatRows = 64;

template <int D>
__global__ void __launch_bounds__(256)
    stats_kernel(const View dout, const View o, const float* lse, float* stats, int64_t plane,
                 int sq_pad, int B, int Hq, int Sq) {
  constexpr int kLanes = D / 8, kRows = 256 / kLanes, kUnroll = kStatRows / kRows;
  pdl_launch_dependents();
  const int lane = static_cast<int>(threadIdx.x) % kLanes;
  const int blocks_s = sq_pad / kStatRows;
  const int bh = static_cast<int>(blockIdx.x) / blocks_s;
  const int s0 = (static_cast<int>(blockIdx.x) - bh * blocks_s) * kStatRows +
                 static_cast<int>(threadIdx.x) / kLanes;
  const int b = bh / Hq, h = bh - b * Hq;
  const uint16_t* x_row = dout.row(b, h, s0) + lane * 8;
  const uint16_t* y_row = o.row(b, h, s0) + lane * 8;
  uint4 x[kUnroll], y[kUnroll];
  float l[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    x[u] = y[u] = make_uint4(0u, 0u, 0u, 0u);
    l[u] = 0.0f;
    if (s0 + u * kRows < Sq) {
      x[u] = __ldg(reinterpret_cast<const uint4*>(x_row + u * kRows * dout.ss));
      y[u] = __ldg(reinterpret_cast<const uint4*>(y_row + u * kRows * o.ss));
      l[u] = __ldg(lse + static_cast<int64_t>(bh) * Sq + s0 + u * kRows);
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const uint32_t a[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
    const uint32_t e[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum = fmaf(__uint_as_float(a[i] << 16), __uint_as_float(e[i] << 16), sum);
      sum = fmaf(__uint_as_float(a[i] & 0xffff0000u), __uint_as_float(e[i] & 0xffff0000u), sum);
    }
#pragma unroll
    for (int m = kLanes / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    if (lane == 0) {
      float* dst = stats + static_cast<int64_t>(bh) * sq_pad + s0 + u * kRows;
      dst[0] = l[u] == -INFINITY ? 0.0f : l[u] * -1.4426950408889634f;
      dst[plane] = -sum;
    }
  }
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
      : "memory");
}

// TMEM loads and stores of a thread's columns.
__device__ __forceinline__ void ld_cols(uint32_t taddr, uint32_t (&r)[32]) { tmem_ld32(taddr, r); }
__device__ __forceinline__ void ld_cols(uint32_t taddr, uint32_t (&r)[16]) { tmem_ld16(taddr, r); }
__device__ __forceinline__ void st_cols(uint32_t taddr, const uint32_t (&r)[16]) {
  tmem_st16(taddr, r);
}
__device__ __forceinline__ void st_cols(uint32_t taddr, const uint32_t (&r)[8]) {
  tmem_st8(taddr, r);
}
__device__ __forceinline__ void written_here(uint32_t (&r)[32]) { reg_written_here(r); }
__device__ __forceinline__ void written_here(uint32_t (&r)[16]) { reg_written_here16(r); }

// Transposes 16-byte pieces among groups of kShare lanes: afterwards piece e of
// lane q is what piece q of lane e was.
template <int kShare>
__device__ __forceinline__ void exchange(uint32_t (&x)[4 * kShare], int lane) {
#pragma unroll
  for (int m = 1; m < kShare; m <<= 1) {
    const bool up = lane & m;
#pragma unroll
    for (int e = 0; e < kShare; ++e) {
      if (e & m) continue;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t& a = x[4 * e + u];
        uint32_t& b = x[4 * (e | m) + u];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? a : b, m);
        if (up)
          a = got;
        else
          b = got;
      }
    }
  }
}

// One owned tile: where it lies and what it streams.
template <bool kKeys>
struct TileItem {
  int b, h;         // h: kv head (kKeys) or query head
  int r0;           // first owned row
  int n, off;       // keys of the request; position of query row 0
  int steps;
  int per_head, t0;             // kKeys: steps of a query head, first 64-query tile
  int first, part;              // kKeys: first step; the part of a divided tile, or -1
  // queries: they see keys of [0, se) and [lo, hi) only; tile i of keys is i for
  // the n_sink tiles before the window's and i + skip after them.
  int se, lo, hi, n_sink, skip;
};

template <bool kKeys>
__device__ __forceinline__ TileItem<kKeys> tile_item(const TileParams& p, int k) {
  TileItem<kKeys> it;
  const int heads = kKeys ? p.Hkv : p.Hq;
  // All (batch, head) of one tile index are adjacent: for keys the first tiles
  // (sinks, seen by most queries) start first, for queries the last ones.
  it.part = -1;
  if (kKeys && p.parts > 0) {
    const int divided = p.B * heads * p.part_tiles * p.parts;
    if (k < divided) {
      it.part = k % p.parts;
      k /= p.parts;
    } else {
      k -= divided - p.B * heads * p.part_tiles;
    }
  }
  int tile = k / (p.B * heads);
  const int bh = k - tile * (p.B * heads);
  if (!kKeys) tile = p.tiles - 1 - tile;
  it.b = bh / heads;
  it.h = bh - it.b * heads;
  it.r0 = tile * kOwn;
  it.n = p.kv_len ? max(0, min(ld_global_l2(p.kv_len + it.b), p.Skv)) : p.Skv;
  it.off = it.n - p.Sq;
  if constexpr (kKeys) {
    const int k1 = min(it.r0 + kOwn, it.n);  // queries [i0, i1) see some of keys [r0, k1)
    const int i0 = max(0, it.r0 - it.off);
    const int i1 = k1 <= it.r0 ? 0
                   : it.r0 < p.sinks ? p.Sq
                                     : min(p.Sq, k1 - 1 + p.window - it.off);
    it.t0 = i0 / 64;
    it.per_head = i1 > i0 ? (i1 + 63) / 64 - it.t0 : 0;
    it.first = 0;
    it.steps = it.per_head * p.group;
    if (it.part >= 0) {
      const int64_t all = it.steps;
      it.first = static_cast<int>(all * it.part / p.parts);
      it.steps = static_cast<int>(all * (it.part + 1) / p.parts) - it.first;
    }
  } else {
    const int last = it.off + min(it.r0 + kOwn, p.Sq) - 1;
    it.hi = max(0, last + 1);
    it.lo = max(0, it.off + it.r0 - p.window + 1);
    if (p.sinks >= it.lo || it.hi == 0) it.lo = 0;
    it.se = it.lo > 0 ? p.sinks : 0;
    const int w0 = it.lo / 128;
    it.per_head = -1;
    it.n_sink = min((it.se + 127) / 128, w0);
    it.skip = w0 - it.n_sink;
    it.steps = it.n_sink + (it.hi + 127) / 128 - w0;
  }
  return it;
}

// P and dS of kCols columns of this thread's row, as bf16 pairs.  kKeys: -lse and
// -delta of the columns at st_l and st_l + n; else the row's own.
template <bool kKeys, bool kMasked, int kCols>
__device__ __forceinline__ void elementwise(const uint32_t (&s)[kCols], const uint32_t (&d)[kCols],
                                            uint64_t c2, const float* st_l, int n, float nlse,
                                            float ndelta, int col0, int va, int vb, int vs,
                                            uint32_t (&pk)[kCols / 2],
                                            uint32_t (&dk)[kCols / 2]) {
#pragma unroll
  for (int e = 0; e < kCols / 2; ++e) {
    uint64_t nl2, nd2;
    if constexpr (kKeys) {
      nl2 = *reinterpret_cast<const uint64_t*>(st_l + 2 * e);
      nd2 = *reinterpret_cast<const uint64_t*>(st_l + n + 2 * e);
    } else {
      nl2 = f2_pack(nlse, nlse);
      nd2 = f2_pack(ndelta, ndelta);
    }
    const uint64_t x2 =
        f2_fma(f2_pack(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), c2, nl2);
    float x0, x1;
    f2_unpack(x2, x0, x1);
    float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
    const uint64_t g2 =
        f2_mul(f2_pack(p0, p1),
               f2_add(f2_pack(__uint_as_float(d[2 * e]), __uint_as_float(d[2 * e + 1])), nd2));
    float g0, g1;
    f2_unpack(g2, g0, g1);
    if constexpr (kMasked) {
      const int u = col0 + 2 * e;
      bool see0 = u >= va && u < vb, see1 = u + 1 >= va && u + 1 < vb;
      if constexpr (!kKeys) {
        see0 |= u < vs;
        see1 |= u + 1 < vs;
      }
      p0 = see0 ? p0 : 0.0f;
      p1 = see1 ? p1 : 0.0f;
      g0 = see0 ? g0 : 0.0f;
      g1 = see1 ? g1 : 0.0f;
    }
    if constexpr (kKeys) pk[e] = pack_bf16x2(p0, p1);
    dk[e] = pack_bf16x2(g0, g1);
  }
}

template <int D, bool kKeys>
__global__ void __launch_bounds__(TileCfg<D, kKeys>::kThreads, 1)
    bwd_tile_kernel(const __grid_constant__ CUtensorMap own1_map,
                    const __grid_constant__ CUtensorMap own2_map,
                    const __grid_constant__ CUtensorMap str1_map,
                    const __grid_constant__ CUtensorMap str2_map,
                    const __grid_constant__ TileParams p) {
  using C = TileCfg<D, kKeys>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* own = smem;
  uint8_t* ring1 = smem + C::kRingOff;
  uint8_t* ring2 = smem + C::kRing2Off;
  float* stat = reinterpret_cast<float*>(smem + C::kStatOff);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t *own_full = bars, *own_empty = bars + 1, *p_free = bars + 2, *sd_ready = bars + 5,
           *dp_free = bars + 6, *p_ready = bars + 7, *acc_full = bars + 10,
           *acc_empty = bars + 11, *drain = bars + 12, *full1 = bars + 13,
           *empty1 = full1 + C::kStages1, *full2 = empty1 + C::kStages1,
           *empty2 = full2 + C::kStages2;
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + C::kSlotOff);
  const int warp = static_cast<int>(warp_id()), lane = static_cast<int>(lane_id());

  if (threadIdx.x == 0) {
    mbar_init(own_full, 1);
    mbar_init(own_empty, 1);
    for (int i = 0; i < 3; ++i) {
      mbar_init(&p_free[i], 1);
      // One for each S buffer: the elementwise warps may be as many steps ahead of
      // the accumulating one as there are buffers, but a buffer's next P waits for
      // the products that this one's phase admits.
      mbar_init(&p_ready[i], C::kWarps);
    }
    mbar_init(sd_ready, 1);
    mbar_init(dp_free, C::kWarps);
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, C::kWarps);
    mbar_init(drain, 2);
    for (int i = 0; i < 2 * (C::kStages1 + C::kStages2); ++i) mbar_init(&full1[i], 1);
    fence_mbar_init();
  }
  if (warp == C::kWarps) {
    tmem_alloc(slot, 512);
    tmem_relinquish();
    if (lane == 0) {
      tma_prefetch_desc(&own1_map);
      tma_prefetch_desc(&own2_map);
      tma_prefetch_desc(&str1_map);
      tma_prefetch_desc(&str2_map);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;
  if constexpr (kKeys) {
    // The row statistics; then the queries' kernel may start where this one's
    // last CTAs leave SMs free (they are complete for it too).
    pdl_wait();
    pdl_launch_dependents();
  }

  // First streamed row of a query head's step i.
  auto str_row = [&](const TileItem<kKeys>& it, int i) {
    if constexpr (kKeys)
      return (it.t0 + i) * 64;
    else
      return (i < it.n_sink ? i : i + it.skip) * 128;
  };

  if (warp == C::kWarps) {
    // ================= TMA producer =================
    if (lane == 0) {
      const uint64_t pol_own = l2_policy_evict_first(), pol_str = l2_policy_evict_last();
      int t = 0, li = 0, n1 = 0, n2 = 0;  // steps; copies issued
      bool ok = true;
      for (int k = static_cast<int>(blockIdx.x); k < p.n_items && ok; k += gridDim.x) {
        const TileItem<kKeys> it = tile_item<kKeys>(p, k);
        if (it.steps == 0) continue;
        ok = mbar_wait(own_empty, (static_cast<uint32_t>(li) & 1u) ^ 1u, kSiteBwdOwn,
                       kDefaultWaitLimitNs, 20000u);
        if (!ok) break;
        mbar_arrive_expect_tx(own_full, 2 * C::kOwnBytes);
        for (int x = 0; x < C::kBoxes; ++x) {
          tma_load_4d(own + x * C::kOwnBox, &own1_map, own_full, x * 64, it.r0, it.h * p.o1_h,
                      it.b * p.o1_b, pol_own);
          tma_load_4d(own + C::kOwnBytes + x * C::kOwnBox, &own2_map, own_full, x * 64, it.r0,
                      it.h * p.o2_h, it.b * p.o2_b, pol_own);
        }
        ++li;
        // Step of a query head; the head.
        int hi = kKeys && it.steps > 0 ? it.first % it.per_head : 0;
        int hq = kKeys ? it.h * p.group + it.first / max(it.per_head, 1) : it.h;
        for (int i = 0; i < it.steps; ++i, ++t) {
          const int st1 = t % C::kStages1, st2 = t % C::kStages2;
          const int row = str_row(it, hi);
          const int h = kKeys ? hq : it.h / p.group;
          ok = mbar_wait(&empty1[st1], (static_cast<uint32_t>(t / C::kStages1) & 1u) ^ 1u,
                         kSiteBwdEmpty, kDefaultWaitLimitNs, 20000u);
          if (!ok) break;
          mbar_arrive_expect_tx(&full1[st1], C::kStrBytes);
          for (int x = 0; x < C::kBoxes; ++x)
            tma_load_4d(ring1 + st1 * C::kStrBytes + x * C::kStrBox, &str1_map, &full1[st1],
                        x * 64, row, h * p.s1_h, it.b * p.s1_b, pol_str);
          n1 = t + 1;
          ok = mbar_wait(&empty2[st2], (static_cast<uint32_t>(t / C::kStages2) & 1u) ^ 1u,
                         kSiteBwdEmpty, kDefaultWaitLimitNs, 20000u);
          if (!ok) break;
          mbar_arrive_expect_tx(&full2[st2], C::kStrBytes + C::kStatBytes);
          for (int x = 0; x < C::kBoxes; ++x)
            tma_load_4d(ring2 + st2 * C::kStrBytes + x * C::kStrBox, &str2_map, &full2[st2],
                        x * 64, row, h * p.s2_h, it.b * p.s2_b, pol_str);
          if constexpr (kKeys) {
            const float* src =
                p.stats + (static_cast<int64_t>(it.b) * p.Hq + hq) * p.sq_pad + row;
            float* sdst = stat + st2 * 2 * C::kN;
            bulk_load(sdst, src, C::kN * 4, &full2[st2]);
            bulk_load(sdst + C::kN, src + p.stat_plane, C::kN * 4, &full2[st2]);
          }
          n2 = t + 1;
          ++hi;
          if (kKeys && hi == it.per_head) {
            hi = 0;
            ++hq;
          }
        }
      }
      if (!ok) {
        // Unwinding: let every copy already issued land before the CTA exits.
        if (li > 0) attn::drain_wait(own_full, static_cast<uint32_t>(li - 1) & 1u);
        for (int i = max(0, n1 - C::kStages1); i < n1; ++i)
          attn::drain_wait(&full1[i % C::kStages1], static_cast<uint32_t>(i / C::kStages1) & 1u);
        for (int i = max(0, n2 - C::kStages2); i < n2; ++i)
          attn::drain_wait(&full2[i % C::kStages2], static_cast<uint32_t>(i / C::kStages2) & 1u);
      }
    }
    __syncwarp();
  } else if (warp == C::kWarps + 1 || warp == C::kWarps + 2) {
    // ================= MMA issuers =================
    const bool acc = warp == C::kWarps + 2;
    const uint32_t own_addr = smem_u32(own);
    const uint64_t d_own1 = sdesc_sw128(own_addr, 16, 1024);
    const uint64_t d_own2 = sdesc_sw128(own_addr + C::kOwnBytes, 16, 1024);
    // Streamed tiles with their rows as N (S, dP) and as K (accumulation).
    const uint64_t d_n1 = sdesc_sw128(smem_u32(ring1), 16, 1024);
    const uint64_t d_n2 = sdesc_sw128(smem_u32(ring2), 16, 1024);
    const uint64_t d_k1 = sdesc_sw128(smem_u32(ring1), C::kStrBox, 1024);
    const uint64_t d_k2 = sdesc_sw128(smem_u32(ring2), C::kStrBox, 1024);
    constexpr uint32_t kStr16 = C::kStrBytes >> 4;
    auto warp_wait = [&](uint64_t* bar, uint32_t parity, uint32_t site) {
      const bool ok = attn::warp_wait(bar, parity, site);
      tc_fence_after();
      return ok;
    };
    int t = 0, li = 0;
    bool ok = true;
    for (int k = static_cast<int>(blockIdx.x); k < p.n_items && ok; k += gridDim.x) {
      const int steps = tile_item<kKeys>(p, k).steps;
      if (steps == 0) continue;
      if (!acc) {
        ok = warp_wait(own_full, static_cast<uint32_t>(li) & 1u, kSiteBwdOwn);
      } else {
        // The epilogue of the item before has read the accumulators.
        ok = warp_wait(acc_empty, (static_cast<uint32_t>(li) & 1u) ^ 1u, kSiteBwdAcc);
      }
      ++li;
      for (int i = 0; i < steps && ok; ++i, ++t) {
        const int st1 = t % C::kStages1, st2 = t % C::kStages2;
        const uint32_t par1 = static_cast<uint32_t>(t / C::kStages1) & 1u;
        const uint32_t par2 = static_cast<uint32_t>(t / C::kStages2) & 1u;
        const int sb = t % C::kSBufs;  // S buffer
        const uint32_t t_s = tmem + static_cast<uint32_t>(sb * C::kN);
        if (!acc) {
          // S(t), once the products of step t - kSBufs have read P and dS there.
          {
            const uint32_t f = smem_u32(&full1[st1]);
            ok = __all_sync(0xffffffffu,
                            mbar_wait3(f, par1, smem_u32(&p_free[sb]),
                                       (static_cast<uint32_t>(t / C::kSBufs) & 1u) ^ 1u, f, par1,
                                       kSiteBwdFull));
          }
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            mma_ss_warp(t_s, d_own1 + (kk >> 2) * (C::kOwnBox >> 4) + (kk & 3) * 2,
                        d_n1 + st1 * kStr16 + (kk >> 2) * (C::kStrBox >> 4) + (kk & 3) * 2,
                        C::kIdescS, kk > 0 ? 1u : 0u);
          // dP(t), once dP(t - 1) is in the registers.
          {
            const uint32_t f = smem_u32(&full2[st2]);
            ok = __all_sync(0xffffffffu,
                            mbar_wait3(f, par2, smem_u32(dp_free),
                                       (static_cast<uint32_t>(t) & 1u) ^ 1u, f, par2,
                                       kSiteBwdFull));
          }
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            mma_ss_warp(tmem + C::kColDp, d_own2 + (kk >> 2) * (C::kOwnBox >> 4) + (kk & 3) * 2,
                        d_n2 + st2 * kStr16 + (kk >> 2) * (C::kStrBox >> 4) + (kk & 3) * 2,
                        C::kIdescS, kk > 0 ? 1u : 0u);
          if constexpr (!kKeys) mma_commit_warp(&empty2[st2]);
          mma_commit_warp(sd_ready);
          if (i + 1 == steps) mma_commit_warp(own_empty);
        } else {
          ok = warp_wait(&p_ready[sb], static_cast<uint32_t>(t / C::kSBufs) & 1u, kSiteBwdP);
          if (!ok) break;
          if constexpr (kKeys) {
#pragma unroll
            for (int kk = 0; kk < C::kN / 16; ++kk)
              mma_ts_warp(tmem + C::kColAcc2, t_s + kk * 8,
                          d_k2 + st2 * kStr16 + kk * (2048 >> 4), C::kIdescAcc,
                          (i > 0 || kk > 0) ? 1u : 0u);
          }
#pragma unroll
          for (int kk = 0; kk < C::kN / 16; ++kk)
            mma_ts_warp(tmem + (kKeys ? C::kColAcc1 : C::kColAcc2), t_s + C::kDs + kk * 8,
                        d_k1 + st1 * kStr16 + kk * (2048 >> 4), C::kIdescAcc,
                        (i > 0 || kk > 0) ? 1u : 0u);
          mma_commit_warp(&empty1[st1]);
          if constexpr (kKeys) mma_commit_warp(&empty2[st2]);
          mma_commit_warp(&p_free[sb]);
          if (i + 1 == steps) mma_commit_warp(acc_full);
        }
      }
    }
    mma_commit_warp(drain);
    attn::drain_wait(drain, 0);
    __syncwarp();
  } else if (warp < C::kWarps) {
    // ================= elementwise and epilogue =================
    const int quad = warp & 3, wg = warp >> 2;
    const int col0 = wg * C::kCols;
    const int row = quad * 32 + lane;
    const uint32_t tlane = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const float c = p.scale_log2;
    const uint64_t c2 = f2_pack(c, c);
    const uint32_t sd_bar = smem_u32(sd_ready), full2_bar = smem_u32(full2);
    // Epilogue: this warpgroup's columns of dQ, or of dK or dV (`second`).
    const bool second = kKeys && wg >= C::kAccGroups;
    const View& out = second ? p.out2 : p.out1;
    const float out_scale = second ? 1.0f : p.scale;
    const int c0 = wg % C::kAccGroups * C::kAccCols;
    const uint32_t tacc = tlane + (kKeys && !second ? C::kColAcc1 : C::kColAcc2) + c0;
    int t = 0, sb = 0, li = 0;  // steps, t % kSBufs, items with steps
    bool ok = true;
    TileItem<kKeys> it{};
    float nlse = 0.0f, ndelta = 0.0f;
    auto open_item = [&](int k) {
      it = tile_item<kKeys>(p, k);
      if (!kKeys && it.r0 + row < p.Sq) {
        const float* src =
            p.stats + (static_cast<int64_t>(it.b) * p.Hq + it.h) * p.sq_pad + it.r0 + row;
        nlse = ld_global_l2(src);
        ndelta = ld_global_l2(src + p.stat_plane);
      }
    };
    if (static_cast<int>(blockIdx.x) < p.n_items) open_item(static_cast<int>(blockIdx.x));
    for (int k = static_cast<int>(blockIdx.x); k < p.n_items && ok; k += gridDim.x) {
      const int my = it.r0 + row;  // this thread's key or query
      // Steps whose pairs are all visible: those with str0 in [clear0, clear1],
      // or (queries) below clear1 and within the sinks.
      int clear0, clear1;
      // The streamed positions [va, vb) that this row meets; queries also
      // those below vs (sinks).
      int va, vb, vs = 0;
      // Live streamed rows: [0, se) and [lo, hi).  The others may hold anything.
      int se, lo, hi;
      if constexpr (kKeys) {
        const bool sinks_only = it.r0 + kOwn <= p.sinks;
        clear0 = it.r0 + kOwn - 1 - it.off;
        clear1 = min(p.Sq - 64, sinks_only ? p.Sq : p.window - 64 + it.r0 - it.off);
        va = my - it.off;
        vb = min(p.Sq, my < p.sinks ? p.Sq : my + p.window - it.off);
        se = 0;
        lo = max(0, -it.off);
        hi = 0x7fffffff;
      } else {
        const int first = it.off + it.r0, pos = it.off + my;
        clear0 = first + kOwn - p.window;
        clear1 = it.r0 + kOwn <= p.Sq ? first - 127 : -1;
        va = pos - p.window + 1;
        vb = pos + 1;
        vs = min(p.sinks, pos + 1);
        if (my >= p.Sq) va = vb = vs = 0;
        se = it.se;
        lo = it.lo;
        hi = it.hi;
      }
      int head_i = kKeys && it.steps > 0 ? it.first % it.per_head : 0;  // step of a head
      int str0 = str_row(it, head_i);
      for (int i = 0; i < it.steps; ++i, ++t) {
        const bool masked =
            str0 > clear1 || (str0 < clear0 && (kKeys || str0 + 128 > p.sinks));
        // S and dP; kKeys: the columns' statistics, which came with dO.
        {
          const uint32_t par = static_cast<uint32_t>(t) & 1u;
          const uint32_t f_bar = kKeys ? full2_bar + 8u * (t % C::kStages2) : sd_bar;
          const uint32_t f_par = kKeys ? static_cast<uint32_t>(t / C::kStages2) & 1u : par;
          ok = __all_sync(0xffffffffu,
                          mbar_wait3(sd_bar, par, f_bar, f_par, sd_bar, par, kSiteBwdS));
        }
        if (!ok) {
          // Another warp of the quadrant may have seen the barrier: it must not
          // wait for this one.  (It gets no further: dP stays taken.)
          named_bar_arrive(kBarQuad + quad, 32 * C::kGroups);
          break;
        }
        tc_fence_after();
        uint32_t s[C::kCols], d[C::kCols];
        const int buf = sb;
        const uint32_t t_s = tlane + static_cast<uint32_t>(buf * C::kN);
        if (++sb == C::kSBufs) sb = 0;
        ld_cols(t_s + col0, s);
        ld_cols(tlane + C::kColDp + col0, d);
        tmem_wait_ld();
        written_here(s);
        written_here(d);
        // The next step's dP may overwrite this one's, and, once the warps of
        // this quadrant have all loaded S, P and dS may overwrite that.
        tc_fence_before();
        __syncwarp();
        mbar_arrive_warp(dp_free);
        named_bar_sync(kBarQuad + quad, 32 * C::kGroups);
        tc_fence_after();
        uint32_t pk[C::kCols / 2], dk[C::kCols / 2];
        const float* st_l = stat + t % C::kStages2 * 2 * C::kN + col0;
        if (masked)
          elementwise<kKeys, true>(s, d, c2, st_l, C::kN, nlse, ndelta, col0, va - str0, vb - str0,
                                   vs - str0, pk, dk);
        else
          elementwise<kKeys, false>(s, d, c2, st_l, C::kN, nlse, ndelta, col0, 0, 0, 0, pk, dk);
        if constexpr (kKeys) st_cols(t_s + (col0 >> 1), pk);
        st_cols(t_s + C::kDs + (col0 >> 1), dk);
        // Streamed rows that nothing sees: zeroed before the accumulating
        // products read them (0 * NaN is NaN).
        if (str0 + C::kN > hi || (str0 < lo && str0 + C::kN > se)) {
          const int st1 = t % C::kStages1, st2 = t % C::kStages2;
          ok = attn::warp_wait(&full1[st1], static_cast<uint32_t>(t / C::kStages1) & 1u,
                               kSiteBwdFull);
          if (!ok) break;
          for (int r = static_cast<int>(threadIdx.x); r < (kKeys ? 2 : 1) * C::kBoxes * C::kN;
               r += 32 * C::kWarps) {
            const int sr = str0 + r % C::kN;
            if (sr >= hi || (sr < lo && sr >= se)) {
              const int x = r / C::kN;  // boxes of the first tensor, then of the second
              uint8_t* box = x < C::kBoxes
                                 ? ring1 + st1 * C::kStrBytes + x * C::kStrBox
                                 : ring2 + st2 * C::kStrBytes + (x - C::kBoxes) * C::kStrBox;
              const uint32_t at = smem_u32(box) + static_cast<uint32_t>(r % C::kN) * 128u;
#pragma unroll
              for (int e = 0; e < 8; ++e) st_shared_v4(at + e * 16, 0u, 0u, 0u, 0u);
            }
          }
          fence_proxy_async_smem();
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        mbar_arrive_warp(&p_ready[buf]);
        if constexpr (kKeys) {
          str0 += 64;
          if (++head_i == it.per_head) {
            head_i = 0;
            str0 = str_row(it, 0);
          }
        } else {
          str0 = i + 1 == it.n_sink ? str_row(it, i + 1) : str0 + 128;
        }
      }
      if (!ok) break;
      const bool any = it.steps > 0;
      const int b = it.b, h = it.h, r0 = it.r0, part = it.part;
      // The next item's request length and statistics, under this one's end.
      if (k + static_cast<int>(gridDim.x) < p.n_items) open_item(k + gridDim.x);
      if (any) {
        ok = attn::warp_wait(acc_full, static_cast<uint32_t>(li) & 1u, kSiteBwdAcc);
        if (!ok) break;
        ++li;
        tc_fence_after();
      }
      float* sums = nullptr;  // a divided tile's row
      if (kKeys && part >= 0)
        sums = p.part_sums + ((((static_cast<int64_t>(b) * p.Hkv + h) * p.part_tiles + r0 / kOwn) *
                                   p.parts + part) * 2 + second) * (kOwn * D) + row * D + c0;
      uint32_t w[C::kAccCols / 2];
#pragma unroll
      for (int cc = 0; cc < C::kAccCols; cc += 16) {
        uint32_t v[16];
        if (any) {
          tmem_ld16(tacc + cc, v);
          tmem_wait_ld();
          written_here(v);
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = 0u;
        }
        if (kKeys && sums) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            reinterpret_cast<uint4*>(sums + cc)[e] =
                make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
          w[cc / 2 + e] = pack_bf16x2(__uint_as_float(v[2 * e]) * out_scale,
                                      __uint_as_float(v[2 * e + 1]) * out_scale);
      }
      if (any) {
        tc_fence_before();
        __syncwarp();
        mbar_arrive_warp(acc_empty);
      }
      if (kKeys && sums) continue;
      // A thread holds kAccCols columns of its row; kShare threads exchange
      // 16-byte pieces so that together they store 64 bytes of a row at a time.
      constexpr int kShare = C::kAccCols >= 32 ? 4 : 2;
      const int rows = kKeys ? p.Skv : p.Sq;
#pragma unroll
      for (int cc = 0; cc < C::kAccCols / 2; cc += 4 * kShare) {
        uint32_t(&x)[4 * kShare] = *reinterpret_cast<uint32_t(*)[4 * kShare]>(&w[cc]);
        exchange<kShare>(x, lane);
        // Now piece e of x is piece lane % kShare of row e of the kShare rows.
#pragma unroll
        for (int e = 0; e < kShare; ++e) {
          const int r = r0 + quad * 32 + (lane & ~(kShare - 1)) + e;
          if (r < rows)
            *reinterpret_cast<uint4*>(out.row(b, h, r) + c0 + 2 * cc +
                                      8 * (lane & (kShare - 1))) =
                make_uint4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == C::kWarps) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  // The queries' grid ends after the keys', so that what follows it follows both.
  if (!kKeys && blockIdx.x + 1 == gridDim.x) pdl_wait();
}

// dK and dV of the divided tiles: the parts' sums, in part order.  Four columns
// to a thread.
template <int D>
__global__ void __launch_bounds__(256) part_sum_kernel(const __grid_constant__ TileParams p) {
  int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int c = static_cast<int>(i % (D / 4)) * 4;
  i /= D / 4;
  const int row = static_cast<int>(i % kOwn);
  i /= kOwn;
  const int which = static_cast<int>(i % 2);
  i /= 2;
  const int tile = static_cast<int>(i % p.part_tiles);
  const int64_t bh = i / p.part_tiles;
  const int key = tile * kOwn + row;
  if (bh >= static_cast<int64_t>(p.B) * p.Hkv || key >= p.Skv) return;
  const float* src = p.part_sums +
                     (((bh * p.part_tiles + tile) * p.parts) * 2 + which) * (kOwn * D) +
                     row * D + c;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int part = 0; part < p.parts; ++part) {
    const float4 x = *reinterpret_cast<const float4*>(src + static_cast<int64_t>(part) * 2 * kOwn * D);
    sum.x += x.x;
    sum.y += x.y;
    sum.z += x.z;
    sum.w += x.w;
  }
  const float scale = which ? 1.0f : p.scale;
  const View& out = which ? p.out2 : p.out1;
  *reinterpret_cast<uint2*>(out.row(bh / p.Hkv, bh % p.Hkv, key) + c) =
      make_uint2(pack_bf16x2(sum.x * scale, sum.y * scale), pack_bf16x2(sum.z * scale, sum.w * scale));
}

}  // namespace bwd
}  // namespace b200
