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
// fixed order: no atomics, equal bits from call to call.
//
// TMEM: S, dP, then P and dS, then the accumulators.  S and dP have one buffer
// each: the registers of the elementwise warps are the second, so the next
// step's S and dP run while this step's P is computed.  kKeys steps are 64
// queries wide: two accumulators of D columns leave no room for 128.
//
// Roles: warps 0-7 elementwise (warp w: lanes 32 (w % 4), columns half w / 4)
// and epilogue; warp 8 TMA; warp 9 issues S and dP; warp 10 the accumulating
// products.  Waits are bounded as in the forward kernel.
#pragma once

#include "attention_kernel.cuh"
#include "ptx.cuh"
#include "view.cuh"

namespace b200 {
namespace bwd {

constexpr int kTileThreads = 384;
constexpr int kOwn = 128;  // owned rows

template <int D, bool kKeys>
struct TileCfg {
  static constexpr int kN = kKeys ? 64 : 128;  // streamed rows of a step
  static constexpr int kStages = (kKeys ? 4 : 2) * (128 / D);
  static constexpr int kBoxes = D / 64;
  static constexpr int kOwnBox = kOwn * 128;
  static constexpr int kOwnBytes = kBoxes * kOwnBox;
  static constexpr int kStrBox = kN * 128;
  static constexpr int kStrBytes = kBoxes * kStrBox;
  static constexpr int kStatBytes = kKeys ? 2 * kN * 4 : 0;  // -lse, -delta of the queries
  static constexpr int kRingOff = 2 * kOwnBytes;
  static constexpr int kStatOff = kRingOff + kStages * 2 * kStrBytes;
  static constexpr int kBarOff = kStatOff + kStages * kStatBytes;
  // own_full own_empty s_ready dp_ready s_free p_ready p_free acc_full acc_empty drain
  static constexpr int kNumBars = 10 + 2 * kStages;
  static constexpr int kSlotOff = kBarOff + kNumBars * 8;
  static constexpr int kSmemBytes = kSlotOff + 16 + 1024;  // + alignment slack
  static_assert(kSmemBytes <= 232448, "exceeds the 227 KiB of shared memory a CTA may use");
  static_assert(kSmemBytes > 116 * 1024, "one CTA per SM: each takes all of TMEM");
  static constexpr uint32_t kColS = 0, kColDp = kN, kColP = 2 * kN;
  static constexpr uint32_t kColDs = kColP + (kKeys ? kN / 2 : 0);
  static constexpr uint32_t kColAcc1 = 512 - 2 * D, kColAcc2 = 512 - D;
  static_assert(kColDs + kN / 2 <= (kKeys ? kColAcc1 : kColAcc2), "TMEM columns");
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
  int window, sinks;
  float scale, scale_log2;
  // Coordinate factors of broadcast axes (own1, own2, str1, str2; batch, head).
  int o1_b, o1_h, o2_b, o2_h, s1_b, s1_h, s2_b, s2_h;
};

enum : uint32_t {
  kSiteBwdOwn = 0x20, kSiteBwdFull, kSiteBwdEmpty, kSiteBwdS, kSiteBwdDp, kSiteBwdSFree,
  kSiteBwdP, kSiteBwdPFree, kSiteBwdAcc
};

// -lse and -delta of every query row, padded with zeros; one warp to a row.
template <int D>
__global__ void __launch_bounds__(256)
    stats_kernel(const View dout, const View o, const float* lse, float* stats, int64_t plane,
                 int sq_pad, int B, int Hq, int Sq) {
  pdl_launch_dependents();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + warp_id();
  if (row >= plane) return;
  const int64_t bh = row / sq_pad, s = row - bh * sq_pad, b = bh / Hq, h = bh - b * Hq;
  float sum = 0.0f, l = 0.0f;
  if (s < Sq) {
    const uint16_t* x = dout.row(b, h, s);
    const uint16_t* y = o.row(b, h, s);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int c = i * 32 + static_cast<int>(lane_id());
      const uint32_t a = reinterpret_cast<const uint32_t*>(x)[c];
      const uint32_t e = reinterpret_cast<const uint32_t*>(y)[c];
      sum = fmaf(__uint_as_float(a << 16), __uint_as_float(e << 16), sum);
      sum = fmaf(__uint_as_float(a & 0xffff0000u), __uint_as_float(e & 0xffff0000u), sum);
    }
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    l = lse[bh * Sq + s];
  }
  if (lane_id() == 0) {
    stats[row] = l == -INFINITY ? 0.0f : l * -1.4426950408889634f;
    stats[plane + row] = -sum;
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

// One owned tile: where it lies and what it streams.
template <bool kKeys>
struct TileItem {
  int b, h;         // h: kv head (kKeys) or query head
  int r0;           // first owned row
  int n, off;       // keys of the request; position of query row 0
  int steps;
  int per_head, t0;             // kKeys: steps of a query head, first 64-query tile
  int se, lo, hi, n_sink, skip;  // queries: as in the forward kernel
};

template <bool kKeys>
__device__ __forceinline__ TileItem<kKeys> tile_item(const TileParams& p, int k) {
  TileItem<kKeys> it;
  const int heads = kKeys ? p.Hkv : p.Hq;
  // All (batch, head) of one tile index are adjacent: for keys the first tiles
  // (sinks, seen by most queries) start first, for queries the last ones.
  int tile = k / (p.B * heads);
  const int bh = k - tile * (p.B * heads);
  if (!kKeys) tile = p.tiles - 1 - tile;
  it.b = bh / heads;
  it.h = bh - it.b * heads;
  it.r0 = tile * kOwn;
  it.n = p.kv_len ? max(0, min(__ldg(p.kv_len + it.b), p.Skv)) : p.Skv;
  it.off = it.n - p.Sq;
  if constexpr (kKeys) {
    const int k1 = min(it.r0 + kOwn, it.n);  // queries [i0, i1) see some of keys [r0, k1)
    const int i0 = max(0, it.r0 - it.off);
    const int i1 = k1 <= it.r0 ? 0
                   : it.r0 < p.sinks ? p.Sq
                                     : min(p.Sq, k1 - 1 + p.window - it.off);
    it.t0 = i0 / 64;
    it.per_head = i1 > i0 ? (i1 + 63) / 64 - it.t0 : 0;
    it.steps = it.per_head * p.group;
  } else {
    const int last = it.off + min(it.r0 + kOwn, p.Sq) - 1;
    it.hi = max(0, last + 1);
    it.lo = max(0, it.off + it.r0 - p.window + 1);
    if (p.sinks >= it.lo || it.hi == 0) it.lo = 0;
    it.se = it.lo > 0 ? p.sinks : 0;
    const int w0 = it.lo / 128;
    it.n_sink = min((it.se + 127) / 128, w0);
    it.skip = w0 - it.n_sink;
    it.steps = it.n_sink + (it.hi + 127) / 128 - w0;
  }
  return it;
}

template <int D, bool kKeys>
__global__ void __launch_bounds__(kTileThreads, 1)
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
  uint8_t* ring = smem + C::kRingOff;
  float* stat = reinterpret_cast<float*>(smem + C::kStatOff);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t *own_full = bars, *own_empty = bars + 1, *s_ready = bars + 2, *dp_ready = bars + 3,
           *s_free = bars + 4, *p_ready = bars + 5, *p_free = bars + 6, *acc_full = bars + 7,
           *acc_empty = bars + 8, *drain = bars + 9, *full = bars + 10,
           *empty = bars + 10 + C::kStages;
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + C::kSlotOff);
  const int warp = static_cast<int>(warp_id()), lane = static_cast<int>(lane_id());

  if (threadIdx.x == 0) {
    mbar_init(own_full, 1);
    mbar_init(own_empty, 1);
    mbar_init(s_ready, 1);
    mbar_init(dp_ready, 1);
    mbar_init(s_free, 8);
    mbar_init(p_ready, 8);
    mbar_init(p_free, 1);
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 8);
    mbar_init(drain, 2);
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    fence_mbar_init();
  }
  if (warp == 8) {
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
  pdl_wait();  // the row statistics

  // Streamed row 0 and the query head of step i.
  auto str_row = [&](const TileItem<kKeys>& it, int i) {
    if constexpr (kKeys)
      return (it.t0 + i % it.per_head) * 64;
    else
      return (i < it.n_sink ? i : i + it.skip) * 128;
  };
  auto query_head = [&](const TileItem<kKeys>& it, int i) {
    if constexpr (kKeys)
      return it.h * p.group + i / it.per_head;
    else
      return it.h;
  };

  if (warp == 8) {
    // ================= TMA producer =================
    if (lane == 0) {
      const uint64_t pol_own = l2_policy_evict_first(), pol_str = l2_policy_evict_last();
      int t = 0, li = 0;
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
        for (int i = 0; i < it.steps; ++i, ++t) {
          const int st = t % C::kStages;
          ok = mbar_wait(&empty[st], (static_cast<uint32_t>(t / C::kStages) & 1u) ^ 1u,
                         kSiteBwdEmpty, kDefaultWaitLimitNs, 20000u);
          if (!ok) break;
          const int row = str_row(it, i), hq = query_head(it, i);
          const int h = kKeys ? hq : it.h / p.group;
          mbar_arrive_expect_tx(&full[st], 2 * C::kStrBytes + C::kStatBytes);
          uint8_t* dst = ring + st * 2 * C::kStrBytes;
          for (int x = 0; x < C::kBoxes; ++x) {
            tma_load_4d(dst + x * C::kStrBox, &str1_map, &full[st], x * 64, row, h * p.s1_h,
                        it.b * p.s1_b, pol_str);
            tma_load_4d(dst + C::kStrBytes + x * C::kStrBox, &str2_map, &full[st], x * 64, row,
                        h * p.s2_h, it.b * p.s2_b, pol_str);
          }
          if constexpr (kKeys) {
            const float* src =
                p.stats + (static_cast<int64_t>(it.b) * p.Hq + hq) * p.sq_pad + row;
            float* sdst = stat + st * 2 * C::kN;
            bulk_load(sdst, src, C::kN * 4, &full[st]);
            bulk_load(sdst + C::kN, src + p.stat_plane, C::kN * 4, &full[st]);
          }
        }
      }
      if (!ok) {
        // Unwinding: let every copy already issued land before the CTA exits.
        if (li > 0) attn::drain_wait(own_full, static_cast<uint32_t>(li - 1) & 1u);
        for (int i = max(0, t - C::kStages); i < t; ++i)
          attn::drain_wait(&full[i % C::kStages], static_cast<uint32_t>(i / C::kStages) & 1u);
      }
    }
    __syncwarp();
  } else if (warp == 9 || warp == 10) {
    // ================= MMA issuers =================
    const bool acc = warp == 10;
    const uint32_t ring_addr = smem_u32(ring), own_addr = smem_u32(own);
    const uint64_t d_own1 = sdesc_sw128(own_addr, 16, 1024);
    const uint64_t d_own2 = sdesc_sw128(own_addr + C::kOwnBytes, 16, 1024);
    const uint64_t d_str = sdesc_sw128(ring_addr, 16, 1024);           // rows as N
    const uint64_t d_acc = sdesc_sw128(ring_addr, C::kStrBox, 1024);   // rows as K
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
        const int st = t % C::kStages;
        const uint32_t stage16 = static_cast<uint32_t>(st * 2 * C::kStrBytes) >> 4;
        if (!acc) {
          ok = warp_wait(&full[st], static_cast<uint32_t>(t / C::kStages) & 1u, kSiteBwdFull) &&
               warp_wait(s_free, (static_cast<uint32_t>(t) & 1u) ^ 1u, kSiteBwdSFree);
          if (!ok) break;
#pragma unroll
          for (int which = 0; which < 2; ++which) {
            const uint64_t da = which ? d_own2 : d_own1;
            const uint64_t db = d_str + stage16 + (which ? C::kStrBytes >> 4 : 0);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              mma_ss_warp(tmem + (which ? C::kColDp : C::kColS),
                          da + (kk >> 2) * (C::kOwnBox >> 4) + (kk & 3) * 2,
                          db + (kk >> 2) * (C::kStrBox >> 4) + (kk & 3) * 2, C::kIdescS,
                          kk > 0 ? 1u : 0u);
            mma_commit_warp(which ? dp_ready : s_ready);
          }
          if (i + 1 == steps) mma_commit_warp(own_empty);
        } else {
          ok = warp_wait(p_ready, static_cast<uint32_t>(t) & 1u, kSiteBwdP);
          if (!ok) break;
          const uint64_t db = d_acc + stage16;
          if constexpr (kKeys) {
#pragma unroll
            for (int kk = 0; kk < C::kN / 16; ++kk)
              mma_ts_warp(tmem + C::kColAcc2, tmem + C::kColP + kk * 8,
                          db + (C::kStrBytes >> 4) + kk * (2048 >> 4), C::kIdescAcc,
                          (i > 0 || kk > 0) ? 1u : 0u);
          }
#pragma unroll
          for (int kk = 0; kk < C::kN / 16; ++kk)
            mma_ts_warp(tmem + (kKeys ? C::kColAcc1 : C::kColAcc2), tmem + C::kColDs + kk * 8,
                        db + kk * (2048 >> 4), C::kIdescAcc, (i > 0 || kk > 0) ? 1u : 0u);
          mma_commit_warp(&empty[st]);
          mma_commit_warp(p_free);
          if (i + 1 == steps) mma_commit_warp(acc_full);
        }
      }
    }
    mma_commit_warp(drain);
    attn::drain_wait(drain, 0);
    __syncwarp();
  } else if (warp < 8) {
    // ================= elementwise and epilogue =================
    const int quad = warp & 3, half = warp >> 2;
    const int row = quad * 32 + lane;
    const uint32_t tlane = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const float c = p.scale_log2;
    const uint64_t c2 = f2_pack(c, c);
    int t = 0, li = 0;
    bool ok = true;
    for (int k = static_cast<int>(blockIdx.x); k < p.n_items && ok; k += gridDim.x) {
      const TileItem<kKeys> it = tile_item<kKeys>(p, k);
      const int my = it.r0 + row;  // this thread's key or query
      float nlse = 0.0f, ndelta = 0.0f;
      if (!kKeys && my < p.Sq) {
        const float* src = p.stats + (static_cast<int64_t>(it.b) * p.Hq + it.h) * p.sq_pad + my;
        nlse = __ldg(src);
        ndelta = __ldg(src + p.stat_plane);
      }
      for (int i = 0; i < it.steps; ++i, ++t) {
        const int st = t % C::kStages;
        const int str0 = str_row(it, i);
        // The streamed columns [va, vb) that this row meets; for queries also
        // those below vs (sinks).  `masked`: some pair of the step is hidden.
        int va, vb, vs = 0;
        bool masked;
        if constexpr (kKeys) {
          va = my - it.off - str0;
          vb = min(p.Sq - str0, my < p.sinks ? 64 : my + p.window - it.off - str0);
          const int first = it.off + str0, last = first + 63;  // positions of the step
          masked = str0 + 64 > p.Sq || first < it.r0 + kOwn - 1 ||
                   (last - it.r0 >= p.window && it.r0 + kOwn > p.sinks);
        } else {
          const int pos = it.off + my;
          va = pos - p.window + 1 - str0;
          vb = (my < p.Sq ? pos : -1) + 1 - str0;
          vs = min(p.sinks, pos + 1) - str0;
          if (my >= p.Sq) vs = va = vb = -1;
          const int first = it.off + it.r0, last = first + kOwn - 1;
          masked = it.r0 + kOwn > p.Sq || str0 + 127 > first ||
                   (last - str0 >= p.window && str0 + 128 > p.sinks);
        }
        ok = attn::warp_wait(s_ready, static_cast<uint32_t>(t) & 1u, kSiteBwdS);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int ch = 0; ch < C::kN / 64; ++ch) {
          const int col0 = half * (C::kN / 2) + ch * 32;
          uint32_t s[32], d[32];
          tmem_ld32(tlane + C::kColS + col0, s);
          if (ch == 0) {
            ok = attn::warp_wait(dp_ready, static_cast<uint32_t>(t) & 1u, kSiteBwdDp);
            if (!ok) {
              tmem_wait_ld(s);
              break;
            }
            tc_fence_after();
          }
          tmem_ld32(tlane + C::kColDp + col0, d);
          tmem_wait_ld(s);
          tmem_wait_ld(d);
          if (ch + 1 == C::kN / 64) {  // the next step's S and dP may overwrite these
            tc_fence_before();
            __syncwarp();
            mbar_arrive_warp(s_free);
          }
          const float* st_l = stat + st * 2 * C::kN + col0;
          uint32_t pk[16], dk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            uint64_t nl2, nd2;
            if constexpr (kKeys) {
              nl2 = *reinterpret_cast<const uint64_t*>(st_l + 2 * e);
              nd2 = *reinterpret_cast<const uint64_t*>(st_l + C::kN + 2 * e);
            } else {
              nl2 = f2_pack(nlse, nlse);
              nd2 = f2_pack(ndelta, ndelta);
            }
            const uint64_t x2 = f2_fma(
                f2_pack(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), c2, nl2);
            float x0, x1;
            f2_unpack(x2, x0, x1);
            float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
            uint64_t g2 = f2_mul(
                f2_pack(p0, p1),
                f2_add(f2_pack(__uint_as_float(d[2 * e]), __uint_as_float(d[2 * e + 1])), nd2));
            float g0, g1;
            f2_unpack(g2, g0, g1);
            if (masked) {
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
          if (ch == 0) {
            // The products of the step before have read P and dS.
            ok = attn::warp_wait(p_free, (static_cast<uint32_t>(t) & 1u) ^ 1u, kSiteBwdPFree);
            if (!ok) break;
            tc_fence_after();
          }
          if constexpr (kKeys) tmem_st16(tlane + C::kColP + (col0 >> 1), pk);
          tmem_st16(tlane + C::kColDs + (col0 >> 1), dk);
        }
        if (!ok) break;
        // Streamed rows that nothing sees may hold anything: zero them before
        // the accumulating products read them (0 * NaN is NaN).
        {
          int se, lo, hi;  // live rows: [0, se) and [lo, hi)
          if constexpr (kKeys) {
            se = 0;
            lo = max(0, -it.off);
            hi = 0x7fffffff;
          } else {
            se = it.se;
            lo = it.lo;
            hi = it.hi;
          }
          if (str0 + C::kN > hi || (str0 < lo && str0 + C::kN > se)) {
            ok = attn::warp_wait(&full[st], static_cast<uint32_t>(t / C::kStages) & 1u,
                                 kSiteBwdFull);
            if (!ok) break;
            for (int r = warp * 32 + lane; r < 2 * C::kBoxes * C::kN; r += 256) {
              const int sr = str0 + r % C::kN;
              if (sr >= hi || (sr < lo && sr >= se)) {
                const uint32_t at = smem_u32(ring + st * 2 * C::kStrBytes) +
                                    static_cast<uint32_t>(r) * 128u;
#pragma unroll
                for (int e = 0; e < 8; ++e) st_shared_v4(at + e * 16, 0u, 0u, 0u, 0u);
              }
            }
            fence_proxy_async_smem();
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        mbar_arrive_warp(p_ready);
      }
      if (!ok) break;
      // Epilogue: kKeys, half 0 writes dK and half 1 dV; queries, each half
      // writes its half of dQ's columns.
      const View& out = kKeys && half ? p.out2 : p.out1;
      const float scale = kKeys && half ? 1.0f : p.scale;
      constexpr int kCols = kKeys ? D : D / 2;
      const int c0 = kKeys ? 0 : half * kCols;
      const bool live = my < (kKeys ? p.Skv : p.Sq);
      uint16_t* dst = out.row(it.b, it.h, live ? my : 0) + c0;
      if (it.steps > 0) {
        ok = attn::warp_wait(acc_full, static_cast<uint32_t>(li) & 1u, kSiteBwdAcc);
        if (!ok) break;
        ++li;
        tc_fence_after();
      }
      const uint32_t tacc = tlane + (kKeys && !half ? C::kColAcc1 : C::kColAcc2) + c0;
#pragma unroll 1
      for (int cc = 0; cc < kCols; cc += 32) {
        uint32_t v[32];
        if (it.steps > 0) {
          tmem_ld32(tacc + cc, v);
          tmem_wait_ld(v);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0u;
        }
        if (live) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t w[4];
#pragma unroll
            for (int f = 0; f < 4; ++f)
              w[f] = pack_bf16x2(__uint_as_float(v[8 * e + 2 * f]) * scale,
                                 __uint_as_float(v[8 * e + 2 * f + 1]) * scale);
            *reinterpret_cast<uint4*>(dst + cc + 8 * e) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (it.steps > 0) {
        tc_fence_before();
        __syncwarp();
        mbar_arrive_warp(acc_empty);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace bwd
}  // namespace b200
