// Gradients of window attention.  With S = Q K^T scale, P = exp(S - lse) over
// the visible keys and delta_i = sum_d dO_id O_id:
//
//   dV = P^T dO      dP = dO V^T      dS = P (dP - delta)
//   dQ = dS K scale  dK = dS^T Q scale
//
// Three kernels without atomics, so that results do not depend on any order:
// delta; dK and dV (a CTA owns 64 keys and walks the query tiles that see
// them, over all query heads that share the keys); dQ (a CTA owns 64 queries
// and walks the key tiles that they see).  S and dP are computed twice, 14 D
// flops per visible pair instead of 10 D.
#pragma once

#include "mma_sync.cuh"
#include "ptx.cuh"
#include "view.cuh"

namespace b200 {
namespace bwd {

constexpr int kThreads = 128;
constexpr int kTile = 64;  // keys or queries of a tile; 16 of the owned ones per warp

template <int D>
struct Cfg {
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kTileBytes = kTile * kRowBytes;
  // The owned pair of tiles, and two stages of the walked pair with the
  // queries' lse and delta.
  static constexpr int kStageBytes = 2 * kTileBytes + 2 * kTile * 4;
  static constexpr int kSmemBytes = 2 * kTileBytes + 2 * kStageBytes;
};

struct Params {
  View dout, q, k, v, o, dq, dk, dv;
  const float* lse;    // [B, Hq, Sq]
  float* delta;        // [B, Hq, Sq]
  const int32_t* kv_len;
  int B, Hq, Hkv, group, Sq, Skv;
  int q_tiles, k_tiles;
  int window, sinks;  // at most Skv
  float scale, scale_log2;
};

__device__ __forceinline__ int batch_len(const Params& p, int b) {
  return p.kv_len ? max(0, min(p.kv_len[b], p.Skv)) : p.Skv;
}

// delta; one warp to a row.
template <int D>
__global__ void __launch_bounds__(256) delta_kernel(const __grid_constant__ Params p) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + warp_id();
  if (row >= static_cast<int64_t>(p.B) * p.Hq * p.Sq) return;
  const int64_t bh = row / p.Sq, s = row - bh * p.Sq, b = bh / p.Hq, h = bh - b * p.Hq;
  const uint16_t* x = p.dout.row(b, h, s);
  const uint16_t* y = p.o.row(b, h, s);
  float sum = 0.0f;
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
  if (lane_id() == 0) p.delta[row] = sum;
}

// Rows [r0, r0 + 64) of one head of a tensor; rows outside [0, se) and
// [lo, hi) are zeroed and not read.
template <int D>
__device__ __forceinline__ void load_tile(uint32_t dst, const View& t, int b, int h, int r0,
                                          int se, int lo, int hi) {
  constexpr int kChunks = D / 8;
  const uint16_t* base = t.row(b, h, 0);
#pragma unroll
  for (int u = 0; u < kTile * kChunks / kThreads; ++u) {
    const int idx = u * kThreads + static_cast<int>(threadIdx.x);
    const int r = idx / kChunks, c = idx % kChunks;
    const int row = r0 + r;
    const bool live = row < hi && (row >= lo || row < se);
    cp_async16(dst + swz<2 * D>(r, c), base + (live ? row : 0) * t.ss + c * 8, live);
  }
}

// acc[t] (16 x 8 each, t = 0..3) = A (16 rows at a_row0 of tile a) x B^T
// (32 rows at b_row0 of tile b), over D.
template <int D>
__device__ __forceinline__ void product_t(float (&acc)[4][4], uint32_t a, int a_row0, uint32_t b,
                                          int b_row0) {
  const int lane = static_cast<int>(lane_id());
  const int ar = a_row0 + (lane & 15), ac = lane >> 4;
  const int br = b_row0 + ((lane >> 4) << 3) + (lane & 7), bc = (lane >> 3) & 1;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[t][e] = 0.0f;
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    uint32_t fa[4], f0[4], f1[4];
    ldsm4(a + swz<2 * D>(ar, 2 * kk + ac), fa);
    ldsm4(b + swz<2 * D>(br, 2 * kk + bc), f0);
    ldsm4(b + swz<2 * D>(br + 16, 2 * kk + bc), f1);
    mma_bf16(acc[0], fa, f0[0], f0[1]);
    mma_bf16(acc[1], fa, f0[2], f0[3]);
    mma_bf16(acc[2], fa, f1[0], f1[1]);
    mma_bf16(acc[3], fa, f1[2], f1[3]);
  }
}

// out (16 x D) += X (16 x 32, as accumulators, rounded to bf16 for the tensor
// cores) x B (32 rows at b_row0 of tile b).
template <int D>
__device__ __forceinline__ void accumulate(float (&out)[D / 8][4], const float (&x)[4][4],
                                           uint32_t b, int b_row0) {
  const int lane = static_cast<int>(lane_id());
  const int br = b_row0 + (lane & 15), bc = lane >> 4;
#pragma unroll
  for (int kc = 0; kc < 2; ++kc) {
    const uint32_t a[4] = {
        pack_bf16x2(x[2 * kc][0], x[2 * kc][1]), pack_bf16x2(x[2 * kc][2], x[2 * kc][3]),
        pack_bf16x2(x[2 * kc + 1][0], x[2 * kc + 1][1]),
        pack_bf16x2(x[2 * kc + 1][2], x[2 * kc + 1][3])};
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      uint32_t f[4];
      ldsm4_trans(b + swz<2 * D>(br + 16 * kc, 2 * d + bc), f);
      mma_bf16(out[2 * d], a, f[0], f[1]);
      mma_bf16(out[2 * d + 1], a, f[2], f[3]);
    }
  }
}

template <int D>
__device__ __forceinline__ void store_rows(const View& t, int b, int h, int r0, int rows,
                                           const float (&x)[D / 8][4], float scale) {
  const int lane = static_cast<int>(lane_id());
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = r0 + (lane >> 2) + 8 * half;
    if (r >= rows) continue;
    uint16_t* dst = t.row(b, h, r) + 2 * (lane & 3);
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
      *reinterpret_cast<uint32_t*>(dst + 8 * d) =
          pack_bf16x2(x[d][2 * half] * scale, x[d][2 * half + 1] * scale);
  }
}

// dK, dV of 64 keys.
template <int D>
__global__ void __launch_bounds__(kThreads) dkdv_kernel(const __grid_constant__ Params p) {
  using C = Cfg<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t ks = smem_u32(smem), vs = ks + C::kTileBytes, ring = vs + C::kTileBytes;
  // The first key tiles (sinks) are seen by the most queries: they start first.
  const int kt = static_cast<int>(blockIdx.x / (p.B * p.Hkv));
  const int bh = static_cast<int>(blockIdx.x % (p.B * p.Hkv));
  const int b = bh / p.Hkv, h = bh - b * p.Hkv;
  const int n = batch_len(p, b), off = n - p.Sq;
  const int k0 = kt * kTile, k1 = min(k0 + kTile, n);
  // Queries [i0, i1) see some of keys [k0, k1).
  const int i0 = max(0, k0 - off);
  const int i1 = k1 <= k0 ? 0 : k0 < p.sinks ? p.Sq : min(p.Sq, k1 - 1 + p.window - off);
  const int t0 = i0 / kTile;
  const int nt = i1 > i0 ? (i1 + kTile - 1) / kTile - t0 : 0;
  const int steps = nt * p.group;
  const int warp = static_cast<int>(warp_id()), lane = static_cast<int>(lane_id());

  float dk[D / 8][4], dv[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) dk[i][e] = dv[i][e] = 0.0f;

  // Step i: query head h * group + i / nt, query tile t0 + i % nt.
  auto load_step = [&](int i) {
    if (i < steps) {
      const int hq = h * p.group + i / nt, r0 = (t0 + i % nt) * kTile;
      const uint32_t dst = ring + (i & 1) * C::kStageBytes;
      const int live0 = max(0, -off);  // earlier rows see nothing
      load_tile<D>(dst, p.q, b, hq, r0, 0, live0, p.Sq);
      load_tile<D>(dst + C::kTileBytes, p.dout, b, hq, r0, 0, live0, p.Sq);
      float* st = reinterpret_cast<float*>(smem + 2 * C::kTileBytes + (i & 1) * C::kStageBytes +
                                           2 * C::kTileBytes);
      if (threadIdx.x < kTile) {
        const int r = r0 + static_cast<int>(threadIdx.x);
        const int64_t at = (static_cast<int64_t>(b) * p.Hq + hq) * p.Sq + r;
        const float lse = r < p.Sq ? p.lse[at] : -INFINITY;
        st[threadIdx.x] = lse == -INFINITY ? 0.0f : lse * 1.4426950408889634f;
        st[kTile + threadIdx.x] = r < p.Sq ? p.delta[at] : 0.0f;
      }
    }
    cp_async_commit();
  };
  if (steps > 0) {
    load_tile<D>(ks, p.k, b, h, k0, 0, 0, n);
    load_tile<D>(vs, p.v, b, h, k0, 0, 0, n);
  }
  load_step(0);
  for (int i = 0; i < steps; ++i) {
    load_step(i + 1);
    cp_async_wait<1>();
    __syncthreads();
    const uint32_t qs = ring + (i & 1) * C::kStageBytes, os = qs + C::kTileBytes;
    const float* st = reinterpret_cast<const float*>(
        smem + 2 * C::kTileBytes + (i & 1) * C::kStageBytes + 2 * C::kTileBytes);
    const int r0 = (t0 + i % nt) * kTile;
#pragma unroll 1
    for (int c0 = 0; c0 < kTile; c0 += 32) {
      float s[4][4], dp[4][4];
      product_t<D>(s, ks, warp * 16, qs, c0);
      product_t<D>(dp, vs, warp * 16, os, c0);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int qi = c0 + 8 * t + 2 * (lane & 3) + (e & 1);
          const int j = k0 + warp * 16 + (lane >> 2) + 8 * (e >> 1);
          const int pos = off + r0 + qi;
          const bool seen = r0 + qi < p.Sq && j <= pos && (pos - j < p.window || j < p.sinks);
          s[t][e] = seen ? ex2_approx(fmaf(s[t][e], p.scale_log2, -st[qi])) : 0.0f;
          dp[t][e] = seen ? s[t][e] * (dp[t][e] - st[kTile + qi]) : 0.0f;
        }
      accumulate<D>(dv, s, os, c0);
      accumulate<D>(dk, dp, qs, c0);
    }
    __syncthreads();  // the stage is free
  }
  cp_async_wait<0>();
  store_rows<D>(p.dk, b, h, k0 + warp * 16, p.Skv, dk, p.scale);
  store_rows<D>(p.dv, b, h, k0 + warp * 16, p.Skv, dv, 1.0f);
}

// dQ of 64 queries.
template <int D>
__global__ void __launch_bounds__(kThreads) dq_kernel(const __grid_constant__ Params p) {
  using C = Cfg<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t qs = smem_u32(smem), os = qs + C::kTileBytes, ring = os + C::kTileBytes;
  const int qt = p.q_tiles - 1 - static_cast<int>(blockIdx.x / (p.B * p.Hq));
  const int bh = static_cast<int>(blockIdx.x % (p.B * p.Hq));
  const int b = bh / p.Hq, hq = bh - b * p.Hq, h = hq / p.group;
  const int n = batch_len(p, b), off = n - p.Sq;
  const int r0 = qt * kTile, r_last = min(r0 + kTile, p.Sq) - 1;
  // Keys [0, se) and [lo, hi) are seen by some of the tile's queries.
  const int hi = max(0, off + r_last + 1);
  int lo = max(0, off + r0 - p.window + 1);
  if (p.sinks >= lo || hi == 0) lo = 0;
  const int se = lo > 0 ? p.sinks : 0;
  const int ns = min((se + kTile - 1) / kTile, lo / kTile);  // sink tiles before the window's
  const int t0 = lo / kTile;
  const int steps = ns + (hi + kTile - 1) / kTile - t0;
  const int warp = static_cast<int>(warp_id()), lane = static_cast<int>(lane_id());

  float dq[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) dq[i][e] = 0.0f;
  auto tile_of = [&](int i) { return i < ns ? i : t0 + i - ns; };
  auto load_step = [&](int i) {
    if (i < steps) {
      const int k0 = tile_of(i) * kTile;
      const uint32_t dst = ring + (i & 1) * C::kStageBytes;
      load_tile<D>(dst, p.k, b, h, k0, se, lo, hi);
      load_tile<D>(dst + C::kTileBytes, p.v, b, h, k0, se, lo, hi);
    }
    cp_async_commit();
  };
  if (steps > 0) {
    load_tile<D>(qs, p.q, b, hq, r0, 0, max(0, -off), p.Sq);
    load_tile<D>(os, p.dout, b, hq, r0, 0, max(0, -off), p.Sq);
  }
  load_step(0);
  float lse[2], delta[2];
  int pos[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = min(r0 + warp * 16 + (lane >> 2) + 8 * half, p.Sq - 1);
    const int64_t at = (static_cast<int64_t>(b) * p.Hq + hq) * p.Sq + r;
    const float x = p.lse[at];
    lse[half] = x == -INFINITY ? 0.0f : x * 1.4426950408889634f;
    delta[half] = p.delta[at];
    pos[half] = off + r;
  }
  for (int i = 0; i < steps; ++i) {
    load_step(i + 1);
    cp_async_wait<1>();
    __syncthreads();
    const uint32_t ks = ring + (i & 1) * C::kStageBytes, vs = ks + C::kTileBytes;
    const int k0 = tile_of(i) * kTile;
#pragma unroll 1
    for (int c0 = 0; c0 < kTile; c0 += 32) {
      float s[4][4], dp[4][4];
      product_t<D>(s, qs, warp * 16, ks, c0);
      product_t<D>(dp, os, warp * 16, vs, c0);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int half = e >> 1;
          const int j = k0 + c0 + 8 * t + 2 * (lane & 3) + (e & 1);
          const bool seen =
              j <= pos[half] && (pos[half] - j < p.window || j < p.sinks);
          const float w =
              seen ? ex2_approx(fmaf(s[t][e], p.scale_log2, -lse[half])) : 0.0f;
          dp[t][e] = seen ? w * (dp[t][e] - delta[half]) : 0.0f;
        }
      accumulate<D>(dq, dp, ks, c0);
    }
    __syncthreads();
  }
  cp_async_wait<0>();
  store_rows<D>(p.dq, b, hq, r0 + warp * 16, p.Sq, dq, p.scale);
}

}  // namespace bwd
}  // namespace b200
