// Attention of a few query rows over a long key range, split over the keys.
//
//   O_i = softmax_j(q_i k_j scale) v_j over the keys that row i sees: with
//   p_i its position, j <= p_i and (p_i - j < window or j < sinks)
//
// after the P keys of a prefix that all requests share (P may be 0), which
// every row sees.
//
// The rows of one (batch, kv head) -- its `group` query heads x Sq tokens --
// are packed into tiles of 16, so that a K/V row is read once for all heads
// that share it.  A unit (batch, kv head, row tile, split) takes a share of
// the 16-key blocks of the prefix, of [0, sinks) and of the window; each of
// its four warps walks its own blocks with its own ring of cp.async stages,
// running maximum, sum and O in registers, and nothing synchronises the warps
// until they merge at the end.  The splits of a row tile are a thread-block
// cluster and merge through distributed shared memory; where more than
// kMaxCluster are needed to fill the GPU, their unnormalised O (fp32) and
// (m, l) go through global memory to combine_kernel instead.
//
// Bound by memory: 4 D flops per row and key against 4 D bytes per key, so
// 16 rows need 16 flops per byte, about 100 TFLOP/s at the card's bandwidth.
// mma.sync (m16n8k16) carries that with a tile that fits the rows; a tcgen05
// tile is at least 64 rows high.  64 tokens, 64/8 heads, windows of 4096:
// 157 us, 6.8 TB/s, in a graph at full clock; called back to back 171 us, 6.3.
#pragma once

#include "mma_sync.cuh"
#include "ptx.cuh"
#include "view.cuh"

namespace b200 {
namespace split {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 16;    // query rows of a tile
constexpr int kKeys = 16;    // keys of a block
constexpr int kMaxCluster = 8;
constexpr int kMaxSplits = 32;  // the combining warp holds one split's (m, l) per lane

template <int D>
struct Cfg {
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kTileBytes = kKeys * kRowBytes;  // K or V of a block
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kRingBytes = kWarps * kStages * kStageBytes;
  static constexpr int kOStride = D + 4;  // floats; merge buffer rows
  static constexpr int kMergeBytes = kWarps * kRows * (kOStride * 4 + 8);
  static constexpr int kSmemBytes = kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes;
};

struct Params {
  View q, k, v, o;
  View kp, vp;            // the prefix, [1, Hkv, P, D]
  int P;
  const int32_t* kv_len;  // [B], or null: Skv
  int B, Hkv, group, Sq, Skv;
  int rows;       // group * Sq
  int row_tiles;  // ceil(rows / 16)
  int nsplit;
  int window, sinks;  // at most Skv
  // Many short units: each warp takes one whole (nsplit is 1), `units` in all.
  // 0: a CTA takes a unit.
  int units;
  float scale_log2;
  float* part_o;    // [B * Hkv][nsplit][rows][D], or null: the nsplit CTAs are a cluster
  float2* part_ml;  // [B * Hkv][nsplit][rows] (m in log2 units, l)
  float* lse;       // [B, Hq, Sq] natural log of each row's sum, or null
  // The launch overlaps the kernel before it (the prefix's tiles): the last CTA
  // ends after that one, so that whatever follows this grid follows both.
  int overlaps;
};

// The natural log of the row sum l 2^m; a row without keys has none (-inf).
__device__ __forceinline__ float row_lse(float m, float l) {
  return l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

// The weight of a partial sum with maximum m among partials whose maximum is
// mx: a partial without keys (m = -inf, l = 0) weighs nothing.
__device__ __forceinline__ float part_weight(float2 ml, float mx) {
  if (ml.x == -INFINITY && ml.y == 0.0f) return 0.0f;
  return ex2_approx(ml.x - (mx == -INFINITY ? 0.0f : mx));
}

template <int D>
__global__ void __launch_bounds__(kThreads, 2)
    split_attention_kernel(const __grid_constant__ Params p) {
  using C = Cfg<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  if (!p.overlaps) pdl_wait();
  pdl_launch_dependents();
  const int lane = static_cast<int>(lane_id());
  const int warp = static_cast<int>(warp_id());
  const int stride = p.units ? 1 : kWarps;      // of a warp's blocks
  const int first = p.units ? 0 : warp;
  int unit = static_cast<int>(blockIdx.x);
  if (p.units) {
    unit = unit * kWarps + warp;
    if (unit >= p.units) return;
  }
  const int split = unit % p.nsplit;
  unit /= p.nsplit;
  const int rt = unit % p.row_tiles;
  const int bh = unit / p.row_tiles;
  const int b = bh / p.Hkv, h = bh - b * p.Hkv;

  const int len = p.kv_len ? ld_global_l2(p.kv_len + b) : p.Skv;
  // The tile's Q rows, through the ring's last stage, which no block takes
  // before the loop.
  const uint32_t ring = smem_u32(smem) + warp * C::kStages * C::kStageBytes;
  const uint32_t q_at = ring + (C::kStages - 1) * C::kStageBytes;
  {
    // Two lanes to a row; those past the last are zeroed, not read.
    const int i = lane >> 1;
    const bool live = rt * kRows + i < p.rows;
    const int r = live ? rt * kRows + i : 0;
    const uint16_t* src = p.q.row(b, h * p.group + r % p.group, r / p.group);
#pragma unroll
    for (int c = lane & 1; c < D / 8; c += 2)
      cp_async16(q_at + swz<C::kRowBytes>(i, c), src + c * 8, live);
  }
  cp_async_commit();

  // The tile's rows and the keys that some of them see.
  const int n = max(0, min(len, p.Skv));
  const int r_last = min(rt * kRows + kRows - 1, p.rows - 1);
  auto position = [&](int r) { return n - p.Sq + r / p.group; };
  const int p_first = position(rt * kRows), p_last = position(r_last);
  const int hi = max(p_last + 1, 0);
  int lo = max(p_first - p.window + 1, 0);
  if (p.sinks >= lo || hi == 0) lo = 0;   // one range
  const int se = lo > 0 ? p.sinks : 0;    // the sinks before the window's range
  const int nb_p = (p.P + kKeys - 1) / kKeys;
  const int nb_s = (se + kKeys - 1) / kKeys;
  const int nb = nb_p + nb_s + (hi - lo + kKeys - 1) / kKeys;
  const int b0 = static_cast<int>(static_cast<int64_t>(nb) * split / p.nsplit);
  const int b1 = static_cast<int>(static_cast<int64_t>(nb) * (split + 1) / p.nsplit);

  // Keys [j0, j1) of block i, of the prefix or of the request.
  auto block_keys = [&](int i, int* j0, int* j1) {
    if (i < nb_p) {
      *j0 = i * kKeys;
      *j1 = min(*j0 + kKeys, p.P);
    } else if (i < nb_p + nb_s) {
      *j0 = (i - nb_p) * kKeys;
      *j1 = min(*j0 + kKeys, se);
    } else {
      *j0 = lo + (i - nb_p - nb_s) * kKeys;
      *j1 = min(*j0 + kKeys, hi);
    }
  };
  // Block i's K and V rows; rows past the range are zeroed, not read (a V row
  // that holds NaN would reach O through 0 * NaN).
  auto load_block = [&](int i, int stage) {
    if (i < b1) {
      int j0, j1;
      block_keys(i, &j0, &j1);
      constexpr int kChunks = D / 8;  // per row
      const bool shared = i < nb_p;
      const int64_t k_ss = shared ? p.kp.ss : p.k.ss, v_ss = shared ? p.vp.ss : p.v.ss;
      const uint16_t* kbase = shared ? p.kp.row(0, h, j0) : p.k.row(b, h, j0);
      const uint16_t* vbase = shared ? p.vp.row(0, h, j0) : p.v.row(b, h, j0);
      const uint32_t dst = ring + stage * C::kStageBytes;
#pragma unroll
      for (int u = 0; u < kKeys * kChunks / 32; ++u) {
        const int idx = u * 32 + lane;
        const int r = idx / kChunks, c = idx % kChunks;
        const bool live = j0 + r < j1;
        const int64_t j = live ? r : 0;
        const uint32_t at = dst + swz<C::kRowBytes>(r, c);
        cp_async16(at, kbase + j * k_ss + c * 8, live);
        cp_async16(at + C::kTileBytes, vbase + j * v_ss + c * 8, live);
      }
    }
    cp_async_commit();
  };
  int next = b0 + first;
#pragma unroll
  for (int s = 0; s < C::kStages - 1; ++s, next += stride) load_block(next, s);

  // Q as the A operand: lane holds rows lane/4 and lane/4 + 8, columns
  // 2 (lane % 4) + {0, 1, 8, 9} of every 16.
  cp_async_wait<C::kStages - 1>();
  __syncwarp();
  uint32_t qa[D / 16][4];
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    ldsm4(q_at + swz<C::kRowBytes>(lane & 15, 2 * kk + (lane >> 4)), qa[kk]);
  const int ra = rt * kRows + (lane >> 2), rb = ra + 8;
  const int ca = 2 * (lane & 3);
  const int pos_a = position(min(ra, p.rows - 1)), pos_b = position(min(rb, p.rows - 1));

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
  float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.0f, l_b = 0.0f;
  // ldmatrix row and chunk of this lane: K (keys 8 (lane/16) + lane % 8,
  // chunk parity (lane/8) & 1) and V (keys 8 ((lane/8) & 1) + lane % 8).
  const int krow = ((lane >> 4) << 3) + (lane & 7), kpar = (lane >> 3) & 1;
  const int vrow = (((lane >> 3) & 1) << 3) + (lane & 7), vpar = lane >> 4;

  int stage = 0;
  for (int i = b0 + first; i < b1; i += stride) {
    cp_async_wait<C::kStages - 2>();
    __syncwarp();
    // The stage consumed in the previous step takes the next block.
    load_block(next, stage == 0 ? C::kStages - 1 : stage - 1);
    next += stride;
    const uint32_t kt = ring + stage * C::kStageBytes;
    const uint32_t vt = kt + C::kTileBytes;
    stage = stage + 1 == C::kStages ? 0 : stage + 1;

    float s[2][4];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e >> 2][e & 3] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t kb[4];
      ldsm4(kt + swz<C::kRowBytes>(krow, 2 * kk + kpar), kb);
      mma_bf16(s[0], qa[kk], kb[0], kb[1]);
      mma_bf16(s[1], qa[kk], kb[2], kb[3]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e >> 2][e & 3] *= p.scale_log2;
    int j0, j1;
    block_keys(i, &j0, &j1);
    // A block that every row sees whole needs no mask.
    const bool shared = i < nb_p;
    if (!(j1 == j0 + kKeys &&
          (shared || (j1 - 1 <= p_first && (p_last - j0 < p.window || j1 <= p.sinks))))) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j0 + 8 * t + ca + (e & 1);
          const int pos = e < 2 ? pos_a : pos_b;
          if (!(j < j1 && (shared || (j <= pos && (pos - j < p.window || j < p.sinks)))))
            s[t][e] = -INFINITY;
        }
    }
    float x_a = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
    float x_b = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
    x_a = fmaxf(x_a, __shfl_xor_sync(0xffffffffu, x_a, 1));
    x_b = fmaxf(x_b, __shfl_xor_sync(0xffffffffu, x_b, 1));
    x_a = fmaxf(x_a, __shfl_xor_sync(0xffffffffu, x_a, 2));
    x_b = fmaxf(x_b, __shfl_xor_sync(0xffffffffu, x_b, 2));
    x_a = fmaxf(m_a, x_a);
    x_b = fmaxf(m_b, x_b);
    if (__any_sync(0xffffffffu, x_a > m_a || x_b > m_b)) {
      const float f_a = x_a > m_a ? ex2_approx(m_a - x_a) : 1.0f;
      const float f_b = x_b > m_b ? ex2_approx(m_b - x_b) : 1.0f;
      m_a = x_a;
      m_b = x_b;
      l_a *= f_a;
      l_b *= f_b;
#pragma unroll
      for (int d = 0; d < D / 8; ++d) {
        o[d][0] *= f_a;
        o[d][1] *= f_a;
        o[d][2] *= f_b;
        o[d][3] *= f_b;
      }
    }
    const float u_a = m_a == -INFINITY ? 0.0f : m_a, u_b = m_b == -INFINITY ? 0.0f : m_b;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t][0] = ex2_approx(s[t][0] - u_a);
      s[t][1] = ex2_approx(s[t][1] - u_a);
      s[t][2] = ex2_approx(s[t][2] - u_b);
      s[t][3] = ex2_approx(s[t][3] - u_b);
      l_a += s[t][0] + s[t][1];
      l_b += s[t][2] + s[t][3];
    }
    // P goes to the tensor cores in bf16, as in the other attention kernels
    // (relative 2^-9 per weight, averaged over the keys); l keeps fp32.
    const uint32_t pa[4] = {pack_bf16x2(s[0][0], s[0][1]), pack_bf16x2(s[0][2], s[0][3]),
                            pack_bf16x2(s[1][0], s[1][1]), pack_bf16x2(s[1][2], s[1][3])};
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      uint32_t vb[4];
      ldsm4_trans(vt + swz<C::kRowBytes>(vrow, 2 * d + vpar), vb);
      mma_bf16(o[2 * d], pa, vb[0], vb[1]);
      mma_bf16(o[2 * d + 1], pa, vb[2], vb[3]);
    }
  }
  l_a += __shfl_xor_sync(0xffffffffu, l_a, 1);
  l_b += __shfl_xor_sync(0xffffffffu, l_b, 1);
  l_a += __shfl_xor_sync(0xffffffffu, l_a, 2);
  l_b += __shfl_xor_sync(0xffffffffu, l_b, 2);

  if (p.units) {
    // The warp's own rows.
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = half ? rb : ra;
      if (r >= p.rows) continue;
      const float m = half ? m_b : m_a, l = half ? l_b : l_a;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const int head = h * p.group + r % p.group, tok = r / p.group;
      if (p.lse && (lane & 3) == 0)
        p.lse[(static_cast<int64_t>(b) * p.Hkv * p.group + head) * p.Sq + tok] = row_lse(m, l);
      uint16_t* dst = p.o.row(b, head, tok) + ca;
#pragma unroll
      for (int d = 0; d < D / 8; ++d)
        *reinterpret_cast<uint32_t*>(dst + 8 * d) =
            pack_bf16x2(o[d][2 * half] * inv, o[d][2 * half + 1] * inv);
    }
    return;
  }

  // Merge the warps through shared memory (the rings are free by then).
  cp_async_wait<0>();
  __syncthreads();
  float* o_sh = reinterpret_cast<float*>(smem);
  float2* ml_sh = reinterpret_cast<float2*>(o_sh + kWarps * kRows * C::kOStride);
  {
    const int row = lane >> 2;
    float* dst = o_sh + (warp * kRows + row) * C::kOStride + ca;
#pragma unroll
    for (int d = 0; d < D / 8; ++d) {
      *reinterpret_cast<float2*>(dst + 8 * d) = make_float2(o[d][0], o[d][1]);
      *reinterpret_cast<float2*>(dst + 8 * C::kOStride + 8 * d) = make_float2(o[d][2], o[d][3]);
    }
    if ((lane & 3) == 0) {
      ml_sh[warp * kRows + row] = make_float2(m_a, l_a);
      ml_sh[warp * kRows + row + 8] = make_float2(m_b, l_b);
    }
  }
  __syncthreads();
  const int row = static_cast<int>(threadIdx.x) >> 3;  // eight threads to a row
  const int r = rt * kRows + row;
  float mx = -INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, ml_sh[w * kRows + row].x);
  float wt[kWarps], l = 0.0f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const float2 ml = ml_sh[w * kRows + row];
    wt[w] = part_weight(ml, mx);
    l = fmaf(ml.y, wt[w], l);
  }
  const int t8 = static_cast<int>(threadIdx.x) & 7;
  float a[D / 64][8];
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) a[c][e] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float4* src = reinterpret_cast<const float4*>(
          o_sh + (w * kRows + row) * C::kOStride + c * 64 + t8 * 8);
      const float4 x = src[0], y = src[1];
      a[c][0] = fmaf(x.x, wt[w], a[c][0]);
      a[c][1] = fmaf(x.y, wt[w], a[c][1]);
      a[c][2] = fmaf(x.z, wt[w], a[c][2]);
      a[c][3] = fmaf(x.w, wt[w], a[c][3]);
      a[c][4] = fmaf(y.x, wt[w], a[c][4]);
      a[c][5] = fmaf(y.y, wt[w], a[c][5]);
      a[c][6] = fmaf(y.z, wt[w], a[c][6]);
      a[c][7] = fmaf(y.w, wt[w], a[c][7]);
    }
  }
  if (p.part_o) {
    if (p.overlaps && blockIdx.x + 1 == gridDim.x) pdl_wait();
    if (r >= p.rows) return;
    const int64_t part = (static_cast<int64_t>(bh) * p.nsplit + split) * p.rows + r;
    if (t8 == 0) p.part_ml[part] = make_float2(mx, l);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      float4* dst = reinterpret_cast<float4*>(p.part_o + part * D + c * 64 + t8 * 8);
      dst[0] = make_float4(a[c][0], a[c][1], a[c][2], a[c][3]);
      dst[1] = make_float4(a[c][4], a[c][5], a[c][6], a[c][7]);
    }
    return;
  }
  if (p.nsplit > 1) {
    // The cluster's splits: each CTA leaves its rows in its shared memory and
    // merges every nsplit-th row of all of them, in split order.
    __syncthreads();  // the warps' parts have been read
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      float4* dst = reinterpret_cast<float4*>(o_sh + row * C::kOStride + c * 64 + t8 * 8);
      dst[0] = make_float4(a[c][0], a[c][1], a[c][2], a[c][3]);
      dst[1] = make_float4(a[c][4], a[c][5], a[c][6], a[c][7]);
    }
    if (t8 == 0) ml_sh[row] = make_float2(mx, l);
    cluster_sync_all();
    constexpr int kCols = D / 32;  // of a lane; a warp to a row
    for (int i = split + warp * p.nsplit; i < kRows; i += kWarps * p.nsplit) {
      const int r_all = rt * kRows + i;
      if (r_all >= p.rows) break;
      const uint32_t at = smem_u32(o_sh + i * C::kOStride + lane * kCols);
      const float2 ml = lane < p.nsplit
                            ? ld_cluster2(mapa_shared(smem_u32(ml_sh + i), lane))
                            : make_float2(-INFINITY, 0.0f);
      float m_all = ml.x;
#pragma unroll
      for (int m = kMaxCluster / 2; m > 0; m >>= 1)
        m_all = fmaxf(m_all, __shfl_xor_sync(0xffffffffu, m_all, m));
      m_all = __shfl_sync(0xffffffffu, m_all, 0);
      const float w_own = part_weight(ml, m_all);
      float l_all = 0.0f, acc[kCols];
#pragma unroll
      for (int e = 0; e < kCols; ++e) acc[e] = 0.0f;
#pragma unroll 4
      for (int s2 = 0; s2 < p.nsplit; ++s2) {
        const float w = __shfl_sync(0xffffffffu, w_own, s2);
        l_all = fmaf(__shfl_sync(0xffffffffu, ml.y, s2), w, l_all);
        const uint32_t src = mapa_shared(at, static_cast<uint32_t>(s2));
#pragma unroll
        for (int e = 0; e < kCols; e += 2) {
          const float2 x = ld_cluster2(src + 4 * e);
          acc[e] = fmaf(x.x, w, acc[e]);
          acc[e + 1] = fmaf(x.y, w, acc[e + 1]);
        }
      }
      const float inv = l_all == 0.0f ? 0.0f : 1.0f / l_all;
      const int head = h * p.group + r_all % p.group, tok = r_all / p.group;
      if (p.lse && lane == 0)
        p.lse[(static_cast<int64_t>(b) * p.Hkv * p.group + head) * p.Sq + tok] =
            row_lse(m_all, l_all);
      uint16_t* dst = p.o.row(b, head, tok) + lane * kCols;
#pragma unroll
      for (int e = 0; e < kCols; e += 2)
        reinterpret_cast<uint32_t*>(dst)[e / 2] = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
    }
    cluster_sync_all();  // the other CTAs have read this one's rows
    return;
  }
  if (r >= p.rows) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const int head = h * p.group + r % p.group, tok = r / p.group;
  if (p.lse && t8 == 0)
    p.lse[(static_cast<int64_t>(b) * p.Hkv * p.group + head) * p.Sq + tok] = row_lse(mx, l);
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
    *reinterpret_cast<uint4*>(p.o.row(b, head, tok) + c * 64 + t8 * 8) = make_uint4(
        pack_bf16x2(a[c][0] * inv, a[c][1] * inv), pack_bf16x2(a[c][2] * inv, a[c][3] * inv),
        pack_bf16x2(a[c][4] * inv, a[c][5] * inv), pack_bf16x2(a[c][6] * inv, a[c][7] * inv));
}

// O = sum_s w_s O_s / sum_s w_s l_s over the splits' partial sums, added in
// split order; one warp to a row.
struct CombineParams {
  View o;
  // a: [B * Hkv][na][rows][D] (split_attention_kernel's)
  const float* part_a;
  const float2* ml_a;
  int na;
  // b: [Hkv][nb][B * rows][D] (a shared prefix's); nb may be 0
  const float* part_b;
  const float2* ml_b;
  int nb;
  int B, Hkv, group, Sq, rows;
  float* lse;  // as split::Params
};

template <int D>
__global__ void __launch_bounds__(128) combine_kernel(const __grid_constant__ CombineParams p) {
  constexpr int kCols = D / 32;  // of a lane
  const int lane = static_cast<int>(lane_id());
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + warp_id();  // (b, hkv, r)
  if (row >= static_cast<int64_t>(p.B) * p.Hkv * p.rows) return;
  const int64_t bh = row / p.rows;
  const int r = static_cast<int>(row - bh * p.rows);
  const int b = static_cast<int>(bh / p.Hkv), h = static_cast<int>(bh - static_cast<int64_t>(b) * p.Hkv);
  const int64_t a0 = bh * p.na * p.rows + r;  // + s * rows
  const int64_t rows_b = static_cast<int64_t>(p.B) * p.rows;
  const int64_t b0 = h * p.nb * rows_b + static_cast<int64_t>(b) * p.rows + r;  // + s * rows_b
  pdl_wait();  // the partial sums
  const float2 none = make_float2(-INFINITY, 0.0f);
  const float2 ml_a = lane < p.na ? p.ml_a[a0 + static_cast<int64_t>(lane) * p.rows] : none;
  const float2 ml_b = lane < p.nb ? p.ml_b[b0 + lane * rows_b] : none;
  float mx = fmaxf(ml_a.x, ml_b.x);
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, m));
  const float wa = part_weight(ml_a, mx), wb = part_weight(ml_b, mx);
  float l = wa * ml_a.y + wb * ml_b.y;
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) l += __shfl_xor_sync(0xffffffffu, l, m);
  float acc[kCols];
#pragma unroll
  for (int e = 0; e < kCols; ++e) acc[e] = 0.0f;
  auto add = [&](const float* src, float w) {
    float x[kCols];
    if constexpr (kCols == 4) {
      const float4 t = *reinterpret_cast<const float4*>(src + 4 * lane);
      x[0] = t.x;
      x[1] = t.y;
      x[2] = t.z;
      x[3] = t.w;
    } else {
      const float2 t = *reinterpret_cast<const float2*>(src + 2 * lane);
      x[0] = t.x;
      x[1] = t.y;
    }
#pragma unroll
    for (int e = 0; e < kCols; ++e) acc[e] = fmaf(x[e], w, acc[e]);
  };
  for (int s = 0; s < p.nb; ++s)
    add(p.part_b + (b0 + s * rows_b) * D, __shfl_sync(0xffffffffu, wb, s));
  for (int s = 0; s < p.na; ++s)
    add(p.part_a + (a0 + static_cast<int64_t>(s) * p.rows) * D, __shfl_sync(0xffffffffu, wa, s));
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (p.lse && lane == 0)
    p.lse[(bh * p.group + r % p.group) * p.Sq + r / p.group] = row_lse(mx, l);
  uint16_t* dst = p.o.row(b, h * p.group + r % p.group, r / p.group);
  if constexpr (kCols == 4) {
    *reinterpret_cast<uint2*>(dst + 4 * lane) = make_uint2(
        pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  } else {
    *reinterpret_cast<uint32_t*>(dst + 2 * lane) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  }
}

}  // namespace split
}  // namespace b200
