// Query/key norm with position rotation, forward and backward.
//
//   r = (mean(x^2) + eps)^-1/2,   y = R(pos) (x r w)
//
// R(pos) turns pair i of the first `rot` columns by pos * inv_freq[i]: columns
// (i, i + rot/2), or (2i, 2i+1) when interleaved; columns from `rot` on pass
// through.  Backward, with g = R(pos)^T dy:
//
//   dw = sum over rows of g x r,   dx = r (g w - x r mean(g w x r))
//
// Both are bound by memory: forward reads and writes each element once (4 B),
// backward reads two and writes one (6 B).  A row of D bf16 values lives in
// D/16 lanes, 16 values each as two 16-byte chunks placed so that a rotated
// pair never crosses lanes: the row statistics take log2(D/16) shuffles and
// the rotation none.  A CTA takes a block of consecutive tokens; it computes
// the block's angles once (shared memory) for all of its heads.
#pragma once

#include "ptx.cuh"
#include "view.cuh"

namespace b200 {
namespace rope {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;  // tokens of a block whose angles shared memory holds
constexpr int kGradCtasPerSm = 2;

struct Params {
  View q, k;            // x
  View qy, ky;          // forward: y; backward: dy
  View qdx, kdx;        // backward: dx
  const void* wq;       // [D]
  const void* wk;
  int w_f32;            // the weights are fp32 (else bf16)
  const float* inv_freq;  // [rot / 2]
  const int32_t* pos;   // pos[b * pos_sb + s]
  int64_t pos_sb;
  int64_t tokens;       // B * S
  int S, Hq, Hkv, rot;
  int block;            // tokens per block
  uint32_t mul_q, mul_k;  // 2^32 / H + 1 for row / H of a block's rows; 0: H is 1
  float eps;
  float* dw_part;       // backward: [CTAs][2][D]
};

__device__ __forceinline__ float2 bf16x2_f32(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = bf16x2_f32(u[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}

__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                    pack_bf16x2(f[6], f[7]));
}

// The chunks (8 columns each) of lane l of a row: c1 = c0's rotation partner
// in the half-split form.
__device__ __forceinline__ void lane_chunks(int l, int rot, int* c0, int* c1) {
  const int nrot = rot >> 4;  // lanes whose chunks are rotated
  if (l < nrot) {
    *c0 = l;
    *c1 = l + nrot;
  } else {
    *c0 = 2 * l;
    *c1 = 2 * l + 1;
  }
}

// (cos, sin) of the block's tokens.  The angle is formed in 64 bits as a
// fraction of a turn, so that far positions keep theirs; sincospi of the
// reduced fraction is then exact to fp32.
template <int D>
__device__ __forceinline__ void block_angles(const Params& p, int64_t t0, int nt, float2* cs) {
  const int half = p.rot >> 1;
  for (int i = threadIdx.x; i < nt * half; i += kThreads) {
    const int tl = i / half, f = i - tl * half;
    const int64_t t = t0 + tl;
    const int64_t b = t / p.S;
    const double turns = static_cast<double>(p.pos[b * p.pos_sb + (t - b * p.S)]) *
                         static_cast<double>(p.inv_freq[f]) * 0.15915494309189533577;
    float s, c;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
    cs[tl * (D / 2) + f] = make_float2(c, s);
  }
}

template <int D>
__device__ __forceinline__ void load_weights(const Params& p, float* w) {
  for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
    const void* src = i < D ? p.wq : p.wk;
    const int j = i < D ? i : i - D;
    w[i] = p.w_f32 ? static_cast<const float*>(src)[j]
                   : __uint_as_float(
                         static_cast<uint32_t>(static_cast<const uint16_t*>(src)[j]) << 16);
  }
}

// v (16 values, chunks c0 and c1 of a rotated lane) turned by the pairs'
// angles; sign = -1 turns back.
template <bool kInterleaved>
__device__ __forceinline__ void rotate16(float* v, const float2* cs, int c0, int c1, float sign) {
  if constexpr (kInterleaved) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4* a4 = reinterpret_cast<const float4*>(cs + 4 * (h ? c1 : c0));
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float4 a = a4[e];
        float* u = v + 8 * h + 4 * e;
        const float x0 = u[0], y0 = u[1], x1 = u[2], y1 = u[3];
        const float s0 = sign * a.y, s1 = sign * a.w;
        u[0] = x0 * a.x - y0 * s0;
        u[1] = y0 * a.x + x0 * s0;
        u[2] = x1 * a.z - y1 * s1;
        u[3] = y1 * a.z + x1 * s1;
      }
    }
  } else {
    const float4* a4 = reinterpret_cast<const float4*>(cs + 8 * c0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 a = a4[e];
      const float s0 = sign * a.y, s1 = sign * a.w;
      const float x0 = v[2 * e], y0 = v[8 + 2 * e], x1 = v[2 * e + 1], y1 = v[8 + 2 * e + 1];
      v[2 * e] = x0 * a.x - y0 * s0;
      v[8 + 2 * e] = y0 * a.x + x0 * s0;
      v[2 * e + 1] = x1 * a.z - y1 * s1;
      v[8 + 2 * e + 1] = y1 * a.z + x1 * s1;
    }
  }
}

// r / H by its reciprocal (exact for r * H < 2^32); H = 1 has none in 32 bits.
__device__ __forceinline__ int block_token(int r, uint32_t mul) {
  return mul == 0u ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), mul));
}

template <int kLanes>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int m = kLanes / 2; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}

// Element offsets of head 0 of the block's tokens in each of n views.
__device__ __forceinline__ void block_offsets(const Params& p, int64_t t0, int nt,
                                              const View* const* views, int n,
                                              int64_t (*off)[kMaxTokens]) {
  if (static_cast<int>(threadIdx.x) < nt) {
    const int64_t t = t0 + threadIdx.x, b = t / p.S, s = t - b * p.S;
    for (int i = 0; i < n; ++i) off[i][threadIdx.x] = b * views[i]->sb + s * views[i]->ss;
  }
}

// One block of tokens per CTA.
template <int D, bool kInterleaved>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const __grid_constant__ Params p) {
  constexpr int kLanes = D / 16;         // lanes of a row
  constexpr int kRows = 32 / kLanes;     // rows of a warp
  __shared__ __align__(16) float2 cs[kMaxTokens * (D / 2)];
  __shared__ __align__(16) float w_sh[2 * D];
  __shared__ int64_t off[4][kMaxTokens];
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.block;
  const int nt = static_cast<int>(min(static_cast<int64_t>(p.block), p.tokens - t0));
  const View* const views[4] = {&p.q, &p.k, &p.qy, &p.ky};
  block_offsets(p, t0, nt, views, 4, off);
  block_angles<D>(p, t0, nt, cs);
  load_weights<D>(p, w_sh);
  __syncthreads();
  const int lane = static_cast<int>(lane_id());
  const int l = lane & (kLanes - 1);
  int c0, c1;
  lane_chunks(l, p.rot, &c0, &c1);
  const bool rotated = l < (p.rot >> 4);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const View& in = which ? p.k : p.q;
    const View& out = which ? p.ky : p.qy;
    const int H = which ? p.Hkv : p.Hq;
    const uint32_t mul = which ? p.mul_k : p.mul_q;
    const float* w = w_sh + which * D;
    const int rows = nt * H;
    for (int r0 = static_cast<int>(warp_id()) * kRows; r0 < rows; r0 += (kThreads / 32) * kRows) {
      const int r = r0 + lane / kLanes;
      const bool live = r < rows;
      const int tl = live ? block_token(r, mul) : 0;
      const int h = live ? r - tl * H : 0;
      const uint4* src = reinterpret_cast<const uint4*>(in.p + off[which][tl] + h * in.sh);
      float v[16];
      unpack8(src[c0], v);
      unpack8(src[c1], v + 8);
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) ss = fmaf(v[i], v[i], ss);
      const float rn = rsqrtf(row_sum<kLanes>(ss) * (1.0f / D) + p.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] *= rn * w[8 * c0 + i];
        v[8 + i] *= rn * w[8 * c1 + i];
      }
      if (rotated) rotate16<kInterleaved>(v, cs + tl * (D / 2), c0, c1, 1.0f);
      if (live) {
        uint4* dst = reinterpret_cast<uint4*>(out.p + off[2 + which][tl] + h * out.sh);
        dst[c0] = pack8(v);
        dst[c1] = pack8(v + 8);
      }
    }
  }
}

// Backward: each CTA walks token blocks blockIdx.x, + gridDim.x, ... and sums
// its rows' weight gradients in registers, in an order that depends only on
// the grid; norm_rope_dw_kernel adds the CTAs' sums in CTA order.
template <int D, bool kInterleaved>
__global__ void __launch_bounds__(kThreads, kGradCtasPerSm)
    norm_rope_bwd_kernel(const __grid_constant__ Params p) {
  constexpr int kLanes = D / 16;
  constexpr int kRows = 32 / kLanes;
  constexpr int kWarps = kThreads / 32;
  __shared__ __align__(16) float2 cs[kMaxTokens * (D / 2)];
  __shared__ __align__(16) float w_sh[2 * D];
  __shared__ float dw_sh[kWarps][2 * D];
  __shared__ int64_t off[6][kMaxTokens];
  const View* const views[6] = {&p.q, &p.k, &p.qy, &p.ky, &p.qdx, &p.kdx};
  load_weights<D>(p, w_sh);
  const int lane = static_cast<int>(lane_id());
  const int warp = static_cast<int>(warp_id());
  const int l = lane & (kLanes - 1);
  int c0, c1;
  lane_chunks(l, p.rot, &c0, &c1);
  const bool rotated = l < (p.rot >> 4);
  float dw[2][16];
#pragma unroll
  for (int i = 0; i < 32; ++i) dw[i >> 4][i & 15] = 0.0f;
  const int64_t blocks = (p.tokens + p.block - 1) / p.block;
  for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const int64_t t0 = blk * p.block;
    const int nt = static_cast<int>(min(static_cast<int64_t>(p.block), p.tokens - t0));
    __syncthreads();  // every warp is done with the previous block's angles
    block_offsets(p, t0, nt, views, 6, off);
    block_angles<D>(p, t0, nt, cs);
    __syncthreads();
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const View& in = which ? p.k : p.q;
      const View& gin = which ? p.ky : p.qy;
      const View& out = which ? p.kdx : p.qdx;
      const int H = which ? p.Hkv : p.Hq;
      const uint32_t mul = which ? p.mul_k : p.mul_q;
      const float* w = w_sh + which * D;
      const int rows = nt * H;
      for (int r0 = warp * kRows; r0 < rows; r0 += kWarps * kRows) {
        const int r = r0 + lane / kLanes;
        const bool live = r < rows;
        const int tl = live ? block_token(r, mul) : 0;
        const int h = live ? r - tl * H : 0;
        const uint4* src = reinterpret_cast<const uint4*>(in.p + off[which][tl] + h * in.sh);
        const uint4* gsrc =
            reinterpret_cast<const uint4*>(gin.p + off[2 + which][tl] + h * gin.sh);
        const uint4 x0 = src[c0], x1 = src[c1], g0 = gsrc[c0], g1 = gsrc[c1];
        float x[16], g[16];
        unpack8(x0, x);
        unpack8(x1, x + 8);
        unpack8(g0, g);
        unpack8(g1, g + 8);
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
        const float rn = rsqrtf(row_sum<kLanes>(ss) * (1.0f / D) + p.eps);
        if (rotated) rotate16<kInterleaved>(g, cs + tl * (D / 2), c0, c1, -1.0f);
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[i] *= rn;
          if (live) dw[which][i] = fmaf(g[i], x[i], dw[which][i]);
          g[i] *= w[8 * (i < 8 ? c0 : c1) + (i & 7)];
          dot = fmaf(g[i], x[i], dot);
        }
        dot = row_sum<kLanes>(dot) * (1.0f / D);
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = rn * fmaf(-x[i], dot, g[i]);
        if (live) {
          uint4* dst = reinterpret_cast<uint4*>(out.p + off[4 + which][tl] + h * out.sh);
          dst[c0] = pack8(g);
          dst[c1] = pack8(g + 8);
        }
      }
    }
  }
  // The warp's rows, then the CTA's warps.
#pragma unroll
  for (int which = 0; which < 2; ++which)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = dw[which][i];
#pragma unroll
      for (int m = 16; m >= kLanes; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
      if (lane < kLanes) dw_sh[warp][which * D + 8 * (i < 8 ? c0 : c1) + (i & 7)] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += kThreads) {
    float v = 0.0f;
#pragma unroll
    for (int wi = 0; wi < kWarps; ++wi) v += dw_sh[wi][i];
    p.dw_part[static_cast<int64_t>(blockIdx.x) * 2 * D + i] = v;
  }
}

// dw[column] = sum over the CTAs' parts; 32 columns per block, eight threads
// to a column.
__global__ void __launch_bounds__(256)
    norm_rope_dw_kernel(const float* part, int parts, int D, float* dwq, float* dwk) {
  __shared__ float sh[8][32];
  const int col = static_cast<int>(blockIdx.x) * 32 + (threadIdx.x & 31);
  const int row = threadIdx.x >> 5;
  float v = 0.0f;
  for (int i = row; i < parts; i += 8) v += part[static_cast<int64_t>(i) * 2 * D + col];
  sh[row][threadIdx.x & 31] = v;
  __syncthreads();
  if (row == 0) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += sh[i][threadIdx.x];
    if (col < D)
      dwq[col] = sum;
    else
      dwk[col - D] = sum;
  }
}

}  // namespace rope
}  // namespace b200
