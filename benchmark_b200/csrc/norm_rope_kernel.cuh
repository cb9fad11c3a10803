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
// the rotation none.  A warp walks the heads of one token, so that its lanes
// keep their angles and weights in registers; it has the next rows in flight
// while it works on its own, and nothing synchronises the warps.  (A first
// form kept both in shared memory for a block of tokens: its reads kept the
// load/store unit 80 % busy, 77 us against 63 for 16384 tokens of 32 + 8
// heads of 128.)  With few heads a warp's lanes would stay empty: then each
// of its rows walks a token of its own (kPerRow).
#pragma once

#include "ptx.cuh"
#include "view.cuh"

namespace b200 {
namespace rope {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
// Resident CTAs, by registers: forward measured 66 / 63 / 68 / 75 us with 6 / 7
// / 8 / 9 (16384 tokens, 32 + 8 heads of 128), backward 114 / 109 / 142 us with
// 3 / 4 / 5.
constexpr int kCtasPerSm = 7;
constexpr int kGradCtasPerSm = 4;

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
  uint32_t tokens;      // B * S
  int S, Hq, Hkv, rot;
  int slices, slice_groups;  // forward: warps of a token, row groups of each
  float eps;
  float* dw_part;       // backward: [CTAs][D]
  int ctas_q;           // backward: CTAs of the queries; the others take the keys
};

template <int D, bool kPerRow>
struct Shape {
  static constexpr int kLanes = D / 16;                 // lanes of a row
  static constexpr int kRows = 32 / kLanes;             // rows of a warp
  static constexpr int kTokens = kPerRow ? kRows : 1;   // tokens of a warp
  static constexpr int kHeads = kPerRow ? 1 : kRows;    // heads of a row group
};

// A lane's share of a row: chunks c0 and c1 (8 columns each), c1 the rotation
// partner of c0 in the half-split form.
struct Lane {
  int row, l, c0, c1;
  bool rotated;
};

template <int kLanes>
__device__ __forceinline__ Lane lane_of(int rot) {
  Lane x;
  x.row = static_cast<int>(lane_id()) / kLanes;
  x.l = static_cast<int>(lane_id()) % kLanes;
  const int nrot = rot >> 4;  // lanes whose chunks are rotated
  x.rotated = x.l < nrot;
  x.c0 = x.rotated ? x.l : 2 * x.l;
  x.c1 = x.rotated ? x.l + nrot : 2 * x.l + 1;
  return x;
}

__device__ __forceinline__ void unpack8(const uint4& v, uint64_t* f) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    f[i] = f2_pack(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
}

__device__ __forceinline__ uint4 pack8(const uint64_t* f) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a, b;
    f2_unpack(f[i], a, b);
    u[i] = pack_bf16x2(a, b);
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// The lane's 16 weights as pairs.
__device__ __forceinline__ void load_weights(const void* w, int w_f32, const Lane& x,
                                             uint64_t (&out)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c = h ? x.c1 : x.c0;
    if (w_f32) {
      const uint4* src = static_cast<const uint4*>(w) + 2 * c;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint4 a = ld_global(src + e);
        out[4 * h + 2 * e] = f2_pack(__uint_as_float(a.x), __uint_as_float(a.y));
        out[4 * h + 2 * e + 1] = f2_pack(__uint_as_float(a.z), __uint_as_float(a.w));
      }
    } else {
      unpack8(ld_global(static_cast<const uint4*>(w) + c), out + 4 * h);
    }
  }
}

// cos and sin of position * frequency.  The angle is formed in 64 bits as a
// fraction of a turn, so that far positions keep theirs; sincospi of the
// reduced fraction is then exact to fp32.
__device__ __forceinline__ void angle(int pos, float freq, float* c, float* s) {
  const double turns =
      static_cast<double>(pos) * static_cast<double>(freq) * 0.15915494309189533577;
  sincospif(2.0f * static_cast<float>(turns - rint(turns)), s, c);
}

// The lane's 8 angles for its token (cos 1, sin 0 where nothing turns), two to
// a word: pairs 8 l + j in the half-split form; 4 c0 + j, then 4 c1 + j - 4,
// interleaved.
struct Angles {
  uint64_t c[4], s[4];
};

// The rows of a shared token compute 8 / kRows of them each and exchange them.
template <int D, bool kInterleaved, bool kPerRow>
__device__ __forceinline__ Angles lane_angles(const float* inv_freq, int pos, const Lane& x) {
  using Sh = Shape<D, kPerRow>;
  auto pair = [&](int j) {
    return kInterleaved ? 4 * (j < 4 ? x.c0 : x.c1) + (j & 3) : 8 * x.l + j;
  };
  constexpr int kOwn = kPerRow ? 8 : 8 / Sh::kRows;
  float oc[kOwn], os[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    oc[i] = 1.0f;
    os[i] = 0.0f;
    if (x.rotated)
      angle(pos, ld_global(inv_freq + pair((kPerRow ? 0 : x.row * kOwn) + i)), &oc[i], &os[i]);
  }
  Angles a;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    float c[2], s[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      c[e] = oc[(j + e) % kOwn];
      s[e] = os[(j + e) % kOwn];
      if constexpr (!kPerRow) {
        const int from = ((j + e) / kOwn) * Sh::kLanes + x.l;
        c[e] = __shfl_sync(0xffffffffu, c[e], from);
        s[e] = __shfl_sync(0xffffffffu, s[e], from);
      }
    }
    a.c[j / 2] = f2_pack(c[0], c[1]);
    a.s[j / 2] = f2_pack(s[0], s[1]);
  }
  return a;
}

// v (16 values as pairs, chunk c0's then chunk c1's) turned by the lane's
// angles; kBack turns back.
template <bool kInterleaved, bool kBack>
__device__ __forceinline__ void rotate16(uint64_t (&v)[8], const Angles& t) {
  if constexpr (kInterleaved) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float a, b, c[2], s[2];
      f2_unpack(v[j], a, b);
      f2_unpack(t.c[j / 2], c[0], c[1]);
      f2_unpack(t.s[j / 2], s[0], s[1]);
      const float cj = c[j & 1], sj = kBack ? -s[j & 1] : s[j & 1];
      v[j] = f2_pack(fmaf(a, cj, -b * sj), fmaf(b, cj, a * sj));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t a = v[i], b = v[4 + i];
      if constexpr (kBack) {
        v[i] = f2_fma(a, t.c[i], f2_mul(b, t.s[i]));
        v[4 + i] = f2_sub(f2_mul(b, t.c[i]), f2_mul(a, t.s[i]));
      } else {
        v[i] = f2_sub(f2_mul(a, t.c[i]), f2_mul(b, t.s[i]));
        v[4 + i] = f2_fma(b, t.c[i], f2_mul(a, t.s[i]));
      }
    }
  }
}

template <int kLanes>
__device__ __forceinline__ float row_sum(uint64_t pairs) {
  float a, b;
  f2_unpack(pairs, a, b);
  a += b;
#pragma unroll
  for (int m = kLanes / 2; m > 0; m >>= 1) a += __shfl_xor_sync(0xffffffffu, a, m);
  return a;
}

// r of the row whose 16 values per lane are v.
template <int D>
__device__ __forceinline__ float row_norm(const uint64_t (&v)[8], float eps) {
  uint64_t e = f2_mul(v[0], v[0]), o = f2_mul(v[1], v[1]);
#pragma unroll
  for (int i = 2; i < 8; i += 2) {
    e = f2_fma(v[i], v[i], e);
    o = f2_fma(v[i + 1], v[i + 1], o);
  }
  return rsqrtf(row_sum<D / 16>(f2_add(e, o)) * (1.0f / D) + eps);
}

// The two chunks of a lane; streamed, since nothing reads them again.
struct Chunks {
  uint4 a, b;
};

__device__ __forceinline__ Chunks load_chunks(const uint16_t* row, const Lane& x, bool live) {
  Chunks r{make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
  if (live) {
    r.a = ld_global_stream(reinterpret_cast<const uint4*>(row) + x.c0);
    r.b = ld_global_stream(reinterpret_cast<const uint4*>(row) + x.c1);
  }
  return r;
}

__device__ __forceinline__ void store_chunks(uint16_t* row, const Lane& x,
                                             const uint64_t (&v)[8]) {
  reinterpret_cast<uint4*>(row)[x.c0] = pack8(v);
  reinterpret_cast<uint4*>(row)[x.c1] = pack8(v + 4);
}

// A warp takes a slice of the row groups (queries, then keys) of its token.
template <int D, bool kInterleaved, bool kPerRow>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) norm_rope_kernel(const __grid_constant__ Params p) {
  using Sh = Shape<D, kPerRow>;
  pdl_wait();
  pdl_launch_dependents();
  const Lane x = lane_of<Sh::kLanes>(p.rot);
  const uint32_t item = blockIdx.x * kWarps + warp_id();
  const uint32_t tg = p.slices == 1 ? item : item / static_cast<uint32_t>(p.slices);
  const int slice = static_cast<int>(item - tg * static_cast<uint32_t>(p.slices));
  const uint32_t t = tg * Sh::kTokens + (kPerRow ? x.row : 0);
  if (tg * Sh::kTokens >= p.tokens) return;  // the whole warp
  const bool live_t = t < p.tokens;
  const uint32_t b = live_t ? t / static_cast<uint32_t>(p.S) : 0u;
  const uint32_t s = live_t ? t - b * static_cast<uint32_t>(p.S) : 0u;
  const int groups_q = (p.Hq + Sh::kHeads - 1) / Sh::kHeads;
  const int groups = groups_q + (p.Hkv + Sh::kHeads - 1) / Sh::kHeads;
  const int row = kPerRow ? 0 : x.row;
  const int g0 = slice * p.slice_groups, g1 = min(groups, g0 + p.slice_groups);
  const int pos = p.rot > 0 && live_t ? ld_global(p.pos + b * p.pos_sb + s) : 0;
  Angles turn;
  uint64_t w[8];
  bool first = true;
  // Row groups [g, end) of one tensor, the next one's rows in flight.
  auto walk = [&](const View& from, const View& to, const void* weight, int H, int g, int end) {
    if (g >= end) return;
    int h = g * Sh::kHeads + row;
    const int64_t step = Sh::kHeads * from.sh, out_step = Sh::kHeads * to.sh;
    const uint16_t* in = from.row(b, h, s);
    uint16_t* out = to.row(b, h, s);
    const int H_live = live_t ? H : 0;
    Chunks next = load_chunks(in, x, h < H_live);
    if (first) turn = lane_angles<D, kInterleaved, kPerRow>(p.inv_freq, pos, x);
    first = false;
    load_weights(weight, p.w_f32, x, w);
    for (int i = end - g; i > 0; --i) {
      uint64_t v[8];
      unpack8(next.a, v);
      unpack8(next.b, v + 4);
      const bool live = h < H_live;
      h += Sh::kHeads;
      in += step;
      next = load_chunks(in, x, h < H_live);
      const float rn = row_norm<D>(v, p.eps);
      const uint64_t rn2 = f2_pack(rn, rn);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = f2_mul(v[e], f2_mul(w[e], rn2));
      rotate16<kInterleaved, false>(v, turn);
      if (live) store_chunks(out, x, v);
      out += out_step;
    }
  };
  walk(p.q, p.qy, p.wq, p.Hq, g0, min(g1, groups_q));
  walk(p.k, p.ky, p.wk, p.Hkv, max(g0 - groups_q, 0), g1 - groups_q);
}

// Backward: the first ctas_q CTAs take the queries, the others the keys.
// Each warp walks its own tokens and sums its rows' weight gradients in
// registers, in an order that depends only on the grid; norm_rope_dw_kernel
// adds the CTAs' sums in CTA order.
template <int D, bool kInterleaved, bool kPerRow>
__global__ void __launch_bounds__(kThreads, kGradCtasPerSm)
    norm_rope_bwd_kernel(const __grid_constant__ Params p) {
  using Sh = Shape<D, kPerRow>;
  __shared__ float dw_sh[kWarps][D];
  pdl_wait();
  pdl_launch_dependents();
  const Lane x = lane_of<Sh::kLanes>(p.rot);
  const bool is_q = static_cast<int>(blockIdx.x) < p.ctas_q;
  const int cta = static_cast<int>(blockIdx.x) - (is_q ? 0 : p.ctas_q);
  const int ctas = is_q ? p.ctas_q : static_cast<int>(gridDim.x) - p.ctas_q;
  const View& in = is_q ? p.q : p.k;
  const View& gin = is_q ? p.qy : p.ky;
  const View& out = is_q ? p.qdx : p.kdx;
  const int H = is_q ? p.Hq : p.Hkv;
  const uint32_t token_groups = (p.tokens + Sh::kTokens - 1) / Sh::kTokens;
  const uint32_t stride = static_cast<uint32_t>(ctas) * kWarps;
  uint64_t w[8], dw[8];
  load_weights(is_q ? p.wq : p.wk, p.w_f32, x, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[i] = 0ull;
  const int row = kPerRow ? 0 : x.row;
  // A token's first rows in the three tensors.
  struct Place {
    bool live;
    int pos;
    const uint16_t *in, *gin;
    uint16_t* out;
  };
  auto place = [&](uint32_t tg) {
    Place r;
    const uint32_t t = tg * Sh::kTokens + (kPerRow ? x.row : 0);
    r.live = t < p.tokens;
    const uint32_t b = r.live ? t / static_cast<uint32_t>(p.S) : 0u;
    const uint32_t s = r.live ? t - b * static_cast<uint32_t>(p.S) : 0u;
    r.pos = p.rot > 0 && r.live ? ld_global(p.pos + b * p.pos_sb + s) : 0;
    r.in = in.row(b, row, s);
    r.gin = gin.row(b, row, s);
    r.out = out.row(b, row, s);
    return r;
  };
  const int64_t in_step = Sh::kHeads * in.sh, gin_step = Sh::kHeads * gin.sh,
                out_step = Sh::kHeads * out.sh;
  Chunks nx, ng;
  uint32_t tg = static_cast<uint32_t>(cta) * kWarps + warp_id();
  Place now{}, then{};
  if (tg < token_groups) {
    now = place(tg);
    nx = load_chunks(now.in, x, now.live && row < H);
    ng = load_chunks(now.gin, x, now.live && row < H);
  }
  for (; tg < token_groups; tg += stride) {
    const bool more = tg + stride < token_groups;
    if (more) then = place(tg + stride);
    const Angles turn = lane_angles<D, kInterleaved, kPerRow>(p.inv_freq, now.pos, x);
    for (int h = row; h - row < H; h += Sh::kHeads) {
      uint64_t v[8], g[8];
      unpack8(nx.a, v);
      unpack8(nx.b, v + 4);
      unpack8(ng.a, g);
      unpack8(ng.b, g + 4);
      if (h - row + Sh::kHeads < H) {
        now.in += in_step;
        now.gin += gin_step;
        nx = load_chunks(now.in, x, now.live && h + Sh::kHeads < H);
        ng = load_chunks(now.gin, x, now.live && h + Sh::kHeads < H);
      } else if (more) {
        nx = load_chunks(then.in, x, then.live && row < H);
        ng = load_chunks(then.gin, x, then.live && row < H);
      }
      const bool live = now.live && h < H;
      // (Without eps the zeros of a row that is not there would give NaN.)
      const float norm = row_norm<D>(v, p.eps), rn = live ? norm : 0.0f;
      const uint64_t rn2 = f2_pack(rn, rn);
      rotate16<kInterleaved, true>(g, turn);
      uint64_t dot2 = 0ull;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = f2_mul(v[i], rn2);
        dw[i] = f2_fma(g[i], v[i], dw[i]);  // a row that is not live adds zeros
        g[i] = f2_mul(g[i], w[i]);
        dot2 = f2_fma(g[i], v[i], dot2);
      }
      const float dot = row_sum<Sh::kLanes>(dot2) * (-1.0f / D);
      const uint64_t d2 = f2_pack(dot, dot);
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = f2_mul(rn2, f2_fma(v[i], d2, g[i]));
      if (live) store_chunks(now.out, x, g);
      now.out += out_step;
    }
    now = then;
  }
  // The warp's rows, then the CTA's warps.
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float lo, hi;
    f2_unpack(dw[i >> 1], lo, hi);
    float v = (i & 1) ? hi : lo;
#pragma unroll
    for (int m = 16; m >= Sh::kLanes; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    if (x.row == 0) dw_sh[warp_id()][8 * (i < 8 ? x.c0 : x.c1) + (i & 7)] = v;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < D; i += kThreads) {
    float v = 0.0f;
#pragma unroll
    for (int wi = 0; wi < kWarps; ++wi) v += dw_sh[wi][i];
    p.dw_part[static_cast<int64_t>(blockIdx.x) * D + i] = v;
  }
}

// dw[column] = sum over the CTAs' parts, queries' and keys'.  A block takes 8
// columns; a column has 64 threads, eight parts in flight each.
__global__ void __launch_bounds__(512)
    norm_rope_dw_kernel(const float* part, int ctas_q, int ctas, int D, float* dwq, float* dwk) {
  __shared__ float sh[64][9];
  const int c = static_cast<int>(threadIdx.x) & 7, row = static_cast<int>(threadIdx.x) >> 3;
  int col = static_cast<int>(blockIdx.x) * 8 + c;
  const bool is_q = col < D;
  if (!is_q) col -= D;
  const int end = is_q ? ctas_q : ctas;
  pdl_wait();
  float v = 0.0f;
  for (int i = (is_q ? 0 : ctas_q) + row; i < end; i += 512) {
    float x[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      x[u] = i + 64 * u < end ? part[static_cast<int64_t>(i + 64 * u) * D + col] : 0.0f;
    v += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
  }
  sh[row][c] = v;
  __syncthreads();
  if (row == 0) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 64; ++i) sum += sh[i][c];
    (is_q ? dwq : dwk)[col] = sum;
  }
}

}  // namespace rope
}  // namespace b200
