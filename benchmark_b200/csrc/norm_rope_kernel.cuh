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
// keep their angles and weights in registers; the next rows are on their way
// through a ring in shared memory, of which each lane copies and reads its own
// slots: nothing synchronises the warps.  16384 tokens of 32 + 8 heads of 128,
// replayed in a graph at full clock: forward 54.3 us (6.2 TB/s), backward 88.3 us
// (5.7 TB/s); called back to back 59 and 97 us.  (With the next rows
// in registers instead, one row group ahead: 63.5 and 107 us.  With angles and
// weights in shared memory for a block of tokens, their reads kept the
// load/store unit 80 % busy: 77 us forward.)  With few heads a warp's lanes
// would stay empty: then each of its rows walks a token of its own (kPerRow).
#pragma once

#include "mma_sync.cuh"
#include "ptx.cuh"
#include "view.cuh"

namespace b200 {
namespace rope {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
// Resident CTAs, by registers, and row groups of a warp's ring.  Measured (us;
// 16384 tokens, 32 + 8 heads of 128): forward with 6 / 7 / 8 / 10 CTAs 55.2 /
// 54.6 / 55.6 / 86, with 2 / 3 / 4 groups 59.3 / 54.6 / 55.2; backward with 3 /
// 4 / 5 CTAs 95 / 88.4 / 146, with 2 / 3 / 4 groups 94.5 / 88.4 / 94.7.
constexpr int kCtasPerSm = 7;
constexpr int kGradCtasPerSm = 4;
constexpr int kStages = 3, kGradStages = 3;

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

// A lane's two chunks of a row on their way through its own slots of a ring in
// shared memory (nothing but its own copies and reads meet there: no barrier).
using Slots = uint4[2][kThreads];

__device__ __forceinline__ void copy_chunks(Slots& to, const uint16_t* row, const Lane& x,
                                            bool live) {
  cp_async16(smem_u32(&to[0][threadIdx.x]), row + 8 * x.c0, live);
  cp_async16(smem_u32(&to[1][threadIdx.x]), row + 8 * x.c1, live);
}

__device__ __forceinline__ void read_chunks(const Slots& from, uint64_t (&v)[8]) {
  unpack8(from[0][threadIdx.x], v);
  unpack8(from[1][threadIdx.x], v + 4);
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
  __shared__ Slots ring[kStages];
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
  // Row groups g0 to g1, the queries' before the keys'; kStages - 1 on their way.
  auto copy = [&](int g, int stage) {
    if (g < g1) {
      const bool is_q = g < groups_q;
      const View& from = is_q ? p.q : p.k;
      const int h = (is_q ? g : g - groups_q) * Sh::kHeads + row;
      const bool live = live_t && h < (is_q ? p.Hq : p.Hkv);
      copy_chunks(ring[stage], from.row(b, live ? h : 0, s), x, live);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) copy(g0 + i, i);
  const Angles turn = lane_angles<D, kInterleaved, kPerRow>(p.inv_freq, pos, x);
  uint64_t w[8];
  int stage = 0;
  for (int g = g0; g < g1; ++g) {
    const bool is_q = g < groups_q;
    if (g == g0 || g == groups_q) load_weights(is_q ? p.wq : p.wk, p.w_f32, x, w);
    cp_async_wait<kStages - 2>();
    uint64_t v[8];
    read_chunks(ring[stage], v);
    copy(g + kStages - 1, stage == 0 ? kStages - 1 : stage - 1);
    stage = stage + 1 == kStages ? 0 : stage + 1;
    const float rn = row_norm<D>(v, p.eps);
    const uint64_t rn2 = f2_pack(rn, rn);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = f2_mul(v[e], f2_mul(w[e], rn2));
    rotate16<kInterleaved, false>(v, turn);
    const int h = (is_q ? g : g - groups_q) * Sh::kHeads + row;
    if (live_t && h < (is_q ? p.Hq : p.Hkv))
      store_chunks((is_q ? p.qy : p.ky).row(b, h, s), x, v);
  }
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
  __shared__ Slots ring[kGradStages][2];
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
    int64_t b, s;
  };
  auto place = [&](uint32_t tg) {
    Place r;
    const uint32_t t = tg * Sh::kTokens + (kPerRow ? x.row : 0);
    r.live = t < p.tokens;
    const uint32_t b = r.live ? t / static_cast<uint32_t>(p.S) : 0u;
    r.b = b;
    r.s = r.live ? t - b * static_cast<uint32_t>(p.S) : 0u;
    r.pos = p.rot > 0 && r.live ? ld_global(p.pos + r.b * p.pos_sb + r.s) : 0;
    return r;
  };
  // The copies run kStages - 1 row groups ahead, through the warp's tokens.
  uint32_t tg = static_cast<uint32_t>(cta) * kWarps + warp_id(), ctg = tg;
  int ch = row;  // head of the next copy
  const uint16_t *c_in = nullptr, *c_gin = nullptr;
  bool c_live = false;
  auto open = [&]() {
    if (ctg >= token_groups) return;
    const Place r = place(ctg);
    c_live = r.live;
    c_in = in.row(r.b, 0, r.s);
    c_gin = gin.row(r.b, 0, r.s);
  };
  auto copy = [&](int stage) {
    if (ctg < token_groups) {
      const bool live = c_live && ch < H;
      const int64_t h = live ? ch : 0;
      copy_chunks(ring[stage][0], c_in + h * in.sh, x, live);
      copy_chunks(ring[stage][1], c_gin + h * gin.sh, x, live);
      ch += Sh::kHeads;
      if (ch - row >= H) {
        ch = row;
        ctg += stride;
        open();
      }
    }
    cp_async_commit();
  };
  open();
#pragma unroll
  for (int i = 0; i < kGradStages - 1; ++i) copy(i);
  int stage = 0;
  Place now = place(tg);
  for (; tg < token_groups; tg += stride) {
    const Place then = place(min(tg + stride, token_groups - 1));
    const Angles turn = lane_angles<D, kInterleaved, kPerRow>(p.inv_freq, now.pos, x);
    for (int h = row; h - row < H; h += Sh::kHeads) {
      uint64_t v[8], g[8];
      cp_async_wait<kGradStages - 2>();
      read_chunks(ring[stage][0], v);
      read_chunks(ring[stage][1], g);
      copy(stage == 0 ? kGradStages - 1 : stage - 1);
      stage = stage + 1 == kGradStages ? 0 : stage + 1;
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
      if (live) store_chunks(out.row(now.b, h, now.s), x, g);
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
