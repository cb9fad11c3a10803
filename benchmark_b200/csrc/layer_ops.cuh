// Host side of the attention layer's operators (include/b200attn.h):
// qk_norm_rope, attention_window and attention_shared_prefix.  Included by
// b200attn.cu, whose helpers it uses.
#pragma once

namespace {

// ---- tensors ----
b200::View view_of(const b200_tensor* t) {
  return b200::View{static_cast<uint16_t*>(const_cast<void*>(t->data)), t->stride_b, t->stride_h,
                    t->stride_s};
}

// A [B, H, S, D] tensor whose D is contiguous.  An output's rows may not
// overlap: each stride has to step over all that the smaller ones reach.
b200_status check_tensor(const char* who, const char* name, const b200_tensor* t, int B, int H,
                         int S, int D, bool output) {
  if (!t || !t->data) return fail(B200_EINVAL, "%s: null tensor %s", who, name);
  if (!aligned16(t->data))
    return fail(B200_EINVAL, "%s: %s must be 16-byte aligned", who, name);
  struct Dim {
    int64_t stride;
    int n;
  } d[3] = {{t->stride_b, B}, {t->stride_h, H}, {t->stride_s, S}};
  for (const Dim& x : d) {
    if (x.n == 1) continue;  // the stride is never used
    if (x.stride < 0 || x.stride % 8 != 0)
      return fail(B200_EINVAL, "%s: strides of %s must be multiples of 8 elements, not negative",
                  who, name);
    if (x.stride >= (int64_t{1} << 39))
      return fail(B200_EUNSUPPORTED, "%s: a stride of %s is 2^39 elements or more", who, name);
  }
  if (S > 1 && t->stride_s == 0)
    return fail(B200_EINVAL, "%s: the tokens of %s may not share a row (stride 0)", who, name);
  if (!output) return B200_OK;
  std::sort(d, d + 3, [](const Dim& a, const Dim& b) { return a.stride < b.stride; });
  int64_t reach = D;
  for (const Dim& x : d) {
    if (x.n == 1) continue;
    if (x.stride < reach) return fail(B200_EINVAL, "%s: rows of output %s overlap", who, name);
    reach = x.stride * (x.n - 1) + reach;
  }
  return B200_OK;
}

b200_status check_workspace(const char* who, const void* ws, size_t have, size_t need) {
  if (need == 0) return B200_OK;
  if (!ws || !aligned16(ws))
    return fail(B200_EINVAL, "%s: needs a 16-byte aligned workspace of %zu bytes", who, need);
  if (have < need)
    return fail(B200_EINVAL, "%s: workspace of %zu bytes is too small; needs %zu", who, have, need);
  return B200_OK;
}

b200_status check_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? B200_OK : cuda_fail(e, what);
}

// Launch on `stream` a kernel that may start while its predecessor there still
// runs.  It waits (pdl_wait) before it touches memory that others use, so only
// its launch overlaps -- but for two kernels that run beside their predecessor
// (the gradients' query tiles, split_attention_kernel with `overlaps`).  Those
// read what the predecessor has waited for, and nothing that it writes: each
// relies on the kernel directly before it calling pdl_wait before
// pdl_launch_dependents.  Their last CTA ends after the predecessor has, so that
// what follows them follows both.  Measured back to back: one token's attention
// over 1024 keys 10.3 -> 7.9 us a call, three requests behind 517 keys 8.2 -> 6.4.
template <typename... P, typename... A>
b200_status launch_dependent(void (*kernel)(P...), unsigned grid, unsigned threads, size_t smem,
                             cudaStream_t stream, const char* what, A... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  return e == cudaSuccess ? B200_OK : cuda_fail(e, what);
}

size_t round16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

// ---- query/key norm with rotation ----
struct RopeArgs {
  b200::rope::Params p;
  bool per_row;     // few heads: a token to each row of a warp
  int groups_q, groups_k;  // row groups of a token
  int64_t token_groups;
};

b200_status rope_args(const char* who, const b200_tensor* q, const b200_tensor* k,
                      const void* q_weight, const void* k_weight, int weight_f32,
                      const float* inv_freq, int rotary_dim, int interleaved,
                      const int32_t* positions, int64_t position_stride_b, float eps, int B,
                      int S, int Hq, int Hkv, int D, bool backward, RopeArgs* out) {
  if (B < 1 || S < 1 || Hq < 1 || Hkv < 1)
    return fail(B200_EINVAL, "%s: invalid shape B=%d S=%d Hq=%d Hkv=%d", who, B, S, Hq, Hkv);
  if (D != 64 && D != 128)
    return fail(B200_EUNSUPPORTED, "%s: head_dim must be 64 or 128; got D=%d", who, D);
  if (static_cast<int64_t>(B) * S > (int64_t{1} << 30))
    return fail(B200_EUNSUPPORTED, "%s: more than 2^30 tokens", who);
  if (Hq > (1 << 20) || Hkv > (1 << 20))
    return fail(B200_EUNSUPPORTED, "%s: more than 2^20 heads", who);
  if (rotary_dim < 0 || rotary_dim > D || rotary_dim % 16 != 0)
    return fail(B200_EUNSUPPORTED, "%s: rotary_dim must be a multiple of 16 in [0, D]; got %d",
                who, rotary_dim);
  if (!q_weight || !k_weight) return fail(B200_EINVAL, "%s: null weight", who);
  if (!aligned16(q_weight) || !aligned16(k_weight))
    return fail(B200_EINVAL, "%s: weights must be 16-byte aligned", who);
  if (rotary_dim > 0 && (!inv_freq || !positions))
    return fail(B200_EINVAL, "%s: null inv_freq or positions", who);
  if (!(eps >= 0.0f) || !std::isfinite(eps))
    return fail(B200_EINVAL, "%s: eps must be finite and not negative", who);
  if (position_stride_b < 0)
    return fail(B200_EINVAL, "%s: negative position stride", who);
  b200_status st;
  if ((st = check_tensor(who, "q", q, B, Hq, S, D, false)) != B200_OK) return st;
  if ((st = check_tensor(who, "k", k, B, Hkv, S, D, false)) != B200_OK) return st;
  b200::rope::Params p{};
  p.q = view_of(q);
  p.k = view_of(k);
  p.wq = q_weight;
  p.wk = k_weight;
  p.w_f32 = weight_f32 ? 1 : 0;
  p.inv_freq = inv_freq;
  p.pos = positions;
  p.pos_sb = position_stride_b;
  p.tokens = static_cast<uint32_t>(B) * static_cast<uint32_t>(S);
  p.S = S;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.rot = rotary_dim;
  p.eps = eps;
  // Rows of a warp hold heads of one token, or a token each (per_row).  The
  // second leaves none empty, but each row forms its own angles and few tokens
  // fill few warps.  Measured (us, first / second form; tokens, heads x D),
  // forward: 2048, 1+1 x 128 4.3 / 3.7; 8192, 4+2 x 128 9.3 / 8.0; 4096, 4+2 x
  // 128 5.6 / 6.3; 16384, 8+8 x 128 25.3 / 25.0, 16+4 x 128 29.8 / 30.9, 16+16 x
  // 64 25.3 / 27.1.  Backward: 2048, 1+1 x 128 7.1 / 5.8; 4096, 16+4 x 128 17.7 /
  // 15.7; 2048, 4+2 x 128 7.3 / 7.0; 666, 10+5 x 64 5.6 / 8.4; 16384, 16+16 x 64
  // 38.2 / 40.8; 8192, 32+8 x 128 47.3 / 53.1.
  const int rows = 512 / D;
  RopeArgs a{p, false, (Hq + rows - 1) / rows, (Hkv + rows - 1) / rows, p.tokens};
  const bool half_empty =
      2ll * (Hq + Hkv) <= static_cast<long long>(a.groups_q + a.groups_k) * rows;
  a.per_row = half_empty ? p.tokens >= 2048
                         : Hq + Hkv <= (backward ? 24 : 16) &&
                               p.tokens >= (backward ? 4096u : 8192u);
  if (a.per_row) {
    a.groups_q = Hq;
    a.groups_k = Hkv;
    a.token_groups = (p.tokens + rows - 1) / rows;
  }
  *out = a;
  return B200_OK;
}

// f(head size, interleaved, per_row) with these as integral constants.
template <typename F>
b200_status rope_dispatch(int D, bool interleaved, bool per_row, F&& f) {
  using T = std::true_type;
  using N = std::false_type;
  auto by_row = [&](auto d, auto il) { return per_row ? f(d, il, T{}) : f(d, il, N{}); };
  auto by_pairs = [&](auto d) { return interleaved ? by_row(d, T{}) : by_row(d, N{}); };
  return D == 128 ? by_pairs(std::integral_constant<int, 128>{})
                  : by_pairs(std::integral_constant<int, 64>{});
}

// CTAs of the backward kernel for the queries and for the keys, by their rows.
struct RopeGrid {
  int q, k;
};

RopeGrid rope_bwd_grid(const RopeArgs& a) {
  const int64_t ctas = (a.token_groups + b200::rope::kWarps - 1) / b200::rope::kWarps;
  const int64_t most = static_cast<int64_t>(sm_count()) * b200::rope::kGradCtasPerSm;
  const int64_t k = std::max<int64_t>(1, most * a.groups_k / (a.groups_q + a.groups_k));
  return RopeGrid{static_cast<int>(std::min(ctas, most - k)), static_cast<int>(std::min(ctas, k))};
}

// ---- window and prefix attention ----
struct WindowShape {
  int B, Hq, Hkv, Sq, Skv, D, window, sinks;
  float scale;
};

b200_status window_shape(const char* who, int B, int Hq, int Hkv, int Sq, int Skv, int D,
                         int window, int sinks, float softmax_scale, WindowShape* out) {
  if (B < 1 || Hq < 1 || Hkv < 1 || Sq < 1 || Skv < 1)
    return fail(B200_EINVAL, "%s: invalid shape B=%d Hq=%d Hkv=%d Sq=%d Skv=%d", who, B, Hq, Hkv,
                Sq, Skv);
  if (Hq % Hkv != 0)
    return fail(B200_EINVAL, "%s: requires Hq %% Hkv == 0; got Hq=%d Hkv=%d", who, Hq, Hkv);
  if (D != 64 && D != 128)
    return fail(B200_EUNSUPPORTED, "%s: head_dim must be 64 or 128; got D=%d", who, D);
  if (window < 1 || sinks < 0)
    return fail(B200_EINVAL, "%s: window must be at least 1 and sinks at least 0; got %d and %d",
                who, window, sinks);
  if (Sq > (1 << 30) || Skv > (1 << 30) ||
      static_cast<int64_t>(Hq / Hkv) * Sq > (int64_t{1} << 30) ||
      static_cast<int64_t>(B) * Hq > (int64_t{1} << 30))
    return fail(B200_EUNSUPPORTED, "%s: a length, group * Sq or B * Hq above 2^30", who);
  const float scale = softmax_scale < 0.0f ? 1.0f / std::sqrt(static_cast<float>(D))
                                           : softmax_scale;
  if (!std::isfinite(scale)) return fail(B200_EINVAL, "%s: softmax_scale is not finite", who);
  // A window of Skv keys or more hides nothing.
  *out = WindowShape{B, Hq, Hkv, Sq, Skv, D, std::min(window, Skv), std::min(sinks, Skv), scale};
  return B200_OK;
}

// Splits of the keys of a row tile: two CTAs per SM, at least two blocks for
// each of a split's warps.  Up to kMaxCluster of them merge as a cluster; more
// go through a workspace and a second kernel, which pays from twice as many
// on.  Measured (us, second kernel / cluster of 8): 32 splits, B 1, 8 kv heads,
// 8192 keys: 12.7 / 17.6; 9 splits, B 4, 32768 keys: 87.8 / 81.7; 8 splits, B 4,
// 8192 keys: 27.1 / 26.1.  Units of few keys go one to a warp, without a merge
// (us, CTA / warp; D 128): 160 units of 16 keys 4.8 / 3.9, of 64: 5.5 / 6.0; 600 of
// 256: 20.2 / 18.9, of 512: 36.0 / 36.7; 4800 of 16: 58.9 / 16.3, of 128: 92 / 59.
struct SplitPlan {
  int nsplit;
  bool cluster;
  int units;  // not 0: this many units, one to a warp
};

SplitPlan split_plan(int64_t units, int64_t keys, bool partial) {
  namespace sp = b200::split;
  const int64_t want = 2 * static_cast<int64_t>(sm_count()) / std::max<int64_t>(units, 1);
  const int64_t most = keys / (2 * sp::kWarps * sp::kKeys);
  const int n =
      static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({want, most, sp::kMaxSplits})));
  if (partial || n >= 2 * sp::kMaxCluster) return SplitPlan{n, false, 0};
  const bool many = units >= 4 * static_cast<int64_t>(sm_count());
  if (n == 1 && units < (1 << 30) && keys <= (many ? 256 : 2 * sp::kKeys))
    return SplitPlan{1, true, static_cast<int>(units)};
  return SplitPlan{std::min(n, sp::kMaxCluster), true, 0};
}

int row_tiles_of(int64_t rows) {
  return static_cast<int>((rows + b200::split::kRows - 1) / b200::split::kRows);
}

// A 128-row tile of a window call: heads of one kv head x tokens.
struct WindowTile {
  int heads, tokens;
  int64_t key_tiles, items;  // tiles of 128 keys of an item, at most; items
};

// How a window call goes by 128-row tiles: splits of an item's keys, and the
// time of its work in us.
struct TilePlan {
  int nsplit;
  double us;
};

// Of the group's divisors the one with the least work: few tokens reach few keys
// beyond the window, but heads x tokens may fall short of 128.  A map cannot
// hold several heads of a broadcast axis (q null: it is none).
WindowTile window_tile(const WindowShape& s, const b200_tensor* q) {
  const int group = s.Hq / s.Hkv;
  const int most = q && s.Hq > 1 && q->stride_h == 0 ? 1 : std::min(group, b200::attn::kBM);
  const bool folded = s.sinks <= b200::attn::kFold;
  WindowTile best{};
  for (int heads = 1; heads <= most; ++heads) {
    if (group % heads != 0) continue;
    WindowTile t{heads, b200::attn::kBM / heads, 0, 0};
    const int64_t reach = static_cast<int64_t>(s.window) + std::min(t.tokens, s.Sq) - 1 +
                          (s.sinks > 0 && folded ? b200::attn::kFold : 0);
    t.key_tiles = (std::min<int64_t>(s.Skv, reach) + 127) / 128 +
                  (folded || reach >= s.Skv ? 0 : (s.sinks + 127) / 128);
    t.items = static_cast<int64_t>(s.B) * (s.Hq / heads) * ((s.Sq + t.tokens - 1) / t.tokens);
    auto work = [](const WindowTile& x) { return static_cast<double>(x.key_tiles) * x.items; };
    if (best.heads == 0 || work(t) < work(best)) best = t;
  }
  return best;
}

// A 128-row tile spends about 0.87 us on 128 keys, whatever its rows, and the
// kernel starts 1.5 us after the 16-row one.  (An item's start and end are not in
// this: one round of nine tiles is 9.3 us by it and 15.9 measured, with masked
// tiles, so that it ranks the kernels, and does not say their times.)  Where items
// leave SMs idle, their keys are split, four tiles at least to a split; the splits'
// sums and the kernel that merges them cost 4 us and their bytes.  Measured (us, whole /
// split; B 1, heads 32/8 of 128): 32768 keys, Sq 64: 227 / 43; 8192 keys, Sq 16:
// 61.0 / 16.2, 256: 62.8 / 43.9, 512: 64.9 / 65.5; window 2048, Sq 64: 22.4 / 16.7;
// window 1024, Sq 128: 15.9 / 17.2.
TilePlan tile_plan(const WindowShape& s) {
  const WindowTile t = window_tile(s, nullptr);
  const int64_t sms = sm_count();
  const double rows = static_cast<double>(s.B) * s.Hq * s.Sq;
  const double rounds = static_cast<double>((t.items + sms - 1) / sms);
  TilePlan best{1, 0.87 * rounds * static_cast<double>(t.key_tiles) + 1.5};
  const int64_t ns = std::min<int64_t>({sms / t.items, t.key_tiles / 4, b200::split::kMaxSplits});
  if (ns < 2) return best;
  const double us = 0.87 * static_cast<double>((t.key_tiles + ns - 1) / ns) + 5.5 +
                    8.0 * rows * static_cast<double>(ns) * s.D / 6.4e6;
  return us < best.us ? TilePlan{static_cast<int>(ns), us} : best;
}

// Whether a window call goes by 128-row tiles: by the time of each kernel's
// work, neither below its bytes'.  The 16-row kernel does 16,500 (D 64: 21,500)
// keys x units a us with the GPU full; it splits the keys, so that few rows fill
// the GPU.  Measured (us, 16-row / 128-row; heads 32/8 of 128): B 1, window 1024,
// Sq 32: 12.5 / 15.5, 64: 16.7 / 15.7, 128: 22.8 / 15.9; B 8, 8192 keys, Sq 4:
// 46.3 / 62.4, 8: 70.5 / 62.7, 16: 128 / 62.7; B 16, window 128, Sq 8: 8.4 / 10.5,
// 16: 14.9 / 10.5; D 64, B 8, window 1024, Sq 8: 13.1 / 14.7, 16: 16.7 / 15.0;
// B 64, heads 64/8, window 4096, Sq 2: 158 / 177, 4: 267 / 178.
bool window_by_tiles(const WindowShape& s, const TilePlan& t) {
  const int64_t rows = static_cast<int64_t>(s.Hq / s.Hkv) * s.Sq;
  const double keys = static_cast<double>(
      std::min<int64_t>(s.Skv, static_cast<int64_t>(s.window) + s.sinks));
  const double heads = static_cast<double>(s.B) * s.Hkv;
  const double bytes_us = 4.0 * heads * keys * s.D / 6.4e6;
  const double split_us = heads * row_tiles_of(rows) * keys / (s.D == 128 ? 16500.0 : 21500.0);
  return std::max(split_us, bytes_us) > std::max(t.us, bytes_us);
}

size_t part_bytes(int64_t rows, int D) {
  return round16(static_cast<size_t>(rows) * D * sizeof(float)) +
         round16(static_cast<size_t>(rows) * sizeof(float2));
}

struct WindowPlan {
  bool tiles;   // 128-row tiles (tcgen05); else 16-row tiles that split the keys
  int nsplit;
  size_t bytes;  // of the splits' partial sums; 0: a cluster merges them
  int units;     // as SplitPlan
};

size_t split_bytes(int64_t rows, const SplitPlan& p, int D) {
  return p.cluster ? 0 : part_bytes(rows * p.nsplit, D);
}

WindowPlan window_plan(const WindowShape& s) {
  const int64_t rows = static_cast<int64_t>(s.Hq / s.Hkv) * s.Sq;
  const int64_t heads = static_cast<int64_t>(s.B) * s.Hkv;
  const TilePlan t = tile_plan(s);
  if (window_by_tiles(s, t))
    return WindowPlan{true, t.nsplit,
                      t.nsplit > 1 ? part_bytes(heads * rows * t.nsplit, s.D) : 0, 0};
  const int64_t keys = std::min<int64_t>(s.Skv, static_cast<int64_t>(s.window) + s.sinks);
  const SplitPlan p = split_plan(heads * row_tiles_of(rows), keys, false);
  return WindowPlan{false, p.nsplit, split_bytes(heads * rows, p, s.D), p.units};
}

template <int D>
b200_status launch_split(const b200::split::Params& p, cudaStream_t stream) {
  using C = b200::split::Cfg<D>;
  static unsigned attr_done = 0;
  auto kernel = b200::split::split_attention_kernel<D>;
  const b200_status st = ensure_smem_attr(kernel, C::kSmemBytes, &attr_done);
  if (st != B200_OK) return st;
  const int64_t grid =
      p.units ? (p.units + b200::split::kWarps - 1) / b200::split::kWarps
              : static_cast<int64_t>(p.B) * p.Hkv * p.row_tiles * p.nsplit;
  if (grid > 0x7fffffffll) return fail(B200_EUNSUPPORTED, "attention: too many work units");
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(p.nsplit);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(b200::split::kThreads, 1, 1);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = !p.part_o && p.nsplit > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  return e == cudaSuccess ? B200_OK : cuda_fail(e, "split attention launch");
}

b200_status launch_combine(const b200::split::CombineParams& p, int D, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(p.B) * p.Hkv * p.rows;
  const int64_t grid = (rows + 3) / 4;
  if (grid > 0x7fffffffll) return fail(B200_EUNSUPPORTED, "attention: too many rows");
  return launch_dependent(
      D == 128 ? b200::split::combine_kernel<128> : b200::split::combine_kernel<64>,
      static_cast<unsigned>(grid), 128, 0, stream, "combine launch", p);
}

b200::split::Params split_params(const WindowShape& s, const b200_tensor* q, const b200_tensor* k,
                                 const b200_tensor* v, const b200_tensor* o,
                                 const int32_t* kv_len, int nsplit, int units) {
  b200::split::Params p{};
  p.units = units;
  p.q = view_of(q);
  p.k = view_of(k);
  p.v = view_of(v);
  p.o = view_of(o);
  p.kv_len = kv_len;
  p.B = s.B;
  p.Hkv = s.Hkv;
  p.group = s.Hq / s.Hkv;
  p.Sq = s.Sq;
  p.Skv = s.Skv;
  p.rows = p.group * s.Sq;
  p.row_tiles = row_tiles_of(p.rows);
  p.nsplit = nsplit;
  p.window = s.window;
  p.sinks = s.sinks;
  p.scale_log2 = s.scale * 1.4426950408889634f;
  return p;
}

// Partial sums of `rows` rows at `ws`: O, then (m, l).
void part_pointers(void* ws, int64_t rows, int D, float** o, float2** ml) {
  *o = static_cast<float*>(ws);
  *ml = reinterpret_cast<float2*>(static_cast<unsigned char*>(ws) +
                                  round16(static_cast<size_t>(rows) * D * sizeof(float)));
}

b200_status check_qkvo(const char* who, const WindowShape& s, const b200_tensor* q,
                       const b200_tensor* k, const b200_tensor* v, const b200_tensor* o) {
  b200_status st;
  if ((st = check_tensor(who, "q", q, s.B, s.Hq, s.Sq, s.D, false)) != B200_OK) return st;
  if ((st = check_tensor(who, "k", k, s.B, s.Hkv, s.Skv, s.D, false)) != B200_OK) return st;
  if ((st = check_tensor(who, "v", v, s.B, s.Hkv, s.Skv, s.D, false)) != B200_OK) return st;
  return check_tensor(who, "o", o, s.B, s.Hq, s.Sq, s.D, true);
}

// ---- the tiled (tcgen05) forms ----
// Map of a [B, H, S, D] tensor with boxes of `rows` tokens.  An axis that is
// broadcast (stride 0) gets extent 1, and its coordinate the factor 0.
b200_status encode_view(CUtensorMap* map, const b200_tensor* t, int B, int H, int S, int D,
                        uint32_t rows, int* mul_b, int* mul_h) {
  const bool wide_b = B > 1 && t->stride_b != 0, wide_h = H > 1 && t->stride_h != 0;
  *mul_b = wide_b;
  *mul_h = wide_h;
  const cuuint64_t any = static_cast<cuuint64_t>(D) * 2;  // stride of an axis of extent 1
  const cuuint64_t d[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(S),
                           static_cast<cuuint64_t>(wide_h ? H : 1),
                           static_cast<cuuint64_t>(wide_b ? B : 1)};
  const cuuint64_t s[3] = {S > 1 ? static_cast<cuuint64_t>(t->stride_s) * 2 : any,
                           wide_h ? static_cast<cuuint64_t>(t->stride_h) * 2 : any,
                           wide_b ? static_cast<cuuint64_t>(t->stride_b) * 2 : any};
  const cuuint32_t box[4] = {64, rows, 1, 1};
  return encode_bf16_4d(map, t->data, d, s, box);
}

// Map of the queries' tensor with boxes of heads x tokens rows, heads innermost.
// An axis that is broadcast as in encode_view; heads is 1 where that one is.
b200_status encode_rows(CUtensorMap* map, const b200_tensor* t, int B, int H, int S, int D,
                        int heads, int tokens, int* mul_b, int* mul_h) {
  const bool wide_b = B > 1 && t->stride_b != 0, wide_h = H > 1 && t->stride_h != 0;
  *mul_b = wide_b;
  *mul_h = wide_h;
  const cuuint64_t any = static_cast<cuuint64_t>(D) * 2;  // stride of an axis of extent 1
  const cuuint64_t d[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(wide_h ? H : 1),
                           static_cast<cuuint64_t>(S), static_cast<cuuint64_t>(wide_b ? B : 1)};
  const cuuint64_t s[3] = {wide_h ? static_cast<cuuint64_t>(t->stride_h) * 2 : any,
                           S > 1 ? static_cast<cuuint64_t>(t->stride_s) * 2 : any,
                           wide_b ? static_cast<cuuint64_t>(t->stride_b) * 2 : any};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(heads), static_cast<cuuint32_t>(tokens),
                             1};
  return encode_bf16_4d(map, t->data, d, s, box);
}

template <int D, int kForm>
b200_status launch_tiles(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm,
                         const CUtensorMap& om, b200::attn::Params p, long long items, int sms,
                         cudaStream_t stream, const b200::attn::FoldOf<kForm>& fold) {
  using C = b200::attn::Cfg<D>;
  static unsigned attr_done = 0;
  auto kernel = b200::attn::attention_fwd_kernel<D, D == 128 ? kDefaultEmuD128 : kDefaultEmuD64,
                                                 false, false, kForm>;
  const b200_status st = ensure_smem_attr(kernel, C::kSmemBytes, &attr_done);
  if (st != B200_OK) return st;
  static const int launch_regs = [kernel] {
    cudaFuncAttributes a{};
    return cudaFuncGetAttributes(&a, kernel) == cudaSuccess ? a.numRegs : -1;
  }();
  if (launch_regs != b200::attn::kLaunchRegs)
    return fail(B200_EUNSUPPORTED,
                "attention: kernel has %d registers per thread at launch; its register split "
                "needs exactly %d",
                launch_regs, b200::attn::kLaunchRegs);
  if (items > 0x3fffffffll) return fail(B200_EUNSUPPORTED, "attention: too many work items");
  p.n_items = static_cast<int>(items);
  const int grid = static_cast<int>(std::min<long long>(items, sms));
  return launch_dependent(kernel, static_cast<unsigned>(grid), b200::attn::kThreads,
                          C::kSmemBytes, stream, "attention tiles launch", qm, km, vm, om, p,
                          fold);
}

b200::attn::Params tile_params(const WindowShape& s) {
  b200::attn::Params p{};
  p.B = s.B;
  p.Hq = s.Hq;
  p.Hkv = s.Hkv;
  p.Sq = s.Sq;
  p.Skv = s.Skv;
  p.group = s.Hq / s.Hkv;
  p.nsplit = 1;
  p.scale_log2 = s.scale * 1.4426950408889634f;
  return p;
}

template <int D>
b200_status launch_window_tiles(const WindowShape& s, const b200_tensor* q, const b200_tensor* k,
                                const b200_tensor* v, const b200_tensor* o, float* lse,
                                const int32_t* kv_len, int nsplit, float* part_o, float2* part_ml,
                                cudaStream_t stream) {
  b200::attn::Params p = tile_params(s);
  p.nsplit = nsplit;
  p.rows = p.group * s.Sq;
  p.ws_o = part_o;
  p.ws_ml = part_ml;
  CUtensorMap qm, km, vm, om;
  int one;
  b200_status st;
  const WindowTile t = window_tile(s, q);
  p.tile_heads = t.heads;
  p.tile_tokens = t.tokens;
  b200::attn::FoldMaps fold;
  constexpr uint32_t kKeys = b200::attn::kBN, kFold = b200::attn::kFold;
  if ((st = encode_rows(&qm, q, s.B, s.Hq, s.Sq, D, t.heads, t.tokens, &p.q_mb, &p.q_mh)) !=
          B200_OK ||
      (st = encode_rows(&om, o, s.B, s.Hq, s.Sq, D, t.heads, t.tokens, &one, &one)) != B200_OK ||
      (st = encode_view(&km, k, s.B, s.Hkv, s.Skv, D, kKeys, &p.k_mb, &p.k_mh)) != B200_OK ||
      (st = encode_view(&vm, v, s.B, s.Hkv, s.Skv, D, kKeys, &p.v_mb, &p.v_mh)) != B200_OK)
    return st;
  fold.k_sinks = fold.k_rest = km;  // not used without sinks
  fold.v_sinks = fold.v_rest = vm;
  if (s.sinks > 0 && s.sinks <= static_cast<int>(kFold)) {
    const CUtensorMap* const maps[2][2] = {{&fold.k_sinks, &fold.k_rest},
                                           {&fold.v_sinks, &fold.v_rest}};
    for (int i = 0; i < 4; ++i)
      if ((st = encode_view(const_cast<CUtensorMap*>(maps[i / 2][i % 2]), i < 2 ? k : v, s.B,
                            s.Hkv, s.Skv, D, i % 2 ? kKeys - kFold : kFold, &one, &one)) != B200_OK)
        return st;
  }
  p.n_qtiles = (s.Sq + t.tokens - 1) / t.tokens;
  p.causal = 1;  // the order of the items, as causal attention's
  // Hidden scores are -inf before the scale: a scale of 0 becomes one that
  // changes no weight of scores below 1e30.
  if (p.scale_log2 == 0.0f) p.scale_log2 = 1e-37f;
  p.window = s.window;
  p.sinks = s.sinks;
  p.kv_len = kv_len;
  p.lse = lse;
  const long long planes = static_cast<long long>(s.B) * (s.Hq / t.heads);
  // Planes of an ordering group: their K/V in use fit in half of the L2 (as
  // for causal attention).
  const double keys = std::min<double>(s.Skv, static_cast<double>(s.window) + b200::attn::kBM);
  const long long g =
      static_cast<long long>(64.0 * (1 << 20) / (4.0 * keys * D)) * (p.group / t.heads);
  p.cgroup = static_cast<int>(std::max<long long>(1, std::min<long long>(g, planes)));
  const long long items = planes * p.n_qtiles * nsplit;
  return nsplit > 1 ? launch_tiles<D, b200::attn::kWindowSplit>(qm, km, vm, om, p, items,
                                                                sm_count(), stream, fold)
                    : launch_tiles<D, b200::attn::kWindow>(qm, km, vm, om, p, items, sm_count(),
                                                           stream, fold);
}

// ---- window attention's gradients ----
struct WindowGrads {
  const b200_tensor *dout, *q, *k, *v, *o, *dq, *dk, *dv;
  const float* lse;
  const int32_t* kv_len;
};

int64_t padded_queries(int Sq) { return (static_cast<int64_t>(Sq) + 63) / 64 * 64; }

// How the steps of the gradients' first key tiles are divided among CTAs (their
// fp32 sums cost 2 x 128 x D floats each): those of the tiles that hold sinks,
// into parts of half of an SM's share of the launch or of a window, or those of
// all tiles, where they are few; up to 8.  What is left is the longest chain of
// steps or an SM's share, and, if divided, about 4 steps' time for the sums'
// kernel.  Measured (us, undivided / divided): heads 32/8 of 128, 4096 queries,
// window 100, 4 sinks 353 / 154 (sinks); heads 8/1 of 128, causal, 128 queries
// 26.8 / 23.9, 512: 69.8 / 24.0, 4000: 470 / 134 (all); heads 8/2 of 128, 2000
// queries, window 256, 4 sinks: 40.2 (sinks) or 51.9 (all).
struct PartPlan {
  int tiles, parts;  // parts 0: not divided
};

PartPlan part_plan(const WindowShape& s) {
  const int64_t group = s.Hq / s.Hkv, heads = static_cast<int64_t>(s.B) * s.Hkv;
  const int64_t sinks = (std::min(s.sinks, s.Skv) + 127) / 128, all = (s.Skv + 127) / 128;
  const int64_t most = group * ((s.Sq + 63) / 64);  // steps of a tile that all queries see
  const int64_t window = std::min(most, group * ((static_cast<int64_t>(s.window) + 127 + 63) / 64));
  const int64_t sms = sm_count();
  const double steps = static_cast<double>(heads) * (static_cast<double>(sinks) * most +
                                                     static_cast<double>(all - sinks) * window);
  const int64_t share = static_cast<int64_t>(std::min(steps / sms, 1e15));
  auto cost = [&](int64_t tiles, int64_t parts) {
    const int64_t rest = tiles < all ? window : 0, longest = tiles > 0 && sinks > 0 ? most : window;
    const int64_t waves = tiles < all ? 1 : (heads * tiles * parts + sms - 1) / sms;
    const int64_t chain = waves * ((longest + parts - 1) / parts + 3);  // 3: a CTA's start
    return static_cast<double>(std::max({chain, rest, share})) + 4.0 +
           0.04 * static_cast<double>(heads * tiles * parts);
  };
  PartPlan best{0, 0};
  double least = static_cast<double>(std::max(sinks > 0 ? most : window, share));
  auto consider = [&](int64_t tiles, int64_t parts) {
    if (tiles == 0 || parts < 2 || cost(tiles, parts) >= least) return;
    least = cost(tiles, parts);
    best = PartPlan{static_cast<int>(tiles), static_cast<int>(parts)};
  };
  const int64_t size = std::max<int64_t>(std::max(window, share / 2), 1);
  consider(sinks, std::min<int64_t>(8, (most + size - 1) / size));
  for (int64_t waves = 1; waves <= 2; ++waves)
    consider(all, std::min<int64_t>({8, waves * sms / (heads * all),
                                     (sinks > 0 ? most : window) / 6}));
  return best;
}

size_t window_stat_bytes(const WindowShape& s) {
  return static_cast<size_t>(s.B) * s.Hq * padded_queries(s.Sq) * 2 * sizeof(float);
}

size_t window_bwd_bytes(const WindowShape& s) {
  const PartPlan k = part_plan(s);
  return window_stat_bytes(s) + static_cast<size_t>(s.B) * s.Hkv * k.tiles * k.parts * 2 *
                                    b200::bwd::kOwn * s.D * sizeof(float);
}

template <int D, bool kKeys>
b200_status launch_bwd_tiles(const CUtensorMap (&m)[4], b200::bwd::TileParams p, int heads,
                             int rows, cudaStream_t stream) {
  using C = b200::bwd::TileCfg<D, kKeys>;
  static unsigned attr_done = 0;
  auto kernel = b200::bwd::bwd_tile_kernel<D, kKeys>;
  const b200_status st = ensure_smem_attr(kernel, C::kSmemBytes, &attr_done);
  if (st != B200_OK) return st;
  p.tiles = (rows + b200::bwd::kOwn - 1) / b200::bwd::kOwn;
  int64_t items = static_cast<int64_t>(p.B) * heads * p.tiles;
  if (kKeys && p.parts > 0)
    items += static_cast<int64_t>(p.B) * heads * p.part_tiles * (p.parts - 1);
  if (items > 0x3fffffffll) return fail(B200_EUNSUPPORTED, "attention_window_bwd: too many tiles");
  p.n_items = static_cast<int>(items);
  // Key tiles differ in length (sinks): a CTA each, so that the next one starts
  // where one ends.  Query tiles are alike: persistent CTAs.
  const unsigned grid = static_cast<unsigned>(kKeys ? items : std::min<int64_t>(items, sm_count()));
  return launch_dependent(kernel, grid, C::kThreads, C::kSmemBytes, stream,
                          "attention_window_bwd launch", m[0], m[1], m[2], m[3], p);
}

template <int D>
b200_status window_bwd_tiles(const WindowShape& s, const WindowGrads& t, void* workspace,
                             cudaStream_t stream) {
  b200::bwd::TileParams p{};
  p.sq_pad = static_cast<int>(padded_queries(s.Sq));
  p.stat_plane = static_cast<int64_t>(s.B) * s.Hq * p.sq_pad;
  float* stats = static_cast<float*>(workspace);
  p.stats = stats;
  p.kv_len = t.kv_len;
  p.B = s.B;
  p.Hq = s.Hq;
  p.Hkv = s.Hkv;
  p.group = s.Hq / s.Hkv;
  p.Sq = s.Sq;
  p.Skv = s.Skv;
  p.window = s.window;
  p.sinks = s.sinks;
  p.scale = s.scale;
  p.scale_log2 = s.scale * 1.4426950408889634f;
  // [0]: 128-row boxes, [1]: 64-row boxes of the queries' tensors.
  CUtensorMap q[2], dout[2], k, v;
  int q_b, q_h, do_b, do_h, k_b, k_h, v_b, v_h;
  b200_status st;
  for (int i = 0; i < 2; ++i) {
    const uint32_t rows = i ? 64 : 128;
    if ((st = encode_view(&q[i], t.q, s.B, s.Hq, s.Sq, D, rows, &q_b, &q_h)) != B200_OK ||
        (st = encode_view(&dout[i], t.dout, s.B, s.Hq, s.Sq, D, rows, &do_b, &do_h)) != B200_OK)
      return st;
  }
  if ((st = encode_view(&k, t.k, s.B, s.Hkv, s.Skv, D, 128, &k_b, &k_h)) != B200_OK ||
      (st = encode_view(&v, t.v, s.B, s.Hkv, s.Skv, D, 128, &v_b, &v_h)) != B200_OK)
    return st;
  const int64_t blocks = p.stat_plane / b200::bwd::kStatRows;
  if (blocks > 0x7fffffffll)
    return fail(B200_EUNSUPPORTED, "attention_window_bwd: too many query rows");
  b200::bwd::stats_kernel<D><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(
      view_of(t.dout), view_of(t.o), t.lse, stats, p.stat_plane, p.sq_pad, s.B, s.Hq, s.Sq);
  if ((st = check_launch("attention_window_bwd statistics")) != B200_OK) return st;
  const PartPlan plan = part_plan(s);
  p.part_tiles = plan.tiles;
  p.parts = plan.parts;
  p.part_sums = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) +
                                         window_stat_bytes(s));
  p.out1 = view_of(t.dk);
  p.out2 = view_of(t.dv);
  p.o1_b = k_b, p.o1_h = k_h, p.o2_b = v_b, p.o2_h = v_h;
  p.s1_b = q_b, p.s1_h = q_h, p.s2_b = do_b, p.s2_h = do_h;
  if ((st = launch_bwd_tiles<D, true>({k, v, q[1], dout[1]}, p, s.Hkv, s.Skv, stream)) != B200_OK)
    return st;
  // Beside the keys' kernel (see launch_dependent): nothing may stand between
  // the two, and this one reads nothing that that one writes.
  p.out1 = p.out2 = view_of(t.dq);
  p.o1_b = q_b, p.o1_h = q_h, p.o2_b = do_b, p.o2_h = do_h;
  p.s1_b = k_b, p.s1_h = k_h, p.s2_b = v_b, p.s2_h = v_h;
  if ((st = launch_bwd_tiles<D, false>({q[0], dout[0], k, v}, p, s.Hq, s.Sq, stream)) != B200_OK)
    return st;
  if (plan.parts == 0) return B200_OK;
  p.out1 = view_of(t.dk);
  p.out2 = view_of(t.dv);
  const int64_t sums = static_cast<int64_t>(s.B) * s.Hkv * plan.tiles * 2 * b200::bwd::kOwn * D / 4;
  b200::bwd::part_sum_kernel<D><<<static_cast<unsigned>((sums + 255) / 256), 256, 0, stream>>>(p);
  return check_launch("attention_window_bwd sums");
}

// Work of the 16-row kernel behind a shared prefix, in us at the rate it was
// measured at with the GPU full (keys x units per us; a unit is a 16-row tile of
// one kv head).
double split_us(int64_t units, int64_t keys, int D) {
  return static_cast<double>(units) * static_cast<double>(keys) / (D == 128 ? 23400.0 : 36400.0);
}

// Tiles of the prefix form: whole batches, up to 128 rows.
struct PrefixTiles {
  int batches, rows, count;  // of a tile; tiles
};

PrefixTiles prefix_tiles(const WindowShape& own) {
  const int rows = own.Hq / own.Hkv * own.Sq;  // of a batch
  const int nb = std::min(own.B, b200::attn::kBM / rows);
  return PrefixTiles{nb, nb * rows, (own.B + nb - 1) / nb};
}

template <int D>
b200_status launch_prefix_tiles(const WindowShape& own, int P, const b200_tensor* q,
                                const b200_tensor* k, const b200_tensor* v, int nsplit, int sms,
                                float* part_o, float2* part_ml, cudaStream_t stream) {
  WindowShape shared = own;
  shared.Skv = P;
  b200::attn::Params p = tile_params(shared);
  const PrefixTiles t = prefix_tiles(own);
  p.n_qtiles = t.count;
  p.tile_batches = t.batches;
  p.tile_rows = t.rows;
  p.rows = own.B * p.group * own.Sq;
  p.nsplit = nsplit;
  p.ws_o = part_o;
  p.ws_ml = part_ml;
  CUtensorMap qm, km, vm;
  b200_status st;
  const cuuint64_t any = static_cast<cuuint64_t>(D) * 2;
  auto stride = [&](int n, int64_t x) { return n > 1 ? static_cast<cuuint64_t>(x) * 2 : any; };
  const cuuint64_t d[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(own.Hq),
                           static_cast<cuuint64_t>(own.Sq), static_cast<cuuint64_t>(own.B)};
  const cuuint64_t str[3] = {stride(own.Hq, q->stride_h), stride(own.Sq, q->stride_s),
                             stride(own.B, q->stride_b)};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(p.group),
                             static_cast<cuuint32_t>(own.Sq), static_cast<cuuint32_t>(t.batches)};
  if ((st = encode_bf16_4d(&qm, q->data, d, str, box)) != B200_OK) return st;
  constexpr uint32_t kKeys = b200::attn::kBN;
  if ((st = encode_view(&km, k, 1, own.Hkv, P, D, kKeys, &p.k_mb, &p.k_mh)) != B200_OK ||
      (st = encode_view(&vm, v, 1, own.Hkv, P, D, kKeys, &p.v_mb, &p.v_mh)) != B200_OK)
    return st;
  return launch_tiles<D, b200::attn::kPrefix>(
      qm, km, vm, qm, p, static_cast<long long>(own.Hkv) * t.count * nsplit, sms, stream, {});
}

// A shared prefix: by 128-row tiles for the whole batch, beside the requests'
// own keys by 16-row tiles, and combined; or all by 16-row tiles, each request
// reading the prefix.
struct PrefixPlan {
  bool tiles;
  int prefix_splits;  // tiles: of the prefix
  int prefix_sms;     // tiles: SMs that they take
  int own_splits;     // of the requests' keys (not tiles: after the prefix)
  int own_units;      // as SplitPlan
  size_t prefix_bytes, own_bytes;
};

// The second form starts one kernel instead of three, and reads the prefix
// (from L2) for each request: it is chosen up to 6 us more work.  Measured (us,
// tiles / 16-row, 128 own keys): heads 32/8, P 512, B 2: 14.0 / 6.7, B 64: 23.3 /
// 26.0; P 2048, B 8: 16.2 / 14.3, B 16: 17.3 / 21.1; P 32768, B 2: 35.0 / 34.6,
// B 4: 35.6 / 62.5; D 64, P 8192, B 4: 17.8 / 15.8, B 8: 18.0 / 24.8.  A tile
// holds whole requests, and the queries' map cannot broadcast; q's strides
// decide that (null: they do not).  So requests of more than 128 rows (heads of a
// kv head x tokens: prompts) go by 16-row tiles, however long the prefix.
PrefixPlan prefix_plan(const WindowShape& own, int P, const b200_tensor* q) {
  const int64_t rows = static_cast<int64_t>(own.Hq / own.Hkv) * own.Sq;
  const int64_t heads = static_cast<int64_t>(own.B) * own.Hkv;
  const int64_t units = heads * row_tiles_of(rows);
  PrefixPlan p{};
  bool tiles = P > 0 && rows <= b200::attn::kBM &&
               !(q && ((own.B > 1 && q->stride_b == 0) || (own.Hq > 1 && q->stride_h == 0)));
  if (tiles) {
    // Least rounds x (tiles of K/V per unit + a unit's fixed cost of about 3);
    // a tile takes about 1 us.
    const int64_t items = static_cast<int64_t>(own.Hkv) * prefix_tiles(own).count;
    const int64_t kv = (P + b200::attn::kBN - 1) / b200::attn::kBN;
    // Where the requests' own keys are long (4 us at the memory's rate), they
    // stream through three tenths of the SMs beside the tiles: one share for all,
    // not the best of each.  Measured (us; 0 / 20 / 44 / 74 SMs left): 64 requests,
    // heads 64/8, P 16384, up to 1024 keys: 67.9 / 68.1 / 66.3 / 66.5; P 4096:
    // 52.7 / 52.6 / 49.7 / 45.9; 32 requests, P 16384, up to 512: 40.3 / 39.8 /
    // 34.9 / 40.5.
    const double own_us = 4.0 * own.B * own.Hkv * static_cast<double>(own.Skv) * own.D / 6.4e6;
    int64_t sms = sm_count();
    if (own_us > 4.0) sms = std::max<int64_t>(1, sms * 7 / 10);
    p.prefix_sms = static_cast<int>(sms);
    int64_t best = INT64_MAX;
    for (int ns = 1; ns <= std::min<int64_t>(kv, b200::split::kMaxSplits); ++ns) {
      const int64_t cost = (items * ns + sms - 1) / sms * ((kv + ns - 1) / ns + 3);
      if (cost < best) {
        best = cost;
        p.prefix_splits = ns;
      }
    }
    tiles = split_us(units, static_cast<int64_t>(P) + own.Skv, own.D) >
            static_cast<double>(best) + split_us(units, own.Skv, own.D) + 6.0;
  }
  p.tiles = tiles;
  if (tiles) {
    const SplitPlan o = split_plan(units, own.Skv, true);
    p.own_splits = o.nsplit;
    p.own_bytes = split_bytes(heads * rows, o, own.D);
    p.prefix_bytes = part_bytes(heads * rows * p.prefix_splits, own.D);
  } else {
    const SplitPlan o = split_plan(units, static_cast<int64_t>(P) + own.Skv, false);
    p.own_splits = o.nsplit;
    p.own_units = o.units;
    p.own_bytes = split_bytes(heads * rows, o, own.D);
    p.prefix_bytes = 0;
  }
  return p;
}

b200_status prefix_shape(const char* who, int B, int Hq, int Hkv, int Sq, int P, int S, int D,
                         float softmax_scale, WindowShape* out) {
  if (P < 0 || P > (1 << 30))
    return fail(B200_EINVAL, "%s: prefix length %d is not in [0, 2^30]", who, P);
  const b200_status st = window_shape(who, B, Hq, Hkv, Sq, S, D, 1 << 30, 0, softmax_scale, out);
  if (st != B200_OK) return st;
  if (static_cast<int64_t>(B) * (Hq / Hkv) * Sq > (int64_t{1} << 30))
    return fail(B200_EUNSUPPORTED, "%s: B * group * Sq above 2^30", who);
  return B200_OK;
}

}  // namespace

extern "C" {

b200_status qk_norm_rope(const b200_tensor* q, const b200_tensor* k, const void* q_weight,
                         const void* k_weight, int weight_f32, const float* inv_freq,
                         int rotary_dim, int interleaved, const int32_t* positions,
                         int64_t position_stride_b, float eps, const b200_tensor* q_out,
                         const b200_tensor* k_out, int B, int S, int Hq, int Hkv, int D,
                         b200_stream_t stream) {
  const char* who = "qk_norm_rope";
  RopeArgs a;
  b200_status st = rope_args(who, q, k, q_weight, k_weight, weight_f32, inv_freq, rotary_dim,
                             interleaved, positions, position_stride_b, eps, B, S, Hq, Hkv, D, false,
                             &a);
  if (st != B200_OK) return st;
  if ((st = check_tensor(who, "q_out", q_out, B, Hq, S, D, true)) != B200_OK) return st;
  if ((st = check_tensor(who, "k_out", k_out, B, Hkv, S, D, true)) != B200_OK) return st;
  a.p.qy = view_of(q_out);
  a.p.ky = view_of(k_out);
  // Slices of a token's heads, so that few tokens still give every SM 24 warps.
  const int groups = a.groups_q + a.groups_k;
  const int64_t warps = static_cast<int64_t>(sm_count()) * 24;
  a.p.slice_groups = static_cast<int>(
      std::min<int64_t>(groups, (groups * a.token_groups + warps - 1) / warps));
  a.p.slices = (groups + a.p.slice_groups - 1) / a.p.slice_groups;
  const int64_t grid =
      (a.token_groups * a.p.slices + b200::rope::kWarps - 1) / b200::rope::kWarps;
  return rope_dispatch(D, interleaved != 0, a.per_row, [&](auto d, auto il, auto per_row) {
    return launch_dependent(b200::rope::norm_rope_kernel<decltype(d)::value, decltype(il)::value,
                                                         decltype(per_row)::value>,
                            static_cast<unsigned>(grid), b200::rope::kThreads, 0,
                            reinterpret_cast<cudaStream_t>(stream), "qk_norm_rope launch", a.p);
  });
}

b200_status qk_norm_rope_bwd_workspace(int B, int S, int D, size_t* bytes) {
  const char* who = "qk_norm_rope_bwd_workspace";
  if (!bytes) return fail(B200_EINVAL, "%s: null result", who);
  if (B < 1 || S < 1) return fail(B200_EINVAL, "%s: invalid shape B=%d S=%d", who, B, S);
  if (D != 64 && D != 128)
    return fail(B200_EUNSUPPORTED, "%s: head_dim must be 64 or 128; got D=%d", who, D);
  // The grid never exceeds its CTAs per SM, whatever the shape.
  *bytes = static_cast<size_t>(sm_count()) * b200::rope::kGradCtasPerSm * D * sizeof(float);
  return B200_OK;
}

b200_status qk_norm_rope_bwd(const b200_tensor* dq_out, const b200_tensor* dk_out,
                             const b200_tensor* q, const b200_tensor* k, const void* q_weight,
                             const void* k_weight, int weight_f32, const float* inv_freq,
                             int rotary_dim, int interleaved, const int32_t* positions,
                             int64_t position_stride_b, float eps, const b200_tensor* dq,
                             const b200_tensor* dk, float* dq_weight, float* dk_weight, int B,
                             int S, int Hq, int Hkv, int D, void* workspace,
                             size_t workspace_bytes, b200_stream_t stream) {
  const char* who = "qk_norm_rope_bwd";
  RopeArgs a;
  b200_status st = rope_args(who, q, k, q_weight, k_weight, weight_f32, inv_freq, rotary_dim,
                             interleaved, positions, position_stride_b, eps, B, S, Hq, Hkv, D, true,
                             &a);
  if (st != B200_OK) return st;
  if ((st = check_tensor(who, "dq_out", dq_out, B, Hq, S, D, false)) != B200_OK) return st;
  if ((st = check_tensor(who, "dk_out", dk_out, B, Hkv, S, D, false)) != B200_OK) return st;
  if ((st = check_tensor(who, "dq", dq, B, Hq, S, D, true)) != B200_OK) return st;
  if ((st = check_tensor(who, "dk", dk, B, Hkv, S, D, true)) != B200_OK) return st;
  if (!dq_weight || !dk_weight) return fail(B200_EINVAL, "%s: null weight gradient", who);
  const RopeGrid ctas = rope_bwd_grid(a);
  const int grid = ctas.q + ctas.k;
  a.p.ctas_q = ctas.q;
  if ((st = check_workspace(who, workspace, workspace_bytes,
                            static_cast<size_t>(grid) * D * sizeof(float))) != B200_OK)
    return st;
  a.p.qy = view_of(dq_out);
  a.p.ky = view_of(dk_out);
  a.p.qdx = view_of(dq);
  a.p.kdx = view_of(dk);
  a.p.dw_part = static_cast<float*>(workspace);
  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  st = rope_dispatch(D, interleaved != 0, a.per_row, [&](auto d, auto il, auto per_row) {
    return launch_dependent(
        b200::rope::norm_rope_bwd_kernel<decltype(d)::value, decltype(il)::value,
                                         decltype(per_row)::value>,
        static_cast<unsigned>(grid), b200::rope::kThreads, 0, cs, "qk_norm_rope_bwd launch", a.p);
  });
  if (st != B200_OK) return st;
  return launch_dependent(b200::rope::norm_rope_dw_kernel, 2 * D / 8, 512, 0, cs,
                          "qk_norm_rope_bwd weight launch", a.p.dw_part, ctas.q, grid, D,
                          dq_weight, dk_weight);
}

b200_status attention_window_fwd_workspace(int B, int Hq, int Hkv, int Sq, int Skv, int D,
                                           int window, int sinks, size_t* bytes) {
  const char* who = "attention_window_fwd_workspace";
  if (!bytes) return fail(B200_EINVAL, "%s: null result", who);
  WindowShape s;
  const b200_status st = window_shape(who, B, Hq, Hkv, Sq, Skv, D, window, sinks, -1.0f, &s);
  if (st != B200_OK) return st;
  *bytes = window_plan(s).bytes;
  return B200_OK;
}

b200_status attention_window_fwd(const b200_tensor* q, const b200_tensor* k, const b200_tensor* v,
                                 const b200_tensor* o, float* lse, const int32_t* kv_len, int B,
                                 int Hq, int Hkv, int Sq, int Skv, int D, int window, int sinks,
                                 float softmax_scale, void* workspace, size_t workspace_bytes,
                                 b200_stream_t stream) {
  const char* who = "attention_window_fwd";
  WindowShape s;
  b200_status st = window_shape(who, B, Hq, Hkv, Sq, Skv, D, window, sinks, softmax_scale, &s);
  if (st != B200_OK) return st;
  if ((st = check_qkvo(who, s, q, k, v, o)) != B200_OK) return st;
  const WindowPlan plan = window_plan(s);
  if ((st = check_workspace(who, workspace, workspace_bytes, plan.bytes)) != B200_OK) return st;
  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  b200::split::Params p = split_params(s, q, k, v, o, kv_len, plan.nsplit, plan.units);
  p.lse = lse;
  const int64_t rows = static_cast<int64_t>(B) * Hkv * plan.nsplit * p.rows;
  if (plan.bytes > 0) part_pointers(workspace, rows, D, &p.part_o, &p.part_ml);
  if (plan.tiles)
    st = D == 128 ? launch_window_tiles<128>(s, q, k, v, o, lse, kv_len, plan.nsplit, p.part_o,
                                             p.part_ml, cs)
                  : launch_window_tiles<64>(s, q, k, v, o, lse, kv_len, plan.nsplit, p.part_o,
                                            p.part_ml, cs);
  else
    st = D == 128 ? launch_split<128>(p, cs) : launch_split<64>(p, cs);
  if (st != B200_OK) return st;
  if (plan.bytes == 0) return B200_OK;
  b200::split::CombineParams c{};
  c.o = p.o;
  c.part_a = p.part_o;
  c.ml_a = p.part_ml;
  c.na = plan.nsplit;
  c.B = B;
  c.Hkv = Hkv;
  c.group = p.group;
  c.Sq = Sq;
  c.rows = p.rows;
  c.lse = lse;
  return launch_combine(c, D, cs);
}

b200_status attention_window_bwd_workspace(int B, int Hq, int Hkv, int Sq, int Skv, int D,
                                           int window, int sinks, size_t* bytes) {
  const char* who = "attention_window_bwd_workspace";
  if (!bytes) return fail(B200_EINVAL, "%s: null result", who);
  WindowShape s;
  const b200_status st = window_shape(who, B, Hq, Hkv, Sq, Skv, D, window, sinks, -1.0f, &s);
  if (st != B200_OK) return st;
  *bytes = window_bwd_bytes(s);
  return B200_OK;
}

b200_status attention_window_bwd(const b200_tensor* dout, const b200_tensor* q,
                                 const b200_tensor* k, const b200_tensor* v, const b200_tensor* o,
                                 const float* lse, const b200_tensor* dq, const b200_tensor* dk,
                                 const b200_tensor* dv, const int32_t* kv_len, int B, int Hq,
                                 int Hkv, int Sq, int Skv, int D, int window, int sinks,
                                 float softmax_scale, void* workspace, size_t workspace_bytes,
                                 b200_stream_t stream) {
  const char* who = "attention_window_bwd";
  WindowShape s;
  b200_status st = window_shape(who, B, Hq, Hkv, Sq, Skv, D, window, sinks, softmax_scale, &s);
  if (st != B200_OK) return st;
  if ((st = check_tensor(who, "dout", dout, B, Hq, Sq, D, false)) != B200_OK) return st;
  if ((st = check_tensor(who, "q", q, B, Hq, Sq, D, false)) != B200_OK) return st;
  if ((st = check_tensor(who, "k", k, B, Hkv, Skv, D, false)) != B200_OK) return st;
  if ((st = check_tensor(who, "v", v, B, Hkv, Skv, D, false)) != B200_OK) return st;
  if ((st = check_tensor(who, "o", o, B, Hq, Sq, D, false)) != B200_OK) return st;
  if ((st = check_tensor(who, "dq", dq, B, Hq, Sq, D, true)) != B200_OK) return st;
  if ((st = check_tensor(who, "dk", dk, B, Hkv, Skv, D, true)) != B200_OK) return st;
  if ((st = check_tensor(who, "dv", dv, B, Hkv, Skv, D, true)) != B200_OK) return st;
  if (!lse) return fail(B200_EINVAL, "%s: null lse", who);
  if ((st = check_workspace(who, workspace, workspace_bytes, window_bwd_bytes(s))) != B200_OK)
    return st;
  const WindowGrads t{dout, q, k, v, o, dq, dk, dv, lse, kv_len};
  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  return D == 128 ? window_bwd_tiles<128>(s, t, workspace, cs)
                  : window_bwd_tiles<64>(s, t, workspace, cs);
}

b200_status attention_shared_prefix_workspace(int B, int Hq, int Hkv, int Sq, int P, int S, int D,
                                              size_t* bytes) {
  const char* who = "attention_shared_prefix_workspace";
  if (!bytes) return fail(B200_EINVAL, "%s: null result", who);
  WindowShape own;
  const b200_status st = prefix_shape(who, B, Hq, Hkv, Sq, P, S, D, -1.0f, &own);
  if (st != B200_OK) return st;
  const b200_tensor shared{nullptr, 0, 0, 0};  // a q that is broadcast
  const PrefixPlan plan = prefix_plan(own, P, nullptr), other = prefix_plan(own, P, &shared);
  *bytes = std::max(plan.prefix_bytes + plan.own_bytes, other.prefix_bytes + other.own_bytes);
  return B200_OK;
}

b200_status attention_shared_prefix(const b200_tensor* q, const b200_tensor* k_prefix,
                                    const b200_tensor* v_prefix, const b200_tensor* k,
                                    const b200_tensor* v, const b200_tensor* o,
                                    const int32_t* kv_len, int B, int Hq, int Hkv, int Sq, int P,
                                    int S, int D, float softmax_scale, void* workspace,
                                    size_t workspace_bytes, b200_stream_t stream) {
  const char* who = "attention_shared_prefix";
  WindowShape own;
  b200_status st = prefix_shape(who, B, Hq, Hkv, Sq, P, S, D, softmax_scale, &own);
  if (st != B200_OK) return st;
  if ((st = check_qkvo(who, own, q, k, v, o)) != B200_OK) return st;
  const PrefixPlan plan = prefix_plan(own, P, q);
  if (P > 0) {
    if ((st = check_tensor(who, "k_prefix", k_prefix, 1, Hkv, P, D, false)) != B200_OK) return st;
    if ((st = check_tensor(who, "v_prefix", v_prefix, 1, Hkv, P, D, false)) != B200_OK) return st;
  }
  if ((st = check_workspace(who, workspace, workspace_bytes,
                            plan.prefix_bytes + plan.own_bytes)) != B200_OK)
    return st;
  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  b200::split::Params p = split_params(own, q, k, v, o, kv_len, plan.own_splits, plan.own_units);
  b200::split::CombineParams c{};
  c.B = B;
  c.Hkv = Hkv;
  c.group = p.group;
  c.Sq = Sq;
  c.rows = p.rows;
  c.o = p.o;
  if (plan.tiles) {
    float* part_o;
    float2* part_ml;
    part_pointers(workspace, static_cast<int64_t>(B) * Hkv * plan.prefix_splits * p.rows, D,
                  &part_o, &part_ml);
    st = D == 128 ? launch_prefix_tiles<128>(own, P, q, k_prefix, v_prefix, plan.prefix_splits,
                                             plan.prefix_sms, part_o, part_ml, cs)
                  : launch_prefix_tiles<64>(own, P, q, k_prefix, v_prefix, plan.prefix_splits,
                                            plan.prefix_sms, part_o, part_ml, cs);
    if (st != B200_OK) return st;
    c.part_b = part_o;
    c.ml_b = part_ml;
    c.nb = plan.prefix_splits;
    // The requests' own keys run beside the tiles (see launch_dependent):
    // nothing may be launched between the two.
    p.overlaps = 1;
  } else if (P > 0) {
    p.kp = view_of(k_prefix);
    p.vp = view_of(v_prefix);
    p.P = P;
  }
  if (plan.own_bytes > 0)
    part_pointers(static_cast<unsigned char*>(workspace) + plan.prefix_bytes,
                  static_cast<int64_t>(B) * Hkv * p.nsplit * p.rows, D, &p.part_o, &p.part_ml);
  if ((st = D == 128 ? launch_split<128>(p, cs) : launch_split<64>(p, cs)) != B200_OK) return st;
  if (plan.own_bytes == 0) return B200_OK;
  c.part_a = p.part_o;
  c.ml_a = p.part_ml;
  c.na = p.nsplit;
  return launch_combine(c, D, cs);
}

}  // extern "C"
