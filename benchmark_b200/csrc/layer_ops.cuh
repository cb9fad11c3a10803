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

size_t round16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

// ---- query/key norm with rotation ----
struct RopeArgs {
  b200::rope::Params p;
  int D;
  bool interleaved;
};

b200_status rope_args(const char* who, const b200_tensor* q, const b200_tensor* k,
                      const void* q_weight, const void* k_weight, int weight_f32,
                      const float* inv_freq, int rotary_dim, int interleaved,
                      const int32_t* positions, int64_t position_stride_b, float eps, int B,
                      int S, int Hq, int Hkv, int D, RopeArgs* out) {
  if (B < 1 || S < 1 || Hq < 1 || Hkv < 1)
    return fail(B200_EINVAL, "%s: invalid shape B=%d S=%d Hq=%d Hkv=%d", who, B, S, Hq, Hkv);
  if (D != 64 && D != 128)
    return fail(B200_EUNSUPPORTED, "%s: head_dim must be 64 or 128; got D=%d", who, D);
  if (Hq > 4096 || Hkv > 4096) return fail(B200_EUNSUPPORTED, "%s: more than 4096 heads", who);
  if (rotary_dim < 0 || rotary_dim > D || rotary_dim % 16 != 0)
    return fail(B200_EUNSUPPORTED, "%s: rotary_dim must be a multiple of 16 in [0, D]; got %d",
                who, rotary_dim);
  if (!q_weight || !k_weight) return fail(B200_EINVAL, "%s: null weight", who);
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
  p.tokens = static_cast<int64_t>(B) * S;
  p.S = S;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.rot = rotary_dim;
  auto reciprocal = [](int H) {
    return H == 1 ? 0u : static_cast<uint32_t>((uint64_t{1} << 32) / static_cast<uint64_t>(H) + 1);
  };
  p.mul_q = reciprocal(Hq);
  p.mul_k = reciprocal(Hkv);
  p.eps = eps;
  // Blocks of tokens: long enough to share the angles among heads, short
  // enough that the grid fills the GPU.
  const int64_t per = p.tokens / (static_cast<int64_t>(sm_count()) * 8);
  p.block = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>(per, b200::rope::kMaxTokens)));
  *out = RopeArgs{p, D, interleaved != 0};
  return B200_OK;
}

int rope_bwd_grid(int64_t tokens, int block) {
  const int64_t blocks = (tokens + block - 1) / block;
  return static_cast<int>(
      std::min<int64_t>(blocks, static_cast<int64_t>(sm_count()) * b200::rope::kGradCtasPerSm));
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
// each of a split's warps.
int split_plan(int64_t units, int64_t keys) {
  const int64_t want = 2 * static_cast<int64_t>(sm_count()) / std::max<int64_t>(units, 1);
  const int64_t most = keys / (2 * b200::split::kWarps * b200::split::kKeys);
  return static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>({want, most, b200::split::kMaxSplits})));
}

size_t part_bytes(int64_t rows, int D) {
  return round16(static_cast<size_t>(rows) * D * sizeof(float)) +
         round16(static_cast<size_t>(rows) * sizeof(float2));
}

int row_tiles_of(int64_t rows) {
  return static_cast<int>((rows + b200::split::kRows - 1) / b200::split::kRows);
}

struct WindowPlan {
  int nsplit;
  size_t bytes;
};

WindowPlan window_plan(const WindowShape& s, bool partial = false) {
  const int64_t rows = static_cast<int64_t>(s.Hq / s.Hkv) * s.Sq;
  const int64_t units = static_cast<int64_t>(s.B) * s.Hkv * row_tiles_of(rows);
  const int64_t keys = std::min<int64_t>(s.Skv, static_cast<int64_t>(s.window) + s.sinks);
  WindowPlan p{split_plan(units, keys), 0};
  if (p.nsplit > 1 || partial)
    p.bytes = part_bytes(static_cast<int64_t>(s.B) * s.Hkv * p.nsplit * rows, s.D);
  return p;
}

template <int D>
b200_status launch_split(const b200::split::Params& p, cudaStream_t stream) {
  using C = b200::split::Cfg<D>;
  static unsigned attr_done = 0;
  auto kernel = b200::split::split_attention_kernel<D>;
  const b200_status st = ensure_smem_attr(kernel, C::kSmemBytes, &attr_done);
  if (st != B200_OK) return st;
  const int64_t grid = static_cast<int64_t>(p.B) * p.Hkv * p.row_tiles * p.nsplit;
  if (grid > 0x7fffffffll) return fail(B200_EUNSUPPORTED, "attention: too many work units");
  kernel<<<static_cast<unsigned>(grid), b200::split::kThreads, C::kSmemBytes, stream>>>(p);
  return check_launch("split attention launch");
}

b200_status launch_combine(const b200::split::CombineParams& p, int D, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(p.B) * p.Hkv * p.rows;
  const int64_t grid = (rows + 3) / 4;
  if (grid > 0x7fffffffll) return fail(B200_EUNSUPPORTED, "attention: too many rows");
  if (D == 128)
    b200::split::combine_kernel<128><<<static_cast<unsigned>(grid), 128, 0, stream>>>(p);
  else
    b200::split::combine_kernel<64><<<static_cast<unsigned>(grid), 128, 0, stream>>>(p);
  return check_launch("combine launch");
}

b200::split::Params split_params(const WindowShape& s, const b200_tensor* q, const b200_tensor* k,
                                 const b200_tensor* v, const b200_tensor* o,
                                 const int32_t* kv_len, int nsplit) {
  b200::split::Params p{};
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
  p.step = 1;
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

// The prefix as one batch whose rows are those of every request's queries.
struct PrefixPlan {
  int prefix_splits;  // 0: no prefix
  int own_splits;
  size_t prefix_bytes, own_bytes;
};

PrefixPlan prefix_plan(const WindowShape& own, int P) {
  PrefixPlan p{};
  if (P > 0) {
    const int64_t rows = static_cast<int64_t>(own.B) * (own.Hq / own.Hkv) * own.Sq;
    p.prefix_splits = split_plan(static_cast<int64_t>(own.Hkv) * row_tiles_of(rows), P);
    p.prefix_bytes = part_bytes(own.Hkv * p.prefix_splits * rows, own.D);
  }
  const WindowPlan w = window_plan(own, P > 0);
  p.own_splits = w.nsplit;
  p.own_bytes = w.bytes;
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
                             interleaved, positions, position_stride_b, eps, B, S, Hq, Hkv, D, &a);
  if (st != B200_OK) return st;
  if ((st = check_tensor(who, "q_out", q_out, B, Hq, S, D, true)) != B200_OK) return st;
  if ((st = check_tensor(who, "k_out", k_out, B, Hkv, S, D, true)) != B200_OK) return st;
  a.p.qy = view_of(q_out);
  a.p.ky = view_of(k_out);
  const int64_t grid = (a.p.tokens + a.p.block - 1) / a.p.block;
  if (grid > 0x7fffffffll) return fail(B200_EUNSUPPORTED, "%s: too many tokens", who);
  using Kernel = void (*)(b200::rope::Params);
  const Kernel kernel =
      D == 128 ? (a.interleaved ? b200::rope::norm_rope_kernel<128, true>
                                : b200::rope::norm_rope_kernel<128, false>)
               : (a.interleaved ? b200::rope::norm_rope_kernel<64, true>
                                : b200::rope::norm_rope_kernel<64, false>);
  kernel<<<static_cast<unsigned>(grid), b200::rope::kThreads, 0,
           reinterpret_cast<cudaStream_t>(stream)>>>(a.p);
  return check_launch("qk_norm_rope launch");
}

b200_status qk_norm_rope_bwd_workspace(int B, int S, int D, size_t* bytes) {
  if (!bytes || B < 1 || S < 1) return fail(B200_EINVAL, "qk_norm_rope_bwd_workspace: bad argument");
  // The grid never exceeds its CTAs per SM, whatever the shape.
  *bytes = static_cast<size_t>(sm_count()) * b200::rope::kGradCtasPerSm * 2 * D * sizeof(float);
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
                             interleaved, positions, position_stride_b, eps, B, S, Hq, Hkv, D, &a);
  if (st != B200_OK) return st;
  if ((st = check_tensor(who, "dq_out", dq_out, B, Hq, S, D, false)) != B200_OK) return st;
  if ((st = check_tensor(who, "dk_out", dk_out, B, Hkv, S, D, false)) != B200_OK) return st;
  if ((st = check_tensor(who, "dq", dq, B, Hq, S, D, true)) != B200_OK) return st;
  if ((st = check_tensor(who, "dk", dk, B, Hkv, S, D, true)) != B200_OK) return st;
  if (!dq_weight || !dk_weight) return fail(B200_EINVAL, "%s: null weight gradient", who);
  const int grid = rope_bwd_grid(a.p.tokens, a.p.block);
  if ((st = check_workspace(who, workspace, workspace_bytes,
                            static_cast<size_t>(grid) * 2 * D * sizeof(float))) != B200_OK)
    return st;
  a.p.qy = view_of(dq_out);
  a.p.ky = view_of(dk_out);
  a.p.qdx = view_of(dq);
  a.p.kdx = view_of(dk);
  a.p.dw_part = static_cast<float*>(workspace);
  using Kernel = void (*)(b200::rope::Params);
  const Kernel kernel =
      D == 128 ? (a.interleaved ? b200::rope::norm_rope_bwd_kernel<128, true>
                                : b200::rope::norm_rope_bwd_kernel<128, false>)
               : (a.interleaved ? b200::rope::norm_rope_bwd_kernel<64, true>
                                : b200::rope::norm_rope_bwd_kernel<64, false>);
  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  kernel<<<grid, b200::rope::kThreads, 0, cs>>>(a.p);
  if ((st = check_launch("qk_norm_rope_bwd launch")) != B200_OK) return st;
  b200::rope::norm_rope_dw_kernel<<<2 * D / 32, 256, 0, cs>>>(a.p.dw_part, grid, D, dq_weight,
                                                              dk_weight);
  return check_launch("qk_norm_rope_bwd weight launch");
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
  b200::split::Params p = split_params(s, q, k, v, o, kv_len, plan.nsplit);
  p.lse = lse;
  const int64_t rows = static_cast<int64_t>(B) * Hkv * plan.nsplit * p.rows;
  if (plan.nsplit > 1) part_pointers(workspace, rows, D, &p.part_o, &p.part_ml);
  if ((st = D == 128 ? launch_split<128>(p, cs) : launch_split<64>(p, cs)) != B200_OK) return st;
  if (plan.nsplit == 1) return B200_OK;
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

b200_status attention_window_bwd_workspace(int B, int Hq, int Sq, size_t* bytes) {
  if (!bytes || B < 1 || Hq < 1 || Sq < 1)
    return fail(B200_EINVAL, "attention_window_bwd_workspace: bad argument");
  *bytes = static_cast<size_t>(B) * Hq * Sq * sizeof(float);
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
  const size_t need = static_cast<size_t>(B) * Hq * Sq * sizeof(float);
  if ((st = check_workspace(who, workspace, workspace_bytes, need)) != B200_OK) return st;
  namespace bw = b200::bwd;
  bw::Params p{};
  p.dout = view_of(dout);
  p.q = view_of(q);
  p.k = view_of(k);
  p.v = view_of(v);
  p.o = view_of(o);
  p.dq = view_of(dq);
  p.dk = view_of(dk);
  p.dv = view_of(dv);
  p.lse = lse;
  p.delta = static_cast<float*>(workspace);
  p.kv_len = kv_len;
  p.B = B;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.group = Hq / Hkv;
  p.Sq = Sq;
  p.Skv = Skv;
  p.q_tiles = (Sq + bw::kTile - 1) / bw::kTile;
  p.k_tiles = (Skv + bw::kTile - 1) / bw::kTile;
  p.window = s.window;
  p.sinks = s.sinks;
  p.scale = s.scale;
  p.scale_log2 = s.scale * 1.4426950408889634f;
  const int64_t g0 = (static_cast<int64_t>(B) * Hq * Sq + 7) / 8;
  const int64_t g1 = static_cast<int64_t>(B) * Hkv * p.k_tiles;
  const int64_t g2 = static_cast<int64_t>(B) * Hq * p.q_tiles;
  if (std::max({g0, g1, g2}) > 0x7fffffffll)
    return fail(B200_EUNSUPPORTED, "%s: too many work units", who);
  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  auto launch = [&](auto d) -> b200_status {
    constexpr int kD = decltype(d)::value;
    static unsigned attr_kv = 0, attr_q = 0;
    constexpr int bytes = bw::Cfg<kD>::kSmemBytes;
    b200_status r = ensure_smem_attr(bw::dkdv_kernel<kD>, bytes, &attr_kv);
    if (r != B200_OK) return r;
    if ((r = ensure_smem_attr(bw::dq_kernel<kD>, bytes, &attr_q)) != B200_OK) return r;
    bw::delta_kernel<kD><<<static_cast<unsigned>(g0), 256, 0, cs>>>(p);
    bw::dkdv_kernel<kD><<<static_cast<unsigned>(g1), bw::kThreads, bytes, cs>>>(p);
    bw::dq_kernel<kD><<<static_cast<unsigned>(g2), bw::kThreads, bytes, cs>>>(p);
    return check_launch("attention_window_bwd launch");
  };
  return D == 128 ? launch(std::integral_constant<int, 128>{})
                  : launch(std::integral_constant<int, 64>{});
}

b200_status attention_shared_prefix_workspace(int B, int Hq, int Hkv, int Sq, int P, int S, int D,
                                              size_t* bytes) {
  const char* who = "attention_shared_prefix_workspace";
  if (!bytes) return fail(B200_EINVAL, "%s: null result", who);
  WindowShape own;
  const b200_status st = prefix_shape(who, B, Hq, Hkv, Sq, P, S, D, -1.0f, &own);
  if (st != B200_OK) return st;
  const PrefixPlan plan = prefix_plan(own, P);
  *bytes = plan.prefix_bytes + plan.own_bytes;
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
  const PrefixPlan plan = prefix_plan(own, P);
  if (P > 0) {
    if ((st = check_tensor(who, "k_prefix", k_prefix, 1, Hkv, P, D, false)) != B200_OK) return st;
    if ((st = check_tensor(who, "v_prefix", v_prefix, 1, Hkv, P, D, false)) != B200_OK) return st;
  }
  if ((st = check_workspace(who, workspace, workspace_bytes,
                            plan.prefix_bytes + plan.own_bytes)) != B200_OK)
    return st;
  const cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
  auto launch = [&](const b200::split::Params& p) {
    return D == 128 ? launch_split<128>(p, cs) : launch_split<64>(p, cs);
  };
  b200::split::CombineParams c{};
  c.B = B;
  c.Hkv = Hkv;
  c.group = Hq / Hkv;
  c.Sq = Sq;
  c.rows = c.group * Sq;
  c.o = view_of(o);
  if (P > 0) {
    WindowShape shared = own;
    shared.Skv = shared.window = P;
    b200::split::Params p =
        split_params(shared, q, k_prefix, v_prefix, o, nullptr, plan.prefix_splits);
    p.B = 1;
    p.step = 0;
    p.rows = B * c.rows;
    p.row_tiles = row_tiles_of(p.rows);
    part_pointers(workspace, static_cast<int64_t>(Hkv) * p.nsplit * p.rows, D, &p.part_o,
                  &p.part_ml);
    if ((st = launch(p)) != B200_OK) return st;
    c.part_b = p.part_o;
    c.ml_b = p.part_ml;
    c.nb = p.nsplit;
  }
  b200::split::Params p = split_params(own, q, k, v, o, kv_len, plan.own_splits);
  if (plan.own_bytes > 0)
    part_pointers(static_cast<unsigned char*>(workspace) + plan.prefix_bytes,
                  static_cast<int64_t>(B) * Hkv * p.nsplit * p.rows, D, &p.part_o, &p.part_ml);
  if ((st = launch(p)) != B200_OK) return st;
  if (plan.own_bytes == 0) return B200_OK;
  c.part_a = p.part_o;
  c.ml_a = p.part_ml;
  c.na = p.nsplit;
  return launch_combine(c, D, cs);
}

}  // extern "C"
