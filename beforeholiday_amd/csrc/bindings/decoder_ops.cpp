// Grouped-query attention (kernels/grouped_attn.hip), query / key norm + rotary embedding
// (kernels/qk_norm_rope.hip) and counter-based dropout (kernels/counter_dropout.hip). Every call checks its
// operands here, runs on the current stream of the operands' device and allocates what it needs per call.
//
// The autograd nodes are C++ ones: a training step of a small call is bound by the host, and with Python nodes
// the step of a 777 x 3-token norm + rotation took 111 us around 42 us of kernels.
#include "common.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <cmath>

#include "bh/grouped_attn_api.h"
#include "bh/qk_rope_api.h"

namespace bhb {
namespace {

constexpr int64_t kMaxLen = int64_t(1) << 29;     // queries / keys of a sequence
constexpr int64_t kMaxStride = int64_t(1) << 24;  // elements between two positions (block offsets are 32-bit)
constexpr int64_t kMaxTiles = int64_t(1) << 22;
constexpr int64_t kMaxTokens = int64_t(1) << 26;  // 64 threads each

const int64_t* step_seed(const c10::optional<at::Tensor>& t, const at::Tensor& like, const char* what) {
  if (!t.has_value() || !t->defined()) return nullptr;
  TORCH_CHECK(t->scalar_type() == at::kLong && t->numel() == 1 && t->device() == like.device(), what,
              ": seed_dev must be an int64 [1] tensor on the operands' device");
  return t->data_ptr<int64_t>();
}

bh::GaView ga_view(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a GPU (HIP) tensor");
  TORCH_CHECK_VALUE(t.dim() == 4, "grouped attention: ", name, " must be [s, b, heads, head_dim]");
  TORCH_CHECK_VALUE(t.device() == like.device() && t.scalar_type() == like.scalar_type(), "grouped attention: ", name,
              " must have the query's device and dtype");
  TORCH_CHECK_VALUE(t.stride(3) == 1, "grouped attention: ", name, " must be contiguous along head_dim");
  bh::GaView v;
  v.p = t.data_ptr();
  const int64_t hn = t.size(3);
  v.st = t.size(0) > 1 ? t.stride(0) : hn;  // a single position: its stride is never used, any value may be there
  v.sb = t.size(1) > 1 ? t.stride(1) : 0;
  v.sh = t.size(2) > 1 ? t.stride(2) : 0;
  TORCH_CHECK_VALUE(v.st % 8 == 0 && v.sb % 8 == 0 && v.sh % 8 == 0 && reinterpret_cast<uintptr_t>(v.p) % 16 == 0,
              "grouped attention: ", name, " strides must be multiples of 8 elements and its base 16-byte aligned");
  TORCH_CHECK_VALUE(v.st >= hn && v.st < kMaxStride, "grouped attention: ", name, " position stride must be in [head_dim, 2^24)");
  return v;
}

bh::GaArgs ga_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool causal, int64_t window,
                   const c10::optional<at::Tensor>& lens, double scale, double p, int64_t seed,
                   const c10::optional<at::Tensor>& seed_dev) {
  TORCH_CHECK_VALUE(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16,
              "grouped attention: fp16 / bf16 tensors only on the GPU, got ", q.scalar_type());
  bh::GaArgs a;
  a.q = ga_view(q, q, "query");
  a.k = ga_view(k, q, "key");
  a.v = ga_view(v, q, "value");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(1) == q.size(1) && k.size(3) == q.size(3),
              "grouped attention: query ", q.sizes(), ", key ", k.sizes(), " and value ", v.sizes(), " do not fit");
  TORCH_CHECK_VALUE(k.size(2) >= 1 && q.size(2) >= 1 && q.size(2) % k.size(2) == 0,
              "grouped attention: query heads (", q.size(2), ") must be a multiple of key heads (", k.size(2), ")");
  TORCH_CHECK_VALUE(q.size(3) >= 8 && q.size(3) <= 128 && q.size(3) % 8 == 0,
              "grouped attention: head_dim must be a multiple of 8 up to 128, got ", q.size(3));
  TORCH_CHECK_VALUE(q.size(0) <= kMaxLen && k.size(0) <= kMaxLen, "grouped attention: sequences of up to 2^29 only");
  TORCH_CHECK_VALUE(scale >= 1e-30 && scale <= 1e30, "grouped attention: scale must be in [1e-30, 1e30], got ", scale);
  TORCH_CHECK_VALUE(p >= 0 && p < 1, "grouped attention: dropout must be in [0, 1), got ", p);
  a.sq = (int)q.size(0); a.b = (int)q.size(1); a.np = (int)q.size(2); a.hn = (int)q.size(3);
  a.sk = (int)k.size(0); a.ng = (int)k.size(2);
  // 128-row tiles of all heads: the largest launch is of 2 * 512 threads a tile, and a launch has fewer than 2^32
  TORCH_CHECK_VALUE(q.size(1) * q.size(2) * ((q.size(0) + 127) / 128) < kMaxTiles &&
                        k.size(1) * k.size(2) * ((k.size(0) + 127) / 128) < kMaxTiles,
                    "grouped attention: too many heads and positions for one launch: query ", q.sizes(), ", key ", k.sizes());
  a.causal = causal;
  TORCH_CHECK_VALUE(window == 0 || (causal && window > 0), "grouped attention: a window needs causal and at least one key");
  a.window = (int)(window > 0 ? std::min(window, 2 * kMaxLen) : 2 * kMaxLen);
  if (lens.has_value() && lens->defined()) {
    TORCH_CHECK_VALUE(lens->device() == q.device() && lens->scalar_type() == at::kInt && lens->dim() == 1 &&
                    lens->size(0) == q.size(1) && lens->is_contiguous(),
                "grouped attention: key_lengths must be a contiguous int32 [batch] tensor on the query's device");
    a.lens = lens->data_ptr<int>();
  }
  a.scale = (float)scale;
  a.p_drop = p;
  a.seed = (uint64_t)seed;
  a.seed_dev = step_seed(seed_dev, q, "grouped attention");
  return a;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// What the kernels cannot address (head_dim not contiguous, strides or base off 16 bytes, positions overlapping
// or 2^24 elements and more apart) is copied.
at::Tensor ga_usable(const at::Tensor& t) {
  bool ok = t.dim() == 4 && t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  if (ok && t.size(0) > 1) ok = t.stride(0) >= t.size(3) && t.stride(0) < kMaxStride;
  for (int d = 0; ok && d < 3; ++d) ok = t.size(d) <= 1 || t.stride(d) % 8 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
at::Tensor rope_usable(const at::Tensor& t) {
  return t.dim() == 4 && t.stride(3) != 1 ? t.clone(at::MemoryFormat::Contiguous) : t;
}

bool wants_grad(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const auto* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// gradients of a function that is differentiable once: under create_graph they carry a node that raises
variable_list once_differentiable(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list in;
  for (const auto& g : grads)
    if (g.defined()) in.push_back(g.detach().set_requires_grad(true));
  auto err = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " is differentiable once only",
                                                             (int64_t)in.size());
  auto out = err->apply(std::move(in));
  size_t n = 0;
  for (auto& g : grads)
    if (g.defined()) g = out[n++];
  return grads;
}

struct GaCall {
  bool causal;
  int64_t window;
  double scale, p;
  int64_t seed;
};

// -> o, lse, and with `train` what the rounding of o left over
std::tuple<at::Tensor, at::Tensor, at::Tensor> ga_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                      const c10::optional<at::Tensor>& lens,
                                                      const c10::optional<at::Tensor>& seed_dev, const GaCall& c,
                                                      bool train) {
  auto a = ga_args(q, k, v, c.causal, c.window, lens, c.scale, c.p, c.seed, seed_dev);
  const c10::DeviceGuard guard(q.device());
  auto o = at::empty(q.sizes(), q.options());
  auto lse = at::empty({q.size(1), q.size(2), q.size(0)}, q.options().dtype(at::kFloat));
  at::Tensor olo = train ? at::empty(q.sizes(), q.options()) : at::Tensor();
  if (o.numel() == 0) return {o, lse, olo};
  if (a.sk == 0) return {o.zero_(), lse.fill_(INFINITY), olo};
  a.o = ga_view(o, q, "output");
  a.olo = train ? olo.data_ptr() : nullptr;
  a.lse = lse.data_ptr<float>();
  const int64_t n = bh::ga_forward_workspace(a);
  at::Tensor ws = n ? at::empty({n}, lse.options()) : at::Tensor();
  bh::ga_forward(dtype_code(q.scalar_type()), a, n ? ws.data_ptr<float>() : nullptr, stream_for(q));
  return {o, lse, olo};
}

variable_list ga_bwd(const at::Tensor& dout, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                     const at::Tensor& o, const at::Tensor& olo, const at::Tensor& lse,
                     const c10::optional<at::Tensor>& lens, const c10::optional<at::Tensor>& seed_dev, const GaCall& c,
                     bool need_kv) {
  auto a = ga_args(q, k, v, c.causal, c.window, lens, c.scale, c.p, c.seed, seed_dev);
  TORCH_CHECK(dout.sizes() == q.sizes(), "grouped attention: gradient shape mismatch");
  const c10::DeviceGuard guard(q.device());
  at::Tensor dq = at::empty(q.sizes(), q.options()), dk, dv;
  if (need_kv) {
    dk = at::empty(k.sizes(), k.options());
    dv = at::empty(v.sizes(), v.options());
  }
  if (q.numel() == 0 || a.sk == 0) {
    dq.zero_();
    if (need_kv) {
      dk.zero_();
      dv.zero_();
    }
    return {dq, dk, dv};
  }
  a.dout = ga_view(dout, q, "output gradient");
  a.o = ga_view(o, q, "output");
  a.olo = olo.data_ptr();
  a.dq = ga_view(dq, q, "dq");
  if (need_kv) {
    a.dk = ga_view(dk, q, "dk");
    a.dv = ga_view(dv, q, "dv");
  }
  a.lse = lse.data_ptr<float>();
  auto delta = at::empty_like(lse);
  a.delta = delta.data_ptr<float>();
  at::Tensor rowh, ws;
  if (a.p_drop > 0) {
    rowh = at::empty(lse.sizes(), lse.options().dtype(at::kInt));
    a.rowh = reinterpret_cast<uint32_t*>(rowh.data_ptr());
  }
  const int64_t n = need_kv ? bh::ga_backward_workspace(a) : 0;
  if (n) ws = at::empty({n}, lse.options());
  bh::ga_backward(dtype_code(q.scalar_type()), a, n ? ws.data_ptr<float>() : nullptr, stream_for(q));
  return {dq, dk, dv};
}

struct GroupedAttention : torch::autograd::Function<GroupedAttention> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                            const c10::optional<at::Tensor>& lens, const c10::optional<at::Tensor>& seed_dev,
                            GaCall c) {
    auto [o, lse, olo] = ga_fwd(q, k, v, lens, seed_dev, c, true);
    ctx->save_for_backward({q, k, v, o, olo, lse, lens.value_or(at::Tensor())});
    // not saved by version: a captured step advances it in place before every forward
    if (seed_dev.has_value()) ctx->saved_data["seed_dev"] = *seed_dev;
    ctx->saved_data["mask"] = std::vector<int64_t>{c.causal, c.window, c.seed};
    ctx->saved_data["num"] = std::vector<double>{c.scale, c.p};
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const auto mask = ctx->saved_data["mask"].toIntVector();
    const auto num = ctx->saved_data["num"].toDoubleVector();
    const auto sd = ctx->saved_data.find("seed_dev");
    c10::optional<at::Tensor> lens, seed_dev;
    if (s[6].defined()) lens = s[6];
    if (sd != ctx->saved_data.end()) seed_dev = sd->second.toTensor();
    const bool nq = ctx->needs_input_grad(0), nk = ctx->needs_input_grad(1), nv = ctx->needs_input_grad(2);
    auto g = ga_bwd(ga_usable(grads[0].detach()), s[0], s[1], s[2], s[3], s[4], s[5], lens, seed_dev,
                    GaCall{mask[0] != 0, mask[1], num[0], num[1], mask[2]}, nk || nv);
    return once_differentiable({nq ? g[0] : at::Tensor(), nk ? g[1] : at::Tensor(), nv ? g[2] : at::Tensor(),
                                at::Tensor(), at::Tensor(), at::Tensor()},
                               "fused_grouped_attention");
  }
};

at::Tensor ga_call(at::Tensor q, at::Tensor k, at::Tensor v, c10::optional<at::Tensor> lens, bool causal, int64_t window,
                   double scale, double p, int64_t seed, c10::optional<at::Tensor> seed_dev) {
  const GaCall c{causal, window, scale, p, seed};
  q = ga_usable(q);
  k = ga_usable(k);
  v = ga_usable(v);
  if (wants_grad({&q, &k, &v})) return GroupedAttention::apply(q, k, v, lens, seed_dev, c);
  return std::get<0>(ga_fwd(q, k, v, lens, seed_dev, c, false));
}

// ---- query / key norm + rotary embedding ---------------------------------------------------------------------
bool rope_view(const at::Tensor& t, const at::Tensor& like, const char* name, bh::HeadView& v) {
  TORCH_CHECK_VALUE(t.is_cuda(), name, " must be a GPU (HIP) tensor");
  TORCH_CHECK_VALUE(t.dim() == 4, "qk_norm_rope: ", name, " must be [s, b, heads, head_dim]");
  TORCH_CHECK_VALUE(t.device() == like.device() && t.scalar_type() == like.scalar_type(), "qk_norm_rope: ", name,
              " must have the query's device and dtype");
  TORCH_CHECK_VALUE(t.stride(3) == 1, "qk_norm_rope: ", name, " must be contiguous along head_dim");
  v.p = t.data_ptr();
  v.st = t.size(0) > 1 ? t.stride(0) : 0;
  v.sb = t.size(1) > 1 ? t.stride(1) : 0;
  v.sh = t.size(2) > 1 ? t.stride(2) : 0;
  return v.st % 4 == 0 && v.sb % 4 == 0 && v.sh % 4 == 0 &&
         reinterpret_cast<uintptr_t>(v.p) % (4 * t.element_size()) == 0;
}

bh::QkRopeArgs rope_args(const at::Tensor& q, const at::Tensor& k, const c10::optional<at::Tensor>& wq,
                         const c10::optional<at::Tensor>& wk, const c10::optional<at::Tensor>& cos,
                         const c10::optional<at::Tensor>& sin, const c10::optional<at::Tensor>& pos, int64_t offset,
                         double eps, bool interleaved) {
  TORCH_CHECK_VALUE(q.scalar_type() == at::kFloat || q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16,
              "qk_norm_rope: fp32 / fp16 / bf16 tensors only on the GPU, got ", q.scalar_type());
  bh::QkRopeArgs a;
  bool vec = rope_view(q, q, "query", a.x[0]);
  vec = rope_view(k, q, "key", a.x[1]) && vec;
  const int64_t hn = q.size(3);
  TORCH_CHECK_VALUE(k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == hn, "qk_norm_rope: query ", q.sizes(),
              " and key ", k.sizes(), " do not fit");
  TORCH_CHECK_VALUE(hn >= 2 && hn <= 512 && hn % 2 == 0, "qk_norm_rope: head_dim must be even and at most 512, got ", hn);
  TORCH_CHECK_VALUE(q.size(0) * q.size(1) < kMaxTokens && q.size(0) < kMaxTokens && q.size(1) < kMaxTokens &&
                        q.size(2) <= kMaxLen && k.size(2) <= kMaxLen,
                    "qk_norm_rope: fewer than 2^26 tokens only, got ", q.sizes());
  a.s = (int)q.size(0); a.b = (int)q.size(1); a.hn = (int)hn;
  a.heads[0] = (int)q.size(2); a.heads[1] = (int)k.size(2);
  const bool norm = wq.has_value() && wq->defined();
  TORCH_CHECK_VALUE(norm == (wk.has_value() && wk->defined()), "qk_norm_rope: give both norm weights or none");
  if (norm) {
    for (const auto* w : {&*wq, &*wk}) {
      TORCH_CHECK_VALUE(w->device() == q.device() && w->dim() == 1 && w->size(0) == hn && w->is_contiguous() &&
                      w->scalar_type() == wq->scalar_type(),
                  "qk_norm_rope: norm weights must be contiguous [head_dim] tensors of one dtype on the query's device");
      TORCH_CHECK_VALUE(w->scalar_type() == at::kFloat || w->scalar_type() == at::kHalf || w->scalar_type() == at::kBFloat16,
                  "qk_norm_rope: norm weights must be fp32 / fp16 / bf16");
      vec = vec && reinterpret_cast<uintptr_t>(w->data_ptr()) % (4 * w->element_size()) == 0;
    }
    a.w[0] = wq->data_ptr();
    a.w[1] = wk->data_ptr();
    a.w_dt = dtype_code(wq->scalar_type());
    TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "qk_norm_rope: eps must be >= 0");
  }
  const bool rot = cos.has_value() && cos->defined();
  TORCH_CHECK_VALUE(rot == (sin.has_value() && sin->defined()), "qk_norm_rope: give both angle tables or none");
  TORCH_CHECK_VALUE(norm || rot, "qk_norm_rope: neither norm weights nor angle tables");
  if (rot) {
    for (const auto* c : {&*cos, &*sin})
      TORCH_CHECK_VALUE(c->device() == q.device() && c->scalar_type() == at::kFloat && c->dim() == 2 && c->is_contiguous() &&
                      c->sizes() == cos->sizes(),
                  "qk_norm_rope: cos / sin must be contiguous fp32 [positions, rot / 2] tables on the query's device");
    TORCH_CHECK_VALUE(cos->size(1) >= 1 && 2 * cos->size(1) <= hn, "qk_norm_rope: the tables rotate ", 2 * cos->size(1),
                " of ", hn, " values");
    a.cos = cos->data_ptr<float>();
    a.sin = sin->data_ptr<float>();
    a.rot = (int)(2 * cos->size(1));
    a.n_pos = cos->size(0);
    if (pos.has_value() && pos->defined()) {
      TORCH_CHECK_VALUE(pos->device() == q.device() && (pos->scalar_type() == at::kLong || pos->scalar_type() == at::kInt) &&
                      ((pos->dim() == 1 && pos->size(0) == q.size(0)) ||
                       (pos->dim() == 2 && pos->size(0) == q.size(0) && pos->size(1) == q.size(1))),
                  "qk_norm_rope: positions must be an int32 / int64 [s] or [s, b] tensor on the query's device");
      a.pos = pos->data_ptr();
      a.pos_i64 = pos->scalar_type() == at::kLong;
      a.pos_st = pos->stride(0);
      a.pos_sb = pos->dim() == 2 ? pos->stride(1) : 0;
      TORCH_CHECK_VALUE(offset == 0, "qk_norm_rope: an offset goes without positions");
    } else {
      TORCH_CHECK_VALUE(offset >= 0 && offset <= a.n_pos - q.size(0), "qk_norm_rope: ", q.size(0), " positions from ",
                        offset, " on do not fit tables of ", a.n_pos);
      a.offset = offset;
    }
  }
  a.eps = (float)eps;
  a.interleaved = interleaved;
  a.vec = vec && hn % 8 == 0 && (interleaved || a.rot % 8 == 0);
  return a;
}

struct RopeCall {
  int64_t offset;
  double eps;
  bool interleaved;
};
using OptTensor = c10::optional<at::Tensor>;

variable_list rope_fwd(const at::Tensor& q, const at::Tensor& k, const OptTensor& wq, const OptTensor& wk,
                       const OptTensor& cos, const OptTensor& sin, const OptTensor& pos, const RopeCall& c) {
  auto a = rope_args(q, k, wq, wk, cos, sin, pos, c.offset, c.eps, c.interleaved);
  const c10::DeviceGuard guard(q.device());
  auto yq = at::empty(q.sizes(), q.options()), yk = at::empty(k.sizes(), k.options());
  const bool v0 = rope_view(yq, q, "output", a.y[0]), v1 = rope_view(yk, q, "output", a.y[1]);
  a.vec = a.vec && v0 && v1;
  if (yq.numel() + yk.numel() > 0) bh::qk_rope_forward(dtype_code(q.scalar_type()), a, stream_for(q));
  return {yq, yk};
}

variable_list rope_bwd(const at::Tensor& dyq, const at::Tensor& dyk, const at::Tensor& q, const at::Tensor& k,
                       const OptTensor& wq, const OptTensor& wk, const OptTensor& cos, const OptTensor& sin,
                       const OptTensor& pos, const RopeCall& c) {
  auto a = rope_args(q, k, wq, wk, cos, sin, pos, c.offset, c.eps, c.interleaved);
  TORCH_CHECK(dyq.sizes() == q.sizes() && dyk.sizes() == k.sizes(), "qk_norm_rope: gradient shape mismatch");
  const c10::DeviceGuard guard(q.device());
  auto dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
  bool vec = rope_view(dq, q, "dq", a.y[0]);
  vec = rope_view(dk, q, "dk", a.y[1]) && vec;
  vec = rope_view(dyq, q, "query gradient", a.dy[0]) && vec;
  vec = rope_view(dyk, q, "key gradient", a.dy[1]) && vec;
  a.vec = a.vec && vec;
  const auto f32 = q.options().dtype(at::kFloat);
  at::Tensor dwq, dwk;
  if (a.w[0]) {
    dwq = at::empty(wq->sizes(), wq->options());
    dwk = at::empty(wk->sizes(), wk->options());
  }
  if (dq.numel() + dk.numel() == 0) {
    if (dwq.defined()) {
      dwq.zero_();
      dwk.zero_();
    }
  } else {
    const int64_t rows = bh::qk_rope_partial_rows(a);
    at::Tensor part = rows ? at::empty({rows * 2 * q.size(3)}, f32) : at::Tensor();
    bh::qk_rope_backward(dtype_code(q.scalar_type()), a, rows ? part.data_ptr<float>() : nullptr,
                         rows ? dwq.data_ptr() : nullptr, rows ? dwk.data_ptr() : nullptr, stream_for(q));
  }
  return {dq, dk, dwq, dwk};
}

struct QkNormRope : torch::autograd::Function<QkNormRope> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const OptTensor& wq,
                               const OptTensor& wk, const OptTensor& cos, const OptTensor& sin, const OptTensor& pos,
                               RopeCall c) {
    auto y = rope_fwd(q, k, wq, wk, cos, sin, pos, c);
    const at::Tensor none;
    ctx->save_for_backward({q, k, wq.value_or(none), wk.value_or(none), cos.value_or(none), sin.value_or(none),
                            pos.value_or(none)});
    ctx->saved_data["int"] = std::vector<int64_t>{c.offset, c.interleaved};
    ctx->saved_data["eps"] = c.eps;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    auto opt = [](const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const auto n = ctx->saved_data["int"].toIntVector();
    auto g = rope_bwd(rope_usable(grads[0].detach()), rope_usable(grads[1].detach()), s[0], s[1], opt(s[2]), opt(s[3]),
                      opt(s[4]), opt(s[5]), opt(s[6]), RopeCall{n[0], ctx->saved_data["eps"].toDouble(), n[1] != 0});
    const at::Tensor none;
    return once_differentiable({g[0], g[1], g[2], g[3], none, none, none, none}, "fused_qk_norm_rope");
  }
};

variable_list rope_call(at::Tensor q, at::Tensor k, OptTensor wq, OptTensor wk, OptTensor cos, OptTensor sin,
                        OptTensor pos, int64_t offset, double eps, bool interleaved) {
  const RopeCall c{offset, eps, interleaved};
  q = rope_usable(q);
  k = rope_usable(k);
  for (auto* t : {&wq, &wk})
    if (t->has_value()) *t = (*t)->contiguous();
  for (auto* t : {&cos, &sin})
    if (t->has_value()) *t = (*t)->detach().contiguous();
  const at::Tensor none, w0 = wq.value_or(none), w1 = wk.value_or(none);
  if (wants_grad({&q, &k, &w0, &w1})) return QkNormRope::apply(q, k, wq, wk, cos, sin, pos, c);
  return rope_fwd(q, k, wq, wk, cos, sin, pos, c);
}

// ---- dropout -------------------------------------------------------------------------------------------------
struct DropCall {
  int64_t thresh;
  double scale;
  int64_t seed;
};

at::Tensor drop_fwd(const at::Tensor& x_, const c10::optional<at::Tensor>& seed_dev, const DropCall& c) {
  const at::Tensor x = x_.contiguous();
  check_cuda(x, "dropout input");
  TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16,
              "counter_dropout: fp32 / fp16 / bf16 tensors only on the GPU, got ", x.scalar_type());
  TORCH_CHECK(c.thresh >= 0 && c.thresh <= UINT32_MAX, "counter_dropout: bad threshold");
  const int64_t* sd = step_seed(seed_dev, x, "counter_dropout");
  const c10::DeviceGuard guard(x.device());
  auto y = at::empty(x.sizes(), x.options());
  bh::counter_dropout(dtype_code(x.scalar_type()), x.data_ptr(), y.data_ptr(), x.numel(), (uint32_t)c.thresh,
                      (float)c.scale, (uint64_t)c.seed, sd, stream_for(x));
  return y;
}

// linear in x, and its own transpose: the backward pass is the same call (and differentiable again)
struct CounterDropout : torch::autograd::Function<CounterDropout> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const c10::optional<at::Tensor>& seed_dev,
                            DropCall c) {
    if (seed_dev.has_value()) ctx->saved_data["seed_dev"] = *seed_dev;
    ctx->saved_data["int"] = std::vector<int64_t>{c.thresh, c.seed};
    ctx->saved_data["scale"] = c.scale;
    return drop_fwd(x, seed_dev, c);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto n = ctx->saved_data["int"].toIntVector();
    const auto sd = ctx->saved_data.find("seed_dev");
    c10::optional<at::Tensor> seed_dev;
    if (sd != ctx->saved_data.end()) seed_dev = sd->second.toTensor();
    const DropCall c{n[0], ctx->saved_data["scale"].toDouble(), n[1]};
    const at::Tensor g = wants_grad({&grads[0]}) ? CounterDropout::apply(grads[0], seed_dev, c)
                                                 : drop_fwd(grads[0], seed_dev, c);
    return {g, at::Tensor(), at::Tensor()};
  }
};

at::Tensor drop_call(at::Tensor x, int64_t thresh, double scale, int64_t seed, c10::optional<at::Tensor> seed_dev) {
  const DropCall c{thresh, scale, seed};
  return wants_grad({&x}) ? CounterDropout::apply(x, seed_dev, c) : drop_fwd(x, seed_dev, c);
}

}  // namespace

void register_decoder_ops(pybind11::module_& root) {
  namespace py = pybind11;
  auto ga = root.def_submodule("grouped_attention", "grouped-query attention, head sizes up to 128");
  ga.def("attention", &ga_call, "softmax(scale q k^T) v, differentiable", py::arg("q"), py::arg("k"), py::arg("v"),
         py::arg("lens"), py::arg("causal"), py::arg("window"), py::arg("scale"), py::arg("p"), py::arg("seed"),
         py::arg("seed_dev"));
  auto qr = root.def_submodule("qk_norm_rope", "query / key RMS norm + rotary embedding");
  qr.def("norm_rope", &rope_call, "-> (query, key), differentiable", py::arg("q"), py::arg("k"), py::arg("wq"),
         py::arg("wk"), py::arg("cos"), py::arg("sin"), py::arg("pos"), py::arg("offset"), py::arg("eps"),
         py::arg("interleaved"));
  auto cd = root.def_submodule("counter_dropout", "Philox dropout, mask regenerated from the seed");
  cd.def("dropout", &drop_call, "differentiable any number of times", py::arg("x"), py::arg("thresh"), py::arg("scale"),
         py::arg("seed"), py::arg("seed_dev"));
}

}  // namespace bhb
