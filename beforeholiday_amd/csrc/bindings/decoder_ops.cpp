// Grouped-query attention (kernels/grouped_attn.hip), query / key norm + rotary embedding
// (kernels/qk_norm_rope.hip) and counter-based dropout (kernels/counter_dropout.hip). Every call checks its
// operands here, runs on the current stream of the operands' device and allocates what it needs per call.
#include "common.h"

#include <cmath>

#include "bh/grouped_attn_api.h"
#include "bh/qk_rope_api.h"

namespace bhb {
namespace {

constexpr int64_t kMaxLen = int64_t(1) << 29;     // queries / keys of a sequence
constexpr int64_t kMaxStride = int64_t(1) << 24;  // elements between two positions (block offsets are 32-bit)
constexpr int64_t kMaxGrid = (int64_t(1) << 31) - 1;

const int64_t* step_seed(const c10::optional<at::Tensor>& t, const at::Tensor& like, const char* what) {
  if (!t.has_value() || !t->defined()) return nullptr;
  TORCH_CHECK(t->scalar_type() == at::kLong && t->numel() == 1 && t->device() == like.device(), what,
              ": seed_dev must be an int64 [1] tensor on the operands' device");
  return t->data_ptr<int64_t>();
}

bh::GaView ga_view(const at::Tensor& t, const at::Tensor& like, const char* name) {
  check_cuda(t, name);
  TORCH_CHECK(t.dim() == 4, "grouped attention: ", name, " must be [s, b, heads, head_dim]");
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == like.scalar_type(), "grouped attention: ", name,
              " must have the query's device and dtype");
  TORCH_CHECK(t.stride(3) == 1, "grouped attention: ", name, " must be contiguous along head_dim");
  bh::GaView v;
  v.p = t.data_ptr();
  const int64_t hn = t.size(3);
  v.st = t.size(0) > 1 ? t.stride(0) : hn;  // a single position: its stride is never used, any value may be there
  v.sb = t.size(1) > 1 ? t.stride(1) : 0;
  v.sh = t.size(2) > 1 ? t.stride(2) : 0;
  TORCH_CHECK(v.st % 8 == 0 && v.sb % 8 == 0 && v.sh % 8 == 0 && reinterpret_cast<uintptr_t>(v.p) % 16 == 0,
              "grouped attention: ", name, " strides must be multiples of 8 elements and its base 16-byte aligned");
  TORCH_CHECK(v.st >= hn && v.st < kMaxStride, "grouped attention: ", name, " position stride must be in [head_dim, 2^24)");
  return v;
}

bh::GaArgs ga_args(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool causal, int64_t window,
                   const c10::optional<at::Tensor>& lens, double scale, double p, int64_t seed,
                   const c10::optional<at::Tensor>& seed_dev) {
  TORCH_CHECK(q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16,
              "grouped attention: fp16 / bf16 tensors only on the GPU, got ", q.scalar_type());
  bh::GaArgs a;
  a.q = ga_view(q, q, "query");
  a.k = ga_view(k, q, "key");
  a.v = ga_view(v, q, "value");
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(1) == q.size(1) && k.size(3) == q.size(3),
              "grouped attention: query ", q.sizes(), ", key ", k.sizes(), " and value ", v.sizes(), " do not fit");
  TORCH_CHECK(k.size(2) >= 1 && q.size(2) >= 1 && q.size(2) % k.size(2) == 0,
              "grouped attention: query heads (", q.size(2), ") must be a multiple of key heads (", k.size(2), ")");
  TORCH_CHECK(q.size(3) >= 8 && q.size(3) <= 128 && q.size(3) % 8 == 0,
              "grouped attention: head_dim must be a multiple of 8 up to 128, got ", q.size(3));
  TORCH_CHECK(q.size(0) <= kMaxLen && k.size(0) <= kMaxLen, "grouped attention: sequences of up to 2^29 only");
  TORCH_CHECK(std::isfinite(scale) && scale > 0, "grouped attention: scale must be positive, got ", scale);
  TORCH_CHECK(p >= 0 && p < 1, "grouped attention: dropout must be in [0, 1), got ", p);
  a.sq = (int)q.size(0); a.b = (int)q.size(1); a.np = (int)q.size(2); a.hn = (int)q.size(3);
  a.sk = (int)k.size(0); a.ng = (int)k.size(2);
  TORCH_CHECK(q.size(1) * q.size(2) * ((q.size(0) + 15) / 16 + (k.size(0) + 15) / 16) <= kMaxGrid,
              "grouped attention: too many rows for one launch");
  a.causal = causal;
  TORCH_CHECK(window == 0 || (causal && window > 0), "grouped attention: a window needs causal and at least one key");
  a.window = (int)(window > 0 ? std::min(window, 2 * kMaxLen) : 2 * kMaxLen);
  if (lens.has_value() && lens->defined()) {
    TORCH_CHECK(lens->device() == q.device() && lens->scalar_type() == at::kInt && lens->dim() == 1 &&
                    lens->size(0) == q.size(1) && lens->is_contiguous(),
                "grouped attention: key_lengths must be a contiguous int32 [batch] tensor on the query's device");
    a.lens = lens->data_ptr<int>();
  }
  a.scale = (float)scale;
  a.p_drop = (float)p;
  a.seed = (uint64_t)seed;
  a.seed_dev = step_seed(seed_dev, q, "grouped attention");
  return a;
}

std::vector<at::Tensor> ga_fwd(at::Tensor q, at::Tensor k, at::Tensor v, bool causal, int64_t window,
                               c10::optional<at::Tensor> lens, double scale, double p, int64_t seed,
                               c10::optional<at::Tensor> seed_dev) {
  auto a = ga_args(q, k, v, causal, window, lens, scale, p, seed, seed_dev);
  const c10::DeviceGuard guard(q.device());
  auto o = at::empty(q.sizes(), q.options());
  auto lse = at::empty({q.size(1), q.size(2), q.size(0)}, q.options().dtype(at::kFloat));
  if (o.numel() == 0) return {o, lse};
  if (a.sk == 0) return {o.zero_(), lse.fill_(INFINITY)};
  a.o = ga_view(o, q, "output");
  a.lse = lse.data_ptr<float>();
  const int64_t n = bh::ga_forward_workspace(a);
  at::Tensor ws = n ? at::empty({n}, lse.options()) : at::Tensor();
  bh::ga_forward(dtype_code(q.scalar_type()), a, n ? ws.data_ptr<float>() : nullptr, stream_for(q));
  return {o, lse};
}

std::vector<c10::optional<at::Tensor>> ga_bwd(at::Tensor dout, at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor o,
                                              at::Tensor lse, bool causal, int64_t window,
                                              c10::optional<at::Tensor> lens, double scale, double p, int64_t seed,
                                              c10::optional<at::Tensor> seed_dev, bool need_q, bool need_kv) {
  auto a = ga_args(q, k, v, causal, window, lens, scale, p, seed, seed_dev);
  TORCH_CHECK(dout.sizes() == q.sizes() && o.sizes() == q.sizes(), "grouped attention: output / gradient shape mismatch");
  TORCH_CHECK(lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                  lse.numel() == q.size(0) * q.size(1) * q.size(2),
              "grouped attention: lse must be the forward's [b, heads, s] fp32 tensor");
  const c10::DeviceGuard guard(q.device());
  c10::optional<at::Tensor> dq, dk, dv;
  if (need_q) dq = at::empty(q.sizes(), q.options());
  if (need_kv) {
    dk = at::empty(k.sizes(), k.options());
    dv = at::empty(v.sizes(), v.options());
  }
  if (q.numel() == 0 || a.sk == 0) {
    if (need_q) dq->zero_();
    if (need_kv) {
      dk->zero_();
      dv->zero_();
    }
    return {dq, dk, dv};
  }
  a.dout = ga_view(dout, q, "output gradient");
  a.o = ga_view(o, q, "output");
  if (need_q) a.dq = ga_view(*dq, q, "dq");
  if (need_kv) {
    a.dk = ga_view(*dk, q, "dk");
    a.dv = ga_view(*dv, q, "dv");
  }
  auto delta = at::empty_like(lse);
  a.lse = lse.data_ptr<float>();
  a.delta = delta.data_ptr<float>();
  at::Tensor rowh;
  if (a.p_drop > 0.f) {
    rowh = at::empty(lse.sizes(), lse.options().dtype(at::kInt));
    a.rowh = reinterpret_cast<uint32_t*>(rowh.data_ptr());
  }
  bh::ga_backward(dtype_code(q.scalar_type()), a, stream_for(q));
  return {dq, dk, dv};
}

// ---- query / key norm + rotary embedding ---------------------------------------------------------------------
bool rope_view(const at::Tensor& t, const at::Tensor& like, const char* name, bh::HeadView& v) {
  check_cuda(t, name);
  TORCH_CHECK(t.dim() == 4, "qk_norm_rope: ", name, " must be [s, b, heads, head_dim]");
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == like.scalar_type(), "qk_norm_rope: ", name,
              " must have the query's device and dtype");
  TORCH_CHECK(t.stride(3) == 1, "qk_norm_rope: ", name, " must be contiguous along head_dim");
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
  TORCH_CHECK(q.scalar_type() == at::kFloat || q.scalar_type() == at::kHalf || q.scalar_type() == at::kBFloat16,
              "qk_norm_rope: fp32 / fp16 / bf16 tensors only on the GPU, got ", q.scalar_type());
  bh::QkRopeArgs a;
  bool vec = rope_view(q, q, "query", a.x[0]);
  vec = rope_view(k, q, "key", a.x[1]) && vec;
  const int64_t hn = q.size(3);
  TORCH_CHECK(k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == hn, "qk_norm_rope: query ", q.sizes(),
              " and key ", k.sizes(), " do not fit");
  TORCH_CHECK(hn >= 2 && hn <= 512 && hn % 2 == 0, "qk_norm_rope: head_dim must be even and at most 512, got ", hn);
  TORCH_CHECK(q.size(0) * q.size(1) <= 4 * kMaxGrid && q.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX &&
                  q.size(2) <= kMaxLen && k.size(2) <= kMaxLen,
              "qk_norm_rope: too many tokens or heads");
  a.s = (int)q.size(0); a.b = (int)q.size(1); a.hn = (int)hn;
  a.heads[0] = (int)q.size(2); a.heads[1] = (int)k.size(2);
  const bool norm = wq.has_value() && wq->defined();
  TORCH_CHECK(norm == (wk.has_value() && wk->defined()), "qk_norm_rope: give both norm weights or none");
  if (norm) {
    for (const auto* w : {&*wq, &*wk}) {
      TORCH_CHECK(w->device() == q.device() && w->dim() == 1 && w->size(0) == hn && w->is_contiguous() &&
                      w->scalar_type() == wq->scalar_type(),
                  "qk_norm_rope: norm weights must be contiguous [head_dim] tensors of one dtype on the query's device");
      TORCH_CHECK(w->scalar_type() == at::kFloat || w->scalar_type() == at::kHalf || w->scalar_type() == at::kBFloat16,
                  "qk_norm_rope: norm weights must be fp32 / fp16 / bf16");
      vec = vec && reinterpret_cast<uintptr_t>(w->data_ptr()) % (4 * w->element_size()) == 0;
    }
    a.w[0] = wq->data_ptr();
    a.w[1] = wk->data_ptr();
    a.w_dt = dtype_code(wq->scalar_type());
    TORCH_CHECK(eps >= 0 && std::isfinite(eps), "qk_norm_rope: eps must be >= 0");
  }
  const bool rot = cos.has_value() && cos->defined();
  TORCH_CHECK(rot == (sin.has_value() && sin->defined()), "qk_norm_rope: give both angle tables or none");
  TORCH_CHECK(norm || rot, "qk_norm_rope: neither norm weights nor angle tables");
  if (rot) {
    for (const auto* c : {&*cos, &*sin})
      TORCH_CHECK(c->device() == q.device() && c->scalar_type() == at::kFloat && c->dim() == 2 && c->is_contiguous() &&
                      c->sizes() == cos->sizes(),
                  "qk_norm_rope: cos / sin must be contiguous fp32 [positions, rot / 2] tables on the query's device");
    TORCH_CHECK(cos->size(1) >= 1 && 2 * cos->size(1) <= hn, "qk_norm_rope: the tables rotate ", 2 * cos->size(1),
                " of ", hn, " values");
    a.cos = cos->data_ptr<float>();
    a.sin = sin->data_ptr<float>();
    a.rot = (int)(2 * cos->size(1));
    a.n_pos = cos->size(0);
    if (pos.has_value() && pos->defined()) {
      TORCH_CHECK(pos->device() == q.device() && (pos->scalar_type() == at::kLong || pos->scalar_type() == at::kInt) &&
                      ((pos->dim() == 1 && pos->size(0) == q.size(0)) ||
                       (pos->dim() == 2 && pos->size(0) == q.size(0) && pos->size(1) == q.size(1))),
                  "qk_norm_rope: positions must be an int32 / int64 [s] or [s, b] tensor on the query's device");
      a.pos = pos->data_ptr();
      a.pos_i64 = pos->scalar_type() == at::kLong;
      a.pos_st = pos->stride(0);
      a.pos_sb = pos->dim() == 2 ? pos->stride(1) : 0;
      TORCH_CHECK(offset == 0, "qk_norm_rope: an offset goes without positions");
    } else {
      TORCH_CHECK(offset >= 0 && offset + q.size(0) <= a.n_pos, "qk_norm_rope: positions ", offset, " .. ",
                  offset + q.size(0) - 1, " do not fit tables of ", a.n_pos);
      a.offset = offset;
    }
  }
  a.eps = (float)eps;
  a.interleaved = interleaved;
  a.vec = vec && hn % 8 == 0 && a.rot % 8 == 0;
  return a;
}

std::vector<at::Tensor> rope_fwd(at::Tensor q, at::Tensor k, c10::optional<at::Tensor> wq, c10::optional<at::Tensor> wk,
                                 c10::optional<at::Tensor> cos, c10::optional<at::Tensor> sin,
                                 c10::optional<at::Tensor> pos, int64_t offset, double eps, bool interleaved) {
  auto a = rope_args(q, k, wq, wk, cos, sin, pos, offset, eps, interleaved);
  const c10::DeviceGuard guard(q.device());
  auto yq = at::empty(q.sizes(), q.options()), yk = at::empty(k.sizes(), k.options());
  const bool v0 = rope_view(yq, q, "output", a.y[0]), v1 = rope_view(yk, q, "output", a.y[1]);
  a.vec = a.vec && v0 && v1;
  if (yq.numel() + yk.numel() > 0) bh::qk_rope_forward(dtype_code(q.scalar_type()), a, stream_for(q));
  return {yq, yk};
}

std::vector<at::Tensor> rope_bwd(at::Tensor dyq, at::Tensor dyk, at::Tensor q, at::Tensor k,
                                 c10::optional<at::Tensor> wq, c10::optional<at::Tensor> wk,
                                 c10::optional<at::Tensor> cos, c10::optional<at::Tensor> sin,
                                 c10::optional<at::Tensor> pos, int64_t offset, double eps, bool interleaved) {
  auto a = rope_args(q, k, wq, wk, cos, sin, pos, offset, eps, interleaved);
  TORCH_CHECK(dyq.sizes() == q.sizes() && dyk.sizes() == k.sizes(), "qk_norm_rope: gradient shape mismatch");
  const c10::DeviceGuard guard(q.device());
  auto dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
  bool vec = rope_view(dq, q, "dq", a.y[0]);
  vec = rope_view(dk, q, "dk", a.y[1]) && vec;
  vec = rope_view(dyq, q, "query gradient", a.dy[0]) && vec;
  vec = rope_view(dyk, q, "key gradient", a.dy[1]) && vec;
  a.vec = a.vec && vec;
  const auto f32 = q.options().dtype(at::kFloat);
  at::Tensor dw = a.w[0] ? at::empty({2, q.size(3)}, f32) : at::empty({0}, f32);
  if (dq.numel() + dk.numel() == 0) return {dq, dk, dw.zero_()};
  const int64_t rows = bh::qk_rope_partial_rows(a);
  at::Tensor part = at::empty({rows * 2 * q.size(3)}, f32);
  bh::qk_rope_backward(dtype_code(q.scalar_type()), a, rows ? part.data_ptr<float>() : nullptr,
                       rows ? dw.data_ptr<float>() : nullptr, stream_for(q));
  return {dq, dk, dw};
}

// ---- dropout -------------------------------------------------------------------------------------------------
at::Tensor dropout(at::Tensor x, int64_t thresh, double scale, int64_t seed, c10::optional<at::Tensor> seed_dev) {
  check_cuda(x, "dropout input");
  TORCH_CHECK(x.is_contiguous(), "counter_dropout: contiguous input only");
  TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16,
              "counter_dropout: fp32 / fp16 / bf16 tensors only on the GPU, got ", x.scalar_type());
  TORCH_CHECK(thresh >= 0 && thresh <= UINT32_MAX, "counter_dropout: bad threshold");
  const int64_t* sd = step_seed(seed_dev, x, "counter_dropout");
  const c10::DeviceGuard guard(x.device());
  auto y = at::empty(x.sizes(), x.options());
  bh::counter_dropout(dtype_code(x.scalar_type()), x.data_ptr(), y.data_ptr(), x.numel(), (uint32_t)thresh,
                      (float)scale, (uint64_t)seed, sd, stream_for(x));
  return y;
}

}  // namespace

void register_decoder_ops(pybind11::module_& root) {
  namespace py = pybind11;
  auto ga = root.def_submodule("grouped_attention", "grouped-query attention, head sizes up to 128");
  ga.def("forward", &ga_fwd, "-> (o, lse)", py::arg("q"), py::arg("k"), py::arg("v"), py::arg("causal"),
         py::arg("window"), py::arg("lens"), py::arg("scale"), py::arg("p"), py::arg("seed"), py::arg("seed_dev"));
  ga.def("backward", &ga_bwd, "-> (dq, dk, dv)", py::arg("dout"), py::arg("q"), py::arg("k"), py::arg("v"),
         py::arg("o"), py::arg("lse"), py::arg("causal"), py::arg("window"), py::arg("lens"), py::arg("scale"),
         py::arg("p"), py::arg("seed"), py::arg("seed_dev"), py::arg("need_q") = true, py::arg("need_kv") = true);
  auto qr = root.def_submodule("qk_norm_rope", "query / key RMS norm + rotary embedding");
  qr.def("forward", &rope_fwd, "-> (query, key)", py::arg("q"), py::arg("k"), py::arg("wq"), py::arg("wk"),
         py::arg("cos"), py::arg("sin"), py::arg("pos"), py::arg("offset"), py::arg("eps"), py::arg("interleaved"));
  qr.def("backward", &rope_bwd, "-> (dq, dk, dw [2, head_dim])", py::arg("dyq"), py::arg("dyk"), py::arg("q"),
         py::arg("k"), py::arg("wq"), py::arg("wk"), py::arg("cos"), py::arg("sin"), py::arg("pos"), py::arg("offset"),
         py::arg("eps"), py::arg("interleaved"));
  auto cd = root.def_submodule("counter_dropout", "Philox dropout, mask regenerated from the seed");
  cd.def("apply", &dropout, py::arg("x"), py::arg("thresh"), py::arg("scale"), py::arg("seed"), py::arg("seed_dev"));
}

}  // namespace bhb
