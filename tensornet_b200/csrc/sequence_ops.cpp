// Layer normalisation and attention as differentiable functions: torch's graph calls the kernels from here, so that a small call
// costs the host little.
#include "sequence_ops.h"

#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime.h>
#include <torch/csrc/autograd/custom_function.h>

#include "attention.h"
#include "tn_ops.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

void told(const char* err) {
  if (err != nullptr) throw std::runtime_error(err);
}
bool wanted(const OptTensor& t) { return t.has_value() && t->defined() && t->requires_grad(); }
// A tensor with a tangent (forward-mode differentiation), which the functions below refuse; without one, and where no graph is
// built, their kernels are called straight away.
bool dual(const at::Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
const OptTensor some(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
void once_differentiable(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " is differentiable once: its backward pass builds no graph");
}

// The runtime's status words, where a wait that runs out is told
int* status_of(const at::Tensor& status, const at::Tensor& x) {
  TORCH_CHECK(status.device() == x.device() && status.scalar_type() == at::kInt, "operands must be on the runtime's GPU, ", status.device(), ", not on ",
              x.device());
  return status.data_ptr<int>();
}

// ---- layer normalisation ------------------------------------------------------------------------------------------------------
// `t` as [rows, C], contiguous from a 16-byte boundary
at::Tensor rows16(const at::Tensor& t, int64_t C) {
  at::Tensor r = t.contiguous();
  if (reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 != 0) r = r.clone();
  return r.view({r.numel() / C, C});
}
float* column_vec(const OptTensor& v, const at::Tensor& x, const char* what, at::Tensor& keep) {
  if (!v || !v->defined()) return nullptr;
  TORCH_CHECK(v->device() == x.device() && v->scalar_type() == at::kFloat && v->dim() == 1 && v->numel() == x.size(-1),
              "layer_norm: ", what, " must be fp32, one value per column");
  keep = v->contiguous();
  return keep.data_ptr<float>();
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static tn::LayerNormArgs args_of(const at::Tensor& x) {
    TORCH_CHECK(x.is_cuda() && (x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf),
                "layer_norm: fp32, bf16 or fp16 rows on the GPU");
    TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= (1LL << 30), "layer_norm: too many columns");
    tn::LayerNormArgs a{};
    a.kind = x.scalar_type() == at::kFloat ? 0 : x.scalar_type() == at::kBFloat16 ? 1 : 2;
    a.rows = x.size(0); a.C = (int)x.size(1); a.x = x.data_ptr();
    return a;
  }

  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& gamma, const OptTensor& beta, double eps, const at::Tensor& status, bool keep) {
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t C = x.size(-1);
    at::Tensor x2 = rows16(x, C), y = at::empty(x.sizes(), x.options()), stats, kg, kb;      // (y is no view: it may be changed in place)
    tn::LayerNormArgs a = args_of(x2);
    a.gamma = column_vec(gamma, x, "gamma", kg); a.beta = column_vec(beta, x, "beta", kb);
    a.eps = (float)eps; a.y = y.data_ptr(); a.status = status_of(status, x);
    if (keep) {
      stats = at::empty({2, a.rows}, x2.options().dtype(at::kFloat));
      a.stats = stats.data_ptr<float>();
    }
    if (a.rows > 0) told(tn::launch_layer_norm_fwd(a, counted_stream()));
    if (keep) {
      const bool has_gamma = gamma && gamma->defined(), has_beta = beta && beta->defined();
      ctx->save_for_backward({x2.data_ptr() == x.data_ptr() ? x : x2, stats, has_gamma ? *gamma : at::Tensor()});
      ctx->saved_data["gamma"] = has_gamma ? 1 : -1;                      // the place among the arguments that are tensors
      ctx->saved_data["status"] = status;
      ctx->saved_data["beta"] = has_beta ? (has_gamma ? 2 : 1) : -1;
    }
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_differentiable("layer_norm");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &stats = saved[1], &gamma = saved[2];
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t C = x.size(-1);
    at::Tensor x2 = x.view({x.numel() / C, C}), dy = rows16(grads[0], C), kg, dx, dg, db, part;
    tn::LayerNormArgs a = args_of(x2);
    a.status = status_of(ctx->saved_data["status"].toTensor(), x);
    a.dy = dy.data_ptr(); a.stats = stats.data_ptr<float>(); a.gamma = column_vec(some(gamma), x2, "gamma", kg);
    const auto f32 = x2.options().dtype(at::kFloat);
    if (ctx->needs_input_grad(0)) { dx = at::empty_like(x2); a.dx = dx.data_ptr(); }
    auto needed = [&](const char* name) { const int64_t i = ctx->saved_data[name].toInt(); return i >= 0 && ctx->needs_input_grad((size_t)i); };
    if (needed("gamma")) { dg = at::empty({C}, f32); a.dgamma = dg.data_ptr<float>(); }
    if (needed("beta")) { db = at::empty({C}, f32); a.dbeta = db.data_ptr<float>(); }
    if (a.rows > 0) {
      if (a.dgamma || a.dbeta) {
        part = at::empty({(int64_t)tn::layer_norm_part_rows(a), 2, C}, f32);
        a.part = part.data_ptr<float>();
        count_launches(1);
      }
      told(tn::launch_layer_norm_bwd(a, counted_stream()));
    } else {
      if (dg.defined()) dg.zero_();
      if (db.defined()) db.zero_();
    }
    return {dx.defined() ? dx.view(grads[0].sizes()) : dx, dg, db, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

at::Tensor layer_norm(const at::Tensor& x, const OptTensor& gamma, const OptTensor& beta, double eps, const at::Tensor& status) {
  const bool keep = at::GradMode::is_enabled() && (x.requires_grad() || wanted(gamma) || wanted(beta));
  if (!keep && !dual(x) && !(gamma && dual(*gamma)) && !(beta && dual(*beta))) return LayerNorm::forward(nullptr, x, gamma, beta, eps, status, false);
  return LayerNorm::apply(x, gamma, beta, eps, status, keep);
}

// ---- attention ------------------------------------------------------------------------------------------------------------------
// The operand in a form that the kernels read: columns behind one another, rows and heads from 16-byte boundaries.  [N, H, D] or
// [B, T, H, D].
at::Tensor operand(const at::Tensor& t) {
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) ok = ok && (t.size(d) == 1 || (t.stride(d) > 0 && t.stride(d) % 8 == 0));
  if (ok) return t;
  at::Tensor c = t.contiguous();
  return c.data_ptr() == t.data_ptr() ? t.clone(at::MemoryFormat::Contiguous) : c;
}
tn::AttnOperand view_of(const at::Tensor& t) {
  const int64_t n = t.dim();
  tn::AttnOperand o{};
  o.p = t.data_ptr();
  o.sh = t.size(-2) > 1 ? t.stride(-2) : t.size(-1);
  o.st = t.size(n - 3) > 1 ? t.stride(n - 3) : t.size(-1) * t.size(-2);
  o.sb = n == 4 ? (t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2) * t.size(3)) : 0;
  return o;
}
const int* ints_of(const OptTensor& t, const at::Tensor& q, int64_t n, const char* what) {
  if (!t || !t->defined()) return nullptr;
  TORCH_CHECK(t->device() == q.device() && t->scalar_type() == at::kInt && t->is_contiguous() && t->numel() == n, "attention: ", what, " must be ",
              n, " contiguous int32 values on the operands' GPU");
  return t->data_ptr<int>();
}

struct Attention : torch::autograd::Function<Attention> {
  static tn::AttnArgs args_of(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptTensor& q_rows, const OptTensor& k_rows,
                              const OptTensor& prefix, const OptTensor& slopes, bool causal, bool newest, double cap, double scale, const at::Tensor& status) {
    for (const at::Tensor* t : {&q, &k, &v})
      TORCH_CHECK(t->is_cuda() && t->device() == q.device() && t->scalar_type() == at::kBFloat16 && (t->dim() == 3 || t->dim() == 4) &&
                      t->size(-1) == q.size(-1), "attention: bf16 operands [N, heads, columns] or [B, T, heads, columns] on one GPU");
    TORCH_CHECK(k.sizes() == v.sizes(), "attention: keys and values differ in shape");
    TORCH_CHECK(q.size(-1) % 8 == 0 && q.size(-1) >= 8 && q.size(-1) <= 128, "attention: 8 to 128 columns, a multiple of 8");
    TORCH_CHECK(k.size(-2) >= 1 && q.size(-2) % k.size(-2) == 0 && q.size(-2) <= 65535, "attention: query heads must be a multiple of the key heads");
    tn::AttnArgs a{};
    a.H = (int)q.size(-2); a.G = (int)k.size(-2); a.D = (int)q.size(-1);
    const bool pq = q.dim() == 3, pk = k.dim() == 3;
    TORCH_CHECK(!pq || q_rows, "attention: packed queries need their offsets");
    TORCH_CHECK(!pk || k_rows, "attention: packed keys need their offsets");
    const int64_t B = pq ? q_rows->numel() - 1 : q.size(0);
    TORCH_CHECK(B >= 0 && B == (pk ? k_rows->numel() - 1 : k.size(0)), "attention: queries and keys have different numbers of sequences");
    for (const at::Tensor* t : {&q, &k})
      TORCH_CHECK(B < (1 << 24) && (t->dim() == 3 ? t->size(0) : B * ((t->size(1) + 127) / 128 * 128)) < (1LL << 31) - (1 << 24), "attention: too many rows");
    a.B = (int)B;
    (pq ? a.rq.off : a.rq.len) = ints_of(q_rows, q, pq ? B + 1 : B, pq ? "offsets" : "lengths");
    (pk ? a.rk.off : a.rk.len) = ints_of(k_rows, q, pk ? B + 1 : B, pk ? "kv_offsets" : "kv_lengths");
    a.rq.T = (int)q.size(pq ? 0 : 1); a.rk.T = (int)k.size(pk ? 0 : 1);
    a.q = view_of(q); a.k = view_of(k); a.v = view_of(v);
    a.prefix = ints_of(prefix, q, B, "prefix");
    if (slopes && slopes->defined()) {
      TORCH_CHECK(slopes->device() == q.device() && slopes->scalar_type() == at::kFloat && slopes->is_contiguous() && slopes->numel() == a.H,
                  "attention: slopes must be fp32, one per query head");
      a.slopes = slopes->data_ptr<float>();
    }
    TORCH_CHECK(!(causal && newest), "attention: newest queries see all keys, causal ones do not");
    a.causal = causal; a.newest = newest; a.step = newest ? 0.f : 1.f; a.cap = (float)cap; a.scale = (float)scale; a.status = status_of(status, q);
    return a;
  }

  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in, const OptTensor& q_rows,
                            const OptTensor& k_rows, const OptTensor& prefix, const OptTensor& slopes, bool causal, bool newest, double cap, double scale,
                            const at::Tensor& status, bool keep) {
    c10::cuda::CUDAGuard guard(q_in.device());
    const at::Tensor q = operand(q_in), k = operand(k_in), v = operand(v_in);
    tn::AttnArgs a = args_of(q, k, v, q_rows, k_rows, prefix, slopes, causal, newest, cap, scale, status);
    at::Tensor out = at::empty(q.sizes(), q.options()), lse, rest;
    a.o = view_of(out);
    if (out.numel() > 0 && k.numel() == 0) out.zero_();
    if (out.numel() > 0 && k.numel() > 0) {
      if (keep) {
        lse = at::empty({a.H, q.numel() / (a.H * a.D)}, q.options().dtype(at::kFloat));
        a.lse = lse.data_ptr<float>();
        rest = at::empty_like(out);
        a.rest = view_of(rest);
      }
      if (tn::attention_few_takes(a)) {
        at::Tensor work;
        if (const long long n = tn::attention_few_floats(a)) {
          work = at::empty({n}, q.options().dtype(at::kFloat));
          count_launches(1);
        }
        told(tn::launch_attention_few(a, work.defined() ? work.data_ptr<float>() : nullptr, counted_stream()));
      } else if (tn::attention_short_takes(a, false)) {
        told(tn::launch_attention_short_fwd(a, counted_stream()));
      } else {
        told(tn::launch_attention_fwd(a, counted_stream()));
      }
    }
    if (keep) {
      auto opt = [](const OptTensor& t) { return t ? *t : at::Tensor(); };
      ctx->save_for_backward({q, k, v, out, lse, rest, opt(q_rows), opt(k_rows), opt(prefix), opt(slopes)});
      ctx->saved_data["causal"] = causal;
      ctx->saved_data["newest"] = newest;
      ctx->saved_data["cap"] = cap;
      ctx->saved_data["scale"] = scale;
      ctx->saved_data["status"] = status;
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_differentiable("attention");
    const auto s = ctx->get_saved_variables();
    const at::Tensor &q = s[0], &k = s[1], &v = s[2], &out = s[3], &lse = s[4], &rest = s[5];
    c10::cuda::CUDAGuard guard(q.device());
    const at::Tensor go = operand(grads[0]);
    tn::AttnArgs a = args_of(q, k, v, some(s[6]), some(s[7]), some(s[8]), some(s[9]), ctx->saved_data["causal"].toBool(),
                             ctx->saved_data["newest"].toBool(), ctx->saved_data["cap"].toDouble(), ctx->saved_data["scale"].toDouble(),
                             ctx->saved_data["status"].toTensor());
    TORCH_CHECK(go.scalar_type() == at::kBFloat16 && go.sizes() == q.sizes(), "attention: the output's gradient must be like the output");
    at::Tensor gq = at::empty(q.sizes(), q.options()), gk = at::empty(k.sizes(), k.options()), gv = at::empty(v.sizes(), v.options());
    if (q.numel() > 0 && k.numel() > 0) {
      at::Tensor delta = at::empty_like(lse);
      a.o = view_of(out); a.rest = view_of(rest); a.go = view_of(go); a.gq = view_of(gq); a.gk = view_of(gk); a.gv = view_of(gv);
      a.lse = lse.data_ptr<float>(); a.delta = delta.data_ptr<float>();
      count_launches(1);
      told(tn::launch_attention_bwd(a, counted_stream()));
    } else {
      for (at::Tensor* t : {&gq, &gk, &gv}) t->zero_();
    }
    variable_list r(13);
    if (ctx->needs_input_grad(0)) r[0] = gq;
    if (ctx->needs_input_grad(1)) r[1] = gk;
    if (ctx->needs_input_grad(2)) r[2] = gv;
    return r;
  }
};

at::Tensor attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const OptTensor& q_rows, const OptTensor& k_rows,
                     const OptTensor& prefix, const OptTensor& slopes, bool causal, bool newest, double cap, double scale, const at::Tensor& status) {
  const bool keep = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
  if (!keep && !dual(q) && !dual(k) && !dual(v))
    return Attention::forward(nullptr, q, k, v, q_rows, k_rows, prefix, slopes, causal, newest, cap, scale, status, false);
  return Attention::apply(q, k, v, q_rows, k_rows, prefix, slopes, causal, newest, cap, scale, status, keep);
}

}  // namespace

void bind_sequence_ops(pybind11::module& m) {
  m.def("layer_norm", &layer_norm);
  m.def("attention", &attention);
}
