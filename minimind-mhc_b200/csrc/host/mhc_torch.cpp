// Host side of the training-step operators for PyTorch: argument checks, allocations
// and autograd nodes around the C entry points.
//
// A small pass of these operators takes the GPU 3 to 10 us.  With the same host work
// done in Python a call of 77 tokens' attention took 38 us (19 from here), a router's
// forward and backward 110 (72, most of it autograd.grad's own) and a clipped AdamW
// step over 14 tensors 57 (20).  The library itself stays free of
// PyTorch: this file is compiled against its C header only and receives the entry
// points' addresses (bind), so it works on whichever library the process has loaded.
#include <ATen/autocast_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>
#include <string>
#include <vector>

#include "mhc_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entry {
  decltype(&mhc_last_error) last_error;
  decltype(&mhc_attn_lse_pitch) attn_lse_pitch;
  decltype(&mhc_attn_fwd_workspace) attn_fwd_workspace;
  decltype(&mhc_attn_fwd) attn_fwd;
  decltype(&mhc_attn_bwd_workspace) attn_bwd_workspace;
  decltype(&mhc_attn_bwd) attn_bwd;
  decltype(&mhc_route_fwd_workspace) route_fwd_workspace;
  decltype(&mhc_route_fwd) route_fwd;
  decltype(&mhc_route_bwd) route_bwd;
  decltype(&mhc_grad_norm_workspace) grad_norm_workspace;
  decltype(&mhc_grad_norm) grad_norm;
  decltype(&mhc_adamw_check) adamw_check;
  decltype(&mhc_adamw_step) adamw_step;
  decltype(&mhc_rotate) rotate;
  decltype(&mhc_append_kv) append_kv;
  decltype(&mhc_keep_drafts) keep_drafts;
  decltype(&mhc_cached_attn_workspace) cached_attn_workspace;
  decltype(&mhc_cached_attn) cached_attn;
  decltype(&mhc_verify_drafts) verify_drafts;
} E{};
volatile int *give_up_flag = nullptr;  // the pinned word a kernel whose bounded wait ran out writes to

void bind(const std::vector<uintptr_t> &a) {
  TORCH_CHECK(a.size() * sizeof(uintptr_t) == sizeof(Entry), "bind: ", a.size(), " entry points");
  std::memcpy(&E, a.data(), sizeof(Entry));
}
void set_flag(uintptr_t p) { give_up_flag = reinterpret_cast<volatile int *>(p); }

// Before every call: an earlier kernel's give-up is raised here.
void ready() {
  TORCH_CHECK(E.last_error, "the mHC native library is not bound");
  const int code = give_up_flag ? *give_up_flag : 0;
  TORCH_CHECK(code == 0, "an mHC kernel gave up on a bounded device wait (code ", code,
              "); the outputs it owned were overwritten with NaN.  Call model._native.clear_device_error() to continue.");
}
void check(int status, const char *what) { TORCH_CHECK(status == 0, what, " failed with status ", status, ": ", E.last_error()); }

int dtype_code(const Tensor &t, const char *who) {
  switch (t.scalar_type()) {
    case at::kFloat: return MHC_F32;
    case at::kBFloat16: return MHC_BF16;
    case at::kHalf: return MHC_F16;
    default: TORCH_CHECK_TYPE(false, who, ": mHC kernels support float32/bfloat16/float16, got ", t.scalar_type());
  }
}
void require_cuda(const Tensor &t) {
  TORCH_CHECK(t.is_cuda(), "mHC B200 kernels run on CUDA tensors only (this build has no CPU path); got a tensor on ", t.device());
}
// What would pass through a call without a trace of it: a tangent (a dual tensor does not require grad, so the call
// would not meet the autograd node, which refuses it), and the launches themselves under a tracer, which sees the
// allocation of the outputs only.
void require_plain(const char *who, std::initializer_list<const Tensor *> ts) {
  for (const Tensor *t : ts)
    TORCH_CHECK(!t->_fw_grad(0).defined(), who, ": forward-mode derivatives are not implemented");
  TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                  !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
              who, " cannot be traced: its kernels are launched outside of torch's operators");
}
void *stream_of(const Tensor &t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
Tensor scratch(const Tensor &like, size_t bytes) { return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)); }
void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// ---- attention -----------------------------------------------------------------

// x (T, heads, D) as the kernels read it: any token and head strides, but contiguous
// rows, and for 16-bit types what TMA can address (rows that begin at multiples of 16
// bytes, heads that do not overlap), where a copy costs less than the kernels that do
// without.
Tensor rows(const Tensor &x) {
  const int64_t st = x.stride(0), sh = x.stride(1), h = x.size(1), d = x.size(2);
  if (x.stride(2) != 1 && d != 1) return x.contiguous();
  if (x.element_size() == 2 && d % 8 == 0 &&
      (st % 8 || sh % 8 || reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 || (h > 1 && sh < d)))
    return x.contiguous();
  return x;
}

struct Attended {
  Tensor q, k, v, out, out_lo, lse;
};
Attended attend(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &cu, int64_t seqlen, double scale,
                bool for_grad) {
  ready();
  const c10::cuda::CUDAGuard guard(q_.device());
  Attended a{rows(q_), rows(k_), rows(v_), {}, {}, {}};
  const int64_t t = a.q.size(0), h = a.q.size(1), d = a.q.size(2), hk = a.k.size(1);
  a.out = at::empty({t, h, d}, a.q.options());
  // the backward's row sums use out before its rounding to 16 bits
  if (for_grad && a.q.scalar_type() != at::kFloat) a.out_lo = at::empty({t, h, d}, a.q.options());
  a.lse = at::empty({h, E.attn_lse_pitch(t)}, a.q.options().dtype(at::kFloat));
  const size_t need = E.attn_fwd_workspace(t);
  const Tensor ws = scratch(a.q, need);
  const int64_t strides[6] = {a.q.stride(0), a.q.stride(1), a.k.stride(0), a.k.stride(1), a.v.stride(0), a.v.stride(1)};
  check(E.attn_fwd(a.q.data_ptr(), a.k.data_ptr(), a.v.data_ptr(), dtype_code(a.q, "packed_attention"), t, (int)h, (int)hk,
                   (int)d, strides, static_cast<const int32_t *>(ptr(cu)), cu.defined() ? (int)cu.numel() - 1 : 0, seqlen,
                   (float)scale, a.out.data_ptr(), ptr(a.out_lo), a.lse.data_ptr<float>(), ws.data_ptr(), need, stream_of(a.q)),
        "mhc_attn_fwd");
  return a;
}

struct AttentionFn : torch::autograd::Function<AttentionFn> {
  static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v,
                        const std::optional<Tensor> &cu_seqlens, int64_t seqlen, double scale) {
    const Tensor cu = cu_seqlens.value_or(Tensor());
    const Attended a = attend(q, k, v, cu, seqlen, scale, true);
    ctx->save_for_backward({a.q, a.k, a.v, cu, a.out, a.out_lo, a.lse});
    ctx->saved_data["seqlen"] = seqlen;
    ctx->saved_data["scale"] = scale;
    return a.out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "packed_attention: second derivatives are not implemented");
    ready();
    const variable_list s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2], &cu = s[3], &out = s[4], &out_lo = s[5], &lse = s[6];
    const c10::cuda::CUDAGuard guard(q.device());
    const int64_t t = q.size(0), h = q.size(1), d = q.size(2), hk = k.size(1), seqlen = ctx->saved_data["seqlen"].toInt();
    const double scale = ctx->saved_data["scale"].toDouble();
    // contiguous, and for 16-bit types at a multiple of 16 bytes, as rows() has it
    Tensor dout = g[0].contiguous();
    if (dout.element_size() == 2 && d % 8 == 0 && reinterpret_cast<uintptr_t>(dout.data_ptr()) % 16) dout = dout.clone();
    // those that this backward is asked for; dk and dv come from one kernel
    Tensor dq, dk, dv;
    if (ctx->needs_input_grad(0)) dq = at::empty({t, h, d}, q.options());
    if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2)) {
      dk = at::empty({t, hk, d}, q.options());
      dv = at::empty({t, hk, d}, q.options());
    }
    const size_t need = E.attn_bwd_workspace(t, (int)h, (int)hk, (int)d);
    const Tensor ws = scratch(q, need);
    const int64_t strides[6] = {q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1)};
    check(E.attn_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), ptr(out_lo), dout.data_ptr(), lse.data_ptr<float>(),
                     dtype_code(q, "packed_attention"), t, (int)h, (int)hk, (int)d, strides, static_cast<const int32_t *>(ptr(cu)),
                     cu.defined() ? (int)cu.numel() - 1 : 0, seqlen, (float)scale, ptr(dq), ptr(dk), ptr(dv),
                     ws.data_ptr(), need, stream_of(q)),
          "mhc_attn_bwd");
    return {dq, dk, dv, Tensor(), Tensor(), Tensor()};
  }
};

Tensor packed_attention(Tensor q, Tensor k, Tensor v, const std::optional<Tensor> &cu_seqlens, std::optional<double> scale_) {
  const char *who = "packed_attention";
  require_plain(who, {&q, &k, &v});
  if (at::autocast::is_autocast_enabled(at::kCUDA)) {  // as scaled_dot_product_attention under autocast
    const at::ScalarType to = at::autocast::get_autocast_dtype(at::kCUDA);
    q = at::autocast::cached_cast(to, q, at::kCUDA);
    k = at::autocast::cached_cast(to, k, at::kCUDA);
    v = at::autocast::cached_cast(to, v, at::kCUDA);
  }
  const bool packed = cu_seqlens.has_value();
  for (const Tensor *t : {&q, &k, &v}) require_cuda(*t);
  if (packed) require_cuda(*cu_seqlens);
  TORCH_CHECK_TYPE(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), who,
                   ": q, k and v must have one type, got ", q.scalar_type(), ", ", k.scalar_type(), ", ", v.scalar_type());
  dtype_code(q, who);
  TORCH_CHECK_VALUE(q.device() == k.device() && q.device() == v.device() && (!packed || cu_seqlens->device() == q.device()), who,
                    ": q, k, v and cu_seqlens must be on one device");
  const int64_t want = packed ? 3 : 4;
  TORCH_CHECK_VALUE(q.dim() == want && k.dim() == want && v.dim() == want, who,
                    ": (T, heads, D) tensors with cu_seqlens or (B, L, heads, D) tensors without are wanted, got ", q.sizes(), ", ",
                    k.sizes(), ", ", v.sizes());
  bool same = k.sizes() == v.sizes() && q.size(-1) == k.size(-1);
  for (int64_t i = 0; i < want - 2; ++i) same = same && q.size(i) == k.size(i);
  TORCH_CHECK_VALUE(same, who, ": shapes do not match: ", q.sizes(), ", ", k.sizes(), ", ", v.sizes());
  const int64_t h = q.size(-2), hk = k.size(-2), d = q.size(-1);
  TORCH_CHECK_VALUE(h >= 1 && hk >= 1 && h % hk == 0, who, ": ", h, " query heads cannot share ", hk, " key heads");
  TORCH_CHECK_VALUE(d >= 1 && d <= 128, who, ": head sizes up to 128 are supported, got ", d);
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)d);
  TORCH_CHECK_VALUE(scale > 0 && std::isfinite(scale), who, ": scale must be positive and finite, got ", scale);
  Tensor cu, q3 = q, k3 = k, v3 = v;
  int64_t seqlen = 0;
  if (packed) {
    TORCH_CHECK_VALUE(cu_seqlens->scalar_type() == at::kInt && cu_seqlens->dim() == 1 && cu_seqlens->numel() >= 2, who,
                      ": cu_seqlens must be int32 with one offset more than there are sequences, got ", cu_seqlens->scalar_type(),
                      " ", cu_seqlens->sizes());
    cu = cu_seqlens->contiguous();
  } else {
    seqlen = q.size(1);
    q3 = q.flatten(0, 1);
    k3 = k.flatten(0, 1);
    v3 = v.flatten(0, 1);
  }
  const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
  const Tensor out = grad ? AttentionFn::apply(q3, k3, v3, packed ? std::optional<Tensor>(cu) : std::nullopt, seqlen, scale) : attend(q3, k3, v3, cu, seqlen, scale, false).out;
  return packed ? out : out.view(q.sizes());
}

// ---- router ----------------------------------------------------------------------

struct Routed {
  Tensor z, weights, experts, counts, loss;
  int64_t row_stride;
};
Routed route(const Tensor &logits, int64_t k, double coef) {
  ready();
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t t = logits.size(0), e = logits.size(1);
  Routed r;
  r.z = t == 0 || (logits.stride(1) == 1 && logits.stride(0) >= e) ? logits : logits.contiguous();
  r.row_stride = t > 1 ? r.z.stride(0) : e;
  r.weights = at::empty({t, k}, r.z.options().dtype(at::kFloat));
  r.experts = at::empty({t, k}, r.z.options().dtype(at::kLong));
  r.counts = at::empty({e}, r.z.options().dtype(at::kLong));
  r.loss = at::empty({}, r.z.options().dtype(at::kFloat));
  const size_t need = E.route_fwd_workspace(t, (int)e);
  const Tensor ws = need ? scratch(r.z, need) : Tensor();
  check(E.route_fwd(r.z.data_ptr(), dtype_code(r.z, "route_topk"), t, (int)e, r.row_stride, (int)k, (float)coef,
                    r.weights.data_ptr<float>(), r.experts.data_ptr<int64_t>(), r.counts.data_ptr<int64_t>(),
                    r.loss.data_ptr<float>(), ptr(ws), need, stream_of(r.z)),
        "mhc_route_fwd");
  return r;
}

struct RouteFn : torch::autograd::Function<RouteFn> {
  static variable_list forward(AutogradContext *ctx, const Tensor &logits, int64_t k, double coef) {
    const Routed r = route(logits, k, coef);
    ctx->save_for_backward({r.z, r.weights, r.experts, r.counts});
    ctx->saved_data["k"] = k;
    ctx->saved_data["coef"] = coef;
    ctx->saved_data["row_stride"] = r.row_stride;
    ctx->mark_non_differentiable({r.experts, r.counts});
    ctx->set_materialize_grads(false);
    return {r.weights, r.experts, r.counts, r.loss};
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "route_topk: second derivatives are not implemented");
    if (!g[0].defined() && !g[3].defined()) return {Tensor(), Tensor(), Tensor()};
    ready();
    const variable_list s = ctx->get_saved_variables();
    const Tensor &z = s[0];
    const c10::cuda::CUDAGuard guard(z.device());
    const int64_t t = z.size(0), e = z.size(1);
    const Tensor dw = g[0].defined() ? g[0].to(at::kFloat).contiguous() : Tensor();
    const Tensor dl = g[3].defined() ? g[3].to(at::kFloat) : Tensor();
    const Tensor dz = at::empty({t, e}, z.options());
    check(E.route_bwd(z.data_ptr(), dtype_code(z, "route_topk"), t, (int)e, ctx->saved_data["row_stride"].toInt(),
                      (int)ctx->saved_data["k"].toInt(), (float)ctx->saved_data["coef"].toDouble(), s[1].data_ptr<float>(),
                      s[2].data_ptr<int64_t>(), s[3].data_ptr<int64_t>(), static_cast<const float *>(ptr(dw)),
                      static_cast<const float *>(ptr(dl)), dz.data_ptr(), stream_of(z)),
          "mhc_route_bwd");
    return {dz, Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> route_topk(const Tensor &logits, int64_t k, double coef) {
  const char *who = "route_topk";
  require_plain(who, {&logits});
  require_cuda(logits);
  TORCH_CHECK_VALUE(logits.dim() >= 1, who, ": logits must have at least one dimension");
  dtype_code(logits, who);
  const int64_t e = logits.size(-1);
  TORCH_CHECK_VALUE(e >= 1 && e <= 512, who, ": 1 to 512 experts are supported, got ", e);
  TORCH_CHECK_VALUE(k >= 1 && k <= e, who, ": k must be in [1, ", e, "], got ", k);
  const Tensor flat = logits.dim() == 2 ? logits : logits.reshape({-1, e});
  Tensor w, idx, counts, loss;
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    const variable_list r = RouteFn::apply(flat, k, coef);
    w = r[0], idx = r[1], counts = r[2], loss = r[3];
  } else {
    const Routed r = route(flat, k, coef);
    w = r.weights, idx = r.experts, counts = r.counts, loss = r.loss;
  }
  if (logits.dim() != 2) {
    std::vector<int64_t> shape = logits.sizes().vec();
    shape.back() = k;
    w = w.view(shape);
    idx = idx.view(shape);
  }
  return {w, idx, counts, loss};
}

// ---- AdamW -----------------------------------------------------------------------

using Tensors = std::vector<Tensor>;
// parameters, gradients, moments, their scales (8 bits), steps (one, or one each), lr, beta1, beta2, eps, weight decay
using Group = std::tuple<Tensors, Tensors, Tensors, Tensors, Tensors, Tensors, std::vector<int64_t>, double, double, double, double, double>;

void check_one(const Tensor &t, const char *what, int64_t numel, c10::DeviceIndex device, bool type_ok) {
  TORCH_CHECK_TYPE(type_ok, "adamw: ", what, " cannot be ", t.scalar_type());
  TORCH_CHECK_VALUE(t.is_cuda() && t.get_device() == device, "adamw: every tensor must be on cuda:", (int)device, "; ", what, " are not");
  TORCH_CHECK_VALUE(t.is_contiguous(), "adamw: ", what, " must be contiguous");
  TORCH_CHECK_VALUE(t.numel() == numel, "adamw: ", what, " and params differ in size");
}
bool is_param_type(const Tensor &t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf;
}

std::optional<Tensor> adamw(const std::vector<Group> &groups, int bits, std::optional<double> max_norm) {
  require_plain("adamw", {});
  TORCH_CHECK_VALUE(!max_norm.has_value() || *max_norm > 0, "adamw: max_grad_norm must be positive or None, got ", max_norm.value_or(0));
  std::vector<std::vector<mhc_adamw_tensor>> tables;
  Tensor like;
  bool any = false;
  for (const Group &g : groups) {
    const auto &[p, gr, m, v, ms, vs, steps, lr, b1, b2, eps, wd] = g;
    const size_t n = p.size();
    TORCH_CHECK_VALUE(gr.size() == n && m.size() == n && v.size() == n && (bits == 32 || (ms.size() == n && vs.size() == n)), "adamw: ",
                      n, " params, ", gr.size(), " grads, ", m.size(), " and ", v.size(), " moments");
    TORCH_CHECK_VALUE(steps.size() == 1 || steps.size() == n, "adamw: ", steps.size(), " steps for ", n, " params");
    if (n == 0) {
      tables.emplace_back();
      continue;
    }
    if (!like.defined()) {
      like = p[0];
      require_cuda(like);
    }
    const auto dev = like.get_device();
    std::vector<mhc_adamw_tensor> table(n);
    for (size_t i = 0; i < n; ++i) {
      const int64_t numel = p[i].numel(), blocks = (numel + 255) / 256;
      check_one(p[i], "params", numel, dev, is_param_type(p[i]));
      check_one(gr[i], "grads", numel, dev, is_param_type(gr[i]));
      check_one(m[i], "exp_avgs", numel, dev, m[i].scalar_type() == (bits == 32 ? at::kFloat : at::kChar));
      check_one(v[i], "exp_avg_sqs", numel, dev, v[i].scalar_type() == (bits == 32 ? at::kFloat : at::kByte));
      mhc_adamw_tensor &t = table[i];
      t = {};
      if (bits == 8) {
        check_one(ms[i], "exp_avgs scales", blocks, dev, ms[i].scalar_type() == at::kFloat);
        check_one(vs[i], "exp_avg_sqs scales", blocks, dev, vs[i].scalar_type() == at::kFloat);
        t.exp_avg_scale = ms[i].data_ptr<float>();
        t.exp_avg_sq_scale = vs[i].data_ptr<float>();
      }
      t.param = p[i].data_ptr();
      t.grad = gr[i].data_ptr();
      t.exp_avg = m[i].data_ptr();
      t.exp_avg_sq = v[i].data_ptr();
      t.n = numel;
      t.step = steps[steps.size() == 1 ? 0 : i];
      t.param_dtype = dtype_code(p[i], "adamw");
      t.grad_dtype = dtype_code(gr[i], "adamw");
      any = any || numel > 0;
    }
    tables.push_back(std::move(table));
  }
  if (!like.defined()) return std::nullopt;
  ready();
  const c10::cuda::CUDAGuard guard(like.device());
  void *stream = stream_of(like);
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  C10_CUDA_CHECK(cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &capture));
  TORCH_CHECK(capture == cudaStreamCaptureStatusNone,
              "adamw: the step number is an argument of the launch, so a step cannot be captured in a CUDA graph");
  // all of them before the first launch: a refused step has changed nothing
  for (size_t i = 0; i < tables.size(); ++i)
    check(E.adamw_check(tables[i].data(), (int)tables[i].size(), bits, std::get<7>(groups[i]), std::get<8>(groups[i]),
                        std::get<9>(groups[i]), std::get<10>(groups[i]), std::get<11>(groups[i])),
          "mhc_adamw_check");
  Tensor ws, norm;
  if (max_norm.has_value()) {
    const size_t need = E.grad_norm_workspace();
    ws = scratch(like, need);
    bool first = true;
    for (const auto &t : tables) {
      if (t.empty()) continue;
      check(E.grad_norm(t.data(), (int)t.size(), first ? 0 : 1, ws.data_ptr(), need, stream), "mhc_grad_norm");
      first = false;
    }
    // written by the step, unless there is nothing to step
    norm = any ? at::empty({}, like.options().dtype(at::kFloat)) : at::zeros({}, like.options().dtype(at::kFloat));
  }
  for (size_t i = 0; i < tables.size(); ++i) {
    if (tables[i].empty()) continue;
    const Group &g = groups[i];
    // written in place, as autograd sees it: a graph that saved one of them must not run on the new values
    for (const Tensors *ts : {&std::get<0>(g), &std::get<2>(g), &std::get<3>(g), &std::get<4>(g), &std::get<5>(g)})
      for (const Tensor &t : *ts)
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    check(E.adamw_step(tables[i].data(), (int)tables[i].size(), bits, std::get<7>(g), std::get<8>(g), std::get<9>(g), std::get<10>(g),
                       std::get<11>(g), max_norm.value_or(0.0), ptr(ws), static_cast<float *>(ptr(norm)), stream),
          "mhc_adamw_step");
  }
  if (!max_norm.has_value()) return std::nullopt;
  return norm;
}

// ---- rotary positions -------------------------------------------------------------

using Maybe = std::optional<Tensor>;
constexpr int64_t MOST_HEADS = 16384;  // of the C entries, which count them in 32 bits

// a dimension's stride; of one element none is needed, and whatever stands there must not cost the wide copies
int64_t step_of(const Tensor &x, int64_t dim) { return x.size(dim) > 1 ? x.stride(dim) : 0; }
// (T, heads, D) rows with contiguous heads
Tensor flat_rows(const Tensor &x) {
  const Tensor y = x.dim() == 4 ? x.flatten(0, 1) : x;
  return y.stride(2) == 1 || y.size(2) == 1 ? y : y.contiguous();
}
void require_index(const Tensor &t, const char *who, const char *what, at::ScalarType type, const Tensor &like) {
  require_cuda(t);
  TORCH_CHECK_TYPE(t.scalar_type() == type, who, ": ", what, " must be ", type, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.device() == like.device(), who, ": ", what, " is on ", t.device(), ", the rest on ", like.device());
}
// what has no backward must not swallow a gradient that somebody waits for
void require_no_grad(const char *who, std::initializer_list<const Tensor *> ts) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor *t : ts)
    TORCH_CHECK(!t->defined() || !t->requires_grad(), who, " has no gradient: call it under torch.no_grad()");
}

struct Turned {
  Tensor q, k;
};
Turned turn(const Tensor &q, const Tensor &k, const Tensor &positions, int64_t period, const Tensor &turns, bool interleaved, double gain,
            bool inverse) {
  ready();
  const Tensor &like = q.defined() ? q : k;
  const c10::cuda::CUDAGuard guard(like.device());
  Tensor q3, k3;
  Turned out;
  int64_t strides[4] = {0, 0, 0, 0}, t = 0;
  if (q.defined()) {
    q3 = flat_rows(q);
    out.q = at::empty(q.sizes(), q.options());
    strides[0] = step_of(q3, 0), strides[1] = step_of(q3, 1), t = q3.size(0);
  }
  if (k.defined()) {
    k3 = flat_rows(k);
    out.k = at::empty(k.sizes(), k.options());
    strides[2] = step_of(k3, 0), strides[3] = step_of(k3, 1), t = k3.size(0);
  }
  const mhc_rotary r{static_cast<const uint64_t *>(turns.data_ptr()), (int32_t)(2 * turns.numel()), interleaved, (float)gain};
  check(E.rotate(&r, ptr(q3), ptr(out.q), q.defined() ? (int)q3.size(1) : 0, ptr(k3), ptr(out.k), k.defined() ? (int)k3.size(1) : 0,
                 dtype_code(like, "rotate"), t, (int)like.size(-1), strides, ptr(positions),
                 positions.defined() ? (int)positions.element_size() : 0, period, inverse, stream_of(like)),
        "mhc_rotate");
  return out;
}

struct RotateFn : torch::autograd::Function<RotateFn> {
  static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Maybe &positions, int64_t period,
                               const Tensor &turns, bool interleaved, double gain) {
    const Tensor pos = positions.value_or(Tensor());
    ctx->save_for_backward({pos, turns});
    ctx->saved_data["period"] = period;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["gain"] = gain;
    ctx->set_materialize_grads(false);
    const Turned out = turn(q, k, pos, period, turns, interleaved, gain, false);
    variable_list frozen;
    if (!q.requires_grad()) frozen.push_back(out.q);
    if (!k.requires_grad()) frozen.push_back(out.k);
    ctx->mark_non_differentiable(frozen);
    return {out.q, out.k};
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "rotate: second derivatives are not implemented");
    const variable_list s = ctx->get_saved_variables();
    const Tensor dq = ctx->needs_input_grad(0) ? g[0] : Tensor(), dk = ctx->needs_input_grad(1) ? g[1] : Tensor();
    Turned out;
    if (dq.defined() || dk.defined())
      out = turn(dq, dk, s[0], ctx->saved_data["period"].toInt(), s[1], ctx->saved_data["interleaved"].toBool(),
                 ctx->saved_data["gain"].toDouble(), true);
    return {out.q, out.k, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> rotate(const Tensor &q, const Tensor &k, const Maybe &positions, const Tensor &turns, bool interleaved,
                                  double gain) {
  const char *who = "rotate";
  require_plain(who, {&q, &k});
  require_cuda(q);
  require_cuda(k);
  TORCH_CHECK_TYPE(q.scalar_type() == k.scalar_type(), who, ": q and k must have one type, got ", q.scalar_type(), " and ", k.scalar_type());
  dtype_code(q, who);
  const int64_t n = q.dim();
  TORCH_CHECK_VALUE((n == 3 || n == 4) && k.dim() == n, who, ": (T, heads, D) or (B, L, heads, D) tensors are wanted, got ", q.sizes(), ", ",
                    k.sizes());
  bool same = q.size(-1) == k.size(-1) && q.size(0) == k.size(0) && (n == 3 || q.size(1) == k.size(1));
  TORCH_CHECK_VALUE(same && q.size(-2) >= 1 && k.size(-2) >= 1, who, ": shapes do not match: ", q.sizes(), ", ", k.sizes());
  TORCH_CHECK_VALUE(q.size(-2) <= MOST_HEADS && k.size(-2) <= MOST_HEADS, who, ": up to ", MOST_HEADS, " heads are supported, got ", q.size(-2), " and ",
                    k.size(-2));
  TORCH_CHECK_VALUE(q.device() == k.device() && turns.device() == q.device(), who, ": q, k and the frequencies must be on one device");
  const int64_t d = q.size(-1), part = 2 * turns.numel();
  TORCH_CHECK_VALUE(part <= d && d <= 256, who, ": heads of ", part, " (what is rotated) to 256 elements are wanted, got ", d);
  Tensor pos;
  int64_t period = n == 4 ? q.size(1) : 0;
  if (positions.has_value()) {
    require_cuda(*positions);
    TORCH_CHECK_TYPE(positions->scalar_type() == at::kInt || positions->scalar_type() == at::kLong, who, ": positions must be int32 or int64, got ",
                     positions->scalar_type());
    TORCH_CHECK_VALUE(positions->device() == q.device(), who, ": positions must be on the device of q and k");
    const bool each = positions->sizes() == q.sizes().slice(0, n - 2), row = n == 4 && positions->dim() == 1 && positions->size(0) == q.size(1);
    TORCH_CHECK_VALUE(each || row, who, ": positions for every token are wanted, got ", positions->sizes(), " for ", q.sizes());
    pos = positions->contiguous();
    if (each) period = 0;
  }
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad())) {
    const variable_list r = RotateFn::apply(q, k, pos.defined() ? Maybe(pos) : std::nullopt, period, turns, interleaved, gain);
    return {r[0], r[1]};
  }
  const Turned r = turn(q, k, pos, period, turns, interleaved, gain, false);
  return {r.q, r.k};
}

// ---- paged cache --------------------------------------------------------------------

struct Step {
  mhc_kv_cache cache;
  mhc_cache_step step;
  Tensor table, lengths, cu;  // what the pointers point to
};
// checks keys and values ((layers,) pages, slots, heads, D) and a step of t rows
Step step_of_cache(const char *who, const Tensor &keys, const Tensor &values, const Tensor &table, const Tensor &lengths, const Tensor &cu,
                   int64_t t, bool layers) {
  require_plain(who, {&keys, &values});
  require_cuda(keys);
  require_cuda(values);
  TORCH_CHECK_TYPE(keys.scalar_type() == values.scalar_type(), who, ": keys and values must have one type, got ", keys.scalar_type(), " and ",
                   values.scalar_type());
  Step s{};
  s.cache.dtype = dtype_code(keys, who);
  const int64_t n = keys.dim(), f = n - 4;
  TORCH_CHECK_VALUE((n == 4 || (layers && n == 5)) && keys.sizes() == values.sizes(), who, ": keys and values must be ",
                    layers ? "(layers, pages, page size, heads, D) or " : "", "(pages, page size, heads, D), got ", keys.sizes(), ", ", values.sizes());
  TORCH_CHECK_VALUE(keys.device() == values.device(), who, ": keys and values must be on one device");
  const int64_t d = keys.size(f + 3);
  TORCH_CHECK_VALUE(keys.size(f + 1) >= 1 && keys.size(f + 2) >= 1 && d >= 1 && d <= 256, who, ": bad cache shape ", keys.sizes());
  TORCH_CHECK_VALUE(keys.size(f + 1) <= 0x7fffffff && keys.size(f + 2) <= MOST_HEADS && keys.size(0) <= 0x7fffffff, who, ": a cache of ", keys.sizes(),
                    " is more than 32 bits count");
  TORCH_CHECK_VALUE((keys.stride(f + 3) == 1 && values.stride(f + 3) == 1) || d == 1, who, ": the cache's heads must be contiguous");
  require_index(table, who, "page_table", at::kInt, keys);
  require_index(lengths, who, "lengths", at::kInt, keys);
  require_index(cu, who, "cu_tokens", at::kInt, keys);
  TORCH_CHECK_VALUE(table.dim() == 2 && lengths.dim() == 1 && cu.dim() == 1 && table.size(0) == lengths.size(0) && cu.size(0) == lengths.size(0) + 1,
                    who, ": page_table (B, pages), lengths (B,) and cu_tokens (B + 1,) are wanted, got ", table.sizes(), ", ", lengths.sizes(), ", ",
                    cu.sizes());
  TORCH_CHECK_VALUE(table.size(1) * keys.size(f + 1) < ((int64_t)1 << 31) - 4096, who, ": a sequence of ", table.size(1), " pages is too long");
  TORCH_CHECK_VALUE(lengths.size(0) <= (int64_t)1 << 30, who, ": ", lengths.size(0), " sequences are too many");
  s.table = table.size(1) > 1 && table.stride(1) != 1 ? table.contiguous() : table;
  s.lengths = lengths.contiguous();
  s.cu = cu.contiguous();
  s.cache.keys = keys.data_ptr();
  s.cache.values = values.data_ptr();
  s.cache.layers = n == 5 ? (int32_t)keys.size(0) : 1;
  s.cache.pages = keys.size(f);
  s.cache.page_size = (int32_t)keys.size(f + 1);
  s.cache.kv_heads = (int32_t)keys.size(f + 2);
  s.cache.dim = (int32_t)d;
  for (int64_t i = 1 - f; i < 4; ++i) {  // layer (of five dimensions), page, slot, head
    s.cache.strides[i] = step_of(keys, i - 1 + f);
    s.cache.strides[4 + i] = step_of(values, i - 1 + f);
  }
  s.step.page_table = static_cast<const int32_t *>(s.table.data_ptr());
  s.step.lengths = static_cast<const int32_t *>(s.lengths.data_ptr());
  s.step.cu_tokens = static_cast<const int32_t *>(s.cu.data_ptr());
  s.step.table_pitch = step_of(s.table, 0);
  s.step.table_width = (int32_t)s.table.size(1);
  s.step.batch = (int32_t)lengths.size(0);
  s.step.T = t;
  return s;
}
// what is written to must not be expanded: two places would be one memory, and which of them comes last is nobody's choice
void require_own_places(const char *who, std::initializer_list<const Tensor *> ts) {
  for (const Tensor *t : ts)
    for (int64_t i = 0; i < t->dim(); ++i)
      TORCH_CHECK_VALUE(t->size(i) <= 1 || t->stride(i) != 0, who, ": keys and values are written to and must not be expanded, got sizes ", t->sizes(),
                        " with strides ", t->strides());
}
void written(const Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Maybe append_kv(const Tensor &keys, const Tensor &values, const Tensor &table, const Tensor &lengths, const Tensor &cu, const Tensor &k,
                const Tensor &v, const Maybe &q_, const Maybe &positions, const Maybe &turns, bool interleaved, double gain) {
  const char *who = "append_kv";
  const Tensor q = q_.value_or(Tensor());
  require_plain(who, {&k, &v});
  if (q.defined()) require_plain(who, {&q});
  require_no_grad(who, {&keys, &values, &k, &v, &q});
  require_cuda(k);
  require_cuda(v);
  TORCH_CHECK_VALUE(k.dim() == 3 && k.sizes() == v.sizes(), who, ": k and v (T, heads, D) are wanted, got ", k.sizes(), ", ", v.sizes());
  Step s = step_of_cache(who, keys, values, table, lengths, cu, k.size(0), false);
  require_own_places(who, {&keys, &values});
  TORCH_CHECK_VALUE(k.size(1) == s.cache.kv_heads && k.size(2) == s.cache.dim, who, ": k and v ", k.sizes(), " do not fit the cache ", keys.sizes());
  TORCH_CHECK_TYPE(k.scalar_type() == keys.scalar_type() && v.scalar_type() == keys.scalar_type(), who, ": k, v and the cache must have one type, got ",
                   k.scalar_type(), ", ", v.scalar_type(), ", ", keys.scalar_type());
  TORCH_CHECK_VALUE(k.device() == keys.device() && v.device() == keys.device(), who, ": k, v and the cache must be on one device");
  TORCH_CHECK_VALUE(turns.has_value() || (!q.defined() && !positions.has_value()), who, ": q and positions are of use with a rotary only");
  Tensor pos;
  if (turns.has_value()) {
    TORCH_CHECK_VALUE(turns->device() == keys.device(), who, ": the frequencies must be on the cache's device");
    TORCH_CHECK_VALUE(2 * turns->numel() <= s.cache.dim, who, ": heads of ", s.cache.dim, " cannot have ", 2 * turns->numel(), " elements rotated");
  }
  if (q.defined()) {
    require_cuda(q);
    TORCH_CHECK_TYPE(q.scalar_type() == keys.scalar_type(), who, ": q and the cache must have one type, got ", q.scalar_type(), ", ", keys.scalar_type());
    TORCH_CHECK_VALUE(q.device() == keys.device() && q.dim() == 3 && q.size(0) == k.size(0) && q.size(1) >= 1 && q.size(2) == k.size(2), who,
                      ": q (T, heads, D) on the cache's device is wanted, got ", q.sizes(), " for k ", k.sizes());
    TORCH_CHECK_VALUE(q.size(1) <= MOST_HEADS, who, ": up to ", MOST_HEADS, " query heads are supported, got ", q.size(1));
  }
  if (positions.has_value()) {
    require_cuda(*positions);
    TORCH_CHECK_TYPE(positions->scalar_type() == at::kInt || positions->scalar_type() == at::kLong, who, ": positions must be int32 or int64, got ",
                     positions->scalar_type());
    TORCH_CHECK_VALUE(positions->device() == keys.device() && positions->dim() == 1 && positions->size(0) == k.size(0), who,
                      ": a position for every token is wanted, got ", positions->sizes());
    pos = positions->contiguous();
  }
  ready();
  const c10::cuda::CUDAGuard guard(keys.device());
  const Tensor k3 = flat_rows(k), v3 = flat_rows(v), q3 = q.defined() ? flat_rows(q) : Tensor();
  Tensor out = q.defined() ? at::empty(q.sizes(), q.options()) : Tensor();
  int64_t strides[6] = {0, 0, step_of(k3, 0), step_of(k3, 1), step_of(v3, 0), step_of(v3, 1)};
  if (q3.defined()) strides[0] = step_of(q3, 0), strides[1] = step_of(q3, 1);
  mhc_rotary r{};
  if (turns.has_value())
    r = mhc_rotary{static_cast<const uint64_t *>(turns->data_ptr()), (int32_t)(2 * turns->numel()), interleaved, (float)gain};
  written(keys);
  written(values);
  check(E.append_kv(&s.cache, &s.step, k3.data_ptr(), v3.data_ptr(), ptr(q3), ptr(out), q3.defined() ? (int)q3.size(1) : 0, strides,
                    turns.has_value() ? &r : nullptr, ptr(pos), pos.defined() ? (int)pos.element_size() : 0, stream_of(keys)),
        "mhc_append_kv");
  return out.defined() ? Maybe(out) : std::nullopt;
}

Tensor cached_attention(const Tensor &q, const Tensor &keys, const Tensor &values, const Tensor &table, const Tensor &lengths, const Tensor &cu,
                        const Maybe &mask, std::optional<double> scale_) {
  const char *who = "cached_attention";
  require_plain(who, {&q});
  require_no_grad(who, {&q, &keys, &values});
  require_cuda(q);
  TORCH_CHECK_VALUE(q.dim() == 3, who, ": q (T, heads, D) is wanted, got ", q.sizes());
  Step s = step_of_cache(who, keys, values, table, lengths, cu, q.size(0), false);
  TORCH_CHECK_TYPE(q.scalar_type() == keys.scalar_type(), who, ": q and the cache must have one type, got ", q.scalar_type(), ", ", keys.scalar_type());
  TORCH_CHECK_VALUE(q.device() == keys.device(), who, ": q and the cache must be on one device");
  const int64_t t = q.size(0), h = q.size(1), d = q.size(2);
  TORCH_CHECK_VALUE(d == s.cache.dim && h >= 1 && h % s.cache.kv_heads == 0, who, ": ", h, " query heads of ", d, " cannot share ", s.cache.kv_heads,
                    " key heads of ", s.cache.dim);
  TORCH_CHECK_VALUE(d <= 128, who, ": head sizes up to 128 are supported, got ", d);
  TORCH_CHECK_VALUE(h <= 0x7fffffff && t <= 0x7fffffff && t * (h / s.cache.kv_heads) <= 0x7fffffff - 4096, who, ": ", t, " tokens of ", h / s.cache.kv_heads,
                    " heads for a key head are more rows than one call takes");
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)d);
  TORCH_CHECK_VALUE((float)scale > 0 && std::isfinite((float)scale), who, ": scale must be positive and finite, got ", scale);
  Tensor bits;
  if (mask.has_value()) {
    require_index(*mask, who, "mask", at::kLong, keys);
    TORCH_CHECK_VALUE(mask->dim() == 1 && mask->size(0) == t, who, ": a mask for every token is wanted, got ", mask->sizes());
    bits = mask->contiguous();
  }
  ready();
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor q3 = rows(q), out = at::empty({t, h, d}, q.options());
  const size_t need = E.cached_attn_workspace(&s.cache, &s.step, (int)h);
  const Tensor ws = need ? scratch(q, need) : Tensor();
  const int64_t strides[2] = {step_of(q3, 0), step_of(q3, 1)};
  check(E.cached_attn(&s.cache, &s.step, ptr(q3), (int)h, strides, static_cast<const int64_t *>(ptr(bits)), (float)scale, out.data_ptr(), ptr(ws),
                      need, stream_of(q)),
        "mhc_cached_attn");
  return out;
}

void keep_drafts(const Tensor &keys, const Tensor &values, const Tensor &table, const Tensor &lengths, const Tensor &cu, const Tensor &path,
                 const Tensor &kept) {
  const char *who = "keep_drafts";
  require_no_grad(who, {&keys, &values});
  TORCH_CHECK_VALUE(path.dim() == 1, who, ": path (T,) is wanted, got ", path.sizes());
  Step s = step_of_cache(who, keys, values, table, lengths, cu, path.size(0), true);
  require_own_places(who, {&keys, &values});
  require_index(path, who, "path", at::kInt, keys);
  require_index(kept, who, "kept", at::kInt, keys);
  TORCH_CHECK_VALUE(kept.sizes() == lengths.sizes(), who, ": a number of kept tokens for every sequence is wanted, got ", kept.sizes());
  ready();
  const c10::cuda::CUDAGuard guard(keys.device());
  const Tensor p = path.contiguous(), n = kept.contiguous();
  written(keys);
  written(values);
  check(E.keep_drafts(&s.cache, &s.step, static_cast<const int32_t *>(ptr(p)), static_cast<const int32_t *>(ptr(n)), stream_of(keys)),
        "mhc_keep_drafts");
}

// ---- verification of drafted tokens -------------------------------------------------

std::tuple<Tensor, Tensor, Tensor> verify_drafts(const Tensor &tokens, const Tensor &parents, const Tensor &cu, const Tensor &target,
                                                 const Maybe &draft, const Tensor &random) {
  const char *who = "verify_drafts";
  require_plain(who, {&target, &random});
  require_cuda(target);
  dtype_code(target, who);
  TORCH_CHECK_VALUE(target.dim() == 2 && target.size(1) >= 1, who, ": target (T, V) is wanted, got ", target.sizes());
  const int64_t t = target.size(0), v = target.size(1);
  if (draft.has_value()) {
    require_plain(who, {&*draft});
    require_index(*draft, who, "draft", target.scalar_type(), target);
    TORCH_CHECK_VALUE(draft->sizes() == target.sizes(), who, ": draft ", draft->sizes(), " and target ", target.sizes(), " must have one shape");
  }
  require_index(tokens, who, "tokens", at::kLong, target);
  require_index(parents, who, "parents", at::kInt, target);
  require_index(cu, who, "cu_tokens", at::kInt, target);
  require_index(random, who, "random", at::kFloat, target);
  for (const Tensor *x : {&tokens, &parents, &random})
    TORCH_CHECK_VALUE(x->dim() == 1 && x->size(0) == t, who, ": tokens, parents and random of ", t, " rows are wanted, got ", x->sizes());
  TORCH_CHECK_VALUE(cu.dim() == 1 && cu.size(0) >= 1, who, ": cu_tokens (B + 1,) is wanted, got ", cu.sizes());
  TORCH_CHECK_VALUE(cu.size(0) - 1 <= 0x7fffffff, who, ": ", cu.size(0) - 1, " sequences are too many");
  ready();
  const c10::cuda::CUDAGuard guard(target.device());
  auto whole = [](const Tensor &x) { return (x.stride(1) == 1 || x.size(1) == 1) && (x.size(0) <= 1 || x.stride(0) >= x.size(1)) ? x : x.contiguous(); };
  const Tensor p = whole(target), q = draft.has_value() ? whole(*draft) : Tensor();
  const Tensor tk = tokens.contiguous(), pr = parents.contiguous(), c = cu.contiguous(), u = random.contiguous();
  const int64_t batch = cu.size(0) - 1;
  const Tensor path = at::empty({t}, pr.options()), kept = at::empty({batch}, pr.options()), next = at::empty({batch}, tk.options());
  check(E.verify_drafts(static_cast<const int64_t *>(ptr(tk)), static_cast<const int32_t *>(ptr(pr)), static_cast<const int32_t *>(ptr(c)), (int)batch,
                        t, ptr(p), t > 1 ? p.stride(0) : v, ptr(q), q.defined() && t > 1 ? q.stride(0) : v, dtype_code(target, who), v,
                        static_cast<const float *>(ptr(u)), static_cast<int32_t *>(ptr(path)), static_cast<int32_t *>(ptr(kept)),
                        static_cast<int64_t *>(ptr(next)), stream_of(target)),
        "mhc_verify_drafts");
  return {path, kept, next};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("set_flag", &set_flag);
  m.def("packed_attention", &packed_attention);
  m.def("route_topk", &route_topk);
  m.def("adamw", &adamw);
  m.def("rotate", &rotate);
  m.def("append_kv", &append_kv);
  m.def("cached_attention", &cached_attention);
  m.def("keep_drafts", &keep_drafts);
  m.def("verify_drafts", &verify_drafts);
}
