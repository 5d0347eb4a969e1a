// torch.ops.d3pm_mi355x.* -- the PyTorch-ROCm extension form of the boundary.
//
// A thin shim: every operator checks its tensors, allocates its outputs (and workspace) with torch's
// allocator, and calls the C ABI of libd3pm_hip.so (include/d3pm_hip.h) on torch's current HIP stream.  No
// arithmetic happens here.  The operators carry the reference function they stand for in their schema comment;
// autograd nodes live in the Python facade, which calls these operators; those of the fine-tuning objectives live
// here.  Status codes of the library become the exceptions the reference raises: D3PM_EINVAL -> ValueError,
// D3PM_EUNSUPPORTED -> NotImplementedError, D3PM_EHIP -> RuntimeError.  Every operator makes the device of its first tensor current for the call and checks
// every tensor's element count against the batch it describes before a pointer reaches the library: a mis-shaped
// call raises, it does not read or write out of bounds.
#include <ATen/ATen.h>
#include <ATen/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <tuple>
#include <vector>

#include "../../include/d3pm_hip.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

void check_rc(int rc) {
  if (rc == D3PM_OK) return;
  const char* msg = d3pm_last_error();
  TORCH_CHECK_VALUE(rc != D3PM_EINVAL, msg);
  TORCH_CHECK_NOT_IMPLEMENTED(rc != D3PM_EUNSUPPORTED, msg);
  TORCH_CHECK(false, "libd3pm_hip: ", msg, " (code ", rc, ")");
}

void* stream() { return (void*)c10::hip::getCurrentHIPStream().stream(); }

void need_device(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), "d3pm_mi355x: ", what, " must live on an MI355X (device='cuda'); there is no CPU path");
  TORCH_CHECK(t.is_contiguous(), "d3pm_mi355x: ", what, " must be contiguous");
}
int tok_bytes(const Tensor& t, const char* what) {
  need_device(t, what);
  if (t.scalar_type() == at::kLong) return 8;
  TORCH_CHECK(t.scalar_type() == at::kInt, "d3pm_mi355x: ", what, " must be int32 or int64");
  return 4;
}
const void* opt_ptr(const OptTensor& t, at::ScalarType st, const char* what) {
  if (!t.has_value() || !t->defined()) return nullptr;
  need_device(*t, what);
  TORCH_CHECK(t->scalar_type() == st, "d3pm_mi355x: ", what, " has the wrong dtype");
  return t->data_ptr();
}
const float* f32(const Tensor& t, const char* what) {
  need_device(t, what);
  TORCH_CHECK(t.scalar_type() == at::kFloat, "d3pm_mi355x: ", what, " must be float32");
  return t.data_ptr<float>();
}

// ---- shape contracts (element counts: the library sees flat [B, npos, ...] buffers)
void need_numel(const Tensor& t, int64_t n, const char* what) {
  TORCH_CHECK_VALUE(t.numel() == n, "d3pm_mi355x: ", what, " has ", t.numel(), " elements, expected ", n);
}
void need_numel(const OptTensor& t, int64_t n, const char* what) {
  if (t.has_value() && t->defined()) need_numel(*t, n, what);
}
void need_same_shape(const Tensor& a, const Tensor& b, const char* what) {
  TORCH_CHECK_VALUE(a.sizes() == b.sizes(), "d3pm_mi355x: ", what, " must have the same shape, got ", a.sizes(), " and ",
                    b.sizes());
}
// rows [B, npos, ld] with ld >= K
int64_t need_rows(const Tensor& rows, int B, long npos, int64_t K, const char* what) {
  TORCH_CHECK_VALUE(rows.dim() >= 1, "d3pm_mi355x: ", what, " needs a trailing class dimension");
  const int64_t ld = rows.size(-1);
  TORCH_CHECK_VALUE(ld >= K, "d3pm_mi355x: ", what, " has rows of ", ld, " < K = ", K, " entries");
  need_numel(rows, (int64_t)B * npos * ld, what);
  return ld;
}
void need_image_tables(at::TensorList tables, int64_t K, int64_t T, bool structured) {
  TORCH_CHECK(tables.size() == 5 || tables.size() == 7,
              "d3pm_mi355x: tables = [qbar_digest, qone_digest, qbar, qoneT, qbarT(, qbar_f16x2, qbarT_f16x2)]");
  TORCH_CHECK_VALUE(K >= 2 && K <= 256 && T >= 1, "d3pm_mi355x: need 2 <= K <= 256 and T >= 1");
  need_numel(tables[0], T * 8 * K, "qbar_digest (float32 [T, 8, K])");
  need_numel(tables[1], T * 8 * K, "qone_digest (float32 [T, 8, K])");
  if (!structured)
    for (int i = 2; i < 5; ++i) need_numel(tables[i], T * K * K, "dense table copy (float32 [T, K, K])");
  if (tables.size() == 7) {
    const bool h0 = tables[5].defined() && tables[5].numel() > 0, h1 = tables[6].defined() && tables[6].numel() > 0;
    TORCH_CHECK_VALUE(h0 == h1, "d3pm_mi355x: the float16 split tables come as a pair (qbar_f16x2, qbarT_f16x2)");
    if (h0) {
      TORCH_CHECK_VALUE(!structured && (K == 64 || K == 128 || K == 256),
                        "d3pm_mi355x: float16 split tables serve dense tables with K = 64, 128 or 256");
      for (int i = 5; i < 7; ++i) {
        need_device(tables[i], "float16 split table");
        TORCH_CHECK(tables[i].scalar_type() == at::kHalf, "d3pm_mi355x: split tables are float16");
        need_numel(tables[i], T * 2 * K * K, "split table (float16 [T, K / 32, K / 16, 2, 64, 8])");
      }
    }
  }
}
void need_protein_tables(const Tensor& qbar_digest, const Tensor& qone_digest, int64_t K, int64_t T) {
  TORCH_CHECK_VALUE(K >= 2 && K <= 256 && T >= 1, "d3pm_mi355x: need 2 <= K <= 256 and T >= 1");
  need_numel(qbar_digest, T * 4 * K, "qbar_digest (float64 [T, 4, K])");
  need_numel(qone_digest, T * 4 * K, "qone_digest (float64 [T, 4, K])");
}
void need_counter(const OptTensor& c, const char* what) {
  if (c.has_value() && c->defined()) need_numel(*c, 1, what);
}
std::vector<int64_t> with_k(const Tensor& tokens, int64_t K) {
  auto s = tokens.sizes().vec();
  s.push_back(K);
  return s;
}

// tables = [qbar_digest, qone_digest, qbar, qoneT, qbarT(, qbar_f16x2, qbarT_f16x2)]; all but the digests may be
// empty tensors (structured tables; no float16 split tables: the float32 matrix instructions serve K = 256)
d3pm_tables_f32 image_tables(at::TensorList tables, int64_t K, int64_t T, bool structured, double eps) {
  need_image_tables(tables, K, T, structured);
  d3pm_tables_f32 tb{};
  tb.K = (int)K; tb.T = (int)T; tb.structured = structured ? 1 : 0; tb.eps = (float)eps;
  auto get = [&](int i, const char* what) -> const float* {
    return tables[i].defined() && tables[i].numel() > 0 ? f32(tables[i], what) : nullptr;
  };
  tb.qbar_digest = get(0, "qbar_digest"); tb.qone_digest = get(1, "qone_digest");
  tb.qbar = get(2, "qbar"); tb.qoneT = get(3, "qoneT"); tb.qbarT = get(4, "qbarT");
  if (tables.size() == 7 && tables[5].defined() && tables[5].numel() > 0) {
    tb.qbar_f16x2 = (const uint16_t*)tables[5].data_ptr();
    tb.qbarT_f16x2 = (const uint16_t*)tables[6].data_ptr();
  }
  return tb;
}
d3pm_tables_f64 protein_tables(const Tensor& qbar_digest, const Tensor& qone_digest, const Tensor& lvb_digest, int64_t K,
                               int64_t T) {
  need_protein_tables(qbar_digest, qone_digest, K, T);
  need_device(qbar_digest, "qbar_digest"); need_device(qone_digest, "qone_digest");
  TORCH_CHECK(qbar_digest.scalar_type() == at::kDouble && qone_digest.scalar_type() == at::kDouble,
              "d3pm_mi355x: protein digests are float64");
  const float* lvb = nullptr;
  if (lvb_digest.defined() && lvb_digest.numel() > 0) {        // empty: no float32 loss digest (K > 32)
    need_numel(lvb_digest, (int64_t)(d3pm_lvb_digest_f32_size((int)T) / sizeof(float)), "lvb_digest");
    lvb = f32(lvb_digest, "lvb_digest");
  }
  return d3pm_tables_f64{(int)K, (int)T, qbar_digest.data_ptr<double>(), qone_digest.data_ptr<double>(), lvb};
}
std::pair<int, long> dims(const Tensor& tokens) {
  const int B = tokens.dim() ? (int)tokens.size(0) : 1;
  return {B, B ? (long)(tokens.numel() / B) : 0};
}

#define D3PM_GUARD(t) const at::DeviceGuard device_guard_((t).device())

// DiscreteDiffusion.q_probs, d3pm/diffusion_discrete.py:250-263
Tensor q_probs(at::TensorList tables, int64_t K, int64_t T, bool structured, double eps, const Tensor& x0, const Tensor& t) {
  D3PM_GUARD(x0);
  auto tb = image_tables(tables, K, T, structured, eps);
  auto [B, npos] = dims(x0);
  need_numel(t, B, "t");
  Tensor out = at::empty(with_k(x0, K), x0.options().dtype(at::kFloat));
  check_rc(d3pm_q_probs(&tb, x0.data_ptr(), tok_bytes(x0, "x0"), t.data_ptr(), tok_bytes(t, "t"), B, npos,
                        out.data_ptr<float>(), stream()));
  return out;
}

// DiscreteDiffusion.q_sample, :266-285
Tensor q_sample(at::TensorList tables, int64_t K, int64_t T, bool structured, double eps, const Tensor& x0, const Tensor& t,
                const OptTensor& noise, int64_t noise_kind, int64_t seed, int64_t offset, const OptTensor& offset_dev) {
  D3PM_GUARD(x0);
  auto tb = image_tables(tables, K, T, structured, eps);
  auto [B, npos] = dims(x0);
  need_numel(t, B, "t");
  need_numel(noise, (int64_t)B * npos * K, "noise");
  need_counter(offset_dev, "offset_dev");
  Tensor out = at::empty(x0.sizes(), x0.options().dtype(at::kLong));
  check_rc(d3pm_q_sample(&tb, x0.data_ptr(), tok_bytes(x0, "x0"), t.data_ptr(), tok_bytes(t, "t"), B, npos,
                         (const float*)opt_ptr(noise, at::kFloat, "noise"), (int)noise_kind, (uint64_t)seed,
                         (uint64_t)offset, (const uint64_t*)opt_ptr(offset_dev, at::kLong, "offset_dev"),
                         out.data_ptr<int64_t>(), stream()));
  return out;
}

// the first two lines of training_losses, :549-556, with device noise: (t int32 [B], x_t int64) in one launch;
// `clear` (a float32 scalar, optional) is zeroed by the launch
std::tuple<Tensor, Tensor> q_sample_draw_t(at::TensorList tables, int64_t K, int64_t T, bool structured, double eps,
                                           const Tensor& x0, int64_t seed, int64_t offset, const OptTensor& offset_dev,
                                           const OptTensor& clear) {
  D3PM_GUARD(x0);
  auto tb = image_tables(tables, K, T, structured, eps);
  auto [B, npos] = dims(x0);
  need_counter(offset_dev, "offset_dev");
  need_counter(clear, "clear");
  Tensor t = at::empty({B}, x0.options().dtype(at::kInt));
  Tensor x_t = at::empty(x0.sizes(), x0.options().dtype(at::kLong));
  check_rc(d3pm_q_sample_draw_t(&tb, x0.data_ptr(), tok_bytes(x0, "x0"), B, npos, (uint64_t)seed, (uint64_t)offset,
                                (const uint64_t*)opt_ptr(offset_dev, at::kLong, "offset_dev"),
                                (float*)opt_ptr(clear, at::kFloat, "clear"), t.data_ptr<int32_t>(),
                                x_t.data_ptr<int64_t>(), stream()));
  return {t, x_t};
}

// DiscreteDiffusion.q_posterior_logits, :312-336 (and p_logits :339-381 with x_start_is_logits)
Tensor q_posterior_logits(at::TensorList tables, int64_t K, int64_t T, bool structured, double eps, const Tensor& x_start,
                          bool x_start_is_logits, const Tensor& x_t, const Tensor& t) {
  D3PM_GUARD(x_t);
  auto tb = image_tables(tables, K, T, structured, eps);
  auto [B, npos] = dims(x_t);
  need_numel(t, B, "t");
  if (x_start_is_logits) need_rows(x_start, B, npos, K, "x_start logits");
  else need_same_shape(x_start, x_t, "x_start and x_t");
  Tensor out = at::empty(with_k(x_t, K), x_t.options().dtype(at::kFloat));
  const void* xs = x_start_is_logits ? (const void*)f32(x_start, "x_start logits") : x_start.data_ptr();
  const int xb = x_start_is_logits ? 8 : tok_bytes(x_start, "x_start");
  check_rc(d3pm_q_posterior_logits(&tb, xs, x_start_is_logits ? 1 : 0, x_start_is_logits ? x_start.size(-1) : K, xb,
                                   x_t.data_ptr(), tok_bytes(x_t, "x_t"), t.data_ptr(), tok_bytes(t, "t"), B, npos,
                                   out.data_ptr<float>(), stream()));
  return out;
}

// gradient of the above with respect to the x_start logits (autograd of :320-336)
Tensor q_posterior_logits_backward(at::TensorList tables, int64_t K, int64_t T, bool structured, double eps,
                                   const Tensor& x_start_logits, const Tensor& t, const Tensor& grad_out) {
  D3PM_GUARD(x_start_logits);
  auto tb = image_tables(tables, K, T, structured, eps);
  TORCH_CHECK_VALUE(x_start_logits.dim() >= 2, "d3pm_mi355x: x_start logits are [B, ..., K]");
  const int B = (int)x_start_logits.size(0);
  const long npos = B ? (long)(x_start_logits.numel() / x_start_logits.size(-1) / B) : 0;
  need_rows(x_start_logits, B, npos, K, "x_start logits");
  need_numel(t, B, "t");
  need_numel(grad_out, (int64_t)B * npos * K, "grad_out");
  Tensor gz = at::empty_like(x_start_logits);
  check_rc(d3pm_q_posterior_logits_backward(&tb, f32(x_start_logits, "x_start logits"), x_start_logits.size(-1),
                                            t.data_ptr(), tok_bytes(t, "t"), B, npos, f32(grad_out, "grad_out"),
                                            gz.data_ptr<float>(), stream()));
  return gz;
}

struct LossShape { int B; long npos; };
LossShape check_loss_args(const Tensor& logits, const Tensor& x0, const Tensor& x_t, const Tensor& t, int64_t K,
                          const OptTensor& grad_out) {
  auto [B, npos] = dims(x0);
  need_same_shape(x0, x_t, "x0 and x_t");
  need_numel(t, B, "t");
  need_rows(logits, B, npos, K, "logits");
  need_numel(grad_out, B, "grad_out");
  return {B, npos};
}

// vb_terms_bpd :462-489 + cross_entropy_start :527-542 + training_losses :558-582, and d/d logits in the same launch
std::tuple<Tensor, Tensor, Tensor, Tensor> hybrid_loss(at::TensorList tables, int64_t K, int64_t T, bool structured,
                                                       double eps, const Tensor& logits, const Tensor& x0,
                                                       const Tensor& x_t, const Tensor& t, int64_t loss_type,
                                                       double hybrid_coeff, double grad_scale, const OptTensor& grad_out,
                                                       bool want_grad) {
  D3PM_GUARD(logits);
  auto tb = image_tables(tables, K, T, structured, eps);
  auto [B, npos] = check_loss_args(logits, x0, x_t, t, K, grad_out);
  auto fo = logits.options().dtype(at::kFloat);
  Tensor loss = at::empty({B}, fo), vb = at::empty({B}, fo), ce = at::empty({B}, fo);
  Tensor dl = want_grad ? at::empty_like(logits) : at::empty({0}, fo);
  const size_t wsb = d3pm_hybrid_loss_workspace(B, npos, (int)K);
  Tensor ws = at::empty({(int64_t)(wsb / 4 + 1)}, fo);
  check_rc(d3pm_hybrid_loss(&tb, f32(logits, "logits"), logits.size(-1), x0.data_ptr(), tok_bytes(x0, "x0"), x_t.data_ptr(),
                            tok_bytes(x_t, "x_t"), t.data_ptr(), tok_bytes(t, "t"), B, npos, (int)loss_type,
                            (float)hybrid_coeff, (float)grad_scale, (const float*)opt_ptr(grad_out, at::kFloat, "grad_out"),
                            vb.data_ptr<float>(), ce.data_ptr<float>(), loss.data_ptr<float>(),
                            want_grad ? dl.data_ptr<float>() : nullptr, nullptr, nullptr, 0, ws.data_ptr(), wsb, stream()));
  return {loss, vb, ce, dl};
}

// the loss launch of a training step: per-example losses and d/d logits only, optionally the batch mean accumulated
// on the device (`loss_mean`, zeroed beforehand) and the Philox counter of q_sample_draw_t advanced by `rng_step`
std::tuple<Tensor, Tensor> hybrid_loss_step(at::TensorList tables, int64_t K, int64_t T, bool structured, double eps,
                                            const Tensor& logits, const Tensor& x0, const Tensor& x_t, const Tensor& t,
                                            int64_t loss_type, double hybrid_coeff, double grad_scale, bool want_grad,
                                            const OptTensor& loss_mean, const OptTensor& rng_counter, int64_t rng_step) {
  D3PM_GUARD(logits);
  auto tb = image_tables(tables, K, T, structured, eps);
  auto [B, npos] = check_loss_args(logits, x0, x_t, t, K, c10::nullopt);
  need_counter(loss_mean, "loss_mean");
  need_counter(rng_counter, "rng_counter");
  auto fo = logits.options().dtype(at::kFloat);
  Tensor loss = at::empty({B}, fo);
  Tensor dl = want_grad ? at::empty_like(logits) : at::empty({0}, fo);
  const size_t wsb = d3pm_hybrid_loss_workspace(B, npos, (int)K);
  Tensor ws = at::empty({(int64_t)(wsb / 4 + 1)}, fo);
  check_rc(d3pm_hybrid_loss(&tb, f32(logits, "logits"), logits.size(-1), x0.data_ptr(), tok_bytes(x0, "x0"), x_t.data_ptr(),
                            tok_bytes(x_t, "x_t"), t.data_ptr(), tok_bytes(t, "t"), B, npos, (int)loss_type,
                            (float)hybrid_coeff, (float)grad_scale, nullptr, nullptr, nullptr, loss.data_ptr<float>(),
                            want_grad ? dl.data_ptr<float>() : nullptr, (float*)opt_ptr(loss_mean, at::kFloat, "loss_mean"),
                            (uint64_t*)opt_ptr(rng_counter, at::kLong, "rng_counter"), (uint64_t)rng_step, ws.data_ptr(),
                            wsb, stream()));
  return {loss, dl};
}

// the same launch carrying the next batch's timestep draw and corruption (training_losses :549-556 of step i + 1):
// returns (losses, dlogits, next_t int32 [B], next_x_t int64)
std::tuple<Tensor, Tensor, Tensor, Tensor> hybrid_loss_then_q_sample(
    at::TensorList tables, int64_t K, int64_t T, bool structured, double eps, const Tensor& logits, const Tensor& x0,
    const Tensor& x_t, const Tensor& t, int64_t loss_type, double hybrid_coeff, double grad_scale, bool want_grad,
    const Tensor& next_x0, int64_t seed, int64_t offset, const OptTensor& offset_dev) {
  D3PM_GUARD(logits);
  auto tb = image_tables(tables, K, T, structured, eps);
  auto [B, npos] = check_loss_args(logits, x0, x_t, t, K, c10::nullopt);
  need_same_shape(next_x0, x0, "next_x0 and x0");
  need_counter(offset_dev, "offset_dev");
  auto fo = logits.options().dtype(at::kFloat);
  Tensor loss = at::empty({B}, fo);
  Tensor dl = want_grad ? at::empty_like(logits) : at::empty({0}, fo);
  Tensor nt = at::empty({B}, x0.options().dtype(at::kInt));
  Tensor nxt = at::empty(x0.sizes(), x0.options().dtype(at::kLong));
  const size_t wsb = d3pm_hybrid_loss_workspace(B, npos, (int)K);
  Tensor ws = at::empty({(int64_t)(wsb / 4 + 1)}, fo);
  check_rc(d3pm_hybrid_loss_then_q_sample(
      &tb, f32(logits, "logits"), logits.size(-1), x0.data_ptr(), tok_bytes(x0, "x0"), x_t.data_ptr(), tok_bytes(x_t, "x_t"),
      t.data_ptr(), tok_bytes(t, "t"), B, npos, (int)loss_type, (float)hybrid_coeff, (float)grad_scale, nullptr, nullptr,
      nullptr, loss.data_ptr<float>(), want_grad ? dl.data_ptr<float>() : nullptr, ws.data_ptr(), wsb, next_x0.data_ptr(),
      tok_bytes(next_x0, "next_x0"), (uint64_t)seed, (uint64_t)offset,
      (const uint64_t*)opt_ptr(offset_dev, at::kLong, "offset_dev"), nt.data_ptr<int32_t>(), nxt.data_ptr<int64_t>(),
      stream()));
  return {loss, dl, nt, nxt};
}

// hybrid_loss into buffers the caller owns, with the library's static scratch instead of a workspace: nothing is
// allocated by the call (callers under HIP graph capture with their own buffers, serving loops)
void hybrid_loss_static_(at::TensorList tables, int64_t K, int64_t T, bool structured, double eps, const Tensor& logits,
                         const Tensor& x0, const Tensor& x_t, const Tensor& t, int64_t loss_type, double hybrid_coeff,
                         double grad_scale, Tensor loss, const OptTensor& dlogits) {
  D3PM_GUARD(logits);
  auto tb = image_tables(tables, K, T, structured, eps);
  auto [B, npos] = check_loss_args(logits, x0, x_t, t, K, c10::nullopt);
  need_numel(loss, B, "loss");
  need_numel(dlogits, logits.numel(), "dlogits");
  check_rc(d3pm_hybrid_loss_static(&tb, f32(logits, "logits"), logits.size(-1), x0.data_ptr(), tok_bytes(x0, "x0"),
                                   x_t.data_ptr(), tok_bytes(x_t, "x_t"), t.data_ptr(), tok_bytes(t, "t"), B, npos,
                                   (int)loss_type, (float)hybrid_coeff, (float)grad_scale, nullptr, nullptr, nullptr,
                                   const_cast<float*>(f32(loss, "loss")), (float*)opt_ptr(dlogits, at::kFloat, "dlogits"),
                                   nullptr, nullptr, 0, stream()));
}

// backward of the loss nodes: g[b,:] *= upstream[b] / baked, in place
void scale_rows_(Tensor g, const Tensor& upstream, double baked) {
  D3PM_GUARD(g);
  const int B = (int)upstream.numel();
  TORCH_CHECK_VALUE(B == 0 || g.numel() % B == 0, "d3pm_mi355x: g has ", g.numel(), " elements, no multiple of the ", B,
                    " upstream gradients");
  check_rc(d3pm_scale_rows(const_cast<float*>(f32(g, "g")), f32(upstream, "upstream"), (float)baked, B,
                           B ? (long)(g.numel() / B) : 0, stream()));
}

// DiscreteDiffusion.p_sample, :384-403
std::tuple<Tensor, Tensor> p_sample(at::TensorList tables, int64_t K, int64_t T, bool structured, double eps,
                                    const Tensor& logits, const Tensor& x_t, const Tensor& t, const OptTensor& noise,
                                    int64_t noise_kind, int64_t seed, int64_t offset, const OptTensor& offset_dev,
                                    bool want_probs) {
  D3PM_GUARD(logits);
  auto tb = image_tables(tables, K, T, structured, eps);
  auto [B, npos] = dims(x_t);
  need_numel(t, B, "t");
  need_rows(logits, B, npos, K, "logits");
  need_numel(noise, (int64_t)B * npos * K, "noise");
  need_counter(offset_dev, "offset_dev");
  TORCH_CHECK_VALUE(!want_probs || logits.size(-1) == K, "d3pm_mi355x: probabilities are returned for rows of exactly K logits");
  Tensor sample = at::empty(x_t.sizes(), x_t.options().dtype(at::kLong));
  Tensor probs = want_probs ? at::empty_like(logits) : at::empty({0}, logits.options());
  check_rc(d3pm_p_sample(&tb, f32(logits, "logits"), logits.size(-1), x_t.data_ptr(), tok_bytes(x_t, "x_t"), t.data_ptr(),
                         tok_bytes(t, "t"), B, npos, (const float*)opt_ptr(noise, at::kFloat, "noise"), (int)noise_kind,
                         (uint64_t)seed, (uint64_t)offset, (const uint64_t*)opt_ptr(offset_dev, at::kLong, "offset_dev"),
                         sample.data_ptr<int64_t>(), want_probs ? probs.data_ptr<float>() : nullptr, stream()));
  return {sample, probs};
}

// DiscreteDiffusion.prior_bpd, :492-524
Tensor prior_bpd(at::TensorList tables, int64_t K, int64_t T, bool structured, double eps, const Tensor& x0, bool absorbing) {
  D3PM_GUARD(x0);
  auto tb = image_tables(tables, K, T, structured, eps);
  auto [B, npos] = dims(x0);
  auto fo = x0.options().dtype(at::kFloat);
  Tensor out = at::empty({B}, fo);
  const size_t wsb = d3pm_hybrid_loss_workspace(B, npos, (int)K);
  Tensor ws = at::empty({(int64_t)(wsb / 4 + 1)}, fo);
  check_rc(d3pm_prior_bpd(&tb, x0.data_ptr(), tok_bytes(x0, "x0"), B, npos, absorbing ? 1 : 0, out.data_ptr<float>(),
                          ws.data_ptr(), wsb, stream()));
  return out;
}

// _get_logits_from_logistic_pars, :288-309 (+ utils.log_min_exp, d3pm/utils.py:15-18)
Tensor logistic_logits(const Tensor& loc, const Tensor& log_scale, const Tensor& centers, double eps) {
  D3PM_GUARD(loc);
  need_same_shape(loc, log_scale, "loc and log_scale");
  const int64_t K = centers.numel();
  TORCH_CHECK_VALUE(K >= 2, "d3pm_mi355x: at least two bin centres");
  Tensor out = at::empty(with_k(loc, K), loc.options().dtype(at::kFloat));
  check_rc(d3pm_logistic_logits(f32(loc, "loc"), f32(log_scale, "log_scale"), f32(centers, "centers"), (long)loc.numel(),
                                (int)K, (float)eps, out.data_ptr<float>(), stream()));
  return out;
}

// its gradient to (loc, log_scale)
std::tuple<Tensor, Tensor> logistic_logits_backward(const Tensor& loc, const Tensor& log_scale, const Tensor& centers,
                                                    const Tensor& dlogits, double eps) {
  D3PM_GUARD(loc);
  need_same_shape(loc, log_scale, "loc and log_scale");
  const int64_t K = centers.numel();
  need_numel(dlogits, loc.numel() * K, "dlogits");
  Tensor dloc = at::empty_like(loc), dls = at::empty_like(log_scale);
  check_rc(d3pm_logistic_logits_backward(f32(loc, "loc"), f32(log_scale, "log_scale"), f32(centers, "centers"),
                                         f32(dlogits, "dlogits"), (long)loc.numel(), (int)K, (float)eps,
                                         dloc.data_ptr<float>(), dls.data_ptr<float>(), stream()));
  return {dloc, dls};
}

// ---- transition tables
const double* f64(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), "d3pm_mi355x: ", what, " must live on an MI355X (device='cuda'); there is no CPU path");
  TORCH_CHECK(t.scalar_type() == at::kDouble, "d3pm_mi355x: ", what, " must be float64");
  return t.data_ptr<double>();
}
void need_table(const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.dim() == 3 && t.size(1) == t.size(2), "d3pm_mi355x: ", what, " must be [T, K, K]");
}

// DiscreteDiffusion.__init__ table construction, :56-99: (one-step Q_t [T,K,K], q_mats [T,K,K]) float64
std::tuple<Tensor, Tensor> build_tables(const Tensor& betas, int64_t kind, int64_t K, int64_t bands) {
  D3PM_GUARD(betas);
  TORCH_CHECK(betas.is_contiguous(), "d3pm_mi355x: betas must be contiguous");
  const int64_t T = betas.numel();
  Tensor one = at::empty({T, K, K}, betas.options().dtype(at::kDouble)), bar = at::empty_like(one);
  check_rc(d3pm_build_tables_f64((int)kind, (int)K, (int)T, (int)bands, f64(betas, "betas"), one.data_ptr<double>(),
                                 bar.data_ptr<double>(), stream()));
  return {one, bar};
}

// Tokenizer.q_uniform_schedule + cumprod_matrix, protein_generation/utils.py:65-83, :7-18: (Q_t, Q_bar) float64
std::tuple<Tensor, Tensor> protein_uniform_tables(const Tensor& off, const Tensor& norm, int64_t K) {
  D3PM_GUARD(off);
  need_same_shape(off, norm, "off and norm");
  const int64_t T = off.numel();
  Tensor one = at::empty({T, K, K}, off.options().dtype(at::kDouble)), bar = at::empty_like(one);
  check_rc(d3pm_protein_uniform_tables_f64((int)K, (int)T, f32(off, "off"), f32(norm, "norm"), one.data_ptr<double>(),
                                           bar.data_ptr<double>(), stream()));
  return {one, bar};
}

// cumprod_matrix, protein_generation/utils.py:7-18, on a (possibly strided) [T,K,K] float64 tensor
Tensor cumprod(const Tensor& mats) {
  D3PM_GUARD(mats);
  need_table(mats, "mats");
  Tensor out = at::empty(mats.sizes(), mats.options().memory_format(at::MemoryFormat::Contiguous));
  check_rc(d3pm_cumprod_f64((int)mats.size(1), (int)mats.size(0), f64(mats, "mats"), mats.stride(0), mats.stride(1),
                            mats.stride(2), out.data_ptr<double>(), stream()));
  return out;
}

// column-structure digests of a (possibly strided) float64 table: (digest, violations int32 [1])
std::tuple<Tensor, Tensor> digest_f32(const Tensor& table, double eps) {
  D3PM_GUARD(table);
  need_table(table, "table");
  const int64_t T = table.size(0), K = table.size(1);
  Tensor dg = at::empty({T, 8, K}, table.options().dtype(at::kFloat));
  Tensor viol = at::zeros({1}, table.options().dtype(at::kInt));
  check_rc(d3pm_digest_f32(f64(table, "table"), table.stride(0), table.stride(1), table.stride(2), (int)T, (int)K,
                           (float)eps, dg.data_ptr<float>(), viol.data_ptr<int>(), stream()));
  return {dg, viol};
}
std::tuple<Tensor, Tensor> digest_f64(const Tensor& table, double rtol) {
  D3PM_GUARD(table);
  need_table(table, "table");
  const int64_t T = table.size(0), K = table.size(1);
  Tensor dg = at::empty({T, 4, K}, table.options().dtype(at::kDouble));
  Tensor viol = at::zeros({1}, table.options().dtype(at::kInt));
  check_rc(d3pm_digest_f64(f64(table, "table"), table.stride(0), table.stride(1), table.stride(2), (int)T, (int)K, rtol,
                           dg.data_ptr<double>(), viol.data_ptr<int>(), stream()));
  return {dg, viol};
}
// per-timestep float32 constants of the training form of the LVB loss, from the two float64 digests
Tensor lvb_digest(const Tensor& qbar_digest, const Tensor& qone_digest, int64_t K, int64_t T) {
  D3PM_GUARD(qbar_digest);
  auto tb = protein_tables(qbar_digest, qone_digest, Tensor(), K, T);
  Tensor out = at::empty({T, (int64_t)(d3pm_lvb_digest_f32_size(1) / (32 * sizeof(float))), 32},
                         qbar_digest.options().dtype(at::kFloat));
  check_rc(d3pm_lvb_digest_f32(&tb, out.data_ptr<float>(), stream()));
  return out;
}

// content fingerprints of several same-device float64 tables in one tensor (int64 [n]): the cache key of callers
// that are handed fresh copies of their tables on every call (notebook cell-12)
Tensor table_fingerprints(at::TensorList tables) {
  TORCH_CHECK(tables.size() >= 1, "d3pm_mi355x: at least one table");
  D3PM_GUARD(tables[0]);
  Tensor out = at::zeros({(int64_t)tables.size()}, tables[0].options().dtype(at::kLong));
  for (size_t i = 0; i < tables.size(); ++i) {
    const Tensor& tb = tables[i];
    need_table(tb, "table");
    TORCH_CHECK(tb.device() == tables[0].device(), "d3pm_mi355x: tables on different devices");
    check_rc(d3pm_table_fingerprint(f64(tb, "table"), tb.stride(0), tb.stride(1), tb.stride(2), (int)tb.size(0),
                                    (int)tb.size(1), (uint64_t*)(out.data_ptr<int64_t>() + i), stream()));
  }
  return out;
}

// the float32 cast of _at / _at_onehot (:218, :242), done once, into a contiguous [T,K,K]
Tensor table_to_f32(const Tensor& table) {
  D3PM_GUARD(table);
  need_table(table, "table");
  Tensor out = at::empty(table.sizes(), table.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
  check_rc(d3pm_table_to_f32(f64(table, "table"), table.stride(0), table.stride(1), table.stride(2), (int)table.size(0),
                             (int)table.size(1), out.data_ptr<float>(), stream()));
  return out;
}

// a contiguous float32 [T,K,K] table of probabilities as two float16 planes (hi, lo of 2^14 x the entry), laid out
// [T, K / 32, K / 16, 2, 64, 8] as the operand image of the float16 matrix instructions: the operand form of
// _at_onehot's matmul (:242-247)
Tensor table_split_f16x2(const Tensor& table) {
  D3PM_GUARD(table);
  TORCH_CHECK_VALUE(table.dim() == 3 && table.size(1) == table.size(2), "d3pm_mi355x: table must be [T, K, K]");
  const int64_t T = table.size(0), K = table.size(1);
  TORCH_CHECK_VALUE(K % 32 == 0, "d3pm_mi355x: the operand image needs K to be a multiple of 32");
  Tensor out = at::empty({T, K / 32, K / 16, 2, 64, 8}, table.options().dtype(at::kHalf));
  check_rc(d3pm_table_split_f16x2(f32(table, "table"), (int)T, (int)K, (uint16_t*)out.data_ptr(), stream()));
  return out;
}

struct ProtShape { int B; long npos; };
ProtShape check_prot_args(const Tensor& pred, const Tensor* x0, const Tensor& x_t, const Tensor& t, int64_t K) {
  auto [B, npos] = dims(x_t);
  if (x0) need_same_shape(*x0, x_t, "x0 and x_t");
  need_numel(t, B, "t");
  need_rows(pred, B, npos, K, "pred");
  return {B, npos};
}

// D3PMLVBLoss.forward / D3PMLVBLossMSA.forward per batch element, protein_generation/losses.py:48-155
std::tuple<Tensor, Tensor> lvb_loss(const Tensor& qbar_digest, const Tensor& qone_digest, const Tensor& lvb_digest, int64_t K, int64_t T,
                                    const Tensor& pred, const Tensor& x0, const Tensor& x_t, const Tensor& t,
                                    const OptTensor& q, int64_t tmax, int64_t msa, double grad_scale, bool want_grad) {
  D3PM_GUARD(pred);
  auto tb = protein_tables(qbar_digest, qone_digest, lvb_digest, K, T);
  auto [B, npos] = check_prot_args(pred, &x0, x_t, t, K);
  need_numel(q, (int64_t)B * npos * K, "q");
  TORCH_CHECK(tok_bytes(x0, "x0") == 8 && tok_bytes(x_t, "x_t") == 8 && tok_bytes(t, "t") == 8,
              "d3pm_mi355x: protein-style tokens and timesteps are int64");
  Tensor per = at::empty({B}, pred.options().dtype(at::kDouble));
  Tensor dp = want_grad ? at::empty_like(pred) : at::empty({0}, pred.options());
  const size_t wsb = d3pm_lvb_loss_workspace(B, npos, (int)K);
  Tensor ws = at::empty({(int64_t)(wsb / 8 + 1)}, pred.options().dtype(at::kDouble));
  check_rc(d3pm_lvb_loss(&tb, f32(pred, "pred"), pred.size(-1), x0.data_ptr<int64_t>(), x_t.data_ptr<int64_t>(),
                         t.data_ptr<int64_t>(), (const double*)opt_ptr(q, at::kDouble, "q"), B, npos, (int)tmax, (int)msa,
                         grad_scale, per.data_ptr<double>(), want_grad ? dp.data_ptr<float>() : nullptr, ws.data_ptr(),
                         wsb, stream()));
  return {per, dp};
}

// the same with the driver's cross-entropy term (Protein Generation Notebook cell-12: (lvb + lambda ce) n_tokens):
// returns (per_seq, ce_seq, dpred)
std::tuple<Tensor, Tensor, Tensor> lvb_hybrid_loss(const Tensor& qbar_digest, const Tensor& qone_digest, const Tensor& lvb_digest, int64_t K, int64_t T,
                                                   const Tensor& pred, const Tensor& x0, const Tensor& x_t, const Tensor& t,
                                                   const OptTensor& q, int64_t tmax, int64_t msa, double grad_scale,
                                                   double ce_grad_scale, bool want_grad) {
  D3PM_GUARD(pred);
  auto tb = protein_tables(qbar_digest, qone_digest, lvb_digest, K, T);
  auto [B, npos] = check_prot_args(pred, &x0, x_t, t, K);
  need_numel(q, (int64_t)B * npos * K, "q");
  TORCH_CHECK(tok_bytes(x0, "x0") == 8 && tok_bytes(x_t, "x_t") == 8 && tok_bytes(t, "t") == 8,
              "d3pm_mi355x: protein-style tokens and timesteps are int64");
  auto dopt = pred.options().dtype(at::kDouble);
  Tensor per = at::empty({B}, dopt), ce = at::empty({B}, dopt);
  Tensor dp = want_grad ? at::empty_like(pred) : at::empty({0}, pred.options());
  const size_t wsb = d3pm_lvb_loss_workspace(B, npos, (int)K);
  Tensor ws = at::empty({(int64_t)(wsb / 8 + 1)}, dopt);
  check_rc(d3pm_lvb_hybrid_loss(&tb, f32(pred, "pred"), pred.size(-1), x0.data_ptr<int64_t>(), x_t.data_ptr<int64_t>(),
                                t.data_ptr<int64_t>(), (const double*)opt_ptr(q, at::kDouble, "q"), B, npos, (int)tmax,
                                (int)msa, grad_scale, ce_grad_scale, per.data_ptr<double>(), ce.data_ptr<double>(),
                                want_grad ? dp.data_ptr<float>() : nullptr, ws.data_ptr(), wsb, stream()));
  return {per, ce, dp};
}

// reverse step of generate_d3pm / generate_msa_d3pm, protein_generation/generate.py:28-40, :70-93
Tensor lvb_reverse_step(const Tensor& qbar_digest, const Tensor& qone_digest, const Tensor& lvb_digest, int64_t K, int64_t T, const Tensor& pred,
                        const Tensor& x_t, const Tensor& t, const OptTensor& expo, int64_t seed, int64_t offset,
                        const OptTensor& offset_dev, double last_class_div, int64_t exclude_last_prefix) {
  D3PM_GUARD(pred);
  auto tb = protein_tables(qbar_digest, qone_digest, lvb_digest, K, T);
  auto [B, npos] = check_prot_args(pred, nullptr, x_t, t, K);
  need_numel(expo, (int64_t)B * npos * K, "expo");
  need_counter(offset_dev, "offset_dev");
  TORCH_CHECK(tok_bytes(x_t, "x_t") == 8 && tok_bytes(t, "t") == 8, "d3pm_mi355x: protein-style tokens are int64");
  Tensor out = at::empty_like(x_t);
  check_rc(d3pm_lvb_reverse_step(&tb, f32(pred, "pred"), pred.size(-1), x_t.data_ptr<int64_t>(), t.data_ptr<int64_t>(), B,
                                 npos, (const double*)opt_ptr(expo, at::kDouble, "expo"), (uint64_t)seed, (uint64_t)offset,
                                 (const uint64_t*)opt_ptr(offset_dev, at::kLong, "offset_dev"), last_class_div,
                                 (long)exclude_last_prefix, out.data_ptr<int64_t>(), stream()));
  return out;
}

// batched sample_transition_matrix as the collaters use it, protein_generation/utils.py:44-52, dataset.py:234-242
std::tuple<Tensor, Tensor> corrupt(const Tensor& qbar_digest, const Tensor& qone_digest, const Tensor& lvb_digest, int64_t K, int64_t T,
                                   const Tensor& x0, const Tensor& t, const OptTensor& expo, int64_t seed, int64_t offset,
                                   bool want_probs) {
  D3PM_GUARD(x0);
  auto tb = protein_tables(qbar_digest, qone_digest, lvb_digest, K, T);
  auto [B, npos] = dims(x0);
  need_numel(t, B, "t");
  need_numel(expo, (int64_t)B * npos * K, "expo");
  TORCH_CHECK(tok_bytes(x0, "x0") == 8 && tok_bytes(t, "t") == 8, "d3pm_mi355x: protein-style tokens are int64");
  Tensor x_t = at::empty_like(x0);
  Tensor probs = want_probs ? at::empty(with_k(x0, K), x0.options().dtype(at::kDouble))
                            : at::empty({0}, x0.options().dtype(at::kDouble));
  check_rc(d3pm_corrupt(&tb, x0.data_ptr<int64_t>(), t.data_ptr<int64_t>(), B, npos,
                        (const double*)opt_ptr(expo, at::kDouble, "expo"), (uint64_t)seed, (uint64_t)offset,
                        x_t.data_ptr<int64_t>(), want_probs ? probs.data_ptr<double>() : nullptr, stream()));
  return {x_t, probs};
}

// ---- fine-tuning objectives: losses at logits [..., V] of float32, float16 or bfloat16, any strides
int float_dtype(const Tensor& t, const char* what) {
  const auto st = t.scalar_type();
  TORCH_CHECK_TYPE(st == at::kFloat || st == at::kHalf || st == at::kBFloat16, "d3pm_mi355x: ", what,
                   " must be float32, float16 or bfloat16, got ", st);
  return st == at::kFloat ? D3PM_F32 : st == at::kHalf ? D3PM_F16 : D3PM_BF16;
}
void need_same_device(const Tensor& t, const Tensor& z, const char* what) {
  TORCH_CHECK(t.device() == z.device(), "d3pm_mi355x: ", what, " is on ", t.device(), ", the logits on ", z.device());
}
// Whether logits [B, ..., V] are rows as the library walks them: classes side by side, the middle dimensions with one
// stride (`inner`; -1: there is one position to a sequence).
bool in_rows(const Tensor& z, int64_t* inner) {
  *inner = -1;
  if (z.dim() < 2) return false;
  bool walk = z.size(-1) == 1 || z.stride(-1) == 1;
  int64_t next = 0;                             // what the next middle dimension's stride must be
  for (int64_t i = z.dim() - 2; i >= 1 && walk; --i) {
    if (z.size(i) == 1) continue;
    if (*inner < 0) *inner = z.stride(i);
    else walk = z.stride(i) == next;
    next = z.stride(i) * z.size(i);
  }
  return walk;
}
// Logits as such rows: themselves, or a copy.  A loss makes it once and keeps it for its gradient.
Tensor as_rows(const Tensor& z) {
  int64_t inner;
  return z.dim() < 2 || in_rows(z, &inner) ? z : z.contiguous();
}
// The library's view of them: `rows` keeps the tensor that it points into.
struct LogitsView { Tensor rows; d3pm_logits desc; };
LogitsView logits_view(const Tensor& z, at::IntArrayRef per_row, const char* per_row_name) {
  TORCH_CHECK(z.is_cuda(), "d3pm_mi355x: logits must live on an MI355X (device='cuda'); there is no CPU path");
  TORCH_CHECK_VALUE(z.dim() >= 2 && z.sizes().slice(0, z.dim() - 1) == per_row,
                    "d3pm_mi355x: logits must have the shape of ", per_row_name, " and a trailing class dimension, got ",
                    z.sizes(), " and ", per_row);
  const int64_t V = z.size(-1);
  TORCH_CHECK_VALUE(V >= 1 && V <= (1 << 27), "d3pm_mi355x: logits have ", V, " classes, need 1 .. 2^27");
  LogitsView v{z, {}};
  v.desc.dtype = float_dtype(z, "logits");
  v.desc.V = (int)V;
  v.desc.B = z.size(0);
  v.desc.L = v.desc.B ? z.numel() / V / v.desc.B : 0;
  int64_t inner;
  const bool walk = in_rows(z, &inner);
  if (!walk) v.rows = z.contiguous();
  v.desc.stride_b = walk ? z.stride(0) : v.desc.L * V;
  v.desc.stride_l = !walk ? V : inner >= 0 ? inner : v.desc.stride_b;
  v.desc.data = v.rows.data_ptr();
  return v;
}
const uint8_t* mask_ptr(const Tensor& m, at::IntArrayRef per_row, const Tensor& z) {
  if (!m.defined()) return nullptr;
  need_device(m, "mask");
  need_same_device(m, z, "mask");
  TORCH_CHECK_TYPE(m.scalar_type() == at::kBool, "d3pm_mi355x: mask must be bool, got ", m.scalar_type());
  TORCH_CHECK_VALUE(m.sizes() == per_row, "d3pm_mi355x: mask must have the shape of the logits' positions, got ",
                    m.sizes(), " and ", per_row);
  return (const uint8_t*)m.data_ptr();
}
// inputs as the library takes them: dense, float32
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }
Tensor dense_f32(const Tensor& t) { return t.defined() ? (t.scalar_type() == at::kFloat ? t : t.to(at::kFloat)).contiguous() : t; }
Tensor opt(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
OptTensor as_opt(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
const float* row_f32(const Tensor& t, const Tensor& per_row, const Tensor& z, const char* what) {
  need_same_device(t, z, what);
  need_same_shape(t, per_row, what);
  return f32(t, what);
}
int token_bytes(const Tensor& t, const Tensor& z, const char* what) {
  need_same_device(t, z, what);
  TORCH_CHECK_TYPE(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, "d3pm_mi355x: ", what,
                   " must be int32 or int64, got ", t.scalar_type());
  return tok_bytes(t, what);
}
const float* upstream_ptr(const Tensor& u, const Tensor& z) {
  need_same_device(u, z, "upstream");
  need_numel(u, 1, "upstream");
  return f32(u, "upstream");
}
int64_t workspace_doubles(const Tensor& z) {
  const long B = z.dim() ? z.size(0) : 0, L = z.dim() > 1 && z.numel() ? z.numel() / z.size(-1) / B : 0;
  return (int64_t)(d3pm_objective_workspace(B, L) / 8 + 1);
}
Tensor objective_workspace(const Tensor& z) { return at::empty({workspace_doubles(z)}, z.options().dtype(at::kDouble)); }
// the workspace of a loss call, for its gradient alone
Tensor need_workspace(const Tensor& ws, const Tensor& z) {
  need_device(ws, "workspace");
  need_same_device(ws, z, "workspace");
  TORCH_CHECK(ws.scalar_type() == at::kDouble, "d3pm_mi355x: workspace must be float64");
  need_numel(ws, workspace_doubles(z), "workspace");
  return ws;
}
void* grad_ptr(const Tensor& dz, const Tensor& z) {
  need_device(dz, "dlogits");
  need_same_device(dz, z, "dlogits");
  need_same_shape(dz, z, "dlogits and logits");
  TORCH_CHECK(dz.scalar_type() == z.scalar_type(), "d3pm_mi355x: dlogits must have the logits' type");
  return dz.data_ptr();
}
Tensor grad_buffer(const Tensor& z) { return at::empty(z.sizes(), z.options().memory_format(at::MemoryFormat::Contiguous)); }

// The autograd nodes of these losses are C++: at the sizes where the host is the bound (a protein batch), a Python
// node and its saved tensors took 40 us of a 96 us forward and backward (57 now, 50 of them torch's engine; in one thread
// 52 and 31, 28 of them the engine).  A node keeps what its gradient needs, and
// the gradient buffer that the loss launch filled for an upstream gradient of 1; backward hands that buffer over
// after a launch that does it again only if the upstream gradient is another number, and a second backward
// (retain_graph) fills a buffer of its own.  So does a backward that is captured into another graph than its forward, or
// captured without it: a replay would find the buffer as the last one left it, not as the forward fills it.
//
// The autograd kernel of an operator calls, through the dispatcher, the operator itself (no gradient wanted) or one of
// underscored name that returns what the node keeps too; backward calls one that fills the gradient.  So dispatch modes
// and transforms see what runs.  Those operators are not differentiable themselves: their derivative is an error.
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

template <typename F>
c10::TypedOperatorHandle<F> op_handle(const char* name, F*) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
// the operator that `run` is the device kernel of
#define D3PM_CALL(name, run, ...)                                            \
  ([&] {                                                                     \
    static const auto op_ = op_handle("d3pm_mi355x::" name, &run);           \
    return op_.call(__VA_ARGS__);                                            \
  }())

// the capture that the current stream of the tensor's device is in, 0 if none
unsigned long long capture_id(const Tensor& on) {
  D3PM_GUARD(on);
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo((hipStream_t)stream(), &status, &id) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return status == hipStreamCaptureStatusActive ? id + 1 : 0;
}

// a gradient, as a function of the logits and the upstream gradient without a derivative
Tensor once_differentiable(const Tensor& grad, const Tensor&, const Tensor&) { return grad.clone(); }

struct ObjectiveNode : public torch::autograd::Node {
  SavedVariable logits_;
  std::vector<SavedVariable> saved_;
  Tensor dz_;
  unsigned long long capture_ = 0;       // that the loss launch was in
  bool released_ = false;

  // rows: the logits, or their copy
  void save(const Tensor& logits, const Tensor& rows, std::initializer_list<Tensor> others) {
    logits_ = SavedVariable(rows, false);
    for (const Tensor& t : others) saved_.emplace_back(t, false);
    set_next_edges(torch::autograd::collect_next_edges(logits));
  }
  void keep_gradient(Tensor&& dz) {
    dz_ = std::move(dz);
    capture_ = capture_id(dz_);
  }
  // the gradient for `upstream` into dz; only_if_rescaled: dz holds that for an upstream gradient of 1
  virtual void fill(const Tensor& logits, const std::vector<Tensor>& saved, const Tensor& upstream,
                    bool only_if_rescaled, Tensor& dz) = 0;

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    TORCH_CHECK(!released_, torch::autograd::ERR_BACKWARD_TWICE);
    if (!grads[0].defined() || !task_should_compute_output(0)) return variable_list(1);
    const bool twice = at::GradMode::is_enabled();
    // (with autograd still in place: a checkpoint computes its part of the model again here)
    const Tensor logits = logits_.unpack(getptr());
    std::vector<Tensor> saved;
    for (const auto& v : saved_) saved.push_back(v.unpack(getptr()));
    Tensor dz;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const Tensor upstream = grads[0].contiguous();
      const bool first = dz_.defined() && capture_ == capture_id(logits);
      dz = first ? std::move(dz_) : at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
      dz_.reset();
      fill(logits, saved, upstream, first, dz);
    }
    if (!twice) return {std::move(dz)};
    // create_graph: the gradient is a value that depends on the logits and on the upstream gradient; differentiating it
    // by either is an error, not a zero, also where it is one term of a sum
    if (dz.key_set().has(c10::DispatchKey::FuncTorchGradWrapper))      // nested transforms: in the graph of each of them
      dz = D3PM_CALL("_once_differentiable", once_differentiable, dz, logits, grads[0]);
    auto edges = torch::autograd::collect_next_edges(grads[0]);
    edges.insert(edges.end(), next_edges().begin(), next_edges().end());
    using torch::autograd::Error;
    torch::autograd::set_history(dz, std::shared_ptr<Error>(new Error("d3pm_mi355x: the gradient of " + name() +
        " cannot be differentiated", std::move(edges)), torch::autograd::deleteNode));
    return {std::move(dz)};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    logits_.reset_data();
    for (auto& v : saved_) v.reset_data();
    dz_.reset();
    released_ = true;
  }
};
template <typename N>
std::shared_ptr<N> new_node() { return std::shared_ptr<N>(new N(), torch::autograd::deleteNode); }
bool differentiated(const Tensor& logits) { return at::GradMode::is_enabled() && logits.requires_grad(); }
// these losses have no forward-mode derivative: a tangent is refused, not dropped
void need_no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(t.defined() && t._fw_grad(0).defined()), "d3pm_mi355x: ", what,
                              " carries a forward-mode tangent, and this loss has no forward-mode derivative");
}
void need_constant(const Tensor& t, const char* what) {
  need_no_tangent(t, what);
  TORCH_CHECK_VALUE(!(t.defined() && at::GradMode::is_enabled() && t.requires_grad()), "d3pm_mi355x: ", what, " is a constant of this loss and must not require a gradient (detach it)");
}

// ---- log_softmax(logits / temperature) at the tokens, float32; stats [.., 4]: what its gradient is made from
std::tuple<Tensor, Tensor> logprobs_run(const Tensor& logits, const Tensor& tokens_, const Tensor& mask,
                                        double temperature, bool want_stats) {
  D3PM_GUARD(logits);
  const Tensor tokens = dense(tokens_), m = dense(mask);
  auto v = logits_view(logits, tokens.sizes(), "tokens");
  auto fo = logits.options().dtype(at::kFloat);
  Tensor lp = at::empty(tokens.sizes(), fo), stats;
  if (want_stats) stats = at::empty({tokens.numel(), 4}, fo);
  check_rc(d3pm_token_logprobs(&v.desc, tokens.data_ptr(), token_bytes(tokens, logits, "tokens"),
                               mask_ptr(m, tokens.sizes(), logits), (float)temperature, lp.data_ptr<float>(),
                               want_stats ? stats.data_ptr<float>() : nullptr, stream()));
  return {lp, stats};
}
Tensor token_logprobs(const Tensor& logits, const Tensor& tokens, const OptTensor& mask, double temperature) {
  return std::get<0>(logprobs_run(logits, tokens, opt(mask), temperature, false));
}
std::tuple<Tensor, Tensor> token_logprobs_stats(const Tensor& logits, const Tensor& tokens, const OptTensor& mask,
                                                double temperature) {
  return logprobs_run(logits, tokens, opt(mask), temperature, true);
}
// the gradient at the logits from the rows' statistics
Tensor& token_grad_(Tensor& dz, const Tensor& logits, const Tensor& tokens, double temperature, const Tensor& stats,
                    const Tensor& upstream, bool per_row, bool only_if_rescaled) {
  D3PM_GUARD(logits);
  auto v = logits_view(logits, tokens.sizes(), "tokens");
  need_numel(stats, tokens.numel() * 4, "stats");
  const float* u = per_row ? row_f32(upstream, tokens, logits, "upstream and tokens") : upstream_ptr(upstream, logits);
  check_rc(d3pm_token_grad(&v.desc, tokens.data_ptr(), token_bytes(tokens, logits, "tokens"), (float)temperature,
                           f32(stats, "stats"), u, per_row, only_if_rescaled, grad_ptr(dz, logits), stream()));
  return dz;
}
struct TokenLogprobsBackward : public ObjectiveNode {
  double temperature;
  std::string name() const override { return "TokenLogprobs"; }
  void fill(const Tensor& logits, const std::vector<Tensor>& s, const Tensor& upstream, bool, Tensor& dz) override {
    D3PM_CALL("_token_grad_", token_grad_, dz, logits, s[0], temperature, s[1], upstream, true, false);
  }
};
Tensor token_logprobs_autograd(const Tensor& logits, const Tensor& tokens_, const OptTensor& mask, double temperature) {
  need_no_tangent(logits, "logits");
  const bool want = differentiated(logits);
  Tensor rows, tokens, lp, stats;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    if (!want) return D3PM_CALL("token_logprobs", token_logprobs, logits, tokens_, mask, temperature);
    rows = as_rows(logits);
    tokens = dense(tokens_);
    std::tie(lp, stats) = D3PM_CALL("_token_logprobs", token_logprobs_stats, rows, tokens, mask, temperature);
  }
  auto node = new_node<TokenLogprobsBackward>();
  node->save(logits, rows, {tokens, stats});
  node->temperature = temperature;
  torch::autograd::set_history(lp, node);
  return lp;
}

// ---- distillation from a teacher's top logits
// loss and per may be null (the gradient alone, times upstream), dz undefined (no gradient); ws: the loss call's workspace
void distill_run(const Tensor& logits, const Tensor& teacher_logits_, const Tensor& teacher_index_, const Tensor& mask_,
                 double temperature, double out_scale, const float* upstream, bool only_if_rescaled, Tensor* loss,
                 Tensor* per, const Tensor& dz, Tensor ws) {
  const Tensor teacher_logits = dense(teacher_logits_), teacher_index = dense(teacher_index_), mask = dense(mask_);
  const auto rows = logits.sizes().slice(0, std::max<int64_t>(logits.dim(), 1) - 1);
  auto v = logits_view(logits, rows, "the teacher's positions");
  need_device(teacher_logits, "teacher_logits");
  need_same_device(teacher_logits, logits, "teacher_logits");
  need_same_shape(teacher_logits, teacher_index, "teacher_logits and teacher_index");
  TORCH_CHECK_VALUE(teacher_logits.dim() == logits.dim() && teacher_logits.sizes().slice(0, logits.dim() - 1) == rows,
                    "d3pm_mi355x: teacher_logits must be [.., k] over the logits' positions, got ",
                    teacher_logits.sizes(), " for ", logits.sizes());
  const int64_t k = teacher_logits.size(-1);
  TORCH_CHECK_VALUE(k >= 1 && k <= 256, "d3pm_mi355x: the teacher's lists have ", k, " entries, need 1 .. 256");
  const int t_dtype = float_dtype(teacher_logits, "teacher_logits");
  const int i_bytes = token_bytes(teacher_index, logits, "teacher_index");
  const uint8_t* m = mask_ptr(mask, rows, logits);
  if (loss) {
    auto fo = logits.options().dtype(at::kFloat);
    *loss = at::empty({}, fo);
    *per = at::empty(rows, fo);
  }
  check_rc(d3pm_topk_distill_loss(&v.desc, teacher_logits.data_ptr(), t_dtype, teacher_index.data_ptr(), i_bytes, (int)k,
                                  m, (float)temperature, (float)out_scale, upstream, only_if_rescaled,
                                  loss ? loss->data_ptr<float>() : nullptr, per ? per->data_ptr<float>() : nullptr,
                                  dz.defined() ? grad_ptr(dz, logits) : nullptr, ws.data_ptr(), ws.nbytes(), stream()));
}
// (loss [], per_token)
std::tuple<Tensor, Tensor> topk_distill_loss(const Tensor& logits, const Tensor& teacher_logits,
                                             const Tensor& teacher_index, const OptTensor& mask, double temperature,
                                             double out_scale) {
  D3PM_GUARD(logits);
  Tensor loss, per;
  distill_run(logits, teacher_logits, teacher_index, opt(mask), temperature, out_scale, nullptr, false, &loss, &per,
              Tensor(), objective_workspace(logits));
  return {loss, per};
}
// (loss, per_token, gradient, workspace)
std::tuple<Tensor, Tensor, Tensor, Tensor> topk_distill_loss_grad(const Tensor& logits, const Tensor& teacher_logits,
                                                                  const Tensor& teacher_index, const OptTensor& mask,
                                                                  double temperature, double out_scale) {
  D3PM_GUARD(logits);
  Tensor loss, per, dz = grad_buffer(logits), ws = objective_workspace(logits);
  distill_run(logits, teacher_logits, teacher_index, opt(mask), temperature, out_scale, nullptr, false, &loss, &per, dz, ws);
  return {loss, per, dz, ws};
}
Tensor& topk_distill_grad_(Tensor& dz, const Tensor& logits, const Tensor& teacher_logits, const Tensor& teacher_index,
                           const OptTensor& mask, double temperature, double out_scale, const Tensor& ws,
                           const Tensor& upstream, bool only_if_rescaled) {
  D3PM_GUARD(logits);
  distill_run(logits, teacher_logits, teacher_index, opt(mask), temperature, out_scale, upstream_ptr(upstream, logits),
              only_if_rescaled, nullptr, nullptr, dz, need_workspace(ws, logits));
  return dz;
}
struct DistillBackward : public ObjectiveNode {
  double temperature, out_scale;
  std::string name() const override { return "TopKDistillLoss"; }
  void fill(const Tensor& logits, const std::vector<Tensor>& s, const Tensor& upstream, bool only, Tensor& dz) override {
    D3PM_CALL("_topk_distill_grad_", topk_distill_grad_, dz, logits, s[0], s[1], as_opt(s[2]), temperature, out_scale, s[3],
              upstream, only);
  }
};
std::tuple<Tensor, Tensor> topk_distill_loss_autograd(const Tensor& logits, const Tensor& teacher_logits_,
                                                      const Tensor& teacher_index_, const OptTensor& mask_,
                                                      double temperature, double out_scale) {
  need_no_tangent(logits, "logits");
  need_constant(teacher_logits_, "teacher_logits");
  const bool want = differentiated(logits);
  Tensor rows, teacher_logits, teacher_index, mask, loss, per, dz, ws;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    if (!want)
      return D3PM_CALL("topk_distill_loss", topk_distill_loss, logits, teacher_logits_, teacher_index_, mask_, temperature,
                       out_scale);
    rows = as_rows(logits);
    teacher_logits = dense(teacher_logits_); teacher_index = dense(teacher_index_); mask = dense(opt(mask_));
    std::tie(loss, per, dz, ws) = D3PM_CALL("_topk_distill_loss", topk_distill_loss_grad, rows, teacher_logits,
                                            teacher_index, as_opt(mask), temperature, out_scale);
  }
  auto node = new_node<DistillBackward>();
  node->save(logits, rows, {teacher_logits, teacher_index, mask, ws});
  node->keep_gradient(std::move(dz));
  node->temperature = temperature;
  node->out_scale = out_scale;
  torch::autograd::set_history(loss, node);
  return {loss, per};
}

// ---- clipped policy loss with a KL term
struct PolicyArgs { double temperature, clip_low, clip_high, kl_coeff, out_scale; };
void policy_run(const Tensor& logits, const Tensor& tokens_, const Tensor& old_logprobs_, const Tensor& advantages_,
                const Tensor& ref_logprobs_, const Tensor& mask_, const PolicyArgs& args, const float* upstream,
                bool only_if_rescaled, Tensor* loss, Tensor* lp, const Tensor& dz, Tensor ws) {
  const Tensor tokens = dense(tokens_), old_logprobs = dense_f32(old_logprobs_), advantages = dense_f32(advantages_),
               ref_logprobs = dense_f32(ref_logprobs_), mask = dense(mask_);
  auto v = logits_view(logits, tokens.sizes(), "tokens");
  const int t_bytes = token_bytes(tokens, logits, "tokens");
  const float* old_lp = row_f32(old_logprobs, tokens, logits, "old_logprobs and tokens");
  const bool per_seq = advantages.dim() == 1 && tokens.dim() > 1;
  if (per_seq) need_numel(advantages, tokens.size(0), "advantages (one per sequence)");
  else need_same_shape(advantages, tokens, "advantages and tokens");
  need_same_device(advantages, logits, "advantages");
  const float* adv = f32(advantages, "advantages");
  const float* ref = ref_logprobs.defined() ? row_f32(ref_logprobs, tokens, logits, "ref_logprobs and tokens") : nullptr;
  const uint8_t* m = mask_ptr(mask, tokens.sizes(), logits);
  if (loss) {
    auto fo = logits.options().dtype(at::kFloat);
    *loss = at::empty({}, fo);
    *lp = at::empty(tokens.sizes(), fo);
  }
  check_rc(d3pm_policy_loss(&v.desc, tokens.data_ptr(), t_bytes, old_lp, adv, per_seq, ref, m, (float)args.temperature,
                            (float)args.clip_low, (float)args.clip_high, (float)args.kl_coeff, (float)args.out_scale,
                            upstream, only_if_rescaled, loss ? loss->data_ptr<float>() : nullptr,
                            lp ? lp->data_ptr<float>() : nullptr, dz.defined() ? grad_ptr(dz, logits) : nullptr,
                            ws.data_ptr(), ws.nbytes(), stream()));
}
// (loss [], logprobs)
std::tuple<Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& tokens, const Tensor& old_logprobs,
                                       const Tensor& advantages, const OptTensor& ref_logprobs, const OptTensor& mask,
                                       double temperature, double clip_low, double clip_high, double kl_coeff,
                                       double out_scale) {
  D3PM_GUARD(logits);
  Tensor loss, lp;
  policy_run(logits, tokens, old_logprobs, advantages, opt(ref_logprobs), opt(mask),
             {temperature, clip_low, clip_high, kl_coeff, out_scale}, nullptr, false, &loss, &lp, Tensor(),
             objective_workspace(logits));
  return {loss, lp};
}
// (loss, logprobs, gradient, workspace)
std::tuple<Tensor, Tensor, Tensor, Tensor> policy_loss_grad(
    const Tensor& logits, const Tensor& tokens, const Tensor& old_logprobs, const Tensor& advantages,
    const OptTensor& ref_logprobs, const OptTensor& mask, double temperature, double clip_low, double clip_high,
    double kl_coeff, double out_scale) {
  D3PM_GUARD(logits);
  Tensor loss, lp, dz = grad_buffer(logits), ws = objective_workspace(logits);
  policy_run(logits, tokens, old_logprobs, advantages, opt(ref_logprobs), opt(mask),
             {temperature, clip_low, clip_high, kl_coeff, out_scale}, nullptr, false, &loss, &lp, dz, ws);
  return {loss, lp, dz, ws};
}
Tensor& policy_grad_(Tensor& dz, const Tensor& logits, const Tensor& tokens, const Tensor& old_logprobs,
                     const Tensor& advantages, const OptTensor& ref_logprobs, const OptTensor& mask, double temperature,
                     double clip_low, double clip_high, double kl_coeff, double out_scale, const Tensor& ws,
                     const Tensor& upstream, bool only_if_rescaled) {
  D3PM_GUARD(logits);
  policy_run(logits, tokens, old_logprobs, advantages, opt(ref_logprobs), opt(mask),
             {temperature, clip_low, clip_high, kl_coeff, out_scale}, upstream_ptr(upstream, logits), only_if_rescaled,
             nullptr, nullptr, dz, need_workspace(ws, logits));
  return dz;
}
struct PolicyBackward : public ObjectiveNode {
  PolicyArgs args;
  std::string name() const override { return "PolicyLoss"; }
  void fill(const Tensor& logits, const std::vector<Tensor>& s, const Tensor& upstream, bool only, Tensor& dz) override {
    D3PM_CALL("_policy_grad_", policy_grad_, dz, logits, s[0], s[1], s[2], as_opt(s[3]), as_opt(s[4]), args.temperature,
              args.clip_low, args.clip_high, args.kl_coeff, args.out_scale, s[5], upstream, only);
  }
};
std::tuple<Tensor, Tensor> policy_loss_autograd(const Tensor& logits, const Tensor& tokens_, const Tensor& old_logprobs_,
                                                const Tensor& advantages_, const OptTensor& ref_logprobs_,
                                                const OptTensor& mask_, double temperature, double clip_low,
                                                double clip_high, double kl_coeff, double out_scale) {
  need_no_tangent(logits, "logits");
  need_constant(old_logprobs_, "old_logprobs");
  need_constant(advantages_, "advantages");
  need_constant(opt(ref_logprobs_), "ref_logprobs");
  const bool want = differentiated(logits);
  Tensor rows, tokens, old_logprobs, advantages, ref_logprobs, mask, loss, lp, dz, ws;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    if (!want)
      return D3PM_CALL("policy_loss", policy_loss, logits, tokens_, old_logprobs_, advantages_, ref_logprobs_, mask_,
                       temperature, clip_low, clip_high, kl_coeff, out_scale);
    rows = as_rows(logits);
    tokens = dense(tokens_); old_logprobs = dense_f32(old_logprobs_); advantages = dense_f32(advantages_);
    ref_logprobs = dense_f32(opt(ref_logprobs_)); mask = dense(opt(mask_));
    std::tie(loss, lp, dz, ws) = D3PM_CALL("_policy_loss", policy_loss_grad, rows, tokens, old_logprobs, advantages,
                                           as_opt(ref_logprobs), as_opt(mask), temperature, clip_low, clip_high, kl_coeff,
                                           out_scale);
  }
  auto node = new_node<PolicyBackward>();
  node->save(logits, rows, {tokens, old_logprobs, advantages, ref_logprobs, mask, ws});
  node->keep_gradient(std::move(dz));
  node->args = {temperature, clip_low, clip_high, kl_coeff, out_scale};
  torch::autograd::set_history(loss, node);
  return {loss, lp};
}

// ---- preference loss of the pairs (p, p + B / 2)
std::tuple<Tensor, Tensor, Tensor> preference_run(const Tensor& logits, const Tensor& tokens_, const Tensor& ref_logprobs_,
                                                  const Tensor& mask_, double beta, double label_smoothing, bool average,
                                                  double out_scale, const Tensor& dz) {
  const Tensor tokens = dense(tokens_), ref_logprobs = dense_f32(ref_logprobs_), mask = dense(mask_);
  auto v = logits_view(logits, tokens.sizes(), "tokens");
  const int t_bytes = token_bytes(tokens, logits, "tokens");
  const float* ref = ref_logprobs.defined() ? row_f32(ref_logprobs, tokens, logits, "ref_logprobs and tokens") : nullptr;
  const uint8_t* m = mask_ptr(mask, tokens.sizes(), logits);
  auto fo = logits.options().dtype(at::kFloat);
  const Tensor loss = at::empty({}, fo), rewards = at::empty({v.desc.B}, fo), stats = at::empty({tokens.numel(), 4}, fo);
  const Tensor ws = objective_workspace(logits);
  check_rc(d3pm_preference_loss(&v.desc, tokens.data_ptr(), t_bytes, ref, m, (float)beta, (float)label_smoothing,
                                average, (float)out_scale, loss.data_ptr<float>(), rewards.data_ptr<float>(),
                                stats.data_ptr<float>(), dz.defined() ? grad_ptr(dz, logits) : nullptr, ws.data_ptr(),
                                ws.nbytes(), stream()));
  return {loss, rewards, stats};
}
// (loss [], rewards [B])
std::tuple<Tensor, Tensor> preference_loss(const Tensor& logits, const Tensor& tokens, const OptTensor& ref_logprobs,
                                           const OptTensor& mask, double beta, double label_smoothing, bool average,
                                           double out_scale) {
  D3PM_GUARD(logits);
  auto [loss, rewards, stats] = preference_run(logits, tokens, opt(ref_logprobs), opt(mask), beta, label_smoothing,
                                               average, out_scale, Tensor());
  return {loss, rewards};
}
// (loss, rewards, gradient, row statistics)
std::tuple<Tensor, Tensor, Tensor, Tensor> preference_loss_grad(const Tensor& logits, const Tensor& tokens,
                                                                const OptTensor& ref_logprobs, const OptTensor& mask,
                                                                double beta, double label_smoothing, bool average,
                                                                double out_scale) {
  D3PM_GUARD(logits);
  const Tensor dz = grad_buffer(logits);
  auto [loss, rewards, stats] = preference_run(logits, tokens, opt(ref_logprobs), opt(mask), beta, label_smoothing,
                                               average, out_scale, dz);
  return {loss, rewards, dz, stats};
}
struct PreferenceBackward : public ObjectiveNode {
  std::string name() const override { return "PreferenceLoss"; }
  void fill(const Tensor& logits, const std::vector<Tensor>& s, const Tensor& upstream, bool only, Tensor& dz) override {
    D3PM_CALL("_token_grad_", token_grad_, dz, logits, s[0], 1.0, s[1], upstream, false, only);
  }
};
std::tuple<Tensor, Tensor> preference_loss_autograd(const Tensor& logits, const Tensor& tokens_,
                                                    const OptTensor& ref_logprobs, const OptTensor& mask, double beta,
                                                    double label_smoothing, bool average, double out_scale) {
  need_no_tangent(logits, "logits");
  need_constant(opt(ref_logprobs), "ref_logprobs");
  const bool want = differentiated(logits);
  Tensor rows, tokens, loss, rewards, stats, dz;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    if (!want)
      return D3PM_CALL("preference_loss", preference_loss, logits, tokens_, ref_logprobs, mask, beta, label_smoothing,
                       average, out_scale);
    rows = as_rows(logits);
    tokens = dense(tokens_);
    std::tie(loss, rewards, dz, stats) = D3PM_CALL("_preference_loss", preference_loss_grad, rows, tokens, ref_logprobs,
                                                   mask, beta, label_smoothing, average, out_scale);
  }
  auto node = new_node<PreferenceBackward>();
  node->save(logits, rows, {tokens, stats});
  node->keep_gradient(std::move(dz));
  torch::autograd::set_history(loss, node);
  return {loss, rewards};
}

}  // namespace

#define D3PM_TB "Tensor[] tables, int K, int T, bool structured, float eps, "
#define D3PM_PT "Tensor qbar_digest, Tensor qone_digest, Tensor lvb_digest, int K, int T, "
#define D3PM_LOSS_ARGS "Tensor logits, Tensor x0, Tensor x_t, Tensor t, int loss_type, float hybrid_coeff, float grad_scale, "

TORCH_LIBRARY(d3pm_mi355x, m) {
  m.def("q_probs(" D3PM_TB "Tensor x0, Tensor t) -> Tensor");
  m.def("q_sample(" D3PM_TB "Tensor x0, Tensor t, Tensor? noise, int noise_kind, int seed, int offset, "
        "Tensor? offset_dev) -> Tensor");
  m.def("q_sample_draw_t(" D3PM_TB "Tensor x0, int seed, int offset, Tensor? offset_dev, Tensor(a!)? clear) -> (Tensor, Tensor)");
  m.def("q_posterior_logits(" D3PM_TB "Tensor x_start, bool x_start_is_logits, Tensor x_t, Tensor t) -> Tensor");
  m.def("q_posterior_logits_backward(" D3PM_TB "Tensor x_start_logits, Tensor t, Tensor grad_out) -> Tensor");
  m.def("hybrid_loss(" D3PM_TB D3PM_LOSS_ARGS "Tensor? grad_out, bool want_grad) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("hybrid_loss_step(" D3PM_TB D3PM_LOSS_ARGS "bool want_grad, Tensor(a!)? loss_mean, Tensor(b!)? rng_counter, "
        "int rng_step) -> (Tensor, Tensor)");
  m.def("hybrid_loss_then_q_sample(" D3PM_TB D3PM_LOSS_ARGS "bool want_grad, Tensor next_x0, int seed, int offset, "
        "Tensor? offset_dev) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("hybrid_loss_static_(" D3PM_TB D3PM_LOSS_ARGS "Tensor(a!) loss, Tensor(b!)? dlogits) -> ()");
  m.def("scale_rows_(Tensor(a!) g, Tensor upstream, float baked) -> ()");
  m.def("p_sample(" D3PM_TB "Tensor logits, Tensor x_t, Tensor t, Tensor? noise, int noise_kind, int seed, int offset, "
        "Tensor? offset_dev, bool want_probs) -> (Tensor, Tensor)");
  m.def("prior_bpd(" D3PM_TB "Tensor x0, bool absorbing) -> Tensor");
  m.def("logistic_logits(Tensor loc, Tensor log_scale, Tensor centers, float eps) -> Tensor");
  m.def("logistic_logits_backward(Tensor loc, Tensor log_scale, Tensor centers, Tensor dlogits, float eps) -> (Tensor, Tensor)");
  m.def("build_tables(Tensor betas, int kind, int K, int bands) -> (Tensor, Tensor)");
  m.def("protein_uniform_tables(Tensor off, Tensor norm, int K) -> (Tensor, Tensor)");
  m.def("cumprod(Tensor mats) -> Tensor");
  m.def("digest_f32(Tensor table, float eps) -> (Tensor, Tensor)");
  m.def("digest_f64(Tensor table, float rtol) -> (Tensor, Tensor)");
  m.def("table_to_f32(Tensor table) -> Tensor");
  m.def("table_split_f16x2(Tensor table) -> Tensor");
  m.def("table_fingerprints(Tensor[] tables) -> Tensor");
  m.def("lvb_digest(Tensor qbar_digest, Tensor qone_digest, int K, int T) -> Tensor");
  m.def("lvb_loss(" D3PM_PT "Tensor pred, Tensor x0, Tensor x_t, Tensor t, Tensor? q, int tmax, int msa, "
        "float grad_scale, bool want_grad) -> (Tensor, Tensor)");
  m.def("lvb_hybrid_loss(" D3PM_PT "Tensor pred, Tensor x0, Tensor x_t, Tensor t, Tensor? q, int tmax, int msa, "
        "float grad_scale, float ce_grad_scale, bool want_grad) -> (Tensor, Tensor, Tensor)");
  m.def("lvb_reverse_step(" D3PM_PT "Tensor pred, Tensor x_t, Tensor t, Tensor? expo, int seed, int offset, "
        "Tensor? offset_dev, float last_class_div, int exclude_last_prefix) -> Tensor");
  m.def("corrupt(" D3PM_PT "Tensor x0, Tensor t, Tensor? expo, int seed, int offset, bool want_probs) -> (Tensor, Tensor)");
#define D3PM_TEMPERATURE "Tensor? mask, float temperature"
#define D3PM_DISTILL "Tensor logits, Tensor teacher_logits, Tensor teacher_index, " D3PM_TEMPERATURE ", float out_scale"
#define D3PM_POLICY "Tensor logits, Tensor tokens, Tensor old_logprobs, Tensor advantages, Tensor? ref_logprobs, " \
                    D3PM_TEMPERATURE ", float clip_low, float clip_high, float kl_coeff, float out_scale"
#define D3PM_PREFERENCE "Tensor logits, Tensor tokens, Tensor? ref_logprobs, Tensor? mask, float beta, " \
                        "float label_smoothing, bool average, float out_scale"
  m.def("token_logprobs(Tensor logits, Tensor tokens, " D3PM_TEMPERATURE ") -> Tensor");
  m.def("topk_distill_loss(" D3PM_DISTILL ") -> (Tensor, Tensor)");
  m.def("policy_loss(" D3PM_POLICY ") -> (Tensor, Tensor)");
  m.def("preference_loss(" D3PM_PREFERENCE ") -> (Tensor, Tensor)");
  // what their autograd kernels call
  m.def("_token_logprobs(Tensor logits, Tensor tokens, " D3PM_TEMPERATURE ") -> (Tensor, Tensor)");
  m.def("_topk_distill_loss(" D3PM_DISTILL ") -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("_policy_loss(" D3PM_POLICY ") -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("_preference_loss(" D3PM_PREFERENCE ") -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("_once_differentiable(Tensor grad, Tensor logits, Tensor upstream) -> Tensor");
  m.def("_token_grad_(Tensor(a!) dlogits, Tensor logits, Tensor tokens, float temperature, Tensor stats, Tensor upstream, "
        "bool per_row, bool only_if_rescaled) -> Tensor(a!)");
  m.def("_topk_distill_grad_(Tensor(a!) dlogits, " D3PM_DISTILL ", Tensor workspace, Tensor upstream, "
        "bool only_if_rescaled) -> Tensor(a!)");
  m.def("_policy_grad_(Tensor(a!) dlogits, " D3PM_POLICY ", Tensor workspace, Tensor upstream, bool only_if_rescaled) -> Tensor(a!)");
}

TORCH_LIBRARY_IMPL(d3pm_mi355x, CUDA, m) {
  m.impl("q_probs", q_probs);
  m.impl("q_sample", q_sample);
  m.impl("q_sample_draw_t", q_sample_draw_t);
  m.impl("q_posterior_logits", q_posterior_logits);
  m.impl("q_posterior_logits_backward", q_posterior_logits_backward);
  m.impl("hybrid_loss", hybrid_loss);
  m.impl("hybrid_loss_step", hybrid_loss_step);
  m.impl("hybrid_loss_then_q_sample", hybrid_loss_then_q_sample);
  m.impl("hybrid_loss_static_", hybrid_loss_static_);
  m.impl("scale_rows_", scale_rows_);
  m.impl("p_sample", p_sample);
  m.impl("prior_bpd", prior_bpd);
  m.impl("logistic_logits", logistic_logits);
  m.impl("logistic_logits_backward", logistic_logits_backward);
  m.impl("build_tables", build_tables);
  m.impl("protein_uniform_tables", protein_uniform_tables);
  m.impl("cumprod", cumprod);
  m.impl("digest_f32", digest_f32);
  m.impl("digest_f64", digest_f64);
  m.impl("table_to_f32", table_to_f32);
  m.impl("table_split_f16x2", table_split_f16x2);
  m.impl("table_fingerprints", table_fingerprints);
  m.impl("lvb_digest", lvb_digest);
  m.impl("lvb_loss", lvb_loss);
  m.impl("lvb_hybrid_loss", lvb_hybrid_loss);
  m.impl("lvb_reverse_step", lvb_reverse_step);
  m.impl("corrupt", corrupt);
  m.impl("token_logprobs", token_logprobs);
  m.impl("topk_distill_loss", topk_distill_loss);
  m.impl("policy_loss", policy_loss);
  m.impl("preference_loss", preference_loss);
  m.impl("_token_logprobs", token_logprobs_stats);
  m.impl("_topk_distill_loss", topk_distill_loss_grad);
  m.impl("_policy_loss", policy_loss_grad);
  m.impl("_preference_loss", preference_loss_grad);
  m.impl("_once_differentiable", once_differentiable);
  m.impl("_token_grad_", token_grad_);
  m.impl("_topk_distill_grad_", topk_distill_grad_);
  m.impl("_policy_grad_", policy_grad_);
}

// the fine-tuning objectives bring their own autograd nodes
TORCH_LIBRARY_IMPL(d3pm_mi355x, AutogradCUDA, m) {
  m.impl("token_logprobs", token_logprobs_autograd);
  m.impl("topk_distill_loss", topk_distill_loss_autograd);
  m.impl("policy_loss", policy_loss_autograd);
  m.impl("preference_loss", preference_loss_autograd);
  for (const char* name : {"_token_logprobs", "_topk_distill_loss", "_policy_loss", "_preference_loss", "_token_grad_",
                           "_topk_distill_grad_", "_policy_grad_", "_once_differentiable"})
    m.impl(name, torch::autograd::autogradNotImplementedFallback());
}
