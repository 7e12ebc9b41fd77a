// Operators of a language model that torch's layers do not cover on this
// device, in the `ocl` namespace: the root-mean-square norm with the residual's
// addition (and its output in 8 bits), the linear layer in 8-bit floating point
// with scales, and the log probabilities of given tokens.  The reference had
// none of them: its norm is layer norm (src/norm_ops.cpp:167-351), its layers
// and log_softmax + nll_loss are fp32 (src/vision_ops.cpp:243-351,
// src/loss_ops.cpp:23-213).
#include <torch/csrc/autograd/custom_function.h>
#include <torch/extension.h>

#include "ocl.h"

namespace ocl {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

static bool float_type(c10::ScalarType t) { return t == at::kFloat || t == at::kHalf || t == at::kBFloat16; }

static bool given(const std::optional<at::Tensor>& t) { return t.has_value() && t->defined(); }

// whether autograd has to see this: a gradient is asked for, or a tangent of
// forward mode is there (which the functions refuse)
static bool differentiated(std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    if (t && t->defined() && ((at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined())) return true;
  return false;
}
static const at::Tensor* pointer(const std::optional<at::Tensor>& t) { return given(t) ? &*t : nullptr; }

static void no_second_gradient(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "ocl ", op, ": the backward pass cannot be differentiated again");
}

// [..., D] as [rows, D] with unit stride along D and rows apart, or a copy
static at::Tensor rows_of(const at::Tensor& t) {
  const int64_t D = t.size(-1);
  int64_t R = 1;
  for (int64_t k = 0; k + 1 < t.dim(); ++k) R *= t.size(k);
  const at::Tensor m = t.reshape({R, D});
  return (D <= 1 || m.stride(1) == 1) && (R <= 1 || m.stride(0) >= D) ? m : contiguous(m);
}

static int64_t groups_of(int64_t D) { return (D + 127) / 128; }

static at::DimVector with_last(c10::IntArrayRef sizes, int64_t last) {
  at::DimVector s(sizes.begin(), sizes.end());
  s.back() = last;
  return s;
}

// codes of this shape, rows on 16-byte boundaries
static at::Tensor empty_codes(c10::IntArrayRef sizes, int dev) {
  at::DimVector strides(sizes.size(), 1);
  int64_t step = (sizes.back() + 15) / 16 * 16;
  for (int64_t k = (int64_t)sizes.size() - 2; k >= 0; --k) {
    strides[k] = step;
    step *= std::max<int64_t>(1, sizes[k]);
  }
  return empty_strided_dev(sizes, strides, at::kByte, dev);
}

// ---------------------------------------------------------------- RMS norm
static void norm_check(const char* op, const at::Tensor& x, const std::optional<at::Tensor>& weight,
                       const std::optional<at::Tensor>& residual) {
  TORCH_CHECK(is_ocl(x) && float_type(x.scalar_type()) && x.dim() >= 1, "ocl ", op,
              ": fp32, fp16 or bf16 rows [..., features] on ocl expected, got ", x.scalar_type(), " ", x.sizes(), " on ",
              x.device());
  if (given(weight))
    TORCH_CHECK(is_ocl(*weight) && weight->device() == x.device() && weight->scalar_type() == x.scalar_type() &&
                    weight->dim() == 1 && weight->size(0) == x.size(-1),
                "ocl ", op, ": weight [features] of the input's type and device expected, got ", weight->scalar_type(), " ",
                weight->sizes(), " on ", weight->device());
  if (given(residual))
    TORCH_CHECK(is_ocl(*residual) && residual->device() == x.device() && residual->scalar_type() == x.scalar_type() &&
                    residual->sizes().equals(x.sizes()),
                "ocl ", op, ": a residual of the input's shape, type and device expected, got ", residual->scalar_type(),
                " ", residual->sizes(), " on ", residual->device());
}

static pvb2_rms_norm_desc norm_desc(const at::Tensor& rows, double eps) {
  pvb2_rms_norm_desc d;
  memset(&d, 0, sizeof(d));
  d.rows = rows.size(0);
  d.D = rows.size(1);
  d.ldx = rows.stride(0);
  d.eps = eps;
  d.dtype = dtype_code(rows.scalar_type());
  return d;
}

struct NormForward {
  at::Tensor y, sum, rstd, scales;  // y: codes where there are scales
};

static NormForward norm_forward(const char* op, const at::Tensor& input, const std::optional<at::Tensor>& weight,
                                const std::optional<at::Tensor>& residual, double eps, bool codes, bool keep) {
  norm_check(op, input, weight, residual);
  const int dev = input.device().index();
  DeviceScope scope(dev);
  OCL_OP(op, dev);
  const at::Tensor x = rows_of(input);
  at::Tensor w, r;
  if (given(weight)) w = contiguous(*weight);
  pvb2_rms_norm_desc d = norm_desc(x, eps);
  NormForward f;
  if (given(residual)) {
    r = rows_of(*residual);
    d.ldr = r.stride(0);
    f.sum = empty(input.sizes(), input.scalar_type(), dev);
  }
  const void* rp = r.defined() ? r.data_ptr() : nullptr;
  const void* wp = w.defined() ? w.data_ptr() : nullptr;
  void* sp = f.sum.defined() ? f.sum.data_ptr() : nullptr;
  if (codes) {
    f.y = empty_codes(input.sizes(), dev);
    f.scales = empty(with_last(input.sizes(), groups_of(d.D)), at::kFloat, dev);
    d.ldc = (d.D + 15) / 16 * 16;
    OCL_CHECK(pvb2_rms_norm_8bit(&d, x.data_ptr(), rp, wp, (uint8_t*)f.y.data_ptr(), (float*)f.scales.data_ptr(), sp,
                                 stream_for(dev)));
    return f;
  }
  f.y = empty(input.sizes(), input.scalar_type(), dev);
  if (keep) f.rstd = empty({d.rows}, at::kFloat, dev);
  OCL_CHECK(pvb2_rms_norm_fwd(&d, x.data_ptr(), rp, wp, f.y.data_ptr(), sp,
                              f.rstd.defined() ? (float*)f.rstd.data_ptr() : nullptr, stream_for(dev)));
  return f;
}

// gradients of the input (and of the residual: the same) and of the weight
static std::tuple<at::Tensor, at::Tensor> norm_backward(const at::Tensor& gy, const at::Tensor& gsum, const at::Tensor& h,
                                                        const at::Tensor& weight, const at::Tensor& rstd, bool need_x,
                                                        bool need_w) {
  const int dev = h.device().index();
  DeviceScope scope(dev);
  OCL_OP("rms_norm_backward", dev);
  const at::Tensor x = rows_of(h), g = rows_of(gy);
  at::Tensor w, gs, dx, dw;
  if (weight.defined()) w = contiguous(weight);
  pvb2_rms_norm_desc d = norm_desc(x, 0.0);
  d.ldg = g.stride(0);
  if (gsum.defined()) {
    gs = rows_of(gsum);
    d.ldr = gs.stride(0);
  }
  if (need_x) dx = empty(h.sizes(), h.scalar_type(), dev);
  if (need_w) dw = empty({d.D}, h.scalar_type(), dev);
  Workspace ws(need_w ? pvb2_rms_norm_bwd_workspace_size(&d) : 0, dev);
  OCL_CHECK(pvb2_rms_norm_bwd(&d, x.data_ptr(), w.defined() ? w.data_ptr() : nullptr, (const float*)rstd.data_ptr(),
                              g.data_ptr(), gs.defined() ? gs.data_ptr() : nullptr, dx.defined() ? dx.data_ptr() : nullptr,
                              dw.defined() ? dw.data_ptr() : nullptr, ws.get(), ws.bytes, stream_for(dev)));
  return {dx, dw};
}

struct RmsNorm : public torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& input, const std::optional<at::Tensor>& weight,
                               const std::optional<at::Tensor>& residual, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    const NormForward f = norm_forward("rms_norm", input, weight, residual, eps, false, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({f.sum.defined() ? f.sum : input, given(weight) ? *weight : at::Tensor(), f.rstd});
    ctx->saved_data["weight"] = given(weight);
    ctx->saved_data["residual"] = given(residual);
    if (f.sum.defined()) return {f.y, f.sum};
    return {f.y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_gradient("rms_norm");
    const variable_list s = ctx->get_saved_variables();
    // needs_input_grad counts the tensors that were passed
    size_t at = 1;
    const bool need_w = ctx->saved_data["weight"].toBool() && ctx->needs_input_grad(at++);
    const bool need_r = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(at);
    const bool need_x = ctx->needs_input_grad(0);
    const at::Tensor gsum = grads.size() > 1 ? grads[1] : at::Tensor();
    at::Tensor dx, dw;
    if (!grads[0].defined()) dx = gsum;  // the norm itself was not used
    else std::tie(dx, dw) = norm_backward(grads[0], gsum, s[0], s[1], s[2], need_x || need_r, need_w);
    const at::Tensor none;
    return {need_x ? dx : none, dw, need_r ? dx : none, none};
  }
};

static at::Tensor rms_norm(const at::Tensor& x, const std::optional<at::Tensor>& weight, double eps) {
  return norm_forward("rms_norm", x, weight, std::nullopt, eps, false, false).y;
}

static at::Tensor rms_norm_autograd(const at::Tensor& x, const std::optional<at::Tensor>& weight, double eps) {
  if (differentiated({&x, pointer(weight)})) return RmsNorm::apply(x, weight, std::optional<at::Tensor>(), eps)[0];
  at::AutoDispatchBelowADInplaceOrView below;
  return rms_norm(x, weight, eps);
}

static std::tuple<at::Tensor, at::Tensor> rms_norm_add(const at::Tensor& x, const at::Tensor& residual,
                                                       const std::optional<at::Tensor>& weight, double eps) {
  const NormForward f = norm_forward("rms_norm", x, weight, residual, eps, false, false);
  return {f.y, f.sum};
}

static std::tuple<at::Tensor, at::Tensor> rms_norm_add_autograd(const at::Tensor& x, const at::Tensor& residual,
                                                                const std::optional<at::Tensor>& weight, double eps) {
  if (differentiated({&x, &residual, pointer(weight)})) {
    const variable_list out = RmsNorm::apply(x, weight, std::optional<at::Tensor>(residual), eps);
    return {out[0], out[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return rms_norm_add(x, residual, weight, eps);
}

static std::vector<at::Tensor> rms_norm_8bit(const at::Tensor& x, const std::optional<at::Tensor>& weight,
                                             const std::optional<at::Tensor>& residual, double eps) {
  const NormForward f = norm_forward("rms_norm_8bit", x, weight, residual, eps, true, false);
  if (f.sum.defined()) return {f.y, f.scales, f.sum};
  return {f.y, f.scales};
}

static void no_gradient(const char* op, bool differentiated) {
  TORCH_CHECK(!differentiated, "ocl ", op, ": codes have no gradient; call it under torch.no_grad() or on detached tensors");
}

static std::vector<at::Tensor> rms_norm_8bit_autograd(const at::Tensor& x, const std::optional<at::Tensor>& weight,
                                                      const std::optional<at::Tensor>& residual, double eps) {
  no_gradient("rms_norm_8bit", differentiated({&x, pointer(weight), pointer(residual)}));
  at::AutoDispatchBelowADInplaceOrView below;
  return rms_norm_8bit(x, weight, residual, eps);
}

// ------------------------------------------------- 8-bit codes with scales
static std::tuple<at::Tensor, at::Tensor> quantize_8bit(const at::Tensor& input, bool tall) {
  TORCH_CHECK(is_ocl(input) && float_type(input.scalar_type()) && input.dim() >= (tall ? 2 : 1),
              "ocl quantize_8bit: fp32, fp16 or bf16 [..., features] on ocl expected, got ", input.scalar_type(), " ",
              input.sizes(), " on ", input.device());
  TORCH_CHECK(!tall || input.dim() == 2, "ocl quantize_8bit: blocks of 128 rows are of a matrix, got ", input.sizes());
  const int dev = input.device().index();
  DeviceScope scope(dev);
  OCL_OP("quantize_8bit", dev);
  const at::Tensor x = rows_of(input);
  const int64_t R = x.size(0), D = x.size(1);
  at::Tensor codes = empty_codes(input.sizes(), dev);
  at::Tensor scales = tall ? empty({groups_of(R), groups_of(D)}, at::kFloat, dev)
                           : empty(with_last(input.sizes(), groups_of(D)), at::kFloat, dev);
  OCL_CHECK(pvb2_quantize_8bit(dtype_code(x.scalar_type()), R, D, x.data_ptr(), x.stride(0), tall ? 1 : 0,
                               (uint8_t*)codes.data_ptr(), (D + 15) / 16 * 16, (float*)scales.data_ptr(), stream_for(dev)));
  return {codes, scales};
}

static std::tuple<at::Tensor, at::Tensor> quantize_8bit_autograd(const at::Tensor& input, bool tall) {
  no_gradient("quantize_8bit", differentiated({&input}));
  at::AutoDispatchBelowADInplaceOrView below;
  return quantize_8bit(input, tall);
}

static void codes_check(const char* op, const char* what, const at::Tensor& codes, const at::Tensor& scales, bool tall,
                        const at::Tensor& lead) {
  TORCH_CHECK(is_ocl(codes) && codes.scalar_type() == at::kByte && codes.dim() >= 1 && is_ocl(scales) &&
                  scales.scalar_type() == at::kFloat && codes.device() == lead.device() && scales.device() == lead.device(),
              "ocl ", op, ": ", what, ": uint8 codes [..., features] and fp32 scales on one ocl device expected, got ",
              codes.scalar_type(), " ", codes.sizes(), " on ", codes.device(), " and ", scales.scalar_type(), " on ",
              scales.device());
  const int64_t groups = groups_of(codes.size(-1));
  const bool fits = tall ? codes.dim() == 2 && scales.dim() == 2 && scales.size(0) == groups_of(codes.size(0)) &&
                               scales.size(1) == groups
                         : scales.sizes().equals(with_last(codes.sizes(), groups));
  TORCH_CHECK(fits, "ocl ", op, ": ", what, ": one scale for every 128 ", tall ? "x 128 codes" : "codes of a row",
              " expected, got codes ", codes.sizes(), " and scales ", scales.sizes());
}

static at::Tensor dequantize_8bit(const at::Tensor& codes, const at::Tensor& scales, at::ScalarType dtype) {
  // scales for blocks of rows: as many as there are blocks, and not rows
  const bool tall = codes.dim() == 2 && scales.dim() == 2 && scales.size(0) != codes.size(0);
  codes_check("dequantize_8bit", "codes", codes, scales, tall, codes);
  TORCH_CHECK(float_type(dtype), "ocl dequantize_8bit: fp32, fp16 or bf16 expected, got ", dtype);
  const int dev = codes.device().index();
  DeviceScope scope(dev);
  OCL_OP("dequantize_8bit", dev);
  const at::Tensor c = rows_of(codes), s = contiguous(scales);
  at::Tensor out = empty(codes.sizes(), dtype, dev);
  OCL_CHECK(pvb2_dequantize_8bit(c.size(0), c.size(1), (const uint8_t*)c.data_ptr(), c.stride(0),
                                 (const float*)s.data_ptr(), tall ? 1 : 0, dtype_code(dtype), out.data_ptr(),
                                 stream_for(dev)));
  return out;
}

static at::Tensor dequantize_8bit_autograd(const at::Tensor& codes, const at::Tensor& scales, at::ScalarType dtype) {
  no_gradient("dequantize_8bit", differentiated({&scales}));
  at::AutoDispatchBelowADInplaceOrView below;
  return dequantize_8bit(codes, scales, dtype);
}

// [rows, K] whose rows begin on 16-byte boundaries, or a copy
static at::Tensor code_rows(const at::Tensor& codes) {
  const at::Tensor c = rows_of(codes);
  if ((reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) == 0 && (c.size(0) <= 1 || c.stride(0) % 16 == 0)) return c;
  at::Tensor out = empty_codes(c.sizes(), c.device().index());
  copy_into(out, c, false);
  return out;
}

static at::Tensor linear_8bit(const at::Tensor& codes, const at::Tensor& scales, const at::Tensor& weight_codes,
                              const at::Tensor& weight_scales, const std::optional<at::Tensor>& bias,
                              at::ScalarType dtype) {
  codes_check("linear_8bit", "input", codes, scales, false, codes);
  codes_check("linear_8bit", "weight", weight_codes, weight_scales, true, codes);
  TORCH_CHECK(float_type(dtype), "ocl linear_8bit: an output in fp32, fp16 or bf16 expected, got ", dtype);
  const int64_t N = weight_codes.size(0), K = weight_codes.size(1);
  TORCH_CHECK(codes.size(-1) == K && K > 0, "ocl linear_8bit: input [..., features] and weight [outputs, features] expected, got ",
              codes.sizes(), " and ", weight_codes.sizes());
  if (given(bias))
    TORCH_CHECK(is_ocl(*bias) && bias->device() == codes.device() && bias->scalar_type() == dtype && bias->dim() == 1 &&
                    bias->size(0) == N,
                "ocl linear_8bit: bias [outputs] of the output's type expected, got ", bias->scalar_type(), " ", bias->sizes());
  const int dev = codes.device().index();
  DeviceScope scope(dev);
  OCL_OP("linear_8bit", dev);
  at::Tensor out = empty(with_last(codes.sizes(), N), dtype, dev);
  if (out.numel() == 0) return out;
  const at::Tensor x = code_rows(codes), w = code_rows(weight_codes), xs = contiguous(scales), ws = contiguous(weight_scales);
  at::Tensor b;
  if (given(bias)) b = contiguous(*bias);
  pvb2_linear8_desc d;
  memset(&d, 0, sizeof(d));
  d.M = x.size(0);
  d.N = N;
  d.K = K;
  d.ldx = x.stride(0);
  d.ldw = w.stride(0);
  d.dtype = dtype_code(dtype);
  OCL_CHECK(pvb2_linear8(&d, (const uint8_t*)x.data_ptr(), (const float*)xs.data_ptr(), (const uint8_t*)w.data_ptr(),
                         (const float*)ws.data_ptr(), b.defined() ? b.data_ptr() : nullptr, out.data_ptr(),
                         stream_for(dev)));
  return out;
}

static at::Tensor linear_8bit_autograd(const at::Tensor& codes, const at::Tensor& scales, const at::Tensor& weight_codes,
                                       const at::Tensor& weight_scales, const std::optional<at::Tensor>& bias,
                                       at::ScalarType dtype) {
  no_gradient("linear_8bit", differentiated({&scales, &weight_scales, pointer(bias)}));
  at::AutoDispatchBelowADInplaceOrView below;
  return linear_8bit(codes, scales, weight_codes, weight_scales, bias, dtype);
}

// --------------------------------------------------- token log probabilities
struct LogProbs {
  at::Tensor logp, entropy, top_logp, top_index, stats;
  variable_list list() const { return {logp, entropy, top_logp, top_index}; }
};

static pvb2_token_logp_desc logp_desc(const at::Tensor& z, int64_t top) {
  pvb2_token_logp_desc d;
  memset(&d, 0, sizeof(d));
  d.N = z.size(0);
  d.V = z.size(1);
  d.ldz = z.stride(0);
  d.dtype = dtype_code(z.scalar_type());
  d.top = (int32_t)top;
  return d;
}

static LogProbs log_probs(const at::Tensor& logits, const at::Tensor& tokens, int64_t top, bool keep) {
  const char* op = "ocl token_log_probs: ";
  TORCH_CHECK(is_ocl(logits) && is_ocl(tokens) && logits.device() == tokens.device(), op,
              "logits and tokens on one ocl device expected, got ", logits.device(), " and ", tokens.device());
  TORCH_CHECK(float_type(logits.scalar_type()) && logits.dim() >= 1 && logits.size(-1) > 0, op,
              "fp32, fp16 or bf16 logits [..., vocabulary] expected, got ", logits.scalar_type(), " ", logits.sizes());
  TORCH_CHECK(tokens.scalar_type() == at::kLong && tokens.sizes().equals(logits.sizes().slice(0, logits.dim() - 1)), op,
              "int64 tokens shaped like the logits without their vocabulary expected, got ", tokens.scalar_type(), " ",
              tokens.sizes());
  TORCH_CHECK_VALUE(top >= 0 && top <= 32 && top <= logits.size(-1), op, "top is 0 to 32 and at most the vocabulary, got ", top);
  const int dev = logits.device().index();
  DeviceScope scope(dev);
  OCL_OP("token_log_probs", dev);
  const at::Tensor z = rows_of(logits), t = contiguous(tokens);
  at::DimVector wide(tokens.sizes().begin(), tokens.sizes().end());
  wide.push_back(top);
  LogProbs r;
  r.logp = empty(tokens.sizes(), at::kFloat, dev);
  r.entropy = empty(tokens.sizes(), at::kFloat, dev);
  r.top_logp = empty(wide, at::kFloat, dev);
  r.top_index = empty(wide, at::kLong, dev);
  if (keep) r.stats = empty({z.size(0), 3}, at::kFloat, dev);
  const pvb2_token_logp_desc d = logp_desc(z, top);
  OCL_CHECK(pvb2_token_logp_fwd(&d, z.data_ptr(), (const int64_t*)t.data_ptr(), (float*)r.logp.data_ptr(),
                                (float*)r.entropy.data_ptr(), keep ? (float*)r.stats.data_ptr() : nullptr,
                                top ? (float*)r.top_logp.data_ptr() : nullptr,
                                top ? (int64_t*)r.top_index.data_ptr() : nullptr, stream_for(dev)));
  return r;
}

struct TokenLogProbs : public torch::autograd::Function<TokenLogProbs> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& tokens, int64_t top) {
    at::AutoDispatchBelowADInplaceOrView below;
    const LogProbs r = log_probs(logits, tokens, top, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, tokens, r.stats});
    ctx->mark_non_differentiable({r.top_logp, r.top_index});
    return r.list();
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_gradient("token_log_probs");
    const at::Tensor none;
    if (!grads[0].defined() && !grads[1].defined()) return {none, none, none};
    const variable_list s = ctx->get_saved_variables();
    const int dev = s[0].device().index();
    DeviceScope scope(dev);
    OCL_OP("token_log_probs_backward", dev);
    const at::Tensor z = rows_of(s[0]), t = contiguous(s[1]);
    const pvb2_token_logp_desc d = logp_desc(z, 0);
    // one number for all rows (a sum's or a mean's gradient) is read where it is
    bool one[2] = {true, true};
    at::Tensor g[2];
    for (int i = 0; i < 2; ++i) {
      if (!grads[i].defined()) continue;
      for (int64_t k = 0; k < grads[i].dim(); ++k) one[i] = one[i] && (grads[i].size(k) == 1 || grads[i].stride(k) == 0);
      g[i] = one[i] ? grads[i] : contiguous(grads[i]);
    }
    at::Tensor dz = empty(s[0].sizes(), s[0].scalar_type(), dev);
    OCL_CHECK(pvb2_token_logp_bwd(&d, z.data_ptr(), (const int64_t*)t.data_ptr(), (const float*)s[2].data_ptr(),
                                  g[0].defined() ? (const float*)g[0].data_ptr() : nullptr, one[0] ? 1 : 0,
                                  g[1].defined() ? (const float*)g[1].data_ptr() : nullptr, one[1] ? 1 : 0, dz.data_ptr(),
                                  stream_for(dev)));
    return {dz, none, none};
  }
};

using FourTensors = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

static FourTensors token_log_probs(const at::Tensor& logits, const at::Tensor& tokens, int64_t top) {
  const LogProbs r = log_probs(logits, tokens, top, false);
  return {r.logp, r.entropy, r.top_logp, r.top_index};
}

static FourTensors token_log_probs_autograd(const at::Tensor& logits, const at::Tensor& tokens, int64_t top) {
  if (differentiated({&logits})) {
    const variable_list r = TokenLogProbs::apply(logits, tokens, top);
    return {r[0], r[1], r[2], r[3]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return token_log_probs(logits, tokens, top);
}

}  // namespace ocl

TORCH_LIBRARY_FRAGMENT(ocl, m) {
  m.def("rms_norm(Tensor input, Tensor? weight, float eps) -> Tensor");
  m.def("rms_norm_add(Tensor input, Tensor residual, Tensor? weight, float eps) -> (Tensor, Tensor)");
  m.def("rms_norm_8bit(Tensor input, Tensor? weight, Tensor? residual, float eps) -> Tensor[]");
  m.def("quantize_8bit(Tensor input, bool tall) -> (Tensor, Tensor)");
  m.def("dequantize_8bit(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
  m.def("linear_8bit(Tensor codes, Tensor scales, Tensor weight_codes, Tensor weight_scales, Tensor? bias, "
        "ScalarType dtype) -> Tensor");
  m.def("token_log_probs(Tensor logits, Tensor tokens, int top) -> (Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(ocl, PrivateUse1, m) {
  m.impl("rms_norm", &ocl::rms_norm);
  m.impl("rms_norm_add", &ocl::rms_norm_add);
  m.impl("rms_norm_8bit", &ocl::rms_norm_8bit);
  m.impl("quantize_8bit", &ocl::quantize_8bit);
  m.impl("dequantize_8bit", &ocl::dequantize_8bit);
  m.impl("linear_8bit", &ocl::linear_8bit);
  m.impl("token_log_probs", &ocl::token_log_probs);
}

TORCH_LIBRARY_IMPL(ocl, AutogradPrivateUse1, m) {
  m.impl("rms_norm", &ocl::rms_norm_autograd);
  m.impl("rms_norm_add", &ocl::rms_norm_add_autograd);
  m.impl("rms_norm_8bit", &ocl::rms_norm_8bit_autograd);
  m.impl("quantize_8bit", &ocl::quantize_8bit_autograd);
  m.impl("dequantize_8bit", &ocl::dequantize_8bit_autograd);
  m.impl("linear_8bit", &ocl::linear_8bit_autograd);
  m.impl("token_log_probs", &ocl::token_log_probs_autograd);
}
