// torch_ops.cpp — the text-conditioning operators as torch operators (fp8_b200::*), with
// their gradients, over the C ABI of include/fp8ops.h.
//
// In C++ rather than in Python like the other operators' bindings: a training step calls
// these on small tensors, where an autograd function written in Python costs more host
// time (110 us for the attention's two directions, without the engine's own) than the
// kernels take.  Every operator has a CUDA kernel (the call of the C ABI), a Meta kernel
// (shapes, for torch.compile) and, where it is differentiable, an Autograd kernel that
// calls the others through the dispatcher.  Outputs and workspaces come from torch's
// caching allocator; launches go to torch's current stream.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <cmath>
#include <limits>
#include <optional>
#include <tuple>

#include "fp8ops.h"

#ifndef FP8_TORCH_MARK
#error "FP8_TORCH_MARK: the torch this is built for (fp8_b200/build.py)"
#endif
extern "C" __attribute__((used, visibility("default"))) const char fp8_torch_mark[] = FP8_TORCH_MARK;

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

const Tensor& or_undefined(const OptTensor& t) {
  static const Tensor none;
  return t.has_value() ? *t : none;
}
OptTensor or_none(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

void call_ok(int status, const char* what) {
  if (status == FP8_OK) return;
  char msg[512];
  fp8_last_error(msg, sizeof(msg));
  TORCH_CHECK(false, what, " failed (status ", status, "): ", msg);
}

fp8_stream_t current_stream() { return reinterpret_cast<fp8_stream_t>(c10::cuda::getCurrentCUDAStream().stream()); }

int dtype_code(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kBFloat16: return FP8_DTYPE_BF16;
    case at::kFloat: return FP8_DTYPE_FP32;
    case at::kHalf: return FP8_DTYPE_FP16;
    default: TORCH_CHECK(false, what, ": expected bfloat16, float16 or float32, got ", t);
  }
}

void same_device(const Tensor& first, const Tensor& t, const char* what) {
  TORCH_CHECK(!t.defined() || t.device() == first.device(), what, ": tensors on different devices: ", t.device(), " vs ",
              first.device());
}

template <typename Fn>
auto typed_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Fn>();
}

// The backward kernels have no gradient of their own.
void not_twice(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the gradient is not differentiable (create_graph=True)");
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// Nor have the operators a forward-mode derivative: a tangent would be lost, that is, taken for zero.
void no_tangent(const char* what, const Tensor& t) {
  TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), what, ": there is no forward-mode derivative");
}

// ------------------------------------------------------------------ cross attention
constexpr const char* kX = "cross attention";

void x_check(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, const Tensor& mask) {
  for (const Tensor* t : {&k, &v, &lengths, &mask}) same_device(q, *t, kX);
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes() && q.size(0) == k.size(0) && q.size(3) == k.size(3),
              kX, ": q ", q.sizes(), ", k ", k.sizes(), " and v ", v.sizes(),
              " are not [batch, tokens, heads, head_dim] of one batch and head size");
  TORCH_CHECK((q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf) && k.scalar_type() == q.scalar_type() &&
                  v.scalar_type() == q.scalar_type(),
              kX, ": q, k and v must all be bfloat16 or all float16, got ", q.scalar_type(), ", ", k.scalar_type(), ", ",
              v.scalar_type());
  const int64_t d = q.size(3);
  TORCH_CHECK(d % 8 == 0 && d >= 8 && d <= 128, kX, ": head_dim must be a multiple of 8 up to 128, got ", d);
  TORCH_CHECK(k.size(2) > 0 && q.size(2) > 0 && q.size(2) % k.size(2) == 0, kX, ": ", q.size(2),
              " heads are not a multiple of ", k.size(2), " key heads");
  TORCH_CHECK(q.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX && k.size(1) <= INT32_MAX, kX, ": too long");
  if (lengths.defined())
    TORCH_CHECK((lengths.scalar_type() == at::kInt || lengths.scalar_type() == at::kLong) && lengths.dim() == 1 &&
                    lengths.size(0) == q.size(0),
                kX, ": key_lengths must be int32 or int64 [", q.size(0), "], got ", lengths.scalar_type(), " ",
                lengths.sizes());
  if (mask.defined())
    TORCH_CHECK(mask.scalar_type() == at::kBool && mask.dim() == 2 && mask.size(0) == q.size(0) &&
                    mask.size(1) == k.size(1),
                kX, ": key_mask must be bool [", q.size(0), ", ", k.size(1), "], got ", mask.scalar_type(), " ",
                mask.sizes());
}

// t, or a copy of it in rows, if the kernels' loads cannot take its strides or address.
Tensor loadable(const Tensor& t) {
  bool fits = reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 && t.stride(3) == 1;
  for (int i = 0; i < 3; ++i) fits = fits && (t.size(i) == 1 || (t.stride(i) > 0 && t.stride(i) % 8 == 0));
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

fp8_head_strides strides_of(const Tensor& t) { return {t.stride(0), t.stride(1), t.stride(2)}; }

// Key lengths as the kernels read them: int32, clamped before a 64-bit one is narrowed.
Tensor lengths_of(const Tensor& lengths, const Tensor& k) {
  if (!lengths.defined()) return lengths;
  return (lengths.scalar_type() == at::kLong ? lengths.clamp(0, k.size(1)).to(at::kInt) : lengths).contiguous();
}
Tensor mask_of(const Tensor& mask) {
  return !mask.defined() || mask.stride(1) == 1 || mask.size(1) == 1 ? mask : mask.contiguous();
}

fp8_cross_attention_args x_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse,
                                const Tensor& lengths, const Tensor& mask, double scale) {
  fp8_cross_attention_args a{};
  a.q = q.const_data_ptr();
  a.k = k.const_data_ptr();
  a.v = v.const_data_ptr();
  a.o = o.data_ptr();
  a.lse = lse.defined() ? lse.data_ptr<float>() : nullptr;
  a.q_stride = strides_of(q);
  a.k_stride = strides_of(k);
  a.v_stride = strides_of(v);
  a.o_stride = strides_of(o);
  if (lengths.defined()) a.key_lengths = lengths.const_data_ptr<int32_t>();
  if (mask.defined()) {
    a.key_mask = static_cast<const uint8_t*>(mask.const_data_ptr());
    a.mask_stride = mask.stride(0);
  }
  a.batch = static_cast<int32_t>(q.size(0));
  a.q_len = static_cast<int32_t>(q.size(1));
  a.k_len = static_cast<int32_t>(k.size(1));
  a.heads = static_cast<int32_t>(q.size(2));
  a.kv_heads = static_cast<int32_t>(k.size(2));
  a.head_dim = static_cast<int32_t>(q.size(3));
  a.dtype = dtype_code(q.scalar_type(), kX);
  a.scale = static_cast<float>(scale);
  return a;
}

Tensor workspace(const fp8_cross_attention_args& a, int backward, const Tensor& like, size_t* bytes) {
  *bytes = fp8_cross_attention_workspace_bytes(&a, backward);
  return *bytes == 0 ? Tensor() : at::empty({static_cast<int64_t>(*bytes)}, like.options().dtype(at::kByte));
}

std::tuple<Tensor, Tensor> x_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& key_lengths,
                                 const OptTensor& key_mask, double scale, bool want_lse) {
  x_check(q, k, v, or_undefined(key_lengths), or_undefined(key_mask));
  const c10::cuda::CUDAGuard guard(q.device());
  Tensor o = at::empty(q.sizes(), q.options());
  Tensor lse;
  if (want_lse) lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
  if (o.numel() == 0 || k.size(1) == 0) {
    o.zero_();
    if (want_lse) lse.fill_(-std::numeric_limits<double>::infinity());
    return {o, lse};
  }
  const Tensor ql = loadable(q), kl = loadable(k), vl = loadable(v), lengths = lengths_of(or_undefined(key_lengths), k),
               mask = mask_of(or_undefined(key_mask));
  const fp8_cross_attention_args a = x_args(ql, kl, vl, o, lse, lengths, mask, scale);
  size_t bytes = 0;
  const Tensor ws = workspace(a, 0, q, &bytes);
  call_ok(fp8_cross_attention_fwd(&a, ws.defined() ? ws.data_ptr() : nullptr, bytes, current_stream()),
          "fp8_cross_attention_fwd");
  return {o, lse};
}

std::tuple<Tensor, Tensor> cross_attention_fwd(const Tensor& q, const Tensor& k, const Tensor& v,
                                               const OptTensor& key_lengths, const OptTensor& key_mask, double scale) {
  return x_fwd(q, k, v, key_lengths, key_mask, scale, true);
}

// -> (dq, dkv [batch][k_len][2][kv_heads][head_dim])
std::tuple<Tensor, Tensor> cross_attention_bwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o,
                                               const Tensor& lse, const Tensor& dout, const OptTensor& key_lengths,
                                               const OptTensor& key_mask, double scale) {
  x_check(q, k, v, or_undefined(key_lengths), or_undefined(key_mask));
  for (const Tensor* t : {&o, &lse, &dout}) same_device(q, *t, kX);
  TORCH_CHECK(o.sizes() == q.sizes() && dout.sizes() == q.sizes() && o.scalar_type() == q.scalar_type() &&
                  dout.scalar_type() == q.scalar_type(),
              kX, " backward: o ", o.sizes(), " ", o.scalar_type(), " and dout ", dout.sizes(), " ", dout.scalar_type(),
              " do not match q ", q.sizes(), " ", q.scalar_type());
  TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.is_contiguous() && lse.numel() == q.size(0) * q.size(2) * q.size(1),
              kX, " backward: lse must be contiguous float32 [batch, heads, q_len], got ", lse.sizes());
  const c10::cuda::CUDAGuard guard(q.device());
  Tensor dq = at::empty(q.sizes(), q.options());
  Tensor dkv = at::empty({k.size(0), k.size(1), 2, k.size(2), k.size(3)}, k.options());
  if (q.numel() == 0 || k.size(1) == 0) return {dq.zero_(), dkv.zero_()};
  const Tensor ql = loadable(q), kl = loadable(k), vl = loadable(v), ol = loadable(o), gl = loadable(dout),
               lengths = lengths_of(or_undefined(key_lengths), k), mask = mask_of(or_undefined(key_mask));
  fp8_cross_attention_args a = x_args(ql, kl, vl, ol, lse, lengths, mask, scale);
  a.dout = gl.const_data_ptr();
  a.dout_stride = strides_of(gl);
  a.dq = dq.data_ptr();
  a.dq_stride = strides_of(dq);
  char* const grads = static_cast<char*>(dkv.data_ptr());
  a.dk = grads;
  a.dv = grads + dkv.stride(2) * dkv.element_size();
  a.dk_stride = a.dv_stride = {dkv.stride(0), dkv.stride(1), dkv.stride(3)};
  size_t bytes = 0;
  const Tensor ws = workspace(a, 1, q, &bytes);
  call_ok(fp8_cross_attention_bwd(&a, ws.defined() ? ws.data_ptr() : nullptr, bytes, current_stream()),
          "fp8_cross_attention_bwd");
  return {dq, dkv};
}

std::tuple<Tensor, Tensor> cross_attention_fwd_meta(const Tensor& q, const Tensor& k, const Tensor&, const OptTensor&,
                                                    const OptTensor&, double) {
  return {at::empty_symint(q.sym_sizes(), q.options()),
          at::empty_symint({q.sym_size(0), q.sym_size(2), q.sym_size(1)}, q.options().dtype(at::kFloat))};
}
std::tuple<Tensor, Tensor> cross_attention_bwd_meta(const Tensor& q, const Tensor& k, const Tensor&, const Tensor&,
                                                    const Tensor&, const Tensor&, const OptTensor&, const OptTensor&,
                                                    double) {
  return {at::empty_symint(q.sym_sizes(), q.options()),
          at::empty_symint({k.sym_size(0), k.sym_size(1), 2, k.sym_size(2), k.sym_size(3)}, k.options())};
}

// Keys and values given apart, or packed [batch][k_len][2][kv_heads][head_dim] (v undefined).
std::tuple<Tensor, Tensor> unpack_kv(const Tensor& k, const Tensor& v) {
  if (v.defined()) return {k, v};
  TORCH_CHECK(k.dim() == 5 && k.size(2) == 2, kX, ": kv must be [batch, tokens, 2, kv_heads, head_dim], got ", k.sizes());
  return {k.select(2, 0), k.select(2, 1)};
}

double scale_of(const Tensor& q, std::optional<double> scale) {
  TORCH_CHECK(q.dim() == 4, kX, ": q must be [batch, tokens, heads, head_dim], got ", q.sizes());
  return scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(3)));
}

Tensor cross_attention_no_grad(const Tensor& q, const Tensor& k, const OptTensor& v, const OptTensor& key_lengths,
                               const OptTensor& key_mask, std::optional<double> scale) {
  const auto [kk, vv] = unpack_kv(k, or_undefined(v));
  return std::get<0>(x_fwd(q, kk, vv, key_lengths, key_mask, scale_of(q, scale), false));
}
Tensor cross_attention_meta(const Tensor& q, const Tensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                            std::optional<double>) {
  return at::empty_symint(q.sym_sizes(), q.options());
}

struct CrossAttention : torch::autograd::Function<CrossAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const OptTensor& opt_v,
                        const OptTensor& lengths, const OptTensor& mask, double scale) {
    static const auto op = typed_op<decltype(cross_attention_fwd)>("fp8_b200::cross_attention_fwd");
    const at::AutoDispatchBelowADInplaceOrView below;
    const Tensor& v = or_undefined(opt_v);
    const auto [kk, vv] = unpack_kv(k, v);
    const auto [o, lse] = op.call(q, kk, vv, lengths, mask, scale);
    ctx->save_for_backward({q, k, v, o, lse, or_undefined(lengths), or_undefined(mask)});
    ctx->saved_data["scale"] = scale;
    return o;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    not_twice(kX);
    static const auto op = typed_op<decltype(cross_attention_bwd)>("fp8_b200::cross_attention_bwd");
    const variable_list s = ctx->get_saved_variables();
    const auto [kk, vv] = unpack_kv(s[1], s[2]);
    const at::AutoDispatchBelowADInplaceOrView below;
    const auto [dq, dkv] = op.call(s[0], kk, vv, s[3], s[4], grads[0], or_none(s[5]), or_none(s[6]),
                                   ctx->saved_data["scale"].toDouble());
    if (!s[2].defined()) return {dq, dkv, Tensor(), Tensor(), Tensor(), Tensor()};
    return {dq, dkv.select(2, 0), dkv.select(2, 1), Tensor(), Tensor(), Tensor()};
  }
};

Tensor cross_attention_autograd(const Tensor& q, const Tensor& k, const OptTensor& v, const OptTensor& key_lengths,
                                const OptTensor& key_mask, std::optional<double> scale) {
  for (const Tensor* t : {&q, &k, &or_undefined(v)}) no_tangent(kX, *t);
  if (at::GradMode::is_enabled() && (wants_grad(q) || wants_grad(k) || wants_grad(or_undefined(v))))
    return CrossAttention::apply(q, k, v, key_lengths, key_mask, scale_of(q, scale));
  static const auto op = typed_op<decltype(cross_attention_no_grad)>("fp8_b200::cross_attention");
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(q, k, v, key_lengths, key_mask, scale);
}

// ------------------------------------------------------------------ token embedding
constexpr const char* kE = "embedding";

void ids_check(const Tensor& ids, const Tensor& other) {
  same_device(other, ids, kE);
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, kE, ": ids must be int64 or int32, got ",
              ids.scalar_type());
}
void weight_check(const Tensor& weight) {
  TORCH_CHECK(weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0 && weight.size(1) <= INT32_MAX, kE,
              ": weight must be [vocab, width], got ", weight.sizes());
}

Tensor embedding_fwd(const Tensor& ids_in, const Tensor& weight_in, double scale, at::ScalarType dtype) {
  ids_check(ids_in, weight_in);
  weight_check(weight_in);
  const int wcode = dtype_code(weight_in.scalar_type(), kE), ocode = dtype_code(dtype, kE);
  const c10::cuda::CUDAGuard guard(weight_in.device());
  const Tensor ids = ids_in.contiguous(),
               weight = weight_in.stride(1) == 1 || weight_in.size(1) == 1 ? weight_in : weight_in.contiguous();
  auto sizes = ids.sizes().vec();
  sizes.push_back(weight.size(1));
  Tensor out = at::empty(sizes, weight.options().dtype(dtype));
  call_ok(fp8_embedding_fwd(ids.const_data_ptr(), ids.scalar_type() == at::kLong, ids.numel(), weight.const_data_ptr(),
                            wcode, weight.size(0), static_cast<int>(weight.size(1)), weight.stride(0),
                            static_cast<float>(scale), out.data_ptr(), ocode, current_stream()),
          "fp8_embedding_fwd");
  return out;
}

Tensor embedding_bwd(const Tensor& ids_in, const Tensor& dout_in, int64_t vocab, double scale, int64_t padding_idx,
                     at::ScalarType dtype) {
  ids_check(ids_in, dout_in);
  TORCH_CHECK(dout_in.dim() == ids_in.dim() + 1 && dout_in.sizes().slice(0, ids_in.dim()) == ids_in.sizes(), kE,
              " backward: dout ", dout_in.sizes(), " does not match ids ", ids_in.sizes());
  TORCH_CHECK(vocab > 0, kE, " backward: vocab must be positive, got ", vocab);
  const int ocode = dtype_code(dout_in.scalar_type(), kE), wcode = dtype_code(dtype, kE);
  const int64_t width = dout_in.size(-1);
  TORCH_CHECK(width > 0 && width <= INT32_MAX, kE, " backward: bad width ", width);
  const c10::cuda::CUDAGuard guard(dout_in.device());
  const Tensor ids = ids_in.contiguous(), dout = dout_in.contiguous();
  Tensor dw = at::empty({vocab, width}, dout.options().dtype(dtype));
  const size_t bytes = fp8_embedding_bwd_workspace_bytes(ids.numel(), vocab, static_cast<int>(width));
  const Tensor ws = bytes == 0 ? Tensor() : at::empty({static_cast<int64_t>(bytes)}, dout.options().dtype(at::kByte));
  call_ok(fp8_embedding_bwd(ids.const_data_ptr(), ids.scalar_type() == at::kLong, ids.numel(), dout.const_data_ptr(),
                            ocode, dw.data_ptr(), wcode, vocab, static_cast<int>(width), static_cast<float>(scale),
                            padding_idx, ws.defined() ? ws.data_ptr() : nullptr, bytes, current_stream()),
          "fp8_embedding_bwd");
  return dw;
}

Tensor embedding_fwd_meta(const Tensor& ids, const Tensor& weight, double, at::ScalarType dtype) {
  auto sizes = ids.sym_sizes().vec();
  sizes.push_back(weight.sym_size(1));
  return at::empty_symint(sizes, weight.options().dtype(dtype));
}
Tensor embedding_bwd_meta(const Tensor&, const Tensor& dout, int64_t vocab, double, int64_t, at::ScalarType dtype) {
  return at::empty_symint({vocab, dout.sym_size(-1)}, dout.options().dtype(dtype));
}

struct TokenEmbedding : torch::autograd::Function<TokenEmbedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale, int64_t padding_idx,
                        at::ScalarType dtype) {
    static const auto op = typed_op<decltype(embedding_fwd)>("fp8_b200::embedding_fwd");
    const at::AutoDispatchBelowADInplaceOrView below;
    weight_check(weight);
    ctx->save_for_backward({ids});
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["pad"] = padding_idx;
    ctx->saved_data["dtype"] = static_cast<int64_t>(weight.scalar_type());
    return op.call(ids, weight, scale, dtype);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    not_twice(kE);
    static const auto op = typed_op<decltype(embedding_bwd)>("fp8_b200::embedding_bwd");
    const variable_list s = ctx->get_saved_variables();
    const at::AutoDispatchBelowADInplaceOrView below;
    auto& d = ctx->saved_data;
    return {Tensor(), op.call(s[0], grads[0], d["vocab"].toInt(), d["scale"].toDouble(), d["pad"].toInt(),
                              static_cast<at::ScalarType>(d["dtype"].toInt())),
            Tensor(), Tensor(), Tensor()};
  }
};

// padding_idx: -1 for none (the caller has resolved one that counts from the end).
Tensor embed_tokens_autograd(const Tensor& ids, const Tensor& weight, double scale, int64_t padding_idx,
                             at::ScalarType dtype) {
  no_tangent(kE, weight);
  if (at::GradMode::is_enabled() && weight.requires_grad())
    return TokenEmbedding::apply(ids, weight, scale, padding_idx, dtype);
  static const auto op = typed_op<decltype(embedding_fwd)>("fp8_b200::embedding_fwd");
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(ids, weight, scale, dtype);
}
Tensor embed_tokens_no_grad(const Tensor& ids, const Tensor& weight, double scale, int64_t, at::ScalarType dtype) {
  static const auto op = typed_op<decltype(embedding_fwd)>("fp8_b200::embedding_fwd");
  return op.call(ids, weight, scale, dtype);
}

// ------------------------------------------------------------------ dropout
constexpr const char* kD = "dropout";

Tensor dropout_apply(const Tensor& x_in, const OptTensor& residual_in, double p, const Tensor& seed) {
  const Tensor& r_in = or_undefined(residual_in);
  same_device(x_in, seed, kD);
  same_device(x_in, r_in, kD);
  const int code = dtype_code(x_in.scalar_type(), kD);
  TORCH_CHECK(p >= 0.0 && p <= 1.0, kD, ": p must be in [0, 1], got ", p);
  TORCH_CHECK(seed.scalar_type() == at::kLong && seed.numel() == 1, kD, ": seed must be one int64 value, got ",
              seed.numel(), " of ", seed.scalar_type());
  TORCH_CHECK(!r_in.defined() || (r_in.scalar_type() == x_in.scalar_type() && r_in.sizes() == x_in.sizes()), kD,
              ": residual does not match x ", x_in.sizes(), " ", x_in.scalar_type());
  const c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = x_in.contiguous(), r = r_in.defined() ? r_in.contiguous() : r_in;
  Tensor y = at::empty(x.sizes(), x.options());
  call_ok(fp8_dropout(x.const_data_ptr(), r.defined() ? r.const_data_ptr() : nullptr, y.data_ptr(), code, x.numel(), p,
                      seed.const_data_ptr<int64_t>(), current_stream()),
          "fp8_dropout");
  return y;
}
Tensor dropout_meta(const Tensor& x, const OptTensor&, double, const Tensor&) {
  return at::empty_symint(x.sym_sizes(), x.options());
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, double p, const Tensor& seed) {
    static const auto op = typed_op<decltype(dropout_apply)>("fp8_b200::dropout_add");
    const at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({seed});
    ctx->saved_data["p"] = p;
    ctx->saved_data["residual"] = or_undefined(residual).defined();
    return op.call(x, residual, p, seed);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    not_twice(kD);
    static const auto op = typed_op<decltype(dropout_apply)>("fp8_b200::dropout_add");
    const at::AutoDispatchBelowADInplaceOrView below;
    const Tensor dx = ctx->needs_input_grad(0)
                          ? op.call(grads[0], std::nullopt, ctx->saved_data["p"].toDouble(), ctx->get_saved_variables()[0])
                          : Tensor();
    return {dx, ctx->saved_data["residual"].toBool() ? grads[0] : Tensor(), Tensor(), Tensor()};
  }
};

Tensor dropout_autograd(const Tensor& x, const OptTensor& residual, double p, const Tensor& seed) {
  no_tangent(kD, x);
  no_tangent(kD, or_undefined(residual));
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(or_undefined(residual))))
    return Dropout::apply(x, residual, p, seed);
  static const auto op = typed_op<decltype(dropout_apply)>("fp8_b200::dropout_add");
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, residual, p, seed);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(fp8_b200, m) {
  m.def("cross_attention(Tensor q, Tensor k, Tensor? v, Tensor? key_lengths, Tensor? key_mask, float? scale) -> Tensor");
  m.def("cross_attention_fwd(Tensor q, Tensor k, Tensor v, Tensor? key_lengths, Tensor? key_mask, float scale) -> "
        "(Tensor, Tensor)");
  m.def("cross_attention_bwd(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor dout, Tensor? key_lengths, "
        "Tensor? key_mask, float scale) -> (Tensor, Tensor)");
  m.def("embed_tokens(Tensor ids, Tensor weight, float scale, int padding_idx, ScalarType dtype) -> Tensor");
  m.def("embedding_fwd(Tensor ids, Tensor weight, float scale, ScalarType dtype) -> Tensor");
  m.def("embedding_bwd(Tensor ids, Tensor dout, int vocab, float scale, int padding_idx, ScalarType dtype) -> Tensor");
  m.def("dropout_add(Tensor x, Tensor? residual, float p, Tensor seed) -> Tensor");
}

TORCH_LIBRARY_IMPL(fp8_b200, CUDA, m) {
  m.impl("cross_attention", cross_attention_no_grad);
  m.impl("cross_attention_fwd", cross_attention_fwd);
  m.impl("cross_attention_bwd", cross_attention_bwd);
  m.impl("embed_tokens", embed_tokens_no_grad);
  m.impl("embedding_fwd", embedding_fwd);
  m.impl("embedding_bwd", embedding_bwd);
  m.impl("dropout_add", dropout_apply);
}

TORCH_LIBRARY_IMPL(fp8_b200, Meta, m) {
  m.impl("cross_attention", cross_attention_meta);
  m.impl("cross_attention_fwd", cross_attention_fwd_meta);
  m.impl("cross_attention_bwd", cross_attention_bwd_meta);
  m.impl("embed_tokens", embed_tokens_no_grad);
  m.impl("embedding_fwd", embedding_fwd_meta);
  m.impl("embedding_bwd", embedding_bwd_meta);
  m.impl("dropout_add", dropout_meta);
}

TORCH_LIBRARY_IMPL(fp8_b200, Autograd, m) {
  m.impl("cross_attention", cross_attention_autograd);
  m.impl("embed_tokens", embed_tokens_autograd);
  m.impl("dropout_add", dropout_autograd);
}
