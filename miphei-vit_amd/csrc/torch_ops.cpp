// torch.ops.mvit.*: the transformer-block operators (RMS norm, row quantisation, rotary positions, linear with activation and residual)
// on the C-ABI of miphei_hip.h -- argument checks, output allocation, autograd formulas and the choice of library, in C++.
//
// Why C++ here: the calls on one token take the GPU 4 to 8 us, and the same host work in Python (checks, allocations, ctypes) took
// 18 to 22 us a call and 190 us for a forward and backward, 60 of them Python run by autograd's device thread.
//
// Conventions: the work goes to the tensors' device, on its current stream; 16-bit operands are bf16 (libmiphei_hip.so) or fp16
// (libmiphei_hip_f16.so, the same sources), never a mixture; scratch memory comes from torch's allocator on the same stream, so that a
// captured graph owns its own.  Wrong arguments raise ValueError in the GPU and in the meta (shape) implementation alike.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "../../include/miphei_hip.h"

namespace {

using at::ScalarType;
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ---------------------------------------------------------------- the two libraries
struct Lib {
#define MVIT_FN(name) decltype(&::name) name = nullptr
  MVIT_FN(mvit_rmsnorm_fwd);
  MVIT_FN(mvit_rmsnorm_fp8_fwd);
  MVIT_FN(mvit_quantize_rows_fp8);
  MVIT_FN(mvit_rmsnorm_bwd_scratch_bytes);
  MVIT_FN(mvit_rmsnorm_bwd);
  MVIT_FN(mvit_rotary);
  MVIT_FN(mvit_linear_act);
  MVIT_FN(mvit_linear_fp8);
  MVIT_FN(mvit_act_bwd_scratch_bytes);
  MVIT_FN(mvit_act_bwd);
  MVIT_FN(mvit_linear_scratch_bytes);
  MVIT_FN(mvit_linear_grad_scratch_bytes);
  MVIT_FN(mvit_linear_grad);
#undef MVIT_FN
};
std::array<Lib, 2> libs;   // [0] bf16, [1] fp16: filled by mvit_torch_bind before the first call
bool bound = false;

const Lib& lib(bool f16) {
  TORCH_CHECK(bound, "libmiphei_hip.so is not bound: import miphei_vit_amd.torch_ops");
  return libs[f16];
}

void ok(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " failed with code ", rc); }

// ---------------------------------------------------------------- checks
#define REQUIRE(cond, op, ...) TORCH_CHECK_VALUE(cond, "mvit::", op, ": ", ##__VA_ARGS__)

bool is_half(ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }

// The one 16-bit type among the operands; a mixture is refused, and so is any type but bf16, fp16 and f32
struct HalfType {
  const char* op;
  std::optional<ScalarType> t;
  void add(ScalarType d) {
    if (d == at::kFloat) return;
    REQUIRE(is_half(d), op, "operands are bfloat16, float16 or float32, got ", d);
    REQUIRE(!t || *t == d, op, "bfloat16 and float16 operands in one call");
    t = d;
  }
  void add(const OptTensor& x) {
    if (x) add(x->scalar_type());
  }
  bool f16() const { return t && *t == at::kHalf; }
};

void same_place(const char* op, const Tensor& x, const OptTensor& y) {
  REQUIRE(!y || y->device() == x.device(), op, "tensors on ", x.device(), " and ", y->device());
}

// A derivative is never dropped: what carries a forward-mode tangent (torch.no_grad() does not stop those) is refused, and so is, by operators
// without a gradient, what requires one.  Asked in the autograd kernels, where functional transforms have their tensors still wrapped.
bool has_tangent(const OptTensor& t) { return t && t->defined() && t->_fw_grad(/*level=*/0).defined(); }
void no_tangent(const char* op, std::initializer_list<OptTensor> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const auto& t : ts) TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(t), "mvit::", op, " has no forward-mode derivative");
}
bool wants_grad(std::initializer_list<OptTensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const auto& t : ts)
    if (t && t->requires_grad()) return true;
  return false;
}
void no_grad(const char* op, std::initializer_list<OptTensor> ts) {
  no_tangent(op, ts);
  TORCH_CHECK(!wants_grad(ts), "mvit::", op, " has no gradient: call it under torch.no_grad() or on detached tensors");
}

constexpr int64_t ROWS_MAX = 1 << 30;

// ---------------------------------------------------------------- tensors as the kernels take them
// [rows, last] view whose rows are dense, any row stride of at least their length; a copy only where there is none
Tensor rows(const Tensor& t) {
  const int64_t d = t.size(-1);
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, d});
  if ((d > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < d)) r = r.contiguous();
  return r;
}
int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }   // (the stride of a single row says nothing)

// the same for the matrix kernels: rows start on 16 bytes and are at most 2^23 bytes apart
Tensor operand(const Tensor& t) {
  Tensor r = rows(t);
  const int64_t es = r.element_size(), step = r.size(0) > 1 ? r.stride(0) * es : 0;
  if (reinterpret_cast<uintptr_t>(r.const_data_ptr()) % 16 || step % 16 || step > (1 << 23)) r = r.clone(at::MemoryFormat::Contiguous);
  return r;
}

const void* ptr(const OptTensor& t) { return t ? t->const_data_ptr() : nullptr; }
int f32(const OptTensor& t) { return t && t->scalar_type() == at::kFloat; }
void* stream(const Tensor& x) { return c10::hip::getCurrentHIPStream(x.device().index()).stream(); }

// Checks and output shapes take sizes as SymInt (plain integers but while a graph is traced with sizes that vary): a model compiled once runs
// at other batch sizes
using Sizes = std::vector<c10::SymInt>;
Sizes with_last(const Tensor& x, const c10::SymInt& n) {
  Sizes s = x.sym_sizes().vec();
  s.back() = n;
  return s;
}
// (straight to the allocator on the GPU: through the dispatcher each output costs a call on one token 0.2 us more of 5 to 6)
Tensor empty(c10::SymIntArrayRef sizes, const Tensor& like, ScalarType t) {
  if (like.device().is_cuda()) return at::detail::empty_cuda(C10_AS_INTARRAYREF_SLOW(sizes), like.options().dtype(t));
  return at::empty_symint(sizes, like.options().dtype(t));
}
Tensor scratch(const Tensor& x, int64_t bytes) { return empty({bytes}, x, at::kByte); }
Tensor none(const Tensor& x, ScalarType t) { return empty({0}, x, t); }

// ================================================================ RMS norm
void rows_check(const char* op, const Tensor& x) {
  REQUIRE(x.dim() >= 1 && x.sym_size(-1) >= 1 && x.sym_size(-1) <= 16384, op, "the last dimension must be 1 .. 16384");
  REQUIRE(x.sym_numel() <= x.sym_size(-1) * ROWS_MAX, op, "more than 2^30 rows");
}
HalfType norm_check(const char* op, const Tensor& x, const OptTensor& residual, const Tensor& weight, std::optional<ScalarType> out) {
  rows_check(op, x);
  REQUIRE(weight.dim() == 1 && weight.sym_size(0) == x.sym_size(-1), op, "weight ", weight.sym_sizes(), " does not match input ", x.sym_sizes());
  REQUIRE(!residual || residual->sym_sizes() == x.sym_sizes(), op, "residual ", residual->sym_sizes(), " and input ", x.sym_sizes(),
          " differ (it is not broadcast)");
  same_place(op, x, residual);
  same_place(op, x, weight);
  HalfType h{op};
  h.add(x), h.add(residual), h.add(weight);
  if (out) h.add(*out);
  const bool xf = x.scalar_type() == at::kFloat;
  REQUIRE(!xf || !residual || f32(residual), op, "a float32 input needs a float32 residual");
  REQUIRE(!out || *out == x.scalar_type() || xf, op, "out_dtype ", *out, " of a ", x.scalar_type(), " input");
  return h;
}

struct NormOut {
  Tensor y, h, row;   // row: one f32 a row (rstd, scale)
};
NormOut norm_out(const Tensor& x, const OptTensor& residual, ScalarType y) {
  return {empty(x.sym_sizes(), x, y), residual ? empty(x.sym_sizes(), x, residual->scalar_type()) : none(x, x.scalar_type()),
          empty(x.sym_sizes().slice(0, x.dim() - 1), x, at::kFloat)};
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_forward(const Tensor& x, const OptTensor& residual, const Tensor& weight, double eps,
                                                    std::optional<ScalarType> out_dtype) {
  const HalfType h = norm_check("rms_norm", x, residual, weight, out_dtype);
  c10::DeviceGuard guard(x.device());
  NormOut o = norm_out(x, residual, out_dtype.value_or(x.scalar_type()));
  const Tensor x2 = rows(x), w = weight.contiguous();
  const OptTensor r2 = residual ? OptTensor(rows(*residual)) : std::nullopt;
  ok(lib(h.f16()).mvit_rmsnorm_fwd(x2.const_data_ptr(), f32(x2), ld(x2), ptr(r2), f32(r2), r2 ? ld(*r2) : 0, w.const_data_ptr(), f32(w),
                                   residual ? o.h.mutable_data_ptr() : nullptr, o.y.mutable_data_ptr(), f32(o.y), o.row.mutable_data_ptr<float>(),
                                   (int)x2.size(0), (int)x2.size(1), (float)eps, stream(x)),
     "mvit_rmsnorm_fwd");
  return {o.y, o.h, o.row};
}
std::tuple<Tensor, Tensor, Tensor> rms_norm_forward_meta(const Tensor& x, const OptTensor& residual, const Tensor& weight, double,
                                                         std::optional<ScalarType> out_dtype) {
  norm_check("rms_norm", x, residual, weight, out_dtype);
  NormOut o = norm_out(x, residual, out_dtype.value_or(x.scalar_type()));
  return {o.y, o.h, o.row};
}

// (dx, dresidual, dweight), empty where not wanted; where x and the stream have one type the two gradients are one tensor, dx
struct NormBwd {
  Tensor dx, dres, dw;
  bool x, res;
};
NormBwd norm_bwd_out(const Tensor& h, const Tensor& weight, ScalarType x_dtype, bool need_x, bool need_residual, bool need_weight) {
  const bool one = x_dtype == h.scalar_type(), x = need_x || (one && need_residual), res = need_residual && !one;
  return {x ? empty(h.sym_sizes(), h, x_dtype) : none(h, x_dtype), res ? empty(h.sym_sizes(), h, h.scalar_type()) : none(h, h.scalar_type()),
          need_weight ? empty(weight.sym_sizes(), weight, weight.scalar_type()) : none(weight, weight.scalar_type()), x, res};
}
std::tuple<Tensor, Tensor, Tensor> rms_norm_backward(const Tensor& dy, const OptTensor& dh, const Tensor& h, const Tensor& weight, const Tensor& rstd,
                                                     ScalarType x_dtype, bool need_x, bool need_residual, bool need_weight) {
  REQUIRE(h.dim() >= 1 && h.size(-1) >= 1 && dy.sizes() == h.sizes() && (!dh || dh->sizes() == h.sizes()) && weight.numel() == h.size(-1) &&
              rstd.numel() == h.numel() / h.size(-1),
          "rms_norm_backward", "sizes ", dy.sizes(), ", ", h.sizes(), ", ", weight.sizes(), ", ", rstd.sizes());
  for (const Tensor* t : {&dy, &weight, &rstd}) same_place("rms_norm_backward", h, *t);
  same_place("rms_norm_backward", h, dh);
  c10::DeviceGuard guard(h.device());
  NormBwd o = norm_bwd_out(h, weight, x_dtype, need_x, need_residual, need_weight);
  const int64_t d = h.size(-1), m = h.numel() / d;
  // the kernel's dx has dy's type: the gradient of a 16-bit output of an f32 x is widened first (a pass of its own, some 30 us of 99 at [21056, 1536])
  const Tensor h2 = h.contiguous(), dy2 = dy.to(x_dtype).contiguous(), w = weight.contiguous();
  const OptTensor dh2 = dh ? OptTensor(dh->to(h.scalar_type()).contiguous()) : std::nullopt;
  HalfType half{"rms_norm"};
  half.add(dy2), half.add(h2), half.add(w);
  const Lib& l = lib(half.f16());
  const long long bytes = need_weight ? l.mvit_rmsnorm_bwd_scratch_bytes((int)m, (int)d) : 0;
  const Tensor s = scratch(h, bytes);
  ok(l.mvit_rmsnorm_bwd(dy2.const_data_ptr(), f32(dy2), ptr(dh2), h2.const_data_ptr(), f32(h2), w.const_data_ptr(), f32(w), rstd.const_data_ptr<float>(),
                        o.x ? o.dx.mutable_data_ptr() : nullptr, o.res ? o.dres.mutable_data_ptr() : nullptr,
                        need_weight ? o.dw.mutable_data_ptr() : nullptr, bytes ? s.mutable_data_ptr() : nullptr, bytes, (int)m, (int)d, stream(h)),
     "mvit_rmsnorm_bwd");
  return {o.dx, o.dres, o.dw};
}
std::tuple<Tensor, Tensor, Tensor> rms_norm_backward_meta(const Tensor&, const OptTensor&, const Tensor& h, const Tensor& weight, const Tensor&,
                                                          ScalarType x_dtype, bool need_x, bool need_residual, bool need_weight) {
  NormBwd o = norm_bwd_out(h, weight, x_dtype, need_x, need_residual, need_weight);
  return {o.dx, o.dres, o.dw};
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_fp8(const Tensor& x, const OptTensor& residual, const Tensor& weight, double eps) {
  const HalfType h = norm_check("rms_norm_fp8", x, residual, weight, std::nullopt);
  c10::DeviceGuard guard(x.device());
  NormOut o = norm_out(x, residual, at::kFloat8_e4m3fn);
  const Tensor x2 = rows(x), w = weight.contiguous();
  const OptTensor r2 = residual ? OptTensor(rows(*residual)) : std::nullopt;
  ok(lib(h.f16()).mvit_rmsnorm_fp8_fwd(x2.const_data_ptr(), f32(x2), ld(x2), ptr(r2), f32(r2), r2 ? ld(*r2) : 0, w.const_data_ptr(), f32(w),
                                       residual ? o.h.mutable_data_ptr() : nullptr, o.y.mutable_data_ptr(), o.row.mutable_data_ptr<float>(),
                                       (int)x2.size(0), (int)x2.size(1), (float)eps, stream(x)),
     "mvit_rmsnorm_fp8_fwd");
  return {o.y, o.row, o.h};
}
std::tuple<Tensor, Tensor, Tensor> rms_norm_fp8_meta(const Tensor& x, const OptTensor& residual, const Tensor& weight, double) {
  norm_check("rms_norm_fp8", x, residual, weight, std::nullopt);
  NormOut o = norm_out(x, residual, at::kFloat8_e4m3fn);
  return {o.y, o.row, o.h};
}

HalfType quantize_check(const Tensor& x) {
  rows_check("quantize_fp8", x);
  HalfType h{"quantize_fp8"};
  h.add(x);
  return h;
}
std::tuple<Tensor, Tensor> quantize_fp8(const Tensor& x) {
  const HalfType h = quantize_check(x);
  c10::DeviceGuard guard(x.device());
  NormOut o = norm_out(x, std::nullopt, at::kFloat8_e4m3fn);
  const Tensor x2 = rows(x);
  ok(lib(h.f16()).mvit_quantize_rows_fp8(x2.const_data_ptr(), f32(x2), ld(x2), o.y.mutable_data_ptr(), o.row.mutable_data_ptr<float>(),
                                         (int)x2.size(0), (int)x2.size(1), stream(x)),
     "mvit_quantize_rows_fp8");
  return {o.y, o.row};
}
std::tuple<Tensor, Tensor> quantize_fp8_meta(const Tensor& x) {
  quantize_check(x);
  NormOut o = norm_out(x, std::nullopt, at::kFloat8_e4m3fn);
  return {o.y, o.row};
}

// ================================================================ rotary positions
HalfType rotary_check(const char* op, const Tensor& x, const Tensor& positions, const Tensor& inv_freq, at::IntArrayRef sections, int64_t rotate_heads,
                      int64_t num_prefix) {
  REQUIRE(x.dim() == 4, op, "x must be [B, N, heads, head_dim], got ", x.sym_sizes());
  const c10::SymInt B = x.sym_size(0), N = x.sym_size(1), H = x.sym_size(2), Dh = x.sym_size(3);
  const int64_t axes = (int64_t)sections.size();
  REQUIRE(Dh % 2 == 0 && Dh >= 2 && Dh <= 1024 && H >= 1 && H <= 1024 && B <= 65535 && N <= ROWS_MAX, op,
          "head_dim must be even and at most 1024, heads 1 .. 1024, batch at most 65535, tokens at most 2^30");
  int64_t pairs = 0;
  bool good = axes >= 1 && axes <= 4;
  for (const int64_t s : sections) good = good && s >= 0 && Dh >= s, pairs += good ? s : 0;
  REQUIRE(good && pairs >= 1 && Dh >= 2 * pairs, op, "sections ", sections, ": 1 to 4 axes, together 1 .. head_dim / 2 pairs");
  REQUIRE(rotate_heads >= 0 && H >= rotate_heads && num_prefix >= 0 && N >= num_prefix, op, "rotate_heads ", rotate_heads, " of ", H, ", num_prefix ",
          num_prefix, " of ", N);
  const int pd = (int)positions.dim();
  REQUIRE((pd == 2 || pd == 3) && positions.sym_size(-1) == axes && positions.sym_size(-2) == N - num_prefix && (pd == 2 || positions.sym_size(0) == B), op,
          "positions must be [N - num_prefix, axes] or [B, N - num_prefix, axes] of ", x.sym_sizes(), " with ", num_prefix, " and ", axes, ", got ",
          positions.sym_sizes());
  const ScalarType pt = positions.scalar_type(), ft = inv_freq.scalar_type();
  REQUIRE(pt == at::kInt || pt == at::kLong || pt == at::kFloat, op, "positions are int32, int64 or float32, got ", pt);
  REQUIRE(inv_freq.dim() == 1 && inv_freq.sym_size(0) == pairs && (ft == at::kFloat || ft == at::kDouble), op, "inv_freq must be float32 or float64 [", pairs,
          "], got ", ft, " ", inv_freq.sym_sizes());
  same_place(op, x, positions);
  same_place(op, x, inv_freq);
  HalfType h{op};
  h.add(x);
  return h;
}

// y of rotary: x's own layout where that is a layout with dense heads (the order of overlapping windows is not), else contiguous
Tensor rotary_out(const Tensor& x) {
  if (x.is_contiguous()) return empty(x.sym_sizes(), x, x.scalar_type());
  Tensor y = at::empty_like(x);
  return y.sym_stride(3) == 1 ? y : empty(x.sym_sizes(), x, x.scalar_type());
}
// no two elements share an address: every stride reaches beyond all that the smaller ones span
bool apart(const Tensor& x) {
  if (x.unsafeGetTensorImpl()->has_symbolic_sizes_strides()) return true;   // (told when it runs)
  std::vector<std::pair<int64_t, int64_t>> dims;
  for (int64_t i = 0; i < x.dim(); ++i)
    if (x.size(i) > 1) dims.emplace_back(x.stride(i), x.size(i));
  std::sort(dims.begin(), dims.end());
  int64_t span = 0;
  for (const auto& [stride, size] : dims) {
    if (stride <= span) return false;
    span += stride * (size - 1);
  }
  return true;
}

void rotary_into(const HalfType& half, const Tensor& x, const Tensor& y, const Tensor& positions, const Tensor& inv_freq, at::IntArrayRef sections,
                 int64_t rotate_heads, int64_t num_prefix, bool interleaved, bool inverse) {
  if (x.numel() == 0) return;
  const Tensor pos = positions.contiguous(), freq = inv_freq.contiguous();
  mvit_rotary_args a = {};
  a.x = x.const_data_ptr(), a.y = y.mutable_data_ptr(), a.positions = pos.const_data_ptr(), a.inv_freq = freq.const_data_ptr();
  a.xb = x.stride(0), a.xn = x.stride(1), a.xh = x.stride(2), a.yb = y.stride(0), a.yn = y.stride(1), a.yh = y.stride(2);
  a.pos_b = pos.dim() == 3 ? pos.stride(0) : 0;
  a.B = (int)x.size(0), a.N = (int)x.size(1), a.H = (int)x.size(2), a.Dh = (int)x.size(3);
  a.rotate_heads = (int)rotate_heads, a.prefix = (int)num_prefix, a.axes = (int)sections.size();
  for (size_t i = 0; i < sections.size(); ++i) a.sections[i] = (int)sections[i];
  const ScalarType pt = pos.scalar_type();
  a.x_f32 = f32(x), a.pos_type = pt == at::kInt ? 0 : pt == at::kLong ? 1 : 2, a.freq_f64 = freq.scalar_type() == at::kDouble;
  a.interleaved = interleaved, a.inverse = inverse;
  ok(lib(half.f16()).mvit_rotary(&a, stream(x)), "mvit_rotary");
}

Tensor rotary_forward(const Tensor& x0, const Tensor& positions, const Tensor& inv_freq, at::IntArrayRef sections, int64_t rotate_heads,
                      int64_t num_prefix, bool interleaved, bool inverse) {
  const HalfType h = rotary_check("rotary", x0, positions, inv_freq, sections, rotate_heads, num_prefix);
  c10::DeviceGuard guard(x0.device());
  const Tensor x = x0.stride(3) == 1 ? x0 : x0.contiguous();
  Tensor y = rotary_out(x);
  rotary_into(h, x, y, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved, inverse);
  return y;
}
Tensor rotary_forward_meta(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, at::IntArrayRef sections, int64_t rotate_heads,
                           int64_t num_prefix, bool, bool) {
  rotary_check("rotary", x, positions, inv_freq, sections, rotate_heads, num_prefix);
  return rotary_out(x.sym_stride(3) == 1 ? x : x.contiguous());
}

void rotary_check_(const Tensor& x) {
  REQUIRE(x.sym_numel() == 0 || (x.sym_stride(3) == 1 && apart(x)), "rotary_", "x must have dense heads and no overlapping elements to be turned in place");
}
void rotary_(Tensor& x, const Tensor& positions, const Tensor& inv_freq, at::IntArrayRef sections, int64_t rotate_heads, int64_t num_prefix,
             bool interleaved) {
  const HalfType h = rotary_check("rotary_", x, positions, inv_freq, sections, rotate_heads, num_prefix);
  rotary_check_(x);
  c10::DeviceGuard guard(x.device());
  rotary_into(h, x, x, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved, false);
  if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}
void rotary_meta_(Tensor& x, const Tensor& positions, const Tensor& inv_freq, at::IntArrayRef sections, int64_t rotate_heads, int64_t num_prefix, bool) {
  rotary_check("rotary_", x, positions, inv_freq, sections, rotate_heads, num_prefix);
  rotary_check_(x);
}

// ================================================================ linear
int activation(const char* op, c10::string_view a) {
  static constexpr std::pair<const char*, int> names[] = {
      {"none", MVIT_ACT_NONE}, {"relu", MVIT_ACT_RELU}, {"silu", MVIT_ACT_SILU}, {"gelu", MVIT_ACT_GELU}, {"gelu_tanh", MVIT_ACT_GELU_TANH}};
  for (const auto& [name, code] : names)
    if (a == name) return code;
  REQUIRE(false, op, "activation '", std::string(a), "': one of none, relu, silu, gelu, gelu_tanh");
}

int linear_check(const char* op, const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, c10::string_view act,
                 int64_t multiple) {
  REQUIRE(x.dim() >= 1 && weight.dim() == 2 && weight.sym_size(1) == x.sym_size(-1) && weight.sym_size(1) % multiple == 0 && weight.sym_numel() > 0, op,
          "weight ", weight.sym_sizes(), " does not match input ", x.sym_sizes(), " (K must be a multiple of ", multiple, ")");
  const c10::SymInt K = weight.sym_size(1), N = weight.sym_size(0);
  REQUIRE(K * (int64_t)weight.element_size() <= (1 << 23) && N <= (1 << 22) && x.sym_numel() <= K * ROWS_MAX, op,
          "K is at most 2^23 bytes, N at most 2^22, the rows of x at most 2^30");
  const int code = activation(op, act);
  REQUIRE(!bias || (bias->dim() == 1 && bias->sym_size(0) == N), op, "bias ", bias->sym_sizes(), ", expected [", N, "]");
  if (residual) {
    const Sizes want = with_last(x, N);
    REQUIRE(residual->sym_sizes() == c10::SymIntArrayRef(want), op, "residual ", residual->sym_sizes(), ", expected ", c10::SymIntArrayRef(want),
            " (it is not broadcast)");
  }
  same_place(op, x, weight);
  same_place(op, x, bias);
  same_place(op, x, residual);
  return code;
}
HalfType linear_half(const char* op, const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual) {
  REQUIRE(is_half(x.scalar_type()) && weight.scalar_type() == x.scalar_type(), op, "x and weight are both bfloat16 or both float16, got ",
          x.scalar_type(), " and ", weight.scalar_type());
  HalfType h{op};
  h.add(x), h.add(bias), h.add(residual);
  return h;
}

// y = res + act(x w^T + b) of [M, K] and [N, K] operands that operand() made fit
void product(const Lib& l, const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& res, const Tensor& y, void* pre, int act,
             const float* xs, const float* ws, int64_t M, int64_t N, void* st) {
  mvit_linear_args a = {};
  a.x = x.const_data_ptr(), a.w = w.const_data_ptr(), a.bias = ptr(bias), a.res = ptr(res), a.y = y.mutable_data_ptr(), a.pre = pre;
  a.x_scale = xs, a.w_scale = ws, a.ldx = ld(x), a.ldw = ld(w), a.ldr = res ? ld(*res) : 0;
  a.M = (int)M, a.N = (int)N, a.K = (int)x.size(1), a.act = act, a.bias_f32 = f32(bias), a.y_f32 = f32(y);
  a.scratch_bytes = l.mvit_linear_scratch_bytes(a.M, a.N, x.size(1) * x.element_size());
  const Tensor s = a.scratch_bytes ? scratch(y, a.scratch_bytes) : Tensor();
  if (a.scratch_bytes) a.scratch = s.mutable_data_ptr();
  if (xs)
    ok(l.mvit_linear_fp8(&a, st), "mvit_linear_fp8");
  else
    ok(l.mvit_linear_act(&a, st), "mvit_linear_act");
}

Tensor linear_out(const Tensor& x, const Tensor& weight, const OptTensor& residual, ScalarType t) {
  return empty(with_last(x, weight.sym_size(0)), x, residual ? residual->scalar_type() : t);
}

std::tuple<Tensor, Tensor> linear_act_forward(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                                              c10::string_view act, bool save_pre) {
  const int code = linear_check("linear_act", x, weight, bias, residual, act, 8);
  const HalfType h = linear_half("linear_act", x, weight, bias, residual);
  c10::DeviceGuard guard(x.device());
  Tensor y = linear_out(x, weight, residual, x.scalar_type());
  Tensor pre = save_pre ? empty(y.sym_sizes(), x, x.scalar_type()) : none(x, x.scalar_type());
  if (y.numel())
    product(lib(h.f16()), operand(x), operand(weight), bias ? OptTensor(bias->contiguous()) : std::nullopt,
            residual ? OptTensor(rows(*residual)) : std::nullopt, y, save_pre ? pre.mutable_data_ptr() : nullptr, code, nullptr, nullptr,
            x.numel() / x.size(-1), weight.size(0), stream(x));
  return {y, pre};
}
std::tuple<Tensor, Tensor> linear_act_forward_meta(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                                                   c10::string_view act, bool save_pre) {
  linear_check("linear_act", x, weight, bias, residual, act, 8);
  linear_half("linear_act", x, weight, bias, residual);
  Tensor y = linear_out(x, weight, residual, x.scalar_type());
  return {y, save_pre ? empty(y.sym_sizes(), x, x.scalar_type()) : none(x, x.scalar_type())};
}

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
// y[M, N] = x W (x [M, K]) or x^T W (x [K, M]) with W [K, N]
void grad_product(const Lib& l, const Tensor& x, bool x_rows, const Tensor& w, const Tensor& y, int64_t M, int64_t N, int64_t K, void* st) {
  mvit_linear_args a = {};
  a.x = x.const_data_ptr(), a.w = w.const_data_ptr(), a.y = y.mutable_data_ptr(), a.ldx = ld(x), a.ldw = ld(w), a.M = (int)M, a.N = (int)N, a.K = (int)K;
  const long long bytes = l.mvit_linear_grad_scratch_bytes(a.M, a.N, a.K);
  const Tensor s = bytes ? scratch(y, bytes) : Tensor();
  ok(l.mvit_linear_grad(&a, x_rows, bytes ? s.mutable_data_ptr() : nullptr, bytes, st), "mvit_linear_grad");
}

std::tuple<Tensor, Tensor, Tensor> linear_act_backward(const Tensor& dy, const Tensor& x, const Tensor& weight, const Tensor& pre, c10::string_view act,
                                                       bool need_x, bool need_w, bool need_b, ScalarType bias_dtype) {
  const int code = linear_check("linear_act_backward", x, weight, std::nullopt, dy, act, 8);
  linear_half("linear_act_backward", x, weight, pre, dy);
  REQUIRE(code == MVIT_ACT_NONE || (pre.sizes() == dy.sizes() && pre.scalar_type() == x.scalar_type() && pre.is_contiguous()), "linear_act_backward",
          "pre ", pre.sizes(), " of ", dy.sizes());
  same_place("linear_act_backward", x, pre);
  c10::DeviceGuard guard(x.device());
  const ScalarType t = x.scalar_type();
  const int64_t N = weight.size(0), K = weight.size(1), M = x.numel() / K;
  REQUIRE(!need_w || M <= (1 << 29), "linear_act_backward", "more than 2^29 rows of x with a gradient of weight");
  Tensor dx = need_x ? empty(x.sym_sizes(), x, t) : none(x, t);
  Tensor dw = need_w ? empty({N, K}, x, t) : none(x, t);
  Tensor db = need_b ? empty({N}, x, bias_dtype) : none(x, bias_dtype);
  if (M == 0) return {dx, dw.zero_(), db.zero_()};
  const Lib& l = lib(t == at::kHalf);
  void* st = stream(x);
  Tensor dz = dy.reshape({M, N}).contiguous();
  const Tensor dy2 = dz;
  // dz is dy itself where there is nothing to multiply, to round or to pad
  const bool make = (need_x || need_w) && (code != MVIT_ACT_NONE || dy2.scalar_type() != t || N % 8);
  if (make) dz = empty({M, up8(N)}, x, t);
  if (make || need_b) {
    const Tensor s = scratch(x, need_b ? l.mvit_act_bwd_scratch_bytes((int)M, (int)N) : 0);
    ok(l.mvit_act_bwd(dy2.const_data_ptr(), f32(dy2), code == MVIT_ACT_NONE ? nullptr : pre.const_data_ptr(), code, make ? dz.mutable_data_ptr() : nullptr,
                      make ? dz.size(1) : 0, need_b ? db.mutable_data_ptr() : nullptr, f32(db), need_b ? s.mutable_data_ptr() : nullptr, (int)M, (int)N, st),
       "mvit_act_bwd");
  }
  dz = operand(dz);
  if (need_x) grad_product(l, dz, false, operand(weight), dx, M, K, N, st);
  if (need_w) grad_product(l, dz, true, operand(x), dw, N, K, M, st);
  return {dx, dw, db};
}
std::tuple<Tensor, Tensor, Tensor> linear_act_backward_meta(const Tensor&, const Tensor& x, const Tensor& weight, const Tensor&, c10::string_view,
                                                            bool need_x, bool need_w, bool need_b, ScalarType bias_dtype) {
  const ScalarType t = x.scalar_type();
  return {need_x ? empty(x.sym_sizes(), x, t) : none(x, t), need_w ? empty(weight.sym_sizes(), x, t) : none(x, t),
          need_b ? empty(weight.sym_sizes().slice(0, 1), x, bias_dtype) : none(x, bias_dtype)};
}

int linear_fp8_check(const Tensor& x, const Tensor& x_scale, const Tensor& weight, const Tensor& w_scale, const OptTensor& bias,
                     const OptTensor& residual, c10::string_view act, ScalarType out_dtype, HalfType& h) {
  const char* op = "linear_fp8";
  REQUIRE(x.scalar_type() == at::kFloat8_e4m3fn && weight.scalar_type() == at::kFloat8_e4m3fn, op, "x and weight are float8_e4m3fn, got ",
          x.scalar_type(), " and ", weight.scalar_type());
  const int code = linear_check(op, x, weight, bias, residual, act, 16);
  const c10::SymIntArrayRef rows = x.sym_sizes().slice(0, x.dim() - 1), columns = weight.sym_sizes().slice(0, 1);
  REQUIRE(x_scale.scalar_type() == at::kFloat && w_scale.scalar_type() == at::kFloat && x_scale.sym_sizes() == rows && w_scale.sym_sizes() == columns, op,
          "float32 scales ", rows, " and ", columns, ", got ", x_scale.scalar_type(), " ", x_scale.sym_sizes(), " and ", w_scale.scalar_type(), " ",
          w_scale.sym_sizes());
  same_place(op, x, x_scale);
  same_place(op, x, w_scale);
  REQUIRE(is_half(out_dtype) || out_dtype == at::kFloat, op, "out_dtype ", out_dtype);
  h.add(bias), h.add(residual);
  if (!residual) h.add(out_dtype);
  return code;
}
Tensor linear_fp8(const Tensor& x, const Tensor& x_scale, const Tensor& weight, const Tensor& w_scale, const OptTensor& bias, const OptTensor& residual,
                  c10::string_view act, ScalarType out_dtype) {
  HalfType h{"linear_fp8"};
  const int code = linear_fp8_check(x, x_scale, weight, w_scale, bias, residual, act, out_dtype, h);
  c10::DeviceGuard guard(x.device());
  Tensor y = linear_out(x, weight, residual, out_dtype);
  if (y.numel()) {
    const Tensor xs = x_scale.contiguous(), ws = w_scale.contiguous();
    product(lib(h.f16()), operand(x), operand(weight), bias ? OptTensor(bias->contiguous()) : std::nullopt,
            residual ? OptTensor(rows(*residual)) : std::nullopt, y, nullptr, code, xs.const_data_ptr<float>(), ws.const_data_ptr<float>(),
            x.numel() / x.size(-1), weight.size(0), stream(x));
  }
  return y;
}
Tensor linear_fp8_meta(const Tensor& x, const Tensor& x_scale, const Tensor& weight, const Tensor& w_scale, const OptTensor& bias,
                       const OptTensor& residual, c10::string_view act, ScalarType out_dtype) {
  HalfType h{"linear_fp8"};
  linear_fp8_check(x, x_scale, weight, w_scale, bias, residual, act, out_dtype, h);
  return linear_out(x, weight, residual, out_dtype);
}

// ================================================================ autograd
template <class Sig>
c10::TypedOperatorHandle<Sig> op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}
const auto& rms_forward_op() {
  static const auto h = op<decltype(rms_norm_forward)>("mvit::rms_norm_forward");
  return h;
}
const auto& rms_backward_op() {
  static const auto h = op<decltype(rms_norm_backward)>("mvit::rms_norm_backward");
  return h;
}
const auto& rotary_op() {
  static const auto h = op<decltype(rotary_forward)>("mvit::rotary_forward");
  return h;
}
const auto& linear_forward_op() {
  static const auto h = op<decltype(linear_act_forward)>("mvit::linear_act_forward");
  return h;
}
const auto& linear_backward_op() {
  static const auto h = op<decltype(linear_act_backward)>("mvit::linear_act_backward");
  return h;
}

OptTensor given(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& residual, const Tensor& weight, double eps,
                               std::optional<ScalarType> out_dtype) {
    at::AutoDispatchBelowAutograd below;
    auto [y, h, rstd] = rms_forward_op().call(x, residual, weight, eps, out_dtype);
    ctx->save_for_backward({residual ? h : x, weight, rstd});
    ctx->saved_data["x_dtype"] = (int64_t)x.scalar_type();
    ctx->saved_data["residual"] = residual.has_value();
    ctx->set_materialize_grads(false);
    if (residual)
      ctx->mark_non_differentiable({rstd});
    else
      ctx->mark_non_differentiable({h, rstd});
    return {y, h, rstd};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &h = saved[0], &weight = saved[1], &rstd = saved[2];
    const auto x_dtype = (ScalarType)ctx->saved_data["x_dtype"].toInt();
    const bool res = ctx->saved_data["residual"].toBool();   // (edges are counted over the tensors that were given)
    const bool need_x = ctx->needs_input_grad(0), need_res = res && ctx->needs_input_grad(1), need_w = ctx->needs_input_grad(1 + res);
    const Tensor &dy = g[0], &dh = g[1];
    Tensor dx, dres, dw;
    if (dy.defined()) {
      std::tie(dx, dres, dw) = rms_backward_op().call(dy, given(dh), h, weight, rstd, x_dtype, need_x, need_res, need_w);
      if (x_dtype == h.scalar_type()) dres = dx;
    } else if (dh.defined()) {   // y was not used: the stream's gradient alone
      dx = dh.to(x_dtype), dres = dh;
      if (need_w) dw = at::zeros_like(weight);
    }
    return {need_x ? dx : Tensor(), need_res ? dres : Tensor(), need_w ? dw : Tensor(), Tensor(), Tensor()};
  }
};
std::tuple<Tensor, Tensor, Tensor> rms_norm_forward_autograd(const Tensor& x, const OptTensor& residual, const Tensor& weight, double eps,
                                                             std::optional<ScalarType> out_dtype) {
  no_tangent("rms_norm", {x, residual, weight});
  if (wants_grad({x, residual, weight})) {
    auto o = RmsNorm::apply(x, residual, weight, eps, out_dtype);
    return {o[0], o[1], o[2]};
  }
  at::AutoDispatchBelowAutograd below;
  return rms_forward_op().call(x, residual, weight, eps, out_dtype);
}

struct Rotary : torch::autograd::Function<Rotary> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& positions, const Tensor& inv_freq, at::IntArrayRef sections,
                        int64_t rotate_heads, int64_t num_prefix, bool interleaved, bool inverse) {
    at::AutoDispatchBelowAutograd below;
    ctx->save_for_backward({positions, inv_freq});
    ctx->saved_data["sections"] = sections.vec();
    ctx->saved_data["heads"] = rotate_heads;
    ctx->saved_data["prefix"] = num_prefix;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    return rotary_op().call(x, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved, inverse);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {   // the turn back, differentiable again by itself
    const auto saved = ctx->get_saved_variables();
    const auto sections = ctx->saved_data["sections"].toIntVector();
    variable_list out(8);
    if (g[0].defined())
      out[0] = rotary_op().call(g[0], saved[0], saved[1], sections, ctx->saved_data["heads"].toInt(), ctx->saved_data["prefix"].toInt(),
                                ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["inverse"].toBool());
    return out;
  }
};
Tensor rotary_forward_autograd(const Tensor& x, const Tensor& positions, const Tensor& inv_freq, at::IntArrayRef sections, int64_t rotate_heads,
                               int64_t num_prefix, bool interleaved, bool inverse) {
  no_tangent("rotary", {x, positions, inv_freq});
  TORCH_CHECK(!wants_grad({positions, inv_freq}), "mvit::rotary has no gradient of positions and inv_freq: detach them");
  if (wants_grad({x})) return Rotary::apply(x, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved, inverse);
  at::AutoDispatchBelowAutograd below;
  return rotary_op().call(x, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved, inverse);
}

struct LinearAct : torch::autograd::Function<LinearAct> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                               std::string act, bool save_pre) {
    // (the K axis of dW = dz^T x)
    REQUIRE(!weight.requires_grad() || x.sym_numel() <= weight.sym_size(1) * (1 << 29), "linear_act", "more than 2^29 rows of x with a gradient of weight");
    at::AutoDispatchBelowAutograd below;
    const bool keep = save_pre || (act != "none" && (x.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad())));
    auto [y, pre] = linear_forward_op().call(x, weight, bias, residual, act, keep);
    ctx->save_for_backward({x, weight, pre});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias_dtype"] = (int64_t)(bias ? bias->scalar_type() : x.scalar_type());
    ctx->saved_data["bias"] = bias.has_value();
    ctx->saved_data["residual"] = residual.has_value();
    ctx->mark_non_differentiable({pre});
    ctx->set_materialize_grads(false);
    return {y, pre};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(6);
    if (!g[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const bool bias = ctx->saved_data["bias"].toBool(), res = ctx->saved_data["residual"].toBool();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = bias && ctx->needs_input_grad(2);
    if (need_x || need_w || need_b) {
      const std::string act = ctx->saved_data["act"].toStringRef();
      auto [dx, dw, db] = linear_backward_op().call(g[0], saved[0], saved[1], saved[2], act, need_x, need_w, need_b,
                                                    (ScalarType)ctx->saved_data["bias_dtype"].toInt());
      if (need_x) out[0] = dx;
      if (need_w) out[1] = dw;
      if (need_b) out[2] = db;
    }
    if (res && ctx->needs_input_grad(2 + bias)) out[3] = g[0];
    return out;
  }
};
std::tuple<Tensor, Tensor> linear_act_forward_autograd(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                                                       c10::string_view act, bool save_pre) {
  no_tangent("linear_act", {x, weight, bias, residual});
  if (wants_grad({x, weight, bias, residual})) {
    auto o = LinearAct::apply(x, weight, bias, residual, std::string(act), save_pre);
    return {o[0], o[1]};
  }
  at::AutoDispatchBelowAutograd below;
  return linear_forward_op().call(x, weight, bias, residual, act, save_pre);
}

// the backward operators are not differentiable themselves: a gradient of a gradient is refused, not silently zero
std::tuple<Tensor, Tensor, Tensor> rms_norm_backward_autograd(const Tensor& dy, const OptTensor& dh, const Tensor& h, const Tensor& weight,
                                                              const Tensor& rstd, ScalarType x_dtype, bool need_x, bool need_residual,
                                                              bool need_weight) {
  no_tangent("rms_norm_backward", {dy, dh, h, weight});
  TORCH_CHECK(!wants_grad({dy, dh, h, weight}), "mvit::rms_norm is differentiable once");
  at::AutoDispatchBelowAutograd below;
  return rms_backward_op().call(dy, dh, h, weight, rstd, x_dtype, need_x, need_residual, need_weight);
}
std::tuple<Tensor, Tensor, Tensor> linear_act_backward_autograd(const Tensor& dy, const Tensor& x, const Tensor& weight, const Tensor& pre,
                                                                c10::string_view act, bool need_x, bool need_w, bool need_b, ScalarType bias_dtype) {
  no_tangent("linear_act_backward", {dy, x, weight});
  TORCH_CHECK(!wants_grad({dy, x, weight}), "mvit::linear_act is differentiable once");
  at::AutoDispatchBelowAutograd below;
  return linear_backward_op().call(dy, x, weight, pre, act, need_x, need_w, need_b, bias_dtype);
}

// the operators without a gradient
std::tuple<Tensor, Tensor, Tensor> rms_norm_fp8_autograd(const Tensor& x, const OptTensor& residual, const Tensor& weight, double eps) {
  static const auto h = op<decltype(rms_norm_fp8)>("mvit::rms_norm_fp8");
  no_grad("rms_norm_fp8", {x, residual, weight});
  at::AutoDispatchBelowAutograd below;
  return h.call(x, residual, weight, eps);
}
std::tuple<Tensor, Tensor> quantize_fp8_autograd(const Tensor& x) {
  static const auto h = op<decltype(quantize_fp8)>("mvit::quantize_fp8");
  no_grad("quantize_fp8", {x});
  at::AutoDispatchBelowAutograd below;
  return h.call(x);
}
void rotary_autograd_(Tensor& x, const Tensor& positions, const Tensor& inv_freq, at::IntArrayRef sections, int64_t rotate_heads, int64_t num_prefix,
                      bool interleaved) {
  static const auto h = op<decltype(rotary_)>("mvit::rotary_");
  no_grad("rotary_", {x, positions, inv_freq});
  at::AutoDispatchBelowAutograd below;
  h.call(x, positions, inv_freq, sections, rotate_heads, num_prefix, interleaved);
}
Tensor linear_fp8_autograd(const Tensor& x, const Tensor& x_scale, const Tensor& weight, const Tensor& w_scale, const OptTensor& bias,
                           const OptTensor& residual, c10::string_view act, ScalarType out_dtype) {
  static const auto h = op<decltype(linear_fp8)>("mvit::linear_fp8");
  no_grad("linear_fp8", {x, x_scale, weight, w_scale, bias, residual});
  at::AutoDispatchBelowAutograd below;
  return h.call(x, x_scale, weight, w_scale, bias, residual, act, out_dtype);
}

}  // namespace

// The two libraries' entry points, from the paths that the Python host names (it has loaded torch's HIP runtime by then); 0, or 1 with
// the reason in dlerror()
extern "C" __attribute__((visibility("default"))) const char* mvit_torch_bind(const char* bf16_path, const char* f16_path) {
  const char* paths[2] = {bf16_path, f16_path};
  std::array<Lib, 2> got;
  for (int i = 0; i < 2; ++i) {
    void* h = dlopen(paths[i], RTLD_NOW | RTLD_LOCAL);
    if (!h) return dlerror();
#define MVIT_FN(name) \
  if (!(got[i].name = reinterpret_cast<decltype(&::name)>(dlsym(h, #name)))) return dlerror()
    MVIT_FN(mvit_rmsnorm_fwd);
    MVIT_FN(mvit_rmsnorm_fp8_fwd);
    MVIT_FN(mvit_quantize_rows_fp8);
    MVIT_FN(mvit_rmsnorm_bwd_scratch_bytes);
    MVIT_FN(mvit_rmsnorm_bwd);
    MVIT_FN(mvit_rotary);
    MVIT_FN(mvit_linear_act);
    MVIT_FN(mvit_linear_fp8);
    MVIT_FN(mvit_act_bwd_scratch_bytes);
    MVIT_FN(mvit_act_bwd);
    MVIT_FN(mvit_linear_scratch_bytes);
    MVIT_FN(mvit_linear_grad_scratch_bytes);
    MVIT_FN(mvit_linear_grad);
#undef MVIT_FN
  }
  libs = got;
  bound = true;
  return nullptr;
}

TORCH_LIBRARY_FRAGMENT(mvit, m) {
  m.def("rms_norm_forward(Tensor x, Tensor? residual, Tensor weight, float eps, ScalarType? out_dtype) -> (Tensor, Tensor, Tensor)");
  m.def("rms_norm_backward(Tensor dy, Tensor? dh, Tensor h, Tensor weight, Tensor rstd, ScalarType x_dtype, bool need_x, bool need_residual, "
        "bool need_weight) -> (Tensor, Tensor, Tensor)");
  m.def("rms_norm_fp8(Tensor x, Tensor? residual, Tensor weight, float eps) -> (Tensor, Tensor, Tensor)");
  m.def("quantize_fp8(Tensor x) -> (Tensor, Tensor)");
  m.def("rotary_forward(Tensor x, Tensor positions, Tensor inv_freq, int[] sections, int rotate_heads, int num_prefix, bool interleaved, "
        "bool inverse) -> Tensor");
  m.def("rotary_(Tensor(a!) x, Tensor positions, Tensor inv_freq, int[] sections, int rotate_heads, int num_prefix, bool interleaved) -> ()");
  m.def("linear_act_forward(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, str activation, bool save_pre) -> (Tensor, Tensor)");
  m.def("linear_act_backward(Tensor dy, Tensor x, Tensor weight, Tensor pre, str activation, bool need_x, bool need_w, bool need_b, "
        "ScalarType bias_dtype) -> (Tensor, Tensor, Tensor)");
  m.def("linear_fp8(Tensor x, Tensor x_scale, Tensor weight, Tensor w_scale, Tensor? bias, Tensor? residual, str activation, "
        "ScalarType out_dtype) -> Tensor");
}
TORCH_LIBRARY_IMPL(mvit, CUDA, m) {   // (torch's name for the ROCm device)
  m.impl("rms_norm_forward", rms_norm_forward);
  m.impl("rms_norm_backward", rms_norm_backward);
  m.impl("rms_norm_fp8", rms_norm_fp8);
  m.impl("quantize_fp8", quantize_fp8);
  m.impl("rotary_forward", rotary_forward);
  m.impl("rotary_", rotary_);
  m.impl("linear_act_forward", linear_act_forward);
  m.impl("linear_act_backward", linear_act_backward);
  m.impl("linear_fp8", linear_fp8);
}
TORCH_LIBRARY_IMPL(mvit, Meta, m) {
  m.impl("rms_norm_forward", rms_norm_forward_meta);
  m.impl("rms_norm_backward", rms_norm_backward_meta);
  m.impl("rms_norm_fp8", rms_norm_fp8_meta);
  m.impl("quantize_fp8", quantize_fp8_meta);
  m.impl("rotary_forward", rotary_forward_meta);
  m.impl("rotary_", rotary_meta_);
  m.impl("linear_act_forward", linear_act_forward_meta);
  m.impl("linear_act_backward", linear_act_backward_meta);
  m.impl("linear_fp8", linear_fp8_meta);
}
TORCH_LIBRARY_IMPL(mvit, Autograd, m) {
  m.impl("rms_norm_forward", rms_norm_forward_autograd);
  m.impl("rms_norm_backward", rms_norm_backward_autograd);
  m.impl("rotary_forward", rotary_forward_autograd);
  m.impl("linear_act_forward", linear_act_forward_autograd);
  m.impl("linear_act_backward", linear_act_backward_autograd);
  m.impl("rms_norm_fp8", rms_norm_fp8_autograd);
  m.impl("quantize_fp8", quantize_fp8_autograd);
  m.impl("rotary_", rotary_autograd_);
  m.impl("linear_fp8", linear_fp8_autograd);
}
