// The operators without a counterpart in the reference (block-scaled 8-bit products, rotary positions,
// group normalisation) as torch functions over the C ABI: argument checks, outputs and workspaces from
// torch's allocator, the tensors' device and current stream, autograd.
//
// They are called once per layer and step, where the host is what a small call waits for.  Through
// ctypes and Python autograd functions a call measured 14 to 24 us of host time and a forward and
// backward pass 130 to 150 us; here 5 to 9 us and 70 us, of which torch's engine takes 42.
//
// ValueError: operands that do not go together, wrong types, tensors that are not on an sm_100 GPU.
// RuntimeError: sizes beyond the supported ones, failed launches, a second or a forward-mode derivative
// that does not exist, calls under a tracer.
#include <torch/extension.h>

#include <ATen/TensorUtils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/AutogradState.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <atomic>
#include <optional>
#include <tuple>

#include "../../include/zimage_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kBlock = 128;
const auto kE4M3 = at::kFloat8_e4m3fn;

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// --- checks ------------------------------------------------------------------------

void status(int rc, const char* what) {
  if (rc == ZIB_OK) return;
  const bool value = rc == ZIB_ERR_INVALID_ARG || rc == ZIB_ERR_ALIGNMENT;
  TORCH_CHECK_VALUE(!value, what, ": ", zib_status_string(rc), ": ", zib_last_error());
  TORCH_CHECK(value, what, ": ", zib_status_string(rc), ": ", zib_last_error());
}

int find_dtype(at::ScalarType t) {
  return t == at::kBFloat16 ? ZIB_BF16 : t == at::kHalf ? ZIB_F16 : t == at::kFloat ? ZIB_F32 : -1;
}
int dtype_of(const Tensor& t, const char* name) {
  const int d = find_dtype(t.scalar_type());
  TORCH_CHECK_VALUE(d >= 0, name, " must be bfloat16, float16 or float32; got ", t.scalar_type());
  return d;
}

// A view whose elements read as their negatives (autograd forms some behind complex products) holds the
// others in memory: refused as an operand, resolved as an upstream gradient.
void materialised(const Tensor& t) {
  TORCH_CHECK_VALUE(!t.is_neg(), "an operand is a view that is not yet negated in memory: pass it through resolve_neg()");
}

void require_device(const Tensor& t) {
  materialised(t);
  TORCH_CHECK_VALUE(t.is_cuda(), "zimage_b200 ops run only on CUDA tensors (sm_100a); got a tensor on ", t.device(),
                    ". There is no CPU path.");
  static std::atomic<bool> checked[64];
  const int dev = t.get_device();
  if (dev < 64 && checked[dev].load(std::memory_order_relaxed)) return;
  status(zib_device_check(dev), "device check");
  if (dev < 64) checked[dev].store(true, std::memory_order_relaxed);
}
void same_device(const Tensor& t, const Tensor& o) {
  materialised(o);
  TORCH_CHECK_VALUE(o.device() == t.device(), "an operand is on ", o.device(), ", expected ", t.device());
}
void same_device(const Tensor& t, const OptTensor& o) {
  if (o) same_device(t, *o);
}

// A tracer records torch's own operations alone: of a call here the allocation of its output and not the
// kernel, so the replay would return memory that nothing has written.
void not_traced(const char* what) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                  !(Modes::any_modes_set() && Modes::get_mode(c10::impl::TorchDispatchModeKey::PROXY)),
              what, " cannot be traced (torch.jit.trace, make_fx): its kernels are not in the trace");
}

// A dual tensor need not require a gradient, so autograd does not see it: the kernel's output would
// silently have no tangent.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const OptTensor& t) { return t && has_tangent(*t); }
template <typename... T>
void no_tangent(const char* what, const T&... t) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  TORCH_CHECK(!(has_tangent(t) || ...), what, " has no forward-mode derivative");
}

bool wants_grad(const Tensor& t) { return t.requires_grad(); }
bool wants_grad(const OptTensor& t) { return t && t->requires_grad(); }
void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return t.data_ptr<float>(); }
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

// the tensor's device for the launch, and its current stream there
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(const Tensor& t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
};

// --- 8-bit operands ------------------------------------------------------------------

// e4m3 [rows, cols] whose rows start on 16-byte boundaries
Tensor e4m3_rows(int64_t rows, int64_t cols, const Tensor& like) {
  const int64_t ld = round_up(cols, 16);
  Tensor t = at::empty({rows, ld}, like.options().dtype(kE4M3));
  return ld == cols ? t : t.narrow(1, 0, cols);
}
int64_t ld_of(const Tensor& t) { return t.size(0) <= 1 ? round_up(t.size(1), 16) : t.stride(0); }

// 8-bit [R, C] with contiguous columns and 16-byte aligned rows: q itself, or a copy.  The products for few
// tokens read whole 16-byte pieces, so the last row's last one has to lie within the storage too.
Tensor aligned(const Tensor& q) {
  const int64_t R = q.size(0), C = q.size(1);
  const bool cols = q.stride(1) == 1 || C == 1;
  const bool rows = R <= 1 || (q.stride(0) % 16 == 0 && q.stride(0) >= C);
  const bool inside = C % 16 == 0 || R == 0 ||
                      q.storage_offset() + (R - 1) * q.stride(0) + round_up(C, 16) <= (int64_t)q.storage().nbytes();
  if (cols && rows && inside && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0) return q;
  Tensor t = e4m3_rows(q.size(0), q.size(1), q);
  if (cols) {
    On on(q);
    status(zib_fp8_align_rows(ptr(q), q.size(0) <= 1 ? q.size(1) : q.stride(0), ptr(t), ld_of(t), q.size(0), q.size(1),
                              on.stream),
           "8-bit operand");
  } else {
    t.copy_(q);
  }
  return t;
}

// x [..., K] itself where its rows are a fixed step apart (contiguous, or a matrix with contiguous
// columns), else a contiguous copy; and that step
Tensor rows_of(const Tensor& x, int64_t K, int64_t& ld) {
  ld = K;
  if (x.is_contiguous()) return x;
  if (x.dim() == 2 && x.stride(1) == 1 && x.stride(0) >= K) {
    ld = x.stride(0);
    return x;
  }
  return x.contiguous();
}

std::tuple<Tensor, Tensor> fp8_block_quantize(const Tensor& x) {
  not_traced("fp8_block_quantize");
  const int dt = dtype_of(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must be [..., K] with K >= 1, got ", x.sizes());
  require_device(x);
  const int64_t K = x.size(-1), M = x.numel() / K, kb = ceil_div(K, kBlock);
  int64_t ld;
  const Tensor xr = rows_of(x.detach(), K, ld);
  Tensor q = e4m3_rows(M, K, x), s = at::empty({kb, M}, x.options().dtype(at::kFloat));
  {
    On on(x);
    status(zib_fp8_quant_rows(ptr(xr), ld, dt, ptr(q), ld_of(q), fptr(s), 1, M, M, K, on.stream), "fp8_block_quantize");
  }
  s = s.t();
  if (x.dim() == 2) return {q, s};
  if (x.dim() == 1) return {q[0], s[0]};
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  return {q.unflatten(0, lead), s.unflatten(0, lead)};
}

std::tuple<Tensor, Tensor> fp8_block_quantize_weight(const Tensor& w) {
  not_traced("fp8_block_quantize_weight");
  const int dt = dtype_of(w, "w");
  TORCH_CHECK_VALUE(w.dim() == 2 && w.numel() > 0, "w must be a non-empty [N, K], got ", w.sizes());
  require_device(w);
  const int64_t N = w.size(0), K = w.size(1);
  int64_t ld;
  const Tensor wr = rows_of(w.detach(), K, ld);
  Tensor q = e4m3_rows(N, K, w);
  Tensor s = at::empty({ceil_div(N, kBlock), ceil_div(K, kBlock)}, w.options().dtype(at::kFloat));
  On on(w);
  status(zib_fp8_quant_blocks(ptr(wr), ld, dt, ptr(q), ld_of(q), fptr(s), s.stride(0), 1, N, K, on.stream),
         "fp8_block_quantize_weight");
  return {q, s};
}

Tensor fp8_block_transpose(const Tensor& w_q) {
  not_traced("fp8_block_transpose");
  TORCH_CHECK_VALUE(w_q.dim() == 2 && w_q.scalar_type() == kE4M3 && w_q.numel() > 0,
                    "w_q must be a non-empty e4m3 [N, K], got ", w_q.scalar_type(), " ", w_q.sizes());
  require_device(w_q);
  const int64_t N = w_q.size(0), K = w_q.size(1);
  int64_t ld;
  const Tensor w = rows_of(w_q, K, ld);
  Tensor t = e4m3_rows(K, N, w_q);
  On on(w_q);
  status(zib_fp8_transpose(ptr(w), ld, ptr(t), ld_of(t), N, K, on.stream), "fp8_block_transpose");
  return t;
}

// refuses a weight that does not go with K columns and outputs of type dt; returns N
int64_t check_weight(int64_t K, const Tensor& w_q, const Tensor& w_scale, const OptTensor& bias, at::ScalarType dt) {
  TORCH_CHECK_VALUE(w_q.dim() == 2 && w_q.scalar_type() == kE4M3 && w_q.size(1) == K && w_q.size(0) >= 1,
                    "w_q must be e4m3 [N, ", K, "], got ", w_q.scalar_type(), " ", w_q.sizes());
  const int64_t N = w_q.size(0), nb = ceil_div(N, kBlock), kb = ceil_div(K, kBlock);
  TORCH_CHECK_VALUE(w_scale.dim() == 2 && w_scale.size(0) == nb && w_scale.size(1) == kb &&
                        w_scale.scalar_type() == at::kFloat,
                    "w_scale must be fp32 [", nb, ", ", kb, "], got ", w_scale.scalar_type(), " ", w_scale.sizes());
  TORCH_CHECK_VALUE(!bias || (bias->dim() == 1 && bias->size(0) == N && bias->scalar_type() == dt), "bias must be ", dt,
                    " [", N, "], got ", bias->scalar_type(), " ", bias->sizes());
  return N;
}

Tensor fp8_block_matmul(const Tensor& x_q, const Tensor& x_scale, const Tensor& w_q, const Tensor& w_scale,
                        const OptTensor& bias, at::ScalarType out) {
  not_traced("fp8_block_matmul");
  TORCH_CHECK_VALUE(x_q.dim() >= 1 && x_q.scalar_type() == kE4M3 && x_q.size(-1) >= 1,
                    "x_q must be e4m3 [..., K], got ", x_q.scalar_type(), " ", x_q.sizes());
  const int64_t K = x_q.size(-1), M = x_q.numel() / K, kb = ceil_div(K, kBlock);
  const auto lead = x_q.sizes().slice(0, x_q.dim() - 1);
  TORCH_CHECK_VALUE(x_scale.dim() == x_q.dim() && x_scale.size(-1) == kb &&
                        x_scale.sizes().slice(0, x_q.dim() - 1) == lead && x_scale.scalar_type() == at::kFloat,
                    "x_scale must be fp32 ", lead, " x ", kb, ", got ", x_scale.scalar_type(), " ", x_scale.sizes());
  const int dt = find_dtype(out);
  TORCH_CHECK_VALUE(dt >= 0, "out_dtype must be bfloat16, float16 or float32, got ", out);
  const int64_t N = check_weight(K, w_q, w_scale, bias, out);
  require_device(x_q);
  same_device(x_q, x_scale);
  same_device(x_q, w_q);
  same_device(x_q, w_scale);
  same_device(x_q, bias);
  const Tensor sx = x_scale.detach().reshape({M, kb}), q = aligned(x_q.detach().reshape({M, K}));
  const Tensor w = aligned(w_q.detach());
  const OptTensor b = bias ? OptTensor(bias->detach().contiguous()) : OptTensor();
  std::vector<int64_t> shape(lead.begin(), lead.end());
  shape.push_back(N);
  Tensor y = at::empty(shape, x_q.options().dtype(out));
  On on(x_q);
  status(zib_fp8_block_gemm(ptr(q), ld_of(q), fptr(sx), sx.stride(0), sx.stride(1), ptr(w), ld_of(w), fptr(w_scale),
                            w_scale.stride(0), w_scale.stride(1), ptr(b), ptr(y), N, dt, M, N, K, on.stream),
         "fp8_block_matmul");
  return y;
}

// x [..., K] through w [N, K] (rows aligned), scales s with strides; the sums of x's columns into col_sum
Tensor linear(const Tensor& x, const Tensor& w, const Tensor& s, int64_t sn, int64_t sk, const OptTensor& bias,
              const Tensor& col_sum) {
  const int64_t N = w.size(0), K = w.size(1), M = x.numel() / K;
  int64_t ld;
  const Tensor xr = rows_of(x, K, ld);
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  Tensor y = at::empty(shape, x.options());
  const bool sum = col_sum.defined();
  const int64_t n = zib_fp8_block_linear_scratch(M, K, sum);
  Tensor scratch;
  if (n) scratch = bytes(n, x);
  On on(x);
  status(zib_fp8_block_linear(ptr(xr), ld, find_dtype(x.scalar_type()), ptr(w), ld_of(w), fptr(s), sn, sk, ptr(bias),
                              ptr(y), N, sum ? ptr(col_sum) : nullptr, n ? ptr(scratch) : nullptr, n, M, N, K,
                              on.stream),
         "fp8_block_linear");
  return y;
}

struct Linear : torch::autograd::Function<Linear> {
  // w_q is kept as it came (an aligned copy of it lives for the call alone), and only where it is needed again
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& bias, const Tensor& w_q,
                        const Tensor& s, const OptTensor& wt) {
    ctx->save_for_backward({wt ? Tensor() : w_q, s, wt ? *wt : Tensor()});
    ctx->saved_data["x"] = wants_grad(x);
    ctx->saved_data["bias"] = wants_grad(bias);
    return linear(x, aligned(w_q), s, s.stride(0), s.stride(1), bias, Tensor());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "fp8_block_linear is differentiable once: its gradient has no gradient of its own");
    no_tangent("the gradient of fp8_block_linear", grads[0]);
    const auto saved = ctx->get_saved_variables();
    const Tensor dy = grads[0].resolve_neg();
    const Tensor &w = saved[0], &s = saved[1];
    const int64_t N = dy.size(-1);
    Tensor dx, db;
    if (ctx->saved_data["bias"].toBool()) db = at::empty({N}, dy.options());
    if (ctx->saved_data["x"].toBool()) {  // the pass that quantises dy adds up its columns too
      const Tensor wt = saved[2].defined() ? aligned(saved[2]) : fp8_block_transpose(w);
      dx = linear(dy, wt, s, s.stride(1), s.stride(0), OptTensor(), db);
    } else if (db.defined()) {
      int64_t ld;
      const Tensor d = rows_of(dy, N, ld);
      Tensor ws = at::empty({64 * N}, dy.options().dtype(at::kFloat));
      On on(dy);
      status(zib_col_sum(ptr(d), ld, find_dtype(dy.scalar_type()), ptr(db), fptr(ws), ws.numel() * 4, dy.numel() / N, N,
                         on.stream),
             "fp8_block_linear");
    }
    return {dx, db, Tensor(), Tensor(), Tensor()};
  }
};

Tensor fp8_block_linear(const Tensor& x, const Tensor& w_q, const Tensor& w_scale, const OptTensor& bias_,
                        const OptTensor& w_q_t) {
  not_traced("fp8_block_linear");
  no_tangent("fp8_block_linear", x, w_scale, bias_);
  dtype_of(x, "x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "x must be [..., K] with K >= 1, got ", x.sizes());
  const int64_t K = x.size(-1), N = check_weight(K, w_q, w_scale, bias_, x.scalar_type());
  TORCH_CHECK_VALUE(!w_q_t || (w_q_t->dim() == 2 && w_q_t->size(0) == K && w_q_t->size(1) == N &&
                               w_q_t->scalar_type() == kE4M3),
                    "w_q_t must be e4m3 [", K, ", ", N, "], got ", w_q_t->scalar_type(), " ", w_q_t->sizes());
  require_device(x);
  same_device(x, w_q);
  same_device(x, w_scale);
  same_device(x, bias_);
  same_device(x, w_q_t);
  const bool grad = at::GradMode::is_enabled();
  TORCH_CHECK_VALUE(!grad || !(w_q.requires_grad() || w_scale.requires_grad()),
                    "the quantised weight of fp8_block_linear is a constant and must not require gradients");
  const OptTensor bias = bias_ && !bias_->is_contiguous() ? OptTensor(bias_->contiguous()) : bias_;
  if (grad && (wants_grad(x) || wants_grad(bias))) return Linear::apply(x, bias, w_q, w_scale, w_q_t);
  return linear(x, aligned(w_q), w_scale, w_scale.stride(0), w_scale.stride(1), bias, Tensor());
}

// --- rotary positions ------------------------------------------------------------------

// one launch over q and k (either may be undefined): fresh contiguous outputs
std::tuple<Tensor, Tensor> rotate(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin,
                                  const OptTensor& positions, bool half, bool inverse) {
  const Tensor& ref = q.defined() ? q : k;
  const int64_t B = ref.size(0), S = ref.size(1), D = ref.size(3);
  const int64_t esize = ref.element_size();
  struct Side {
    Tensor x, out;
    int64_t sb = 0, ss = 0, sh = 0, H = 0;
  } side[2];
  for (int i = 0; i < 2; ++i) {
    const Tensor& t = i ? k : q;
    if (!t.defined()) continue;
    Side& s = side[i];
    s.x = t;
    // features side by side; interleaved, a pair is one access (a copy even of a contiguous tensor that
    // starts between two pairs)
    if ((t.stride(3) != 1 && D != 1) ||
        (!half && (((t.stride(0) | t.stride(1) | t.stride(2)) & 1) ||
                   reinterpret_cast<uintptr_t>(t.data_ptr()) % (2 * esize))))
      s.x = t.clone(at::MemoryFormat::Contiguous);
    s.out = at::empty(t.sizes(), t.options());
    s.sb = s.x.stride(0), s.ss = s.x.stride(1), s.sh = s.x.stride(2), s.H = t.size(2);
  }
  const bool batched = cos.dim() == 3;
  const int64_t cs_b = batched && cos.size(0) > 1 ? cos.stride(0) : 0;
  On on(ref);
  auto p = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  status(zib_rotary(p(side[0].x), side[0].sb, side[0].ss, side[0].sh, p(side[0].out), side[0].H, p(side[1].x),
                    side[1].sb, side[1].ss, side[1].sh, p(side[1].out), side[1].H, find_dtype(ref.scalar_type()),
                    fptr(cos), fptr(sin), cs_b, cos.stride(-2), cos.size(-2), ptr(positions),
                    positions && positions->scalar_type() == at::kLong, positions ? positions->stride(0) : 0,
                    positions ? positions->stride(1) : 0, B, S, D, 2 * cos.size(-1), half, inverse, on.stream),
         "rotary_embed");
  return {side[0].out, side[1].out};
}

struct Rotary : torch::autograd::Function<Rotary> {
  // q or k may be undefined: the rotation back of one gradient alone
  static variable_list forward(AutogradContext* ctx, const OptTensor& q, const OptTensor& k, const Tensor& cos,
                               const Tensor& sin, const OptTensor& positions, bool half, bool inverse) {
    ctx->save_for_backward({cos, sin, positions ? *positions : Tensor()});
    ctx->saved_data["conf"] = (q ? 1 : 0) | (k ? 2 : 0) | (wants_grad(q) ? 4 : 0) | (wants_grad(k) ? 8 : 0) |
                              (half ? 16 : 0) | (inverse ? 32 : 0);
    ctx->set_materialize_grads(false);
    auto [oq, ok] = rotate(q ? *q : Tensor(), k ? *k : Tensor(), cos, sin, positions, half, inverse);
    variable_list out;
    if (q) out.push_back(oq);
    if (k) out.push_back(ok);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const int64_t conf = ctx->saved_data["conf"].toInt();
    size_t at = 0;
    Tensor dq, dk;
    if (conf & 1) dq = grads[at++];
    if (conf & 2) dk = grads[at++];
    if (!(conf & 4)) dq = Tensor();
    if (!(conf & 8)) dk = Tensor();
    if (dq.defined()) dq = dq.resolve_neg();
    if (dk.defined()) dk = dk.resolve_neg();
    no_tangent("the gradient of rotary_embed", dq, dk);
    Tensor gq, gk;
    if (dq.defined() || dk.defined()) {
      const auto saved = ctx->get_saved_variables();
      const OptTensor pos = saved[2].defined() ? OptTensor(saved[2]) : OptTensor();
      const bool half = conf & 16, back = !(conf & 32);
      // the transposed map of a rotation is the rotation back, itself differentiable
      if (at::GradMode::is_enabled()) {
        const auto r = Rotary::apply(dq.defined() ? OptTensor(dq) : OptTensor(), dk.defined() ? OptTensor(dk) : OptTensor(),
                                     saved[0], saved[1], pos, half, back);
        size_t n = 0;
        if (dq.defined()) gq = r[n++];
        if (dk.defined()) gk = r[n++];
      } else {
        std::tie(gq, gk) = rotate(dq, dk, saved[0], saved[1], pos, half, back);
      }
    }
    return {gq, gk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, OptTensor> rotary_embed(const Tensor& q, const OptTensor& k, const Tensor& cos_, const Tensor& sin_,
                                           const OptTensor& positions_, bool half) {
  not_traced("rotary_embed");
  no_tangent("rotary_embed", q, k, cos_, sin_);
  TORCH_CHECK_VALUE(q.dim() == 4, "q must be [B, S, H, D], got ", q.sizes());
  const int64_t B = q.size(0), S = q.size(1), D = q.size(3);
  TORCH_CHECK_VALUE(!k || (k->dim() == 4 && k->size(0) == B && k->size(1) == S && k->size(3) == D &&
                           k->scalar_type() == q.scalar_type()),
                    "k ", k->sizes(), " ", k->scalar_type(), " does not go with q ", q.sizes(), " ", q.scalar_type());
  Tensor cos = cos_, sin = sin_;
  TORCH_CHECK_VALUE(cos.sizes() == sin.sizes() && (cos.dim() == 2 || cos.dim() == 3) &&
                        cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat,
                    "cos and sin must be fp32 tables of one shape, [L, R/2] or [B, L, R/2]; got ", cos.sizes(), " ",
                    cos.scalar_type(), " and ", sin.sizes(), " ", sin.scalar_type());
  TORCH_CHECK_VALUE(cos.dim() == 2 || cos.size(0) == 1 || cos.size(0) == B, "a table of ", cos.size(0),
                    " batch entries does not go with a batch of ", B);
  TORCH_CHECK_VALUE(cos.size(-1) >= 1 && cos.size(-1) <= D / 2, "tables of ", cos.size(-1),
                    " pairs do not go with heads of ", D, " features");
  OptTensor positions;
  if (!positions_) {
    TORCH_CHECK_VALUE(cos.size(-2) >= S, "a table of ", cos.size(-2), " rows is too short for ", S, " tokens");
  } else {
    const Tensor& p = *positions_;
    TORCH_CHECK_VALUE(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong,
                      "positions must be int32 or int64, got ", p.scalar_type());
    bool fits = p.dim() <= 2;
    for (int64_t i = 1; fits && i <= p.dim(); ++i) fits = p.size(-i) == 1 || p.size(-i) == (i == 1 ? S : B);
    TORCH_CHECK_VALUE(fits, "positions ", p.sizes(), " do not broadcast to [", B, ", ", S, "]");
    TORCH_CHECK_VALUE(cos.size(-2) >= 1, "empty table");
    positions = p.dim() == 2 && p.size(0) == B && p.size(1) == S ? p : p.expand({B, S});
  }
  dtype_of(q, "q");
  TORCH_CHECK_VALUE(half || D % 2 == 0, "the interleaved layout needs an even head size, got ", D);
  TORCH_CHECK_VALUE(D <= 1024, "heads of at most 1024 features, got ", D);
  require_device(q);
  same_device(q, k);
  same_device(q, cos);
  same_device(q, sin);
  same_device(q, positions);
  const bool grad = at::GradMode::is_enabled();
  TORCH_CHECK_VALUE(!grad || !(cos.requires_grad() || sin.requires_grad()),
                    "the tables of rotary_embed are constants: cos and sin must not require gradients");
  if (cos.stride(-1) != 1 || cos.strides() != sin.strides()) {
    cos = cos.contiguous();
    sin = sin.contiguous();
  }
  if (grad && (wants_grad(q) || wants_grad(k))) {
    const auto r = Rotary::apply(OptTensor(q), k, cos, sin, positions, half, false);
    return {r[0], k ? OptTensor(r[1]) : OptTensor()};
  }
  auto [oq, ok] = rotate(q, k ? *k : Tensor(), cos, sin, positions, half, false);
  return {oq, k ? OptTensor(ok) : OptTensor()};
}

std::tuple<Tensor, Tensor> rotary_table(const OptTensor& positions, int64_t T, at::Device device, int64_t dim,
                                        double theta, int scaling, double factor, double original, double beta_fast,
                                        double beta_slow, double attention_factor) {
  not_traced("rotary_table");
  if (positions) {
    TORCH_CHECK_VALUE(positions->dim() == 1 && (positions->scalar_type() == at::kInt ||
                                                positions->scalar_type() == at::kLong),
                      "positions must be an int32 or int64 vector, got ", positions->scalar_type(), " ",
                      positions->sizes());
    require_device(*positions);
    T = positions->size(0);
    device = positions->device();
  }
  TORCH_CHECK_VALUE(device.is_cuda(), "zimage_b200 ops run only on CUDA tensors (sm_100a); got device ", device);
  const auto opt = at::TensorOptions().dtype(at::kFloat).device(device);
  Tensor cos = at::empty({T, dim / 2}, opt), sin = at::empty({T, dim / 2}, opt);
  require_device(cos);
  On on(cos);
  status(zib_rotary_table(ptr(positions), positions && positions->scalar_type() == at::kLong,
                          positions ? positions->stride(0) : 0, 0, T, dim, theta, scaling, factor, original, beta_fast,
                          beta_slow, attention_factor, fptr(cos), fptr(sin), on.stream),
         "rotary_table");
  return {cos, sin};
}

// --- group normalisation ------------------------------------------------------------------

// x [B, ..., C] with its batch and position strides; a contiguous copy where it has no single one
Tensor positions_of(const Tensor& x, int64_t P, int64_t& sb, int64_t& sp) {
  const int64_t C = x.size(-1);
  sb = P * C, sp = C;
  if (x.is_contiguous()) return x;
  const std::vector<int64_t> shape = {x.size(0), P, C};
  const auto strides = at::detail::computeStride(x.sizes(), x.strides(), shape);
  if (!strides || ((*strides)[2] != 1 && C != 1)) return x.contiguous();
  sb = (*strides)[0], sp = (*strides)[1];
  return x;
}

// mean and 1 / sqrt(var + eps), fp32 [B, G] each, at the start of `buffer`
Tensor group_norm(const Tensor& x, const OptTensor& w, const OptTensor& b, int64_t G, double eps, int64_t act,
                  int64_t P, Tensor& buffer) {
  const int64_t B = x.size(0), C = x.size(-1), stats = round_up(8 * B * G, 16);
  Tensor y = at::empty(x.sizes(), x.options());
  int64_t sb, sp;
  const Tensor xs = positions_of(x, P, sb, sp);
  On on(x);
  const int64_t n = zib_group_norm_workspace(B, P, C, G, 0);
  buffer = bytes(stats + n + 16, x);
  char* at = static_cast<char*>(ptr(buffer));
  const OptTensor& p = w ? w : b;
  status(zib_group_norm(ptr(xs), sb, sp, ptr(y), ptr(w), ptr(b), p ? find_dtype(p->scalar_type()) : ZIB_F32,
                        reinterpret_cast<float*>(at), reinterpret_cast<float*>(at) + B * G, at + stats, n, B, P, C, G,
                        find_dtype(x.scalar_type()), (float)eps, (int)act, on.stream),
         "group_norm_act");
  return y;
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w, const OptTensor& b, int64_t G,
                        double eps, int64_t act, int64_t P) {
    Tensor buffer;
    Tensor y = group_norm(x, w, b, G, eps, act, P, buffer);
    ctx->save_for_backward({x, w ? *w : Tensor(), b ? *b : Tensor(), buffer});
    ctx->saved_data["G"] = G;
    ctx->saved_data["P"] = P;
    ctx->saved_data["conf"] = act * 8 + (wants_grad(x) ? 1 : 0) + (wants_grad(w) ? 2 : 0) + (wants_grad(b) ? 4 : 0);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "group_norm_act is differentiable once: its gradient has no gradient of its own");
    no_tangent("the gradient of group_norm_act", grads[0]);
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &buffer = saved[3];
    const int64_t G = ctx->saved_data["G"].toInt(), P = ctx->saved_data["P"].toInt();
    const int64_t conf = ctx->saved_data["conf"].toInt(), B = x.size(0), C = x.size(-1);
    Tensor dx, dw, db;
    const bool empty = x.numel() == 0;
    if (conf & 1) dx = at::empty(x.sizes(), x.options());
    if (conf & 2) dw = empty ? at::zeros({C}, w.options()) : at::empty({C}, w.options());
    if (conf & 4) db = empty ? at::zeros({C}, b.options()) : at::empty({C}, b.options());
    if (!empty) {
      int64_t xsb, xsp, dsb, dsp;
      const Tensor xs = positions_of(x, P, xsb, xsp), ds = positions_of(grads[0].resolve_neg(), P, dsb, dsp);
      On on(x);
      const int64_t n = zib_group_norm_workspace(B, P, C, G, 1);
      const Tensor ws = bytes(n, x);
      auto p = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
      const Tensor& param = w.defined() ? w : b;
      const float* mean = static_cast<const float*>(ptr(buffer));
      status(zib_group_norm_backward(ptr(xs), xsb, xsp, ptr(ds), dsb, dsp, p(dx), p(w), p(b),
                                     param.defined() ? find_dtype(param.scalar_type()) : ZIB_F32, p(dw), p(db), mean,
                                     mean + B * G, ptr(ws), n, B, P, C, G, find_dtype(x.scalar_type()),
                                     (int)(conf / 8), on.stream),
             "group_norm_act");
    }
    return {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

constexpr int64_t kMaxChannels = 8192;

Tensor group_norm_act(const Tensor& x, int64_t G, const OptTensor& w_, const OptTensor& b_, double eps, int64_t act) {
  not_traced("group_norm_act");
  no_tangent("group_norm_act", x, w_, b_);
  TORCH_CHECK_VALUE(x.dim() >= 2, "x must be [B, ..., C], got ", x.sizes());
  const int64_t C = x.size(-1);
  TORCH_CHECK_VALUE(G >= 1 && C >= 1 && C % G == 0, C, " channels do not split into ", G, " groups");
  TORCH_CHECK(C <= kMaxChannels, "group_norm_act takes at most ", kMaxChannels, " channels, got ", C);
  dtype_of(x, "x");
  auto param = [&](const OptTensor& t, const char* name) {
    if (!t) return;
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == C, name, " must have shape [", C, "], got ", t->sizes());
    dtype_of(*t, name);
  };
  param(w_, "weight");
  param(b_, "bias");
  TORCH_CHECK_VALUE(!w_ || !b_ || w_->scalar_type() == b_->scalar_type(), "weight and bias must have one type, got ",
                    w_->scalar_type(), " and ", b_->scalar_type());
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative, got ", eps);
  require_device(x);
  same_device(x, w_);
  same_device(x, b_);
  int64_t P = 1;
  for (int64_t i = 1; i + 1 < x.dim(); ++i) P *= x.size(i);
  const OptTensor w = w_ && !w_->is_contiguous() ? OptTensor(w_->contiguous()) : w_;
  const OptTensor b = b_ && !b_->is_contiguous() ? OptTensor(b_->contiguous()) : b_;
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b)))
    return GroupNorm::apply(x, w, b, G, eps, act, P);
  Tensor buffer;
  return group_norm(x, w, b, G, eps, act, P, buffer);
}

}  // namespace

PYBIND11_MODULE(_ops, m) {
  m.def("fp8_block_quantize", &fp8_block_quantize);
  m.def("fp8_block_quantize_weight", &fp8_block_quantize_weight);
  m.def("fp8_block_transpose", &fp8_block_transpose);
  m.def("fp8_block_matmul", [](const Tensor& x_q, const Tensor& x_scale, const Tensor& w_q, const Tensor& w_scale,
                               const OptTensor& bias, const py::object& out) {
    return fp8_block_matmul(x_q, x_scale, w_q, w_scale, bias, torch::python::detail::py_object_to_dtype(out));
  });
  m.def("fp8_block_linear", &fp8_block_linear);
  m.def("rotary_embed", &rotary_embed);
  m.def("rotary_table", [](const OptTensor& positions, int64_t T, const py::object& device, int64_t dim, double theta,
                           int scaling, double factor, double original, double fast, double slow, double attention) {
    return rotary_table(positions, T, torch::python::detail::py_object_to_device(device), dim, theta, scaling, factor,
                        original, fast, slow, attention);
  });
  m.def("group_norm_act", &group_norm_act);
}
