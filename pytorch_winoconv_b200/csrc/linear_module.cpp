#include "linear_module.h"

#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <vector>

#include "winoconv_b200.h"

namespace {

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return WINOCONV_F32;
    case at::kHalf: return WINOCONV_F16;
    case at::kBFloat16: return WINOCONV_BF16;
    default: return -1;
  }
}
bool is16(const at::Tensor &t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
void check_abi(int st, const char *what) {
  if (st == WINOCONV_OK) return;
  char buf[1024];
  winoconv_last_error(buf, sizeof buf);
  TORCH_CHECK(false, what, " failed (", winoconv_status_string(st), "): ", buf);
}
void *stream_of() { return (void *)at::cuda::getCurrentCUDAStream().stream(); }
at::TensorOptions plain(const at::Tensor &like) { return like.options().requires_grad(false); }
int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }

// Row stride of a matrix whose rows are contiguous; 0 where they are not or overlap.
int64_t row_stride(const at::Tensor &t) {
  const int64_t cols = t.size(1);
  if (cols > 1 && t.stride(1) != 1) return 0;
  if (t.size(0) == 1) return round8(cols);      // of no meaning
  return t.stride(0) >= cols ? t.stride(0) : 0;
}
// A matrix with contiguous rows.
at::Tensor with_rows(const at::Tensor &t) { return row_stride(t) ? t : t.contiguous(); }
bool on16(const at::Tensor &t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }

at::Tensor as_rows(const at::Tensor &t, int64_t cols) { return t.dim() == 2 ? t : t.reshape({-1, cols}); }

// A matrix as the C ABI takes it.
struct Mat {
  void *p = nullptr;
  int64_t ld = 0;
};
// The scratch of a call, allocated once, and the copies that its operands need, made by one launch: matrices whose rows do not
// start on 16 bytes as the tensor cores' loads want them, and float weights, which are rounded.
class Scratch {
 public:
  Scratch(int dtype, const at::Tensor &like) : dtype_(dtype), like_(like) {}
  // The matrix itself, or a copy of it; `anywhere`: its rows need not start on 16 bytes.
  void operand(const at::Tensor &in, Mat *m, bool anywhere = false) {
    const at::Tensor t = with_rows(in);
    const bool same = code_of(t.scalar_type()) == dtype_;
    if (same && (anywhere || (row_stride(t) % 8 == 0 && on16(t)))) {
      *m = {t.data_ptr(), row_stride(t)};
    } else {
      const int64_t rows = t.size(0), cols = t.size(1);
      winoconv_rows_t &r = copies_[n_copies_];
      r = {t.data_ptr(), rows == 1 ? 0 : row_stride(t), nullptr, round8(cols), rows, (int32_t)cols, code_of(t.scalar_type()), dtype_, 0};
      at_[n_copies_] = take(rows * r.y_stride * 2);
      to_[n_copies_++] = m;
    }
    alive_.push_back(t);
  }
  // Bytes for something else; pointer() of the result once allocate() has been called.
  int64_t take(int64_t bytes) {
    const int64_t at = bytes_;
    bytes_ += (bytes + 255) / 256 * 256;
    return at;
  }
  void allocate() {
    if (bytes_ == 0) return;
    buffer_ = at::empty({bytes_}, plain(like_).dtype(at::kByte));
    for (int i = 0; i < n_copies_; ++i) {
      copies_[i].y = pointer(at_[i]);
      *to_[i] = {copies_[i].y, copies_[i].y_stride};
    }
    if (n_copies_ > 0) check_abi(winoconv_pad_rows(copies_, n_copies_, stream_of()), "winoconv_pad_rows");
  }
  void *pointer(int64_t at) const { return (uint8_t *)buffer_.data_ptr() + at; }

 private:
  int dtype_;
  const at::Tensor &like_;
  at::Tensor buffer_;
  std::vector<at::Tensor> alive_;      // of views and copies that torch made
  winoconv_rows_t copies_[2];
  Mat *to_[2];
  int64_t at_[2], bytes_ = 0;
  int n_copies_ = 0;
};

winoconv_linear_desc_t describe(int64_t rows, int64_t k, int64_t n, at::ScalarType type, int act) {
  winoconv_linear_desc_t d = {};
  TORCH_CHECK(rows <= 0x7fffffffLL && k <= 0x7fffffffLL && n <= 0x7fffffffLL, "linear: matrix too large");
  d.rows = rows;
  d.in_features = (int32_t)k;
  d.out_features = (int32_t)n;
  d.dtype = code_of(type);
  d.activation = act;
  return d;
}

// What a layer keeps for its backward pass: x and z, or one buffer with their eight bits and the scales.
struct Kept {
  at::Tensor x, z, packed;
};
// Where the parts lie in that buffer, each on 16 bytes (sizes as kept; a part that is not kept has none).
struct PackedAt {
  int64_t x = 0, x_scale = 0, z = 0, z_scale = 0, bytes = 0;
  PackedAt(int64_t rows, int64_t k, int64_t n, bool keep_x, bool keep_z) {
    auto take = [&](int64_t b) {
      const int64_t at = bytes;
      bytes += (b + 15) / 16 * 16;
      return at;
    };
    if (keep_x) {
      x = take(rows * k);
      x_scale = take(rows * ((k + 31) / 32));
    }
    if (keep_z) {
      z = take(rows * n);
      z_scale = take(rows * ((n + 31) / 32));
    }
  }
};

at::Tensor forward(const at::Tensor &x, const at::Tensor &weight, const at::Tensor &bias, const at::Tensor &residual, int act, bool pack, bool keep_x,
                   bool keep_z, Kept *kept) {
  const at::ScalarType type = x.scalar_type();
  const int64_t k = weight.size(1), n = weight.size(0);
  const at::Tensor x2 = as_rows(x, k);
  const int64_t rows = x2.size(0);
  at::Tensor y;
  if (x.dim() == 2) y = at::empty({rows, n}, plain(x));
  else {
    std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = n;
    y = at::empty(sizes, plain(x));
  }
  const bool z = kept && keep_z, z8 = z && pack;
  const PackedAt lies(rows, k, n, kept && pack && keep_x, z8);
  uint8_t *packed = nullptr;
  if (kept && pack) {
    kept->packed = at::empty({lies.bytes}, plain(x).dtype(at::kByte));
    packed = (uint8_t *)kept->packed.data_ptr();
  }
  if (kept && keep_x && !pack) kept->x = x;
  if (z && !pack) kept->z = at::empty({rows, n}, plain(x));
  if (rows == 0) return y;
  winoconv_linear_desc_t d = describe(rows, k, n, type, act);
  const bool anywhere = rows <= 2 && !z8;      // one or two rows are read as they lie
  Scratch scratch(d.dtype, x);
  Mat xm, wm;
  scratch.operand(x2, &xm, anywhere);
  scratch.operand(weight, &wm, anywhere);
  scratch.allocate();
  const at::Tensor b = bias.defined() ? bias.contiguous() : bias;
  const at::Tensor r = residual.defined() ? with_rows(as_rows(residual, n)) : residual;
  d.bias_f32 = b.defined() && b.scalar_type() == at::kFloat;
  d.x_stride = xm.ld;
  d.w_stride = wm.ld;
  if (r.defined() && rows > 1) d.residual_stride = row_stride(r);
  check_abi(winoconv_linear_forward(&d, xm.p, wm.p, b.defined() ? b.data_ptr() : nullptr, r.defined() ? r.data_ptr() : nullptr, y.data_ptr(),
                                    z && !pack ? kept->z.data_ptr() : nullptr, z8 ? packed + lies.z : nullptr, z8 ? packed + lies.z_scale : nullptr, stream_of()),
            "winoconv_linear_forward");
  if (kept && keep_x && pack) {
    const at::Tensor xr = with_rows(x2);
    check_abi(winoconv_e4m3_pack(d.dtype, xr.data_ptr(), rows > 1 ? row_stride(xr) : 0, rows, (int32_t)k, packed + lies.x, packed + lies.x_scale, stream_of()),
              "winoconv_e4m3_pack");
  }
  return y;
}

struct LinearFn : public torch::autograd::Function<LinearFn> {
  // what the node remembers beside tensors, in one list of numbers: these, then the sizes of x
  enum { X_TYPE, W_TYPE, B_TYPE, ACT, PACK, HAS_BIAS, HAS_RESIDUAL, KEEPS_X, KEEPS_Z, OUT, IN, SIZES };

  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &x, const at::Tensor &weight, const std::optional<at::Tensor> &bias,
                            const std::optional<at::Tensor> &residual, int64_t act, bool pack) {
    const bool nx = x.requires_grad(), nw = weight.requires_grad(), nb = bias && bias->requires_grad();
    Kept kept;
    at::Tensor y;
    {
      at::AutoDispatchBelowADInplaceOrView no_graph;
      y = ::forward(x, weight, bias ? *bias : at::Tensor(), residual ? *residual : at::Tensor(), (int)act, pack, nw,
                    act != WINOCONV_ACT_NONE && (nx || nw || nb), &kept);
    }
    ctx->save_for_backward({kept.x, kept.z, kept.packed, nx ? weight : at::Tensor()});
    std::vector<int64_t> layer{(int64_t)x.scalar_type(), (int64_t)weight.scalar_type(), bias ? (int64_t)bias->scalar_type() : -1, act, pack,
                               bias.has_value(), residual.has_value(), nw, act != WINOCONV_ACT_NONE && (nx || nw || nb), weight.size(0), weight.size(1)};
    layer.insert(layer.end(), x.sizes().begin(), x.sizes().end());
    ctx->saved_data["layer"] = std::move(layer);
    return y;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(6);
    if (!grads[0].defined()) return out;
    TORCH_CHECK(!at::GradMode::is_enabled(), "linear: the gradients are not differentiable again (create_graph=True)");
    auto saved = ctx->get_saved_variables();      // (hooks on them may compute anew what was not kept, with graphs of their own)
    at::AutoDispatchBelowADInplaceOrView no_graph;
    const auto layer = ctx->saved_data["layer"].toIntVector();
    for (int i = 1; i < 3; ++i)      // dense, unless a hook on saved tensors has laid them out anew
      if (saved[i].defined()) saved[i] = saved[i].contiguous();
    const auto type = (at::ScalarType)layer[X_TYPE], w_type = (at::ScalarType)layer[W_TYPE];
    const int act = (int)layer[ACT];
    const bool pack = layer[PACK] != 0, slope = act != WINOCONV_ACT_NONE;
    // numbered by the tensors among the arguments of apply
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nb = layer[HAS_BIAS] && ctx->needs_input_grad(2),
               nr = layer[HAS_RESIDUAL] && ctx->needs_input_grad(2 + layer[HAS_BIAS]);
    c10::cuda::CUDAGuard guard(grads[0].device());
    const at::Tensor gy = grads[0].resolve_neg();
    if (nr) out[3] = gy;
    if (!nx && !nw && !nb) return out;
    const int64_t n = layer[OUT], k = layer[IN];
    const at::Tensor g = with_rows(as_rows(gy, n));
    const int64_t rows = g.size(0);
    at::Tensor dx, dw, db;
    if (nw) dw = at::empty({n, k}, plain(gy).dtype(w_type));
    if (nb) db = at::empty({n}, plain(gy).dtype((at::ScalarType)layer[B_TYPE]));
    if (nx) dx = at::empty(at::IntArrayRef(layer.data() + SIZES, layer.size() - SIZES), plain(gy));
    out[0] = dx;
    out[1] = dw;
    out[2] = db;
    if (rows == 0) {
      if (nw) dw.zero_();
      if (nb) db.zero_();
      return out;
    }
    winoconv_linear_desc_t d = describe(rows, k, n, type, act);
    void *stream = stream_of();
    const PackedAt lies(rows, k, n, pack && layer[KEEPS_X], pack && layer[KEEPS_Z]);
    const uint8_t *packed = saved[2].defined() ? (const uint8_t *)saved[2].data_ptr() : nullptr;
    Scratch scratch(d.dtype, gy);
    Mat dz{g.data_ptr(), row_stride(g)}, w, x;
    // without an activation dz is gy as it lies, or a copy on 16 bytes
    const bool write = (nx || nw) && (slope || dz.ld % 8 != 0 || !on16(g));
    int64_t dz_at = 0, ws_at = 0, x_at = 0;
    uint64_t ws_bytes = 0;
    if (write) dz_at = scratch.take(rows * round8(n) * 2);
    if (nb) {
      check_abi(winoconv_linear_backward_ws(&d, &ws_bytes), "winoconv_linear_backward_ws");
      ws_at = scratch.take((int64_t)ws_bytes);
    }
    if (nx) scratch.operand(saved[3], &w);
    if (nw) {
      if (pack) x_at = scratch.take(rows * round8(k) * 2);
      else scratch.operand(as_rows(saved[0], k), &x);
    }
    scratch.allocate();
    if (write || nb) {
      if (write) dz = {scratch.pointer(dz_at), round8(n)};
      check_abi(winoconv_linear_backward_activation(&d, g.data_ptr(), rows > 1 ? row_stride(g) : 0, slope && !pack ? saved[1].data_ptr() : nullptr,
                                                    slope && pack ? packed + lies.z : nullptr, slope && pack ? packed + lies.z_scale : nullptr,
                                                    write ? dz.p : nullptr, write ? dz.ld : 0, nb ? db.data_ptr() : nullptr, nb ? code_of(db.scalar_type()) : 0,
                                                    nb ? scratch.pointer(ws_at) : nullptr, ws_bytes, stream),
                "winoconv_linear_backward_activation");
    }
    if (nx) {
      d.w_stride = w.ld;
      check_abi(winoconv_linear_backward_data(&d, dz.p, dz.ld, w.p, dx.data_ptr(), 0, stream), "winoconv_linear_backward_data");
    }
    if (nw) {
      if (pack) {
        x = {scratch.pointer(x_at), round8(k)};
        check_abi(winoconv_e4m3_unpack(d.dtype, packed + lies.x, packed + lies.x_scale, rows, (int32_t)k, x.p, x.ld, stream), "winoconv_e4m3_unpack");
      }
      d.x_stride = x.ld;
      check_abi(winoconv_linear_backward_weight(&d, dz.p, dz.ld, x.p, dw.data_ptr(), code_of(w_type), stream), "winoconv_linear_backward_weight");
    }
    return out;
  }
};

}  // namespace

void check_eager(const char *what, std::initializer_list<const at::Tensor *> tensors) {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  bool recorded = torch::jit::tracer::isTracing();
  if (Modes::any_modes_set())      // (a mode that only watches is no hindrance)
    for (Key k : {Key::FAKE, Key::PROXY, Key::FUNCTIONAL}) recorded = recorded || Modes::get_mode(k).has_value();
  TORCH_CHECK(!recorded, what, ": the call cannot be recorded by a tracer: run it eagerly, or capture it into a CUDA graph");
  for (const at::Tensor *t : tensors)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what, ": there is no forward-mode differentiation");
}

at::Tensor linear_call(const at::Tensor &x, const at::Tensor &weight, const std::optional<at::Tensor> &bias, const std::optional<at::Tensor> &residual,
                       int64_t act, bool pack) {
  check_eager("linear", {&x, &weight});
  if (bias) check_eager("linear", {&*bias});
  if (residual) check_eager("linear", {&*residual});
  if (x.is_neg() || weight.is_neg() || (bias && bias->is_neg()) || (residual && residual->is_neg())) {      // memory that holds minus the values
    auto of = [](const std::optional<at::Tensor> &t) { return t ? std::optional<at::Tensor>(t->resolve_neg()) : t; };
    return linear_call(x.resolve_neg(), weight.resolve_neg(), of(bias), of(residual), act, pack);
  }
  TORCH_CHECK(x.is_cuda(), "linear runs on CUDA devices only: there is no CPU path");
  TORCH_CHECK(is16(x), "linear: x must be float16 or bfloat16, got ", x.scalar_type());
  TORCH_CHECK(weight.dim() == 2, "linear: weight must be [out_features, in_features], got ", weight.sizes());
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) == weight.size(1), "linear: x ", x.sizes(), " does not end in the weight's ", weight.size(1), " input features");
  TORCH_CHECK(weight.size(0) > 0 && weight.size(1) > 0, "linear: weight must not be empty, got ", weight.sizes());
  TORCH_CHECK(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat, "linear: weight must be of x's type or float32, got ", weight.scalar_type());
  TORCH_CHECK(weight.device() == x.device(), "linear: weight is on ", weight.device(), ", x on ", x.device());
  if (bias) {
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == weight.size(0), "linear: bias must be [", weight.size(0), "], got ", bias->sizes());
    TORCH_CHECK(bias->scalar_type() == x.scalar_type() || bias->scalar_type() == at::kFloat, "linear: bias must be of x's type or float32, got ", bias->scalar_type());
    TORCH_CHECK(bias->device() == x.device(), "linear: bias is on ", bias->device(), ", x on ", x.device());
  }
  if (residual) {
    std::vector<int64_t> want(x.sizes().begin(), x.sizes().end());
    want.back() = weight.size(0);
    TORCH_CHECK(residual->sizes() == at::IntArrayRef(want), "linear: residual must have the output's shape ", at::IntArrayRef(want), ", got ", residual->sizes());
    TORCH_CHECK(residual->scalar_type() == x.scalar_type(), "linear: residual must be of x's type, got ", residual->scalar_type());
    TORCH_CHECK(residual->device() == x.device(), "linear: residual is on ", residual->device(), ", x on ", x.device());
  }
  TORCH_CHECK(act >= WINOCONV_ACT_NONE && act <= WINOCONV_ACT_SILU, "linear: bad activation");
  c10::cuda::CUDAGuard guard(x.device());
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad()) || (residual && residual->requires_grad())))
    return LinearFn::apply(x, weight, bias, residual, act, pack);
  at::AutoDispatchBelowADInplaceOrView no_graph;
  return forward(x, weight, bias ? *bias : at::Tensor(), residual ? *residual : at::Tensor(), (int)act, false, false, false, nullptr);
}

std::tuple<at::Tensor, at::Tensor> e4m3_pack(const at::Tensor &x_in) {
  check_eager("checkpoint.pack", {&x_in});
  TORCH_CHECK(x_in.is_cuda(), "checkpoint.pack runs on CUDA devices only: there is no CPU path");
  TORCH_CHECK(is16(x_in), "checkpoint.pack: x must be float16 or bfloat16, got ", x_in.scalar_type());
  TORCH_CHECK(x_in.dim() >= 1 && x_in.size(-1) > 0, "checkpoint.pack: x must have a last dimension that is not empty, got ", x_in.sizes());
  at::AutoDispatchBelowADInplaceOrView no_graph;
  c10::cuda::CUDAGuard guard(x_in.device());
  const int64_t cols = x_in.size(-1);
  const at::Tensor x = with_rows(as_rows(x_in.resolve_neg(), cols));
  std::vector<int64_t> sizes(x_in.sizes().begin(), x_in.sizes().end());
  at::Tensor q = at::empty(sizes, plain(x).dtype(at::kFloat8_e4m3fn));
  sizes.back() = (cols + 31) / 32;
  at::Tensor scale = at::empty(sizes, plain(x).dtype(at::kFloat8_e8m0fnu));
  TORCH_CHECK(cols <= 0x7fffffffLL, "checkpoint.pack: rows too long");
  if (x.size(0) > 0)
    check_abi(winoconv_e4m3_pack(code_of(x.scalar_type()), x.data_ptr(), x.size(0) > 1 ? row_stride(x) : 0, x.size(0), (int32_t)cols, q.data_ptr(), scale.data_ptr(), stream_of()),
              "winoconv_e4m3_pack");
  return {q, scale};
}

at::Tensor e4m3_unpack(const at::Tensor &q_in, const at::Tensor &scale_in, at::ScalarType type) {
  check_eager("checkpoint.unpack", {&q_in, &scale_in});
  TORCH_CHECK(q_in.is_cuda() && scale_in.device() == q_in.device(), "checkpoint.unpack runs on CUDA devices only, q and scale on the same one");
  TORCH_CHECK(q_in.scalar_type() == at::kFloat8_e4m3fn && scale_in.scalar_type() == at::kFloat8_e8m0fnu,
              "checkpoint.unpack: q must be float8_e4m3fn and scale float8_e8m0fnu, got ", q_in.scalar_type(), " and ", scale_in.scalar_type());
  TORCH_CHECK(type == at::kHalf || type == at::kBFloat16, "checkpoint.unpack: dtype must be float16 or bfloat16, got ", type);
  TORCH_CHECK(q_in.dim() >= 1 && q_in.size(-1) > 0, "checkpoint.unpack: q must have a last dimension that is not empty, got ", q_in.sizes());
  std::vector<int64_t> sizes(q_in.sizes().begin(), q_in.sizes().end());
  const int64_t cols = sizes.back();
  sizes.back() = (cols + 31) / 32;
  TORCH_CHECK(scale_in.sizes() == at::IntArrayRef(sizes), "checkpoint.unpack: scale must be ", at::IntArrayRef(sizes), " for q ", q_in.sizes(), ", got ", scale_in.sizes());
  TORCH_CHECK(cols <= 0x7fffffffLL, "checkpoint.unpack: rows too long");
  at::AutoDispatchBelowADInplaceOrView no_graph;
  c10::cuda::CUDAGuard guard(q_in.device());
  const at::Tensor q = q_in.contiguous(), scale = scale_in.contiguous();
  at::Tensor x = at::empty(q.sizes(), plain(q).dtype(type));
  const int64_t rows = q.numel() / cols;
  if (rows > 0)
    check_abi(winoconv_e4m3_unpack(code_of(type), q.data_ptr(), scale.data_ptr(), rows, (int32_t)cols, x.data_ptr(), 0, stream_of()), "winoconv_e4m3_unpack");
  return x;
}
