// Differentiable entry points of the training operators: argument checks, row
// views, workspaces and autograd nodes over the C entry points of the kernel
// library (b200_train.h).
//
// They are C++ because a training step calls them hundreds of times on small
// tensors: a Python autograd.Function costs about 35 us a forward and backward
// more than a node of this kind (its backward pass takes the interpreter lock on
// autograd's thread), several times the kernels' own time there.
//
// The kernel library is not linked: bind() takes its entry points' addresses, so
// that whichever build of it Python loaded (release or checked) is the one called.
// Checks run for any device; a call on CPU tensors returns None, and the Python
// side answers it from the reference.
#include <ATen/TracerMode.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <atomic>
#include <optional>
#include <unordered_set>
#include <vector>

#include "b200_train.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct KernelFailure : std::runtime_error {
  using std::runtime_error::runtime_error;
};

#define B200_ENTRIES(X)                                                                                         \
  X(b200_dropout) X(b200_block_norms) X(b200_block_norms_bwd) X(b200_block_norms_max_width)                      \
  X(b200_block_norms_bwd_grid) X(b200_lce_saved_bytes) X(b200_lce_forward_bytes) X(b200_lce_backward_bytes)      \
  X(b200_lce_forward) X(b200_lce_backward)

struct Entries {
#define X(name) decltype(&::name) name = nullptr;
  B200_ENTRIES(X)
#undef X
  bool bound = false;
} lib;

void bind(const py::dict& addresses) {
#define X(name) lib.name = reinterpret_cast<decltype(&::name)>(addresses[#name].cast<uintptr_t>());
  B200_ENTRIES(X)
#undef X
  lib.bound = true;
}

void check(int rc, const char* what) {
  if (rc != 0) throw KernelFailure(std::string(what) + " failed with code " + std::to_string(rc));
}

int num_sms(const at::Device& dev) {
  constexpr int kMax = 64;
  static std::atomic<int> known[kMax];
  const int i = dev.index();
  TORCH_CHECK(i >= 0 && i < kMax, "device index ", i);
  int n = known[i].load(std::memory_order_relaxed);
  if (n == 0) {
    TORCH_CHECK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, i) == cudaSuccess, "no device ", i);
    known[i].store(n, std::memory_order_relaxed);
  }
  return n;
}

// The tensors' device is current for the scope (a launch goes to the calling
// thread's device, whatever its stream); `stream` is torch's current one there.
struct Launch {
  c10::cuda::CUDAGuard guard;
  cudaStream_t stream;
  explicit Launch(const Tensor& t)
      : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {
    if (!lib.bound) throw KernelFailure("the kernel library is not loaded");
  }
};

int elem_code(const Tensor& t, const char* what) {  // ElemType
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: TORCH_CHECK_TYPE(false, what, " must be bfloat16, float16 or float32, not ", t.scalar_type());
  }
}

void same_device(const char* what, const Tensor& a, const Tensor& b) {
  if (b.defined()) TORCH_CHECK_VALUE(a.device() == b.device(), what, ": tensors on ", a.device(), " and ", b.device());
}

// t as it stands in memory: a lazily negated view (complex numbers' .conj().imag) becomes a tensor.
Tensor plain(const Tensor& t) { return t.defined() ? t.resolve_neg() : t; }
// t [..., width] as [rows, width] with neighbouring columns: a view where the
// strides allow it, else a copy. width > 0.
Tensor rows2d(const Tensor& t_, int64_t width) {
  const Tensor t = plain(t_);
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, width});
  return width <= 1 || r.stride(1) == 1 ? r : r.contiguous();
}

Tensor empty(const Tensor& like, at::IntArrayRef shape, at::ScalarType type) {
  return at::empty(shape, like.options().dtype(type).requires_grad(false));
}
Tensor packed_like(const Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false)); }
// What a kernel reads or writes has memory: fake tensors and wrappers of other tensors have
// none, and null would be their address.
bool has_memory(const Tensor& t) {
  return t.has_storage() && t.storage().unsafeGetStorageImpl()->_mutable_data_ptr_no_checks().get() != nullptr;
}
void in_memory(const Tensor& t) {
  TORCH_CHECK_TYPE(!t.defined() || t.numel() == 0 || has_memory(t),
                   "a training operator on a tensor without memory (a fake tensor or a wrapper)");
}
template <typename T = void>
T* ptr(const Tensor& t) {
  in_memory(t);
  return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
// Inputs that the kernels can answer for: in memory, and without forward-mode tangents,
// which a kernel would drop. Nor is the call traced: a trace would hold the empty outputs and
// not the launch.
void computable(const char* what, std::initializer_list<Tensor> inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(!at::tracer::impl::is_dispatch_enabled(), what, ": torch.jit.trace on CUDA");
  for (const Tensor& t : inputs) {
    in_memory(t);
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), what, ": forward-mode derivatives on CUDA");
  }
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
// autograd's argument lists hold no undefined tensors
using Maybe = std::optional<Tensor>;
Tensor opt(const Maybe& t) { return t.has_value() ? *t : Tensor(); }
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }

// A node of the inputs' graph that was made on another stream, outside the capture, and still
// lives: a leaf's accumulation that an eager graph keeps, or an eager part of this graph. The
// engine would make the captured backward pass wait for its stream, which a capture cannot, and
// from its thread that ends the process. The forward call of such a step is refused while it
// can be.
void capturable(const char* what, std::initializer_list<Tensor> inputs) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  std::vector<std::shared_ptr<torch::autograd::Node>> todo;
  for (const Tensor& t : inputs)
    if (wants_grad(t) && t.is_cuda())
      todo.push_back(t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn());
  std::unordered_set<const torch::autograd::Node*> seen;
  while (!todo.empty()) {
    const auto node = std::move(todo.back());
    todo.pop_back();
    if (!node || !seen.insert(node.get()).second) continue;
    const auto stream = node->stream();
    if (stream && stream->device_type() == c10::DeviceType::CUDA) {
      const c10::cuda::CUDAStream made(*stream);
      cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
      if (made != c10::cuda::getCurrentCUDAStream(made.device_index()) && made.stream() != nullptr &&
          cudaStreamIsCapturing(made.stream(), &status) != cudaSuccess)
        status = cudaStreamCaptureStatusNone, cudaGetLastError();
      TORCH_CHECK(made == c10::cuda::getCurrentCUDAStream(made.device_index()) || status == cudaStreamCaptureStatusActive, what,
                  ": a graph of the same leaf, made on another stream, is still alive; drop its outputs before the capture");
    }
    for (const auto& edge : node->next_edges()) todo.push_back(edge.function);
  }
}

// A backward pass's incoming gradients.
void once(const char* what, const variable_list& grads) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the gradient is not differentiable a second time");
  for (const Tensor& g : grads) computable(what, {g});
}

// What autograd gives back of a saved tensor, which hooks of the caller may have replaced: the
// kernels read it by the sizes, type and device that it had.
Tensor kept(const char* what, const Tensor& t, const at::Device& device, at::ScalarType type, at::IntArrayRef sizes) {
  TORCH_CHECK(t.defined() && t.device() == device && t.scalar_type() == type && t.sizes() == sizes, what,
              ": a saved tensor came back changed");
  return t;
}

// ------------------------------------------------------------------ dropout
Tensor dropout_run(const Tensor& x, int64_t cut, uint64_t seed, uint64_t offset, const Tensor& offset_t, const Tensor& residual) {
  if (cut == 65536)  // nothing stays
    return residual.defined() ? residual.clone(at::MemoryFormat::Contiguous) : at::zeros(x.sizes(), x.options().requires_grad(false));
  Tensor y = packed_like(x);
  if (x.numel() == 0) return y;
  const int64_t K = x.dim() ? x.size(-1) : 1;
  const Tensor x2 = rows2d(x, K), r2 = residual.defined() ? rows2d(residual, K) : residual;
  const Launch on(x);
  check(lib.b200_dropout(ptr(x2), x2.stride(0), ptr(r2), r2.defined() ? r2.stride(0) : 0, ptr(y), K, x2.size(0),
                         (int)K, elem_code(x, "dropout"), seed, offset, ptr<int64_t>(offset_t), (int)cut,
                         (float)(65536.0 / (65536 - cut)), num_sms(x.device()), on.stream),
        "dropout");
  return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual_, int64_t cut, int64_t seed, int64_t offset,
                        const Maybe& offset_) {
    const Tensor residual = opt(residual_), offset_t = opt(offset_);
    // a device counter may have moved on by the time the gradient is taken: its value is kept, not the tensor
    const Tensor off = offset_t.defined() ? offset_t.clone() : offset_t;
    ctx->saved_data["call"] = std::vector<int64_t>{cut, seed, offset, wants_grad(x), wants_grad(residual)};
    if (off.defined()) ctx->saved_data["offset"] = off;
    return dropout_run(x, cut, (uint64_t)seed, (uint64_t)offset, off, residual);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("dropout", grads);
    const auto call = ctx->saved_data["call"].toIntVector();
    const auto off = ctx->saved_data.find("offset");
    Tensor dx, dr;
    if (call[3])
      dx = dropout_run(grads[0], call[0], (uint64_t)call[1], (uint64_t)call[2],
                       off == ctx->saved_data.end() ? Tensor() : off->second.toTensor(), Tensor());
    if (call[4]) dr = grads[0];
    return {dx, dr, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Maybe dropout(const Tensor& x, double p, uint64_t seed, uint64_t offset, const Maybe& offset_t,
                              const Maybe& residual_) {
  const Tensor residual = opt(residual_), off = plain(opt(offset_t));
  TORCH_CHECK_VALUE(p >= 0.0 && p <= 1.0, "dropout probability ", p, " is not in [0, 1]");
  elem_code(x, "dropout");
  if (residual.defined()) {
    same_device("dropout", x, residual);
    TORCH_CHECK_VALUE(residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type(), "dropout: residual ",
                      residual.sizes(), " ", residual.scalar_type(), " for x ", x.sizes(), " ", x.scalar_type());
  }
  if (off.defined()) {
    TORCH_CHECK_VALUE(off.scalar_type() == at::kLong && off.numel() == 1, "dropout: a tensor offset is one int64 element");
    same_device("dropout", x, off);
  }
  if (!x.is_cuda()) return std::nullopt;
  computable("dropout", {x, residual, off});
  TORCH_CHECK_VALUE((x.dim() ? x.size(-1) : 1) <= INT32_MAX, "dropout: rows of ", x.size(-1), " columns");
  const int64_t cut = (int64_t)(p * 65536 + 0.5);
  if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(residual))) {
    capturable("dropout", {x, residual});
    return Dropout::apply(x, maybe(residual), cut, (int64_t)seed, (int64_t)offset, maybe(off));
  }
  return dropout_run(x, cut, seed, offset, off, residual);
}

// ------------------------------------------------------------------ block norms
enum GateKind { kNone = 0, kChannel = 1, kRow = 2, kElement = 3 };

struct NormCall {
  int64_t kind;
  double eps, scale;
  bool offset_one, round_branch;
};

Tensor gate_rows(const Tensor& gate, int64_t kind, int64_t H) {
  return !gate.defined() ? gate : kind == kElement ? rows2d(gate, H) : plain(gate).contiguous();
}
Tensor packed(const Tensor& w) { return w.defined() ? plain(w).contiguous() : w; }

// An in-place call reads `t` ([rows, cols] with rows `ld` apart) while other CTAs write rows of
// x. That is sound where t's elements are none of x's, or (aligned: one for each of x's) where
// each is the very element of x that its thread writes, which reads it before.
void inplace_reads(const char* what, const Tensor& x2, const Tensor& t, int64_t rows, int64_t cols, int64_t ld, bool aligned) {
  if (!t.defined() || x2.numel() == 0 || rows == 0 || !has_memory(x2) || !has_memory(t)) return;
  const int64_t xs = x2.element_size(), ts = t.element_size();
  const int64_t xp = (int64_t)reinterpret_cast<uintptr_t>(ptr(x2)), tp = (int64_t)reinterpret_cast<uintptr_t>(t.data_ptr());
  const int64_t width = x2.size(1) * xs, step = x2.stride(0) * xs;
  if (tp >= xp + (x2.size(0) - 1) * step + width || tp + (rows - 1) * ld * ts + cols * ts <= xp) return;
  if (aligned && tp == xp && (rows == 1 || ld * ts == step)) return;
  if (x2.size(0) > 1 && (rows == 1 || ld * ts == step)) {  // beside x's columns in the rows of one buffer
    const int64_t off = ((tp - xp) % step + step) % step;
    if (off >= width && off + cols * ts <= step) return;
  }
  TORCH_CHECK_VALUE(false, "block_norms: inplace writes x, whose memory ", what, " shares");
}

// {y, h, r1, r2}; y is written into `into` when given. r1 / r2 (the reciprocal RMS of
// delta and y) are kept for the backward pass with `save`.
std::array<Tensor, 4> norms_run(const Tensor& x, const Tensor& delta, const Tensor& post, const Tensor& pre, const Tensor& gate,
                                const NormCall& c, const Tensor& into, bool save) {
  const int64_t H = x.size(-1);
  const Tensor x2 = rows2d(x, H), d2 = rows2d(delta, H);
  const int64_t T = x2.size(0);
  const Tensor y = into.defined() ? into : packed_like(x), y2 = rows2d(y, H);
  Tensor h, r1, r2;
  if (pre.defined()) h = packed_like(x);
  if (save && post.defined()) r1 = empty(x, {T}, at::kFloat);
  if (save && pre.defined()) r2 = empty(x, {T}, at::kFloat);
  if (T) {
    const Tensor pw = packed(post), qw = packed(pre), g = gate_rows(gate, c.kind, H);
    const Tensor& w = pw.defined() ? pw : qw;
    const Launch on(x);
    check(lib.b200_block_norms(ptr(x2), x2.stride(0), ptr(d2), d2.stride(0), ptr(pw), ptr(qw),
                               elem_code(w.defined() ? w : x, "block_norms weight"), ptr(g), c.kind == kElement ? g.stride(0) : 0,
                               (int)c.kind, ptr(y2), y2.stride(0), ptr(h), H, ptr<float>(r1), ptr<float>(r2), T, (int)H,
                               elem_code(x, "block_norms"), (float)c.eps, (float)c.scale, c.offset_one, c.round_branch,
                               num_sms(x.device()), on.stream),
          "block_norms");
  }
  return {y, h, r1, r2};
}

struct BlockNorms : torch::autograd::Function<BlockNorms> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& delta, const Maybe& post_, const Maybe& pre_,
                               const Maybe& gate_, int64_t kind, double eps, double scale, bool offset_one, bool round_branch) {
    const Tensor post = opt(post_), pre = opt(pre_), gate = opt(gate_);
    ctx->set_materialize_grads(false);
    auto [y, h, r1, r2] = norms_run(x, delta, post, pre, gate, {kind, eps, scale, offset_one, round_branch}, Tensor(), true);
    ctx->save_for_backward({y, delta, post, pre, gate, r1, r2});
    ctx->saved_data["call"] = std::vector<int64_t>{kind, offset_one, wants_grad(x), wants_grad(delta), wants_grad(post),
                                                   wants_grad(pre), wants_grad(gate), post.defined(), pre.defined(),
                                                   (int64_t)(post.defined() ? post : pre.defined() ? pre : x).scalar_type()};
    ctx->saved_data["scale"] = scale;
    if (gate.defined()) ctx->saved_data["gate"] = gate.sizes().vec();
    if (h.defined()) return {y, h};
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("block_norms", grads);
    const auto saved = ctx->get_saved_variables();
    const auto call = ctx->saved_data["call"].toIntVector();
    const Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
    variable_list out(10);
    if (!dy.defined() && !dh.defined()) return out;
    // the engine has given either gradient y's sizes, type and device
    const Tensor& like = dy.defined() ? dy : dh;
    const int64_t kind = call[0], H = like.size(-1), rows = like.numel() / H;
    auto back = [&](int i, at::ScalarType type, at::IntArrayRef sizes) {
      return kept("block_norms", saved[i], like.device(), type, sizes);
    };
    const auto w_type = (at::ScalarType)call[9];
    const Tensor y = back(0, like.scalar_type(), like.sizes()), delta = back(1, like.scalar_type(), like.sizes());
    const Tensor post = call[7] ? back(2, w_type, {H}) : Tensor(), pre = call[8] ? back(3, w_type, {H}) : Tensor();
    const Tensor gate = kind != kNone ? back(4, like.scalar_type(), ctx->saved_data["gate"].toIntVector()) : Tensor();
    const Tensor r1 = call[7] ? back(5, at::kFloat, {rows}).contiguous() : Tensor();
    const Tensor r2 = call[8] ? back(6, at::kFloat, {rows}).contiguous() : Tensor();
    Tensor &dx = out[0], &dd = out[1], &dpost = out[2], &dpre = out[3], &dgate = out[4];
    if (call[2]) dx = packed_like(y);
    if (call[3]) dd = packed_like(delta);
    if (call[4]) dpost = packed_like(post);
    if (call[5] && dh.defined()) dpre = packed_like(pre);
    if (call[6]) dgate = packed_like(gate);
    const Tensor y2 = rows2d(y, H), d2 = rows2d(delta, H);
    const int64_t T = y2.size(0);
    if (T == 0) {
      for (Tensor* t : {&dpost, &dpre, &dgate})
        if (t->defined()) t->zero_();
      return out;
    }
    const Tensor dy2 = dy.defined() ? rows2d(dy, H) : dy, dh2 = dh.defined() ? rows2d(dh, H) : dh;
    const Tensor pw = packed(post), qw = packed(pre), g = gate_rows(gate, kind, H);
    const Tensor& w = pw.defined() ? pw : qw;
    const int type = elem_code(y, "block_norms"), sms = num_sms(y.device());
    const int parts = dpost.defined() + dpre.defined() + (dgate.defined() && kind == kChannel);
    const Launch on(y);
    Tensor part;
    if (parts) part = empty(y, {(int64_t)parts * lib.b200_block_norms_bwd_grid(T, (int)H, type, sms) * H}, at::kFloat);
    check(lib.b200_block_norms_bwd(ptr(y2), y2.stride(0), ptr(d2), d2.stride(0), ptr(pw), ptr(qw),
                                   elem_code(w.defined() ? w : y, "block_norms weight"), ptr(g),
                                   kind == kElement ? g.stride(0) : 0, (int)kind, ptr<float>(r1), ptr<float>(r2), ptr(dy2),
                                   dy2.defined() ? dy2.stride(0) : 0, ptr(dh2), dh2.defined() ? dh2.stride(0) : 0, ptr(dx),
                                   ptr(dd), ptr(dgate), ptr(dpost), ptr(dpre), ptr<float>(part), T, (int)H, type,
                                   (float)ctx->saved_data["scale"].toDouble(), (int)call[1], sms, on.stream),
          "block_norms backward");
    return out;
  }
};

// (y, h) with h undefined without pre_w, or nothing for CPU tensors.
std::optional<std::pair<Tensor, Maybe>> block_norms(
    const Tensor& x, const Tensor& delta, const Maybe& post_, const Maybe& pre_, double eps,
    const Maybe& gate_, double scale, bool offset_one, bool round_branch, bool inplace) {
  const Tensor post = opt(post_), pre = opt(pre_), gate = opt(gate_);
  TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "block_norms: x needs at least one column");
  const int64_t H = x.size(-1);
  elem_code(x, "block_norms");
  TORCH_CHECK_VALUE(delta.sizes() == x.sizes() && delta.scalar_type() == x.scalar_type(), "block_norms: delta ", delta.sizes(),
                    " ", delta.scalar_type(), " for x ", x.sizes(), " ", x.scalar_type());
  int64_t kind = kNone;
  if (gate.defined()) {
    std::vector<int64_t> row(x.sizes().begin(), x.sizes().end());
    row.back() = 1;
    kind = gate.sizes() == x.sizes().slice(x.dim() - 1) ? kChannel
           : gate.sizes() == at::IntArrayRef(row)       ? kRow
           : gate.sizes() == x.sizes()                  ? kElement
                                                        : -1;
    TORCH_CHECK_VALUE(kind >= 0, "block_norms: gate ", gate.sizes(), " is neither [", H, "], ", at::IntArrayRef(row), " nor ",
                      x.sizes());
    same_device("block_norms", x, gate);
    TORCH_CHECK_TYPE(gate.scalar_type() == x.scalar_type(), "block_norms: gate ", gate.scalar_type(), " for x ", x.scalar_type());
  }
  for (const Tensor* w : {&post, &pre})
    if (w->defined()) {
      TORCH_CHECK_VALUE(w->dim() == 1 && w->size(0) == H, "block_norms: weight ", w->sizes(), " for rows of ", H);
      TORCH_CHECK_TYPE(w->scalar_type() == x.scalar_type() || w->scalar_type() == at::kFloat, "block_norms: weight ",
                       w->scalar_type(), " for x ", x.scalar_type());
      same_device("block_norms", x, *w);
    }
  if (post.defined() && pre.defined())
    TORCH_CHECK_TYPE(post.scalar_type() == pre.scalar_type(), "block_norms: post_w ", post.scalar_type(), ", pre_w ",
                     pre.scalar_type());
  same_device("block_norms", x, delta);
  const bool grad = at::GradMode::is_enabled() &&
                    (x.requires_grad() || delta.requires_grad() || wants_grad(post) || wants_grad(pre) || wants_grad(gate));
  if (inplace) {
    TORCH_CHECK_VALUE(!grad, "block_norms: inplace takes no gradients");
    TORCH_CHECK_VALUE(!x.is_neg(), "block_norms: inplace on a lazily negated view");
    const Tensor rows = x.view({-1, H});
    TORCH_CHECK_VALUE(x.numel() == 0 || ((H == 1 || rows.stride(1) == 1) && (rows.size(0) == 1 || rows.stride(0) >= H)),
                      "block_norms: inplace needs rows of neighbouring columns that do not overlap");
    if (x.numel()) {
      const int64_t T = rows.size(0);
      const Tensor d2 = rows2d(delta, H), g = gate_rows(gate, kind, H);
      inplace_reads("delta", rows, d2, T, H, d2.stride(0), true);
      inplace_reads("post_w", rows, packed(post), 1, H, H, false);
      inplace_reads("pre_w", rows, packed(pre), 1, H, H, false);
      if (kind == kElement) inplace_reads("the gate", rows, g, T, H, g.stride(0), true);
      else inplace_reads("the gate", rows, g, 1, kind == kChannel ? H : T, 0, false);
    }
  }
  if (!x.is_cuda()) return std::nullopt;
  computable("block_norms", {x, delta, post, pre, gate});
  if (!lib.bound) throw KernelFailure("the kernel library is not loaded");
  TORCH_CHECK_VALUE(H <= lib.b200_block_norms_max_width(), "block_norms: ", H, " columns, at most ",
                    lib.b200_block_norms_max_width());
  if (grad) {
    capturable("block_norms", {x, delta, post, pre, gate});
    const auto out = BlockNorms::apply(x, delta, maybe(post), maybe(pre), maybe(gate), kind, eps, scale, offset_one, round_branch);
    return std::make_pair(out[0], out.size() > 1 ? Maybe(out[1]) : std::nullopt);
  }
  const auto out = norms_run(x, delta, post, pre, gate, {kind, eps, scale, offset_one, round_branch}, inplace ? x : Tensor(), false);
  // a node that saved x before has to see that it changed (inference tensors have no counter)
  if (inplace && !x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
  return std::make_pair(out[0], maybe(out[1]));
}

// ------------------------------------------------------------------ linear cross entropy
enum Reduction { kEach = 0, kSum = 1, kMean = 2 };

// The head as TMA reads it (16-byte aligned rows of neighbouring columns): itself, or a
// copy in padded rows.
Tensor aligned_head(const Tensor& w) {
  const int64_t V = w.size(0), K = w.size(1);
  if (!w.is_neg() && (K == 1 || w.stride(1) == 1) && w.stride(0) % 8 == 0 && w.stride(0) >= K &&
      (reinterpret_cast<uintptr_t>(ptr(w)) & 15) == 0)
    return w.detach();
  Tensor out = empty(w, {V, (K + 7) / 8 * 8}, at::kBFloat16).narrow(1, 0, K);
  out.copy_(w.detach());
  return out;
}

struct CeOut {
  Tensor out, saved;
};
CeOut ce_forward(const Tensor& h2, const Tensor& w_, const Tensor& targets, double cap, int64_t ignore, int64_t reduction) {
  const int64_t T = h2.size(0), K = h2.size(1), V = w_.size(0), Kp = (K + 7) / 8 * 8;
  const Tensor w = aligned_head(w_);
  const Launch on(h2);
  const Tensor saved = empty(h2, {lib.b200_lce_saved_bytes((int)T, (int)Kp)}, at::kByte);
  const Tensor part = empty(h2, {lib.b200_lce_forward_bytes((int)T, (int)V)}, at::kByte);
  const Tensor loss = empty(h2, {T}, at::kFloat);
  Tensor total;
  if (reduction != kEach) total = empty(h2, {}, at::kFloat);
  check(lib.b200_lce_forward(ptr(h2), h2.stride(0), ptr(w), w.stride(0), ptr<int64_t>(targets), ignore, (int)T,
                             (int)V, (int)K, (int)Kp, (float)cap, ptr(saved), ptr(part), ptr<float>(loss),
                             ptr<float>(total), reduction == kMean, num_sms(h2.device()), on.stream),
        "linear_cross_entropy");
  return {total.defined() ? total : loss, saved};
}

struct LinearCe : torch::autograd::Function<LinearCe> {
  static Tensor forward(AutogradContext* ctx, const Tensor& h2, const Tensor& w, const Tensor& targets, double cap, int64_t ignore,
                        int64_t reduction, int64_t piece) {
    const CeOut r = ce_forward(h2, w, targets, cap, ignore, reduction);
    ctx->save_for_backward({w, r.saved});
    ctx->saved_data["call"] =
        std::vector<int64_t>{h2.size(0), h2.size(1), reduction, piece, wants_grad(h2), wants_grad(w), w.size(0)};
    ctx->saved_data["cap"] = cap;
    return r.out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once("linear_cross_entropy", grads);
    const auto call = ctx->saved_data["call"].toIntVector();
    const int64_t T = call[0], K = call[1], V = call[6], Kp = (K + 7) / 8 * 8, piece = call[3];
    const auto back = ctx->get_saved_variables();
    const at::Device device = grads[0].device();
    const Tensor w_ = kept("linear_cross_entropy", back[0], device, at::kBFloat16, {V, K});
    const Tensor saved =
        kept("linear_cross_entropy", back[1], device, at::kByte, {lib.b200_lce_saved_bytes((int)T, (int)Kp)}).contiguous();
    const Tensor w = aligned_head(w_), g = plain(grads[0]).reshape(-1);
    const int sms = num_sms(w.device());
    const Launch on(w);
    const int64_t room = lib.b200_lce_backward_bytes((int)T, (int)V, (int)K, (int)Kp, (int)piece, (int)call[4], (int)call[5], sms);
    const Tensor scratch = empty(w, {room}, at::kByte);
    Tensor dh, dw;
    if (call[4]) dh = empty(w, {T, K}, at::kBFloat16);
    if (call[5]) {  // rows as TMA stores them
      dw = empty(w, {V, Kp}, at::kBFloat16);
      if (Kp != K) dw = dw.narrow(1, 0, K);
    }
    check(lib.b200_lce_backward(ptr(saved), ptr(w), w.stride(0), ptr<float>(g),
                                T > 1 && g.numel() == T ? g.stride(0) : 0, call[2] == kMean, (int)T, (int)V, (int)K, (int)Kp,
                                (float)ctx->saved_data["cap"].toDouble(), (int)piece, ptr(scratch), ptr(dh), ptr(dw), Kp,
                                sms, on.stream),
          "linear_cross_entropy backward");
    return {dh, dw, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Maybe linear_cross_entropy(const Tensor& h, const Tensor& w, const Tensor& targets, double cap, int64_t ignore,
                                           const std::string& reduction_, int64_t piece_bytes, int64_t min_piece) {
  const int64_t reduction = reduction_ == "none" ? kEach : reduction_ == "sum" ? kSum : reduction_ == "mean" ? kMean : -1;
  TORCH_CHECK_VALUE(reduction >= 0, "linear_cross_entropy: reduction '", reduction_, "'");
  TORCH_CHECK_VALUE(h.dim() > 0 && w.dim() == 2 && w.size(1) == h.size(-1) && w.size(0) > 0 && w.size(1) > 0,
                    "linear_cross_entropy: hidden rows ", h.sizes(), ", head ", w.sizes());
  TORCH_CHECK_VALUE(targets.sizes() == h.sizes().slice(0, h.dim() - 1), "linear_cross_entropy: targets ", targets.sizes(),
                    " for hidden rows ", h.sizes());
  TORCH_CHECK_TYPE(targets.scalar_type() == at::kLong, "linear_cross_entropy: targets ", targets.scalar_type(), ", int64 needed");
  TORCH_CHECK_TYPE(h.scalar_type() == w.scalar_type() && h.is_floating_point(), "linear_cross_entropy: hidden rows ",
                   h.scalar_type(), ", head ", w.scalar_type());
  // the kernels hold it and its reciprocal in 32 bits: neither may round to 0 (no cap) or inf
  TORCH_CHECK_VALUE(cap == 0.0 || (cap >= 0x1p-126 && cap <= 0x1p126), "linear_cross_entropy: softcap ", cap,
                    ", 0 or a value from 2^-126 to 2^126 needed");
  same_device("linear_cross_entropy", h, w);
  same_device("linear_cross_entropy", h, targets);
  if (!h.is_cuda()) return std::nullopt;
  TORCH_CHECK_TYPE(h.scalar_type() == at::kBFloat16, "linear_cross_entropy: ", h.scalar_type(),
                   "; the CUDA kernels take bfloat16");
  computable("linear_cross_entropy", {h, w, targets});
  const int64_t T = targets.numel(), K = w.size(1), V = w.size(0);
  constexpr int64_t kMost = INT32_MAX - 65536;  // tile counts and coordinates are 32-bit
  TORCH_CHECK_VALUE(T <= kMost && V <= kMost && K <= kMost, "linear_cross_entropy: ", T, " rows, ", V, " x ", K, " head");
  if (!lib.bound) throw KernelFailure("the kernel library is not loaded");
  if (T == 0) {
    // sums of nothing: both stay in the graph, with zero gradients
    const Tensor zero = h.to(at::kFloat).sum() + w.narrow(0, 0, 0).to(at::kFloat).sum();
    return reduction == kEach ? zero.expand(targets.sizes()) : zero;
  }
  const Tensor h2 = rows2d(h, K), t1 = plain(targets).reshape(-1).contiguous();
  Tensor out;
  if (at::GradMode::is_enabled() && (h.requires_grad() || w.requires_grad())) {
    capturable("linear_cross_entropy", {h, w});
    constexpr int64_t kTile = 256;  // pieces of the vocabulary are whole tiles
    const int64_t piece = std::min(std::max(min_piece, piece_bytes / (2 * T) / kTile * kTile), (V + kTile - 1) / kTile * kTile);
    out = LinearCe::apply(h2, w, t1, cap, ignore, reduction, piece);
  } else {
    out = ce_forward(h2, w, t1, cap, ignore, reduction).out;
  }
  return reduction == kEach && targets.dim() != 1 ? out.reshape(targets.sizes()) : out;
}

}  // namespace

PYBIND11_MODULE(_b200torch, m) {
  m.doc() = "Differentiable training operators over the sm_100a kernel library.";
  m.def("bind", [](const py::dict& addresses) { bind(addresses); });
  m.def("raise_as", [](const py::object& kernel_error) {
    static py::object* error = new py::object(kernel_error);  // raised for a kernel entry point's error code
    py::register_exception_translator([](std::exception_ptr p) {
      try {
        if (p) std::rethrow_exception(p);
      } catch (const KernelFailure& e) {
        PyErr_SetString(error->ptr(), e.what());
      } catch (const c10::ValueError& e) {
        PyErr_SetString(PyExc_ValueError, e.what_without_backtrace());
      } catch (const c10::NotImplementedError& e) {
        PyErr_SetString(PyExc_NotImplementedError, e.what_without_backtrace());
      } catch (const c10::TypeError& e) {
        PyErr_SetString(PyExc_TypeError, e.what_without_backtrace());
      }
    });
  });
  const auto unlocked = py::call_guard<py::gil_scoped_release>();
  m.def("dropout", &dropout, unlocked, py::arg("x"), py::arg("p"), py::arg("seed"), py::arg("offset"), py::arg("offset_t"),
        py::arg("residual"));
  m.def("block_norms", &block_norms, unlocked, py::arg("x"), py::arg("delta"), py::arg("post_w"), py::arg("pre_w"),
        py::arg("eps"), py::arg("gate"), py::arg("scale"), py::arg("offset_one"), py::arg("round_branch"), py::arg("inplace"));
  m.def("linear_cross_entropy", &linear_cross_entropy, unlocked, py::arg("h"), py::arg("w"), py::arg("targets"),
        py::arg("softcap"), py::arg("ignore_index"), py::arg("reduction"), py::arg("piece_bytes"), py::arg("min_piece"));
}
