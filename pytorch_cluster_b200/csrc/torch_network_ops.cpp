// Torch operators of gather_rows, norm_rotate and attention, differentiable once: tensor checks, output and workspace
// allocation, the caller's current stream.  The autograd nodes are C++: a training step of a small call is bound by the
// host, and nodes written in Python cost 30 of its 105 us (gather_rows of 1100 edges).  No CPU branch.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/script.h>
#include <nvtx3/nvToolsExt.h>

#include <cmath>
#include <tuple>
#include <vector>

#include "b200_cluster.h"

namespace {

#define CHECK_CUDA(x) TORCH_CHECK(x.device().is_cuda(), #x " must be CUDA tensor")
#define CHECK_INPUT(x) TORCH_CHECK(x, "Input mismatch")

using OptTensor = std::optional<torch::Tensor>;

struct OpRange {
  explicit OpRange(const char *name) { nvtxRangePushA(name); }
  ~OpRange() { nvtxRangePop(); }
  OpRange(const OpRange &) = delete;
  OpRange &operator=(const OpRange &) = delete;
};

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Derivatives are taken backward only.  A tangent would be dropped without a word, which makes the derivative zero.
void refuse_tangents(const char *op, std::initializer_list<const torch::Tensor *> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const torch::Tensor *t : tensors)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), op, " has no forward-mode derivative");
}

bool wants_gradient(std::initializer_list<const torch::Tensor *> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const torch::Tensor *t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// The gradients carry no graph of their own.  Where one is asked for, they come out of this node, which hangs on what
// they were formed from and whose own backward pass refuses, instead of as constants.
struct OnceDifferentiable : torch::autograd::Function<OnceDifferentiable> {
  static variable_list forward(AutogradContext *, at::TensorList tensors, int64_t count) {
    return {tensors.begin(), tensors.begin() + count};
  }
  static variable_list backward(AutogradContext *, variable_list) {
    TORCH_CHECK(false, "trying to differentiate twice a function that is differentiable once");
    return {};
  }
};

variable_list once(variable_list grads, const variable_list &sources) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list tensors;
  for (const auto &g : grads)
    if (g.defined()) tensors.push_back(g);
  const int64_t count = (int64_t)tensors.size();
  bool any = false;
  for (const auto &t : sources)
    if (t.defined()) {
      tensors.push_back(t);
      any = any || t.requires_grad();
    }
  if (!any) return grads;
  variable_list out = OnceDifferentiable::apply(at::TensorList(tensors), count);
  size_t at = 0;
  for (auto &g : grads)
    if (g.defined()) g = out[at++];
  return grads;
}

void check_status(int status) { TORCH_CHECK(status == B200C_OK, "b200_cluster: ", b200c_last_error()); }

int dtype_code(const torch::Tensor &t, const char *op) {
  switch (t.scalar_type()) {
    case at::kFloat: return B200C_F32;
    case at::kHalf: return B200C_F16;
    case at::kBFloat16: return B200C_BF16;
    default: TORCH_CHECK(false, op, " covers float, half and bfloat16 tensors, got ", t.scalar_type());
  }
  return -1;
}

torch::Tensor workspace(size_t bytes, const torch::Tensor &like) {
  return torch::empty({(int64_t)bytes}, like.options().dtype(torch::kByte));
}

// rows whose channels are contiguous are taken as they stand (a slice of a joint projection), others are copied
torch::Tensor rows_of(const torch::Tensor &t) {
  return t.numel() == 0 || t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous();
}

// ---- gather_rows -------------------------------------------------------------------------------------------------

torch::Tensor gather_rows_forward(torch::Tensor x, torch::Tensor index, double scale) {
  OpRange range("torch_cluster::gather_rows");
  CHECK_CUDA(x);
  CHECK_CUDA(index);
  CHECK_INPUT(x.dim() == 2 && index.dim() == 1);
  CHECK_INPUT(x.get_device() == index.get_device());
  TORCH_CHECK(index.scalar_type() == at::kLong, "index must be an int64 tensor");
  const int dtype = dtype_code(x, "gather_rows");
  c10::cuda::CUDAGuard guard(x.device());
  x = x.contiguous();
  index = index.contiguous();
  auto out = torch::empty({index.numel(), x.size(1)}, x.options());
  if (out.numel() == 0) return out;
  if (x.size(0) == 0) return out.zero_();
  check_status(b200c_gather_rows(x.data_ptr(), index.data_ptr<int64_t>(), x.size(0), index.numel(), x.size(1),
                                 (float)scale, dtype, out.data_ptr(), at::cuda::getCurrentCUDAStream().stream()));
  return out;
}

torch::Tensor gather_rows_backward(torch::Tensor dout, torch::Tensor index, int64_t rows, double scale) {
  OpRange range("torch_cluster::gather_rows_backward");
  at::NoGradGuard no_grad;
  CHECK_CUDA(dout);
  CHECK_CUDA(index);
  CHECK_INPUT(dout.dim() == 2 && index.dim() == 1 && dout.size(0) == index.numel() && rows >= 0);
  CHECK_INPUT(dout.get_device() == index.get_device());
  TORCH_CHECK(index.scalar_type() == at::kLong, "index must be an int64 tensor");
  const int dtype = dtype_code(dout, "gather_rows");
  c10::cuda::CUDAGuard guard(dout.device());
  dout = dout.contiguous();
  index = index.contiguous();
  const int64_t edges = index.numel(), channels = dout.size(1);
  auto dx = torch::empty({rows, channels}, dout.options());
  if (dx.numel() == 0) return dx;
  const size_t bytes = b200c_gather_rows_workspace_bytes(rows, edges, channels);
  auto ws = workspace(bytes, dout);
  check_status(b200c_gather_rows_backward(dout.data_ptr(), index.data_ptr<int64_t>(), rows, edges, channels,
                                          (float)scale, dtype, dx.data_ptr(), ws.data_ptr(), bytes,
                                          at::cuda::getCurrentCUDAStream().stream()));
  return dx;
}

struct GatherRows : torch::autograd::Function<GatherRows> {
  static torch::Tensor forward(AutogradContext *ctx, torch::Tensor x, torch::Tensor index, double scale) {
    ctx->save_for_backward({index});
    ctx->saved_data["rows"] = x.size(0);
    ctx->saved_data["scale"] = scale;
    return gather_rows_forward(x, index, scale);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    auto dx = gather_rows_backward(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["rows"].toInt(),
                                   ctx->saved_data["scale"].toDouble());
    return once({dx, {}, {}}, {grads[0]});  // x itself is not in it
  }
};

torch::Tensor gather_rows(torch::Tensor x, torch::Tensor index, double scale) {
  refuse_tangents("gather_rows", {&x});
  CHECK_INPUT(x.dim() == 2);
  if (wants_gradient({&x})) return GatherRows::apply(x, index, scale);
  return gather_rows_forward(x, index, scale);
}

// ---- norm_rotate -------------------------------------------------------------------------------------------------

struct Rotation {
  torch::Tensor x[2], pos[2], freq;
  OptTensor weight[2];
  b200c_norm_rotate_side_t side[2];
  int dims = 0, channels = 0, pos_f64 = 0, freq_f64 = 0, dtype = 0;
};

void prepare_rotation(Rotation &r, const torch::Tensor &q, const torch::Tensor &k, const torch::Tensor &pos_q,
                      const torch::Tensor &pos_k, const torch::Tensor &freq, const OptTensor &weight_q,
                      const OptTensor &weight_k) {
  const torch::Tensor in[2] = {q, k}, pos[2] = {pos_q, pos_k};
  const OptTensor weight[2] = {weight_q, weight_k};
  CHECK_CUDA(freq);
  CHECK_INPUT(freq.dim() == 2);
  TORCH_CHECK(freq.scalar_type() == at::kFloat || freq.scalar_type() == at::kDouble, "freq must be float or double");
  r.freq = freq.contiguous();
  r.freq_f64 = freq.scalar_type() == at::kDouble;
  r.dims = (int)freq.size(0);
  r.channels = (int)q.size(-1);
  r.dtype = dtype_code(q, "norm_rotate");
  CHECK_INPUT(q.dim() == 3 && k.dim() == 3 && q.size(2) == k.size(2) && q.scalar_type() == k.scalar_type());
  TORCH_CHECK(q.size(2) % 2 == 0 && q.size(2) >= 2 && q.size(2) <= 256, "channels must be even and at most 256");
  TORCH_CHECK(freq.size(1) * 2 == q.size(2), "freq must be [coordinates, channels / 2]");
  TORCH_CHECK(freq.size(0) >= 1 && freq.size(0) <= 8, "1 to 8 coordinates are supported");
  CHECK_INPUT(pos_q.scalar_type() == pos_k.scalar_type());
  TORCH_CHECK(pos_q.scalar_type() == at::kFloat || pos_q.scalar_type() == at::kDouble,
              "positions must be float or double");
  r.pos_f64 = pos_q.scalar_type() == at::kDouble;
  const bool same = pos_q.is_same(pos_k);
  for (int i = 0; i < 2; ++i) {
    TORCH_CHECK(in[i].is_cuda(), i == 0 ? "q" : "k", " must be CUDA tensor");
    TORCH_CHECK(pos[i].is_cuda(), i == 0 ? "pos_q" : "pos_k", " must be CUDA tensor");
    CHECK_INPUT(pos[i].dim() == 2 && pos[i].size(0) == in[i].size(0) && pos[i].size(1) == freq.size(0));
    CHECK_INPUT(in[i].get_device() == q.get_device() && pos[i].get_device() == q.get_device() &&
                freq.get_device() == q.get_device());
    CHECK_INPUT(in[i].size(1) >= 1);
    r.x[i] = rows_of(in[i]);
    r.pos[i] = i == 1 && same ? r.pos[0] : pos[i].contiguous();
    if (weight[i].has_value()) {
      const torch::Tensor &w = weight[i].value();
      CHECK_INPUT(w.is_cuda() && w.get_device() == q.get_device() && w.dim() == 1 && w.size(0) == q.size(2) &&
                  w.scalar_type() == at::kFloat);
      r.weight[i] = w.contiguous();
    }
    b200c_norm_rotate_side_t &s = r.side[i];
    s = {};
    s.x = r.x[i].data_ptr();
    s.rows = in[i].size(0);
    s.row_stride = r.x[i].stride(0);
    s.head_stride = r.x[i].stride(1);
    s.heads = (int)in[i].size(1);
    s.pos = r.pos[i].data_ptr();
    s.weight = r.weight[i].has_value() ? r.weight[i].value().data_ptr<float>() : nullptr;
  }
}

std::tuple<torch::Tensor, torch::Tensor> norm_rotate_forward(torch::Tensor q, torch::Tensor k, torch::Tensor pos_q,
                                                             torch::Tensor pos_k, torch::Tensor freq,
                                                             OptTensor weight_q, OptTensor weight_k, double eps) {
  OpRange range("torch_cluster::norm_rotate");
  CHECK_CUDA(q);
  CHECK_INPUT(q.dim() == 3);
  c10::cuda::CUDAGuard guard(q.device());
  Rotation r;
  prepare_rotation(r, q, k, pos_q, pos_k, freq, weight_q, weight_k);
  auto yq = torch::empty(q.sizes(), q.options()), yk = torch::empty(k.sizes(), k.options());
  r.side[0].y = yq.data_ptr();
  r.side[1].y = yk.data_ptr();
  check_status(b200c_norm_rotate(&r.side[0], &r.side[1], r.freq.data_ptr(), r.dims, r.channels, r.pos_f64, r.freq_f64,
                                 (float)eps, r.dtype, at::cuda::getCurrentCUDAStream().stream()));
  return {yq, yk};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor> norm_rotate_backward(
    torch::Tensor dyq, torch::Tensor dyk, torch::Tensor q, torch::Tensor k, torch::Tensor pos_q, torch::Tensor pos_k,
    torch::Tensor freq, OptTensor weight_q, OptTensor weight_k, double eps) {
  OpRange range("torch_cluster::norm_rotate_backward");
  at::NoGradGuard no_grad;
  CHECK_CUDA(q);
  CHECK_INPUT(q.dim() == 3);
  CHECK_INPUT(dyq.sizes() == q.sizes() && dyk.sizes() == k.sizes() && dyq.scalar_type() == q.scalar_type() &&
              dyk.scalar_type() == k.scalar_type() && dyq.device() == q.device() && dyk.device() == q.device());
  c10::cuda::CUDAGuard guard(q.device());
  Rotation r;
  prepare_rotation(r, q, k, pos_q, pos_k, freq, weight_q, weight_k);
  dyq = dyq.contiguous();
  dyk = dyk.contiguous();
  auto dq = torch::empty(q.sizes(), q.options()), dk = torch::empty(k.sizes(), k.options());
  const auto fopts = q.options().dtype(torch::kFloat);
  auto dwq = torch::empty({weight_q.has_value() ? r.channels : 0}, fopts);
  auto dwk = torch::empty({weight_k.has_value() ? r.channels : 0}, fopts);
  r.side[0].dy = dyq.data_ptr();
  r.side[1].dy = dyk.data_ptr();
  r.side[0].dx = dq.data_ptr();
  r.side[1].dx = dk.data_ptr();
  r.side[0].dweight = weight_q.has_value() ? dwq.data_ptr<float>() : nullptr;
  r.side[1].dweight = weight_k.has_value() ? dwk.data_ptr<float>() : nullptr;
  const size_t bytes = weight_q.has_value() || weight_k.has_value() ? b200c_norm_rotate_workspace_bytes(r.channels) : 0;
  auto ws = workspace(bytes, q);
  check_status(b200c_norm_rotate_backward(&r.side[0], &r.side[1], r.freq.data_ptr(), r.dims, r.channels, r.pos_f64,
                                          r.freq_f64, (float)eps, r.dtype, bytes ? ws.data_ptr() : nullptr, bytes,
                                          at::cuda::getCurrentCUDAStream().stream()));
  return {dq, dk, dwq, dwk};
}

// an absent tensor is saved, and comes back, as an undefined one
torch::Tensor or_undefined(const OptTensor &t) { return t.has_value() ? t.value() : torch::Tensor(); }
OptTensor or_none(const torch::Tensor &t) { return t.defined() ? OptTensor(t) : std::nullopt; }

struct NormRotate : torch::autograd::Function<NormRotate> {
  static variable_list forward(AutogradContext *ctx, torch::Tensor q, torch::Tensor k, torch::Tensor pos_q,
                               torch::Tensor pos_k, torch::Tensor freq, OptTensor weight_q, OptTensor weight_k,
                               double eps) {
    ctx->save_for_backward({q, k, pos_q, pos_k, freq, or_undefined(weight_q), or_undefined(weight_k)});
    ctx->saved_data["eps"] = eps;
    auto [yq, yk] = norm_rotate_forward(q, k, pos_q, pos_k, freq, weight_q, weight_k, eps);
    return {yq, yk};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto t = ctx->get_saved_variables();
    const OptTensor wq = or_none(t[5]), wk = or_none(t[6]);
    auto [dq, dk, dwq, dwk] = norm_rotate_backward(grads[0], grads[1], t[0], t[1], t[2], t[3], t[4], wq, wk,
                                                   ctx->saved_data["eps"].toDouble());
    return once(
        {dq, dk, {}, {}, {}, wq.has_value() ? dwq : torch::Tensor(), wk.has_value() ? dwk : torch::Tensor(), {}},
        {grads[0], grads[1], t[0], t[1], t[5], t[6]});
  }
};

std::tuple<torch::Tensor, torch::Tensor> norm_rotate(torch::Tensor q, torch::Tensor k, torch::Tensor pos_q,
                                                     torch::Tensor pos_k, torch::Tensor freq, OptTensor weight_q,
                                                     OptTensor weight_k, double eps) {
  const torch::Tensor wq = or_undefined(weight_q), wk = or_undefined(weight_k);
  refuse_tangents("norm_rotate", {&q, &k, &pos_q, &pos_k, &freq, &wq, &wk});
  if (!wants_gradient({&q, &k, &wq, &wk}))
    return norm_rotate_forward(q, k, pos_q, pos_k, freq, weight_q, weight_k, eps);
  auto y = NormRotate::apply(q, k, pos_q, pos_k, freq, weight_q, weight_k, eps);
  return {y[0], y[1]};
}

// ---- attention -----------------------------------------------------------------------------------------------------

// The word in which a kernel says that a bounded wait of its ran out: read before each call, never waited for.  A caller
// of the C ABI who has set one of their own keeps it.
void check_waits() {
  static int32_t *const word = [] {
    int32_t *mine = b200c_attention_report();
    if (mine != nullptr) return mine;
    void *p = nullptr;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // a first call may be a captured one
    C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
    const cudaError_t error = cudaHostAlloc(&p, sizeof(int32_t), cudaHostAllocPortable | cudaHostAllocMapped);
    C10_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
    C10_CUDA_CHECK(error);
    mine = static_cast<int32_t *>(p);
    *mine = 0;
    b200c_attention_set_report(mine);
    return mine;
  }();
  volatile int32_t *seen = word;
  if (*seen == 0) return;
  *seen = 0;
  TORCH_CHECK(false, "b200_cluster: a bounded wait of an earlier attention call ran out; its rows are NaN");
}

struct Attention {
  torch::Tensor q, k, v, ptr_q, ptr_k, pos_q, pos_k, slope;
  b200c_attention_t a{};
};

void prepare_attention(Attention &t, const torch::Tensor &q, const torch::Tensor &k, const torch::Tensor &v,
                       const OptTensor &ptr_q, const OptTensor &ptr_k, const OptTensor &pos_q, const OptTensor &pos_k,
                       const OptTensor &slope, double scale, double cap) {
  CHECK_CUDA(q);
  CHECK_CUDA(k);
  CHECK_CUDA(v);
  CHECK_INPUT(q.dim() == 3 && k.dim() == 3 && v.dim() == 3);
  CHECK_INPUT(k.sizes() == v.sizes() && q.size(2) == k.size(2));
  CHECK_INPUT(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type());
  CHECK_INPUT(q.get_device() == k.get_device() && q.get_device() == v.get_device());
  b200c_attention_t &a = t.a;
  a.dtype = dtype_code(q, "attention");
  TORCH_CHECK(q.size(2) >= 1 && q.size(2) <= 128, "attention covers 1 to 128 channels per head, got ", q.size(2));
  TORCH_CHECK(k.size(1) >= 1 && q.size(1) >= 1 && q.size(1) % k.size(1) == 0 && q.size(1) <= 1024,
              "the heads of q must be a multiple of the heads of k and v, at most 1024");
  t.q = rows_of(q);
  t.k = rows_of(k);
  t.v = rows_of(v);
  a.q = t.q.data_ptr();
  a.k = t.k.data_ptr();
  a.v = t.v.data_ptr();
  a.q_row = t.q.stride(0), a.q_head = t.q.stride(1);
  a.k_row = t.k.stride(0), a.k_head = t.k.stride(1);
  a.v_row = t.v.stride(0), a.v_head = t.v.stride(1);
  a.m = q.size(0), a.n = k.size(0);
  a.heads = (int)q.size(1), a.groups = (int)k.size(1), a.channels = (int)q.size(2);
  a.scale = (float)scale, a.cap = (float)cap;
  TORCH_CHECK(std::isfinite(a.scale) && std::isfinite(a.cap) && (cap > 0) == (a.cap > 0),
              "scale and cap must be finite numbers of 32 bits");
  a.num_segments = 1;
  CHECK_INPUT(ptr_q.has_value() == ptr_k.has_value());
  if (ptr_q.has_value()) {
    t.ptr_q = ptr_q.value().contiguous();
    t.ptr_k = ptr_k.value().contiguous();
    CHECK_INPUT(t.ptr_q.is_cuda() && t.ptr_k.is_cuda() && t.ptr_q.get_device() == q.get_device() &&
                t.ptr_k.get_device() == q.get_device());
    CHECK_INPUT(t.ptr_q.dim() == 1 && t.ptr_k.dim() == 1 && t.ptr_q.numel() == t.ptr_k.numel() && t.ptr_q.numel() >= 2);
    TORCH_CHECK(t.ptr_q.scalar_type() == at::kLong && t.ptr_k.scalar_type() == at::kLong,
                "ptr_q and ptr_k must be int64 tensors");
    a.ptr_q = t.ptr_q.data_ptr<int64_t>();
    a.ptr_k = t.ptr_k.data_ptr<int64_t>();
    a.num_segments = t.ptr_q.numel() - 1;
  }
  CHECK_INPUT(pos_q.has_value() == pos_k.has_value() && pos_q.has_value() == slope.has_value());
  if (pos_q.has_value()) {
    t.pos_q = pos_q.value().contiguous();
    t.pos_k = pos_k.value().contiguous();
    t.slope = slope.value().contiguous();
    for (const auto &p : {t.pos_q, t.pos_k, t.slope})
      CHECK_INPUT(p.is_cuda() && p.get_device() == q.get_device() && p.scalar_type() == at::kFloat);
    CHECK_INPUT(t.pos_q.dim() == 2 && t.pos_k.dim() == 2 && t.pos_q.size(0) == a.m && t.pos_k.size(0) == a.n &&
                t.pos_q.size(1) == t.pos_k.size(1));
    TORCH_CHECK(t.pos_q.size(1) >= 1 && t.pos_q.size(1) <= 8, "1 to 8 coordinates are supported");
    CHECK_INPUT(t.slope.dim() == 1 && t.slope.size(0) == a.heads);
    a.dims = (int)t.pos_q.size(1);
    a.pos_q = t.pos_q.data_ptr<float>();
    a.pos_k = t.pos_k.data_ptr<float>();
    a.slope = t.slope.data_ptr<float>();
  }
}

// training: also the statistics and, for 16-bit types, what rounding took from the output
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> attention_forward(
    torch::Tensor q, torch::Tensor k, torch::Tensor v, OptTensor ptr_q, OptTensor ptr_k, OptTensor pos_q,
    OptTensor pos_k, OptTensor slope, double scale, double cap, bool training) {
  OpRange range("torch_cluster::attention_forward");
  CHECK_CUDA(q);
  c10::cuda::CUDAGuard guard(q.device());
  check_waits();
  Attention t;
  prepare_attention(t, q, k, v, ptr_q, ptr_k, pos_q, pos_k, slope, scale, cap);
  auto out = torch::empty(q.sizes(), q.options());
  auto lse = torch::empty({training ? t.a.heads : 0, t.a.m}, q.options().dtype(torch::kFloat));
  const bool keep = training && t.a.dtype != B200C_F32;
  auto rest = keep ? torch::empty(q.sizes(), q.options()) : torch::empty({0}, q.options());
  const size_t bytes = b200c_attention_workspace_bytes(&t.a);
  auto ws = workspace(bytes, q);
  check_status(b200c_attention_forward(&t.a, out.data_ptr(), keep ? rest.data_ptr() : nullptr,
                                       training ? lse.data_ptr<float>() : nullptr,
                                       bytes ? ws.data_ptr() : nullptr, bytes,
                                       at::cuda::getCurrentCUDAStream().stream()));
  return {out, rest, lse};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> attention_backward(
    torch::Tensor dout, torch::Tensor q, torch::Tensor k, torch::Tensor v, torch::Tensor out, torch::Tensor rest,
    torch::Tensor lse, OptTensor ptr_q, OptTensor ptr_k, OptTensor pos_q, OptTensor pos_k, OptTensor slope, double scale,
    double cap, bool need_q, bool need_kv) {
  OpRange range("torch_cluster::attention_backward");
  at::NoGradGuard no_grad;
  CHECK_CUDA(q);
  c10::cuda::CUDAGuard guard(q.device());
  check_waits();
  Attention t;
  prepare_attention(t, q, k, v, ptr_q, ptr_k, pos_q, pos_k, slope, scale, cap);
  CHECK_INPUT(dout.sizes() == q.sizes() && out.sizes() == q.sizes() && dout.scalar_type() == q.scalar_type() &&
              out.scalar_type() == q.scalar_type() && dout.device() == q.device() && out.device() == q.device());
  CHECK_INPUT(lse.device() == q.device() && lse.scalar_type() == at::kFloat && lse.dim() == 2 &&
              lse.size(0) == q.size(1) && lse.size(1) == q.size(0));
  dout = dout.contiguous();
  out = out.contiguous();
  lse = lse.contiguous();
  const bool kept = rest.numel() > 0;
  CHECK_INPUT(!kept ||
              (rest.sizes() == q.sizes() && rest.scalar_type() == q.scalar_type() && rest.device() == q.device()));
  rest = rest.contiguous();
  auto none = torch::empty({0}, q.options());
  auto dq = need_q ? torch::empty(q.sizes(), q.options()) : none;
  auto dk = need_kv ? torch::empty(k.sizes(), k.options()) : none;
  auto dv = need_kv ? torch::empty(v.sizes(), v.options()) : none;
  const size_t bytes = b200c_attention_backward_workspace_bytes(&t.a);
  auto ws = workspace(bytes, q);
  check_status(b200c_attention_backward(&t.a, out.data_ptr(), kept ? rest.data_ptr() : nullptr, lse.data_ptr<float>(),
                                        dout.data_ptr(), need_q ? dq.data_ptr() : nullptr, need_kv ? dk.data_ptr() : nullptr,
                                        need_kv ? dv.data_ptr() : nullptr, bytes ? ws.data_ptr() : nullptr, bytes,
                                        at::cuda::getCurrentCUDAStream().stream()));
  return {dq, dk, dv};
}

struct SoftmaxAttention : torch::autograd::Function<SoftmaxAttention> {
  static torch::Tensor forward(AutogradContext *ctx, torch::Tensor q, torch::Tensor k, torch::Tensor v, OptTensor ptr_q,
                               OptTensor ptr_k, OptTensor pos_q, OptTensor pos_k, OptTensor slope, double scale,
                               double cap) {
    auto [out, rest, lse] = attention_forward(q, k, v, ptr_q, ptr_k, pos_q, pos_k, slope, scale, cap, true);
    ctx->save_for_backward({q, k, v, out, rest, lse, or_undefined(ptr_q), or_undefined(ptr_k), or_undefined(pos_q),
                            or_undefined(pos_k), or_undefined(slope)});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["cap"] = cap;
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto t = ctx->get_saved_variables();
    const bool need_q = ctx->needs_input_grad(0), need_k = ctx->needs_input_grad(1), need_v = ctx->needs_input_grad(2);
    auto [dq, dk, dv] = attention_backward(grads[0], t[0], t[1], t[2], t[3], t[4], t[5], or_none(t[6]), or_none(t[7]),
                                           or_none(t[8]), or_none(t[9]), or_none(t[10]),
                                           ctx->saved_data["scale"].toDouble(), ctx->saved_data["cap"].toDouble(),
                                           need_q, need_k || need_v);
    variable_list result(10);
    if (need_q) result[0] = dq;
    if (need_k) result[1] = dk;
    if (need_v) result[2] = dv;
    return once(result, {grads[0], t[0], t[1], t[2]});
  }
};

torch::Tensor attention(torch::Tensor q, torch::Tensor k, torch::Tensor v, OptTensor ptr_q, OptTensor ptr_k,
                        OptTensor pos_q, OptTensor pos_k, OptTensor slope, double scale, double cap) {
  const torch::Tensor pq = or_undefined(pos_q), pk = or_undefined(pos_k), sl = or_undefined(slope);
  refuse_tangents("attention", {&q, &k, &v, &pq, &pk, &sl});
  if (wants_gradient({&q, &k, &v}))
    return SoftmaxAttention::apply(q, k, v, ptr_q, ptr_k, pos_q, pos_k, slope, scale, cap);
  return std::get<0>(attention_forward(q, k, v, ptr_q, ptr_k, pos_q, pos_k, slope, scale, cap, false));
}

}  // namespace

static auto registry = torch::RegisterOperators()
                           .op("torch_cluster::gather_rows", &gather_rows)
                           .op("torch_cluster::norm_rotate", &norm_rotate)
                           .op("torch_cluster::attention", &attention);
