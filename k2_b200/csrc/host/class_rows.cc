// Scores of given classes and distillation from a teacher's top classes on torch tensors: checks
// of arguments, layouts, outputs, and one node each of torch's autograd graph.  Nothing here
// computes; the work is k2b200_token_scores* and k2b200_distillation* (include/k2b200.h).
#include "class_rows.h"

#include <ATen/SavedTensorHooks.h>
#include <ATen/core/DimVector.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <cmath>
#include <mutex>
#include <string>
#include <vector>

#include "../../../include/k2b200.h"
#include "node_name.h"

namespace py = pybind11;

namespace {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

void Check(int32_t status) {
  if (status != 0) throw std::runtime_error(k2b200_last_error());
}

// Arguments are refused as the Python layer does it: with an AssertionError.
void Require(bool ok, const char *what) {
  if (ok) return;
  PyErr_SetString(PyExc_AssertionError, what);
  throw py::error_already_set();
}

void RequireCuda(const at::Tensor &t, const char *what) {
  if (!t.is_cuda())
    throw std::runtime_error(std::string(what) +
                             " must be a CUDA tensor: k2_b200 runs on sm_100a only and has no "
                             "CPU path");
}

// at::empty on the device without the way through the dispatcher (0.6 of 1.3 us each; a call has up
// to five).
at::Tensor NewOn(at::IntArrayRef sizes, at::ScalarType type, at::Device device) {
  return at::detail::empty_cuda(sizes, type, device, c10::nullopt);
}

int32_t FloatType(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return K2B200_F32;
    case at::kHalf: return K2B200_F16;
    case at::kBFloat16: return K2B200_BF16;
    default: return -1;
  }
}

// Dimensions [from, to) of a tensor as one: its stride in elements, or false where there is none.
bool OneStride(const at::Tensor &t, int64_t from, int64_t to, int64_t *stride) {
  bool any = false;
  int64_t expect = 0;
  *stride = 0;
  if (t.numel() == 0) return true;  // (nothing is read by it)
  for (int64_t d = to; d-- > from;) {
    if (t.size(d) == 1) continue;
    if (!any) {
      *stride = t.stride(d);
      any = true;
    } else if (t.stride(d) != expect) {
      return false;
    }
    expect = t.stride(d) * t.size(d);
  }
  return true;
}

int64_t SizeOf(const at::Tensor &t, int64_t from, int64_t to) {
  int64_t n = 1;
  for (int64_t d = from; d < to; ++d) n *= t.size(d);
  return n;
}

// A tensor as adjacent numbers: itself, or a copy.
at::Tensor Plain(const at::Tensor &t) { return (t.is_neg() ? t.resolve_neg() : t).contiguous(); }

// What a node keeps of a tensor between the passes: hooks of the caller may hold it elsewhere, so
// that nothing else here may.  It may come back with other strides, but is read as what it was.
class Saved {
 public:
  void Keep(const at::Tensor &t) {
    // (a teacher's of inference mode have no version that torch could compare: a copy)
    variable_ = SavedVariable(t.is_inference() ? t.clone() : t, false);
    sizes_ = at::DimVector(t.sizes());
    type_ = t.scalar_type();
    device_ = t.device();
    there_ = true;
  }
  bool there() const { return there_; }
  at::Device device() const { return device_; }
  at::Tensor Get() const {
    const at::Tensor t = variable_.unpack();
    TORCH_CHECK(t.defined() && t.layout() == at::kStrided && t.sizes() == at::IntArrayRef(sizes_) &&
                    t.scalar_type() == type_ && t.device() == device_,
                "hooks gave back a saved tensor of other sizes, type or device than they got");
    return t;
  }
  void Release() { variable_.reset_data(); }

 private:
  SavedVariable variable_;
  at::DimVector sizes_;
  at::ScalarType type_ = at::kFloat;
  at::Device device_ = at::kCPU;
  bool there_ = false;
};

// k2b200_class_rows of a tensor of scores, and what it points to.  The rows are the dimensions
// before the last, the first `split` of them the outer ones.
struct RowsOf {
  k2b200_class_rows rows{};
  at::Tensor scores, lengths;
  int64_t split = 0;
};

// Scores of adjacent classes whose rows lie at two strides are read in place, others are copied.
// (what is refused here, with Python's lock held, cannot come up in a backward pass, which has no such
// lock: Saved gives back sizes, types and devices that have been through here)
RowsOf MakeRows(const at::Tensor &scores, const c10::optional<at::Tensor> &lengths) {
  RequireCuda(scores, "logits");
  Require(scores.dim() >= 1 && FloatType(scores) >= 0,
          "logits must be [..., classes] of float32, float16 or bfloat16");
  Require(scores.size(-1) >= 1 && scores.size(-1) <= ((int64_t)1 << 30),
          "logits must have 1 to 2^30 classes");
  const int64_t lead = scores.dim() - 1;
  RowsOf r;
  r.scores = scores.is_neg() ? scores.resolve_neg() : scores;
  int64_t outer_stride = 0, inner_stride = 0;
  const auto splits = [&](int64_t s) {
    return OneStride(r.scores, 0, s, &outer_stride) &&
           OneStride(r.scores, s, lead, &inner_stride);
  };
  bool ok = r.scores.size(-1) == 1 || r.scores.stride(-1) == 1;
  if (lengths.has_value()) {
    Require(scores.dim() == 3, "lengths go with logits of [sequences, frames, classes]");
    r.split = 1;
    ok = ok && splits(1);
  } else if (ok) {
    for (ok = false, r.split = 0; r.split <= lead; ++r.split)
      if ((ok = splits(r.split))) break;
  }
  if (!ok) {
    r.scores = r.scores.contiguous();
    if (!lengths.has_value()) r.split = 0;
    splits(r.split);
  }
  r.rows.scores = r.scores.data_ptr();
  r.rows.type = FloatType(scores);
  r.rows.num_classes = (int32_t)scores.size(-1);
  r.rows.outer = SizeOf(scores, 0, r.split);
  r.rows.inner = SizeOf(scores, r.split, lead);
  Require(r.rows.outer < ((int64_t)1 << 28) && r.rows.inner < ((int64_t)1 << 28) &&
              r.rows.outer * r.rows.inner < ((int64_t)1 << 28),
          "logits must have fewer than 2^28 rows");
  r.rows.outer_stride = outer_stride;
  r.rows.inner_stride = inner_stride;
  if (lengths.has_value()) {
    const at::Tensor &l = *lengths;
    Require(l.dim() == 1 && l.size(0) == scores.size(0) &&
                (l.scalar_type() == at::kInt || l.scalar_type() == at::kLong),
            "lengths must be one int32 or int64 per sequence");
    Require(l.device() == scores.device() || l.is_cpu(),
            "lengths must be on the CPU or on the device of the logits");
    if (l.is_cpu()) {
      // as kernel parameters: the stream is not waited for
      const at::Tensor host = l.clamp(0, scores.size(1)).to(at::kInt).contiguous();
      r.lengths = NewOn({l.size(0)}, at::kInt, scores.device());
      if (l.size(0) > 0)
        Check(k2b200_upload_i32(
            host.data_ptr<int32_t>(), l.size(0), r.lengths.data_ptr<int32_t>(),
            c10::cuda::getCurrentCUDAStream(scores.device().index()).stream()));
    } else {
      r.lengths = Plain(l);
    }
    // (an address even where there are no sequences: lengths are given)
    r.rows.lengths = r.lengths.data_ptr();
    r.rows.lengths_64 = r.lengths.scalar_type() == at::kLong;
  }
  return r;
}

// Whole numbers of the rows, adjacent.
at::Tensor Classes(const at::Tensor &t, const RowsOf &r, const char *what) {
  Require(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, what);
  RequireCuda(t, "tokens");
  Require(t.device() == r.scores.device(), "tokens must be on the device of the logits");
  return Plain(t);
}

bool LeadingSizesAre(const at::Tensor &t, const at::Tensor &scores, int64_t more) {
  return t.dim() == scores.dim() - 1 + more &&
         t.sizes().slice(0, scores.dim() - 1) == scores.sizes().slice(0, scores.dim() - 1);
}

// The gradient of the scores: with their strides, where they fill their storage.
at::Tensor GradLike(const at::Tensor &scores) {
  return at::empty_like(scores, scores.options(), at::MemoryFormat::Preserve);
}

// Upstream gradients as the kernels read them: any strides that the rows' split allows.
k2b200_row_grad RowGrad(at::Tensor &g, const RowsOf &r, bool top) {
  k2b200_row_grad out{};
  if (!g.defined()) return out;
  if (g.scalar_type() != at::kFloat) g = g.to(at::kFloat);
  if (g.is_neg()) g = g.resolve_neg();
  const int64_t lead = r.scores.dim() - 1;
  if (!OneStride(g, 0, r.split, &out.outer) || !OneStride(g, r.split, lead, &out.inner)) {
    g = g.contiguous();
    OneStride(g, 0, r.split, &out.outer);
    OneStride(g, r.split, lead, &out.inner);
  }
  if (top && g.size(-1) > 1) out.top = g.stride(-1);
  out.grad = g.data_ptr<float>();
  return out;
}

// Strides of a gradient that GradLike made.
void GradStrides(const at::Tensor &grad, const RowsOf &r, int64_t *outer, int64_t *inner) {
  const int64_t lead = grad.dim() - 1;
  TORCH_CHECK((grad.size(-1) == 1 || grad.stride(-1) == 1) &&
                  OneStride(grad, 0, r.split, outer) && OneStride(grad, r.split, lead, inner),
              "no strides for the gradient");
}

// A gradient whose rows lie at two strides.
at::Tensor NewGrad(const RowsOf &r) {
  at::Tensor grad = GradLike(r.scores);
  int64_t stride;
  const int64_t lead = grad.dim() - 1;
  if ((grad.size(-1) > 1 && grad.stride(-1) != 1) || !OneStride(grad, 0, r.split, &stride) ||
      !OneStride(grad, r.split, lead, &stride))
    grad = at::empty(r.scores.sizes(), r.scores.options());
  return grad;
}

// The norm of a forward pass, which is read in vectors of 16 bytes.
at::Tensor NormOf(const Saved &norm) {
  const at::Tensor t = Plain(norm.Get());
  return (uintptr_t)t.data_ptr() % 16 == 0 ? t : t.clone();
}

c10::optional<at::Tensor> LengthsOf(const Saved &lengths) {
  return lengths.there() ? c10::optional<at::Tensor>(lengths.Get()) : c10::nullopt;
}

void RefuseForwardMode(const at::Tensor &t) {
  TORCH_CHECK(!t._fw_grad(0).defined(), "k2_b200 has no forward-mode derivatives");
}

// (a gradient without a graph of its own would be taken for a constant)
void RefuseSecondOrder() {
  TORCH_CHECK(!at::GradMode::is_enabled(),
              "k2_b200 has no derivatives of second order (create_graph=True)");
}

// The capture that a stream is in, 0 for none.
unsigned long long CaptureOf(cudaStream_t stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(stream, &status, &id) != cudaSuccess) {
    cudaGetLastError();  // (the legacy stream, while another one is captured)
    return 0;
  }
  return status == cudaStreamCaptureStatusNone ? 0 : id;
}

// A leaf's gradient is added on the stream on which its first graph was made.  If that is the default
// one, which no capture can wait for, a captured backward pass would break its capture there, in a
// thread of torch's that ends the process.
void RefuseLeafOfDefaultStream(const torch::autograd::Node &node, cudaStream_t stream) {
  if (CaptureOf(stream) == 0) return;
  for (const auto &edge : node.next_edges()) {
    const auto leaf = dynamic_cast<torch::autograd::AccumulateGrad *>(edge.function.get());
    if (leaf == nullptr) continue;
    const auto its = leaf->stream();
    TORCH_CHECK(!its.has_value() || c10::cuda::CUDAStream(*its) !=
                                        c10::cuda::getDefaultCUDAStream(its->device_index()),
                "a backward pass cannot be captured while another graph of the same logits lives "
                "that was made on the default stream: delete what holds it, or make it on another "
                "stream");
  }
}

// ---------------------------------------------------------------------------
// token_log_probs
// ---------------------------------------------------------------------------
struct TokenNode : public torch::autograd::Node {
  Saved scores, lengths, tokens, top, norm;
  int32_t top_k = 0;
  // which output the gradients arrive for
  int32_t log_probs_at = -1, entropy_at = -1, top_at = -1;
  bool released = false;

  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(1);
    RefuseSecondOrder();
    at::Tensor g_log_probs, g_entropy, g_top;
    if (log_probs_at >= 0) g_log_probs = grads[log_probs_at];
    if (entropy_at >= 0) g_entropy = grads[entropy_at];
    if (top_at >= 0) g_top = grads[top_at];
    if (!g_log_probs.defined() && !g_entropy.defined() && !g_top.defined()) return out;
    TORCH_CHECK(!released,
                "the scores were already differentiated and their buffers freed "
                "(retain_graph=True keeps them)");
    if (!task_should_compute_output(0)) return out;
    // (hooks run here, under no guard of ours)
    const at::Tensor x = scores.Get();
    const c10::optional<at::Tensor> l = LengthsOf(lengths);
    at::Tensor given = g_log_probs.defined() ? tokens.Get() : at::Tensor(),
               classes = g_top.defined() ? top.Get() : at::Tensor();
    const at::Device device = scores.device();
    c10::cuda::CUDAGuard guard(device);
    at::AutoDispatchBelowADInplaceOrView below_autograd;
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    RefuseLeafOfDefaultStream(*this, stream);
    const RowsOf r = MakeRows(x, l);
    const at::Tensor n = NormOf(norm);
    if (given.defined()) given = Plain(given);
    if (classes.defined()) classes = Plain(classes);
    const k2b200_row_grad a = RowGrad(g_log_probs, r, false), b = RowGrad(g_entropy, r, false),
                          c = RowGrad(g_top, r, true);
    out[0] = NewGrad(r);
    int64_t outer = 0, inner = 0;
    GradStrides(out[0], r, &outer, &inner);
    Check(k2b200_token_scores_backward(
        &r.rows, given.defined() ? given.data_ptr() : nullptr,
        given.defined() && given.scalar_type() == at::kLong, top_k,
        classes.defined() ? classes.data_ptr<int32_t>() : nullptr, n.data_ptr<float>(), &a, &b,
        &c, out[0].data_ptr(), outer, inner, stream));
    return out;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    released = true;
    for (Saved *t : {&scores, &lengths, &tokens, &top, &norm}) t->Release();
  }
};

py::tuple TokenLogProbs(const at::Tensor &scores, const c10::optional<at::Tensor> &given,
                        int64_t top_k, bool want_entropy,
                        const c10::optional<at::Tensor> &lengths) {
  RequireCuda(scores, "logits");
  const at::Device device = scores.device();
  c10::cuda::CUDAGuard guard(device);
  RefuseForwardMode(scores);
  const bool graded = torch::autograd::compute_requires_grad(scores);
  at::Tensor log_probs, entropy, top_log_probs, top_tokens, tokens, norm;
  RowsOf r;
  {
    at::AutoDispatchBelowADInplaceOrView below_autograd;
    r = MakeRows(scores, lengths);
    Require(top_k >= 0 && top_k <= K2B200_MAX_TOP && top_k <= scores.size(-1),
            "top_k must be 0 to 128, and at most the number of classes");
    Require(given.has_value() || top_k > 0 || want_entropy,
            "nothing is asked for: give tokens, top_k or entropy");
    if (given.has_value()) {
      Require(LeadingSizesAre(*given, scores, 0), "tokens must have the shape of logits[..., 0]");
      tokens = Classes(*given, r, "tokens must be int32 or int64");
    }
    const auto lead = scores.sizes().slice(0, scores.dim() - 1);
    std::vector<int64_t> lead_top(lead.begin(), lead.end());
    lead_top.push_back(top_k);
    if (tokens.defined()) log_probs = NewOn(lead, at::kFloat, device);
    if (want_entropy) entropy = NewOn(lead, at::kFloat, device);
    if (top_k > 0) {
      top_log_probs = NewOn(lead_top, at::kFloat, device);
      top_tokens = NewOn(lead_top, at::kInt, device);
    }
    if (graded) norm = NewOn({r.rows.outer * r.rows.inner, 4}, at::kFloat, device);
    const auto floats = [](at::Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    Check(k2b200_token_scores(&r.rows, tokens.defined() ? tokens.data_ptr() : nullptr,
                              tokens.defined() && tokens.scalar_type() == at::kLong,
                              (int32_t)top_k, floats(log_probs), floats(entropy),
                              floats(top_log_probs),
                              top_tokens.defined() ? top_tokens.data_ptr<int32_t>() : nullptr,
                              floats(norm), stream));
  }
  if (graded) {
    const std::shared_ptr<TokenNode> node(new TokenNode(), torch::autograd::deleteNode);
    node->scores.Keep(r.scores);
    if (r.lengths.defined()) node->lengths.Keep(r.lengths);
    if (tokens.defined()) node->tokens.Keep(tokens);
    if (top_k > 0) node->top.Keep(top_tokens);
    node->norm.Keep(norm);
    node->top_k = (int32_t)top_k;
    node->set_next_edges(torch::autograd::collect_next_edges(scores));
    int32_t k = 0;
    for (auto [t, at] : {std::pair{&log_probs, &node->log_probs_at},
                         std::pair{&entropy, &node->entropy_at},
                         std::pair{&top_log_probs, &node->top_at}}) {
      if (!t->defined()) continue;
      torch::autograd::set_history(*t, node);
      *at = k++;
    }
  }
  const auto give = [](const at::Tensor &t) -> py::object {
    return t.defined() ? py::cast(t) : py::none();
  };
  return py::make_tuple(give(log_probs), give(entropy), give(top_log_probs), give(top_tokens));
}

// ---------------------------------------------------------------------------
// distillation_loss
// ---------------------------------------------------------------------------
struct DistilNode : public torch::autograd::Node {
  Saved scores, lengths, tokens, teacher_scores, norm;
  k2b200_teacher teacher{};
  at::Tensor workspace, ready;  // ready: for an upstream of 1
  unsigned long long capture = 0;  // that the forward pass was in
  bool released = false;

  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(1);
    at::Tensor g = grads[0];
    if (!g.defined()) return out;
    RefuseSecondOrder();
    TORCH_CHECK(!released,
                "the loss was already differentiated and its buffers freed (retain_graph=True "
                "keeps them)");
    if (!task_should_compute_output(0)) return out;
    // (hooks run here, under no guard of ours)
    const at::Tensor x = scores.Get();
    const c10::optional<at::Tensor> l = LengthsOf(lengths);
    at::Tensor classes = tokens.Get(), of_teacher = teacher_scores.Get();
    const at::Device device = scores.device();
    c10::cuda::CUDAGuard guard(device);
    at::AutoDispatchBelowADInplaceOrView below_autograd;
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    RefuseLeafOfDefaultStream(*this, stream);
    const RowsOf r = MakeRows(x, l);
    const at::Tensor n = NormOf(norm);
    classes = Plain(classes);
    of_teacher = Plain(of_teacher);
    k2b200_teacher t = teacher;
    t.tokens = classes.data_ptr();
    t.scores = of_teacher.data_ptr();
    k2b200_row_grad up{};
    if (t.reduction == 0) {
      up = RowGrad(g, r, false);
    } else {
      if (g.scalar_type() != at::kFloat) g = g.to(at::kFloat);
      if (g.is_neg()) g = g.resolve_neg();
      up.grad = g.data_ptr<float>();
    }
    // What the forward pass made is given away once: whoever gets it may add to it.  And only if
    // both passes are in one capture, or neither is in any: a forward pass that is replayed by
    // itself would write to the gradient of an earlier one, and a backward pass would find there
    // what its last replay left.
    const bool made = ready.defined() && capture == CaptureOf(stream);
    out[0] = made ? std::move(ready) : NewGrad(r);
    if (made) ready = at::Tensor();
    int64_t outer = 0, inner = 0;
    GradStrides(out[0], r, &outer, &inner);
    const bool work = workspace.defined();
    Check(k2b200_distillation_backward(
        &r.rows, &t, n.data_ptr<float>(), &up, made, out[0].data_ptr(), outer, inner,
        work ? workspace.data_ptr() : nullptr, work ? (size_t)workspace.numel() : 0, stream));
    return out;
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    released = true;
    for (Saved *t : {&scores, &lengths, &tokens, &teacher_scores, &norm}) t->Release();
    workspace.reset();
    ready.reset();
  }
};

at::Tensor DistillationLoss(const at::Tensor &scores, const at::Tensor &teacher_tokens,
                            const at::Tensor &teacher_log_probs, double temperature,
                            double weight, const std::string &reduction,
                            const c10::optional<at::Tensor> &lengths) {
  RequireCuda(scores, "logits");
  const at::Device device = scores.device();
  c10::cuda::CUDAGuard guard(device);
  RefuseForwardMode(scores);
  RefuseForwardMode(teacher_log_probs);
  const bool graded = torch::autograd::compute_requires_grad(scores);
  at::Tensor loss, tokens, teacher_scores, workspace, norm, ready;
  RowsOf r;
  k2b200_teacher t{};
  unsigned long long capture = 0;
  {
    at::AutoDispatchBelowADInplaceOrView below_autograd;
    r = MakeRows(scores, lengths);
    t.reduction = reduction == "none" ? 0 : reduction == "sum" ? 1 : reduction == "mean" ? 2 : -1;
    Require(t.reduction >= 0, "reduction must be \"none\", \"sum\" or \"mean\"");
    // (1e-6 to 1e6 as float32: beyond them the scaled scores overflow)
    Require(temperature >= 1e-6 && temperature <= 1e6, "temperature must be 1e-6 to 1e6");
    Require(std::isfinite((float)weight), "weight must be finite");
    Require(LeadingSizesAre(teacher_tokens, scores, 1),
            "teacher_tokens must be [..., entries] over the rows of the logits");
    const int64_t entries = teacher_tokens.size(-1);
    Require(entries >= 1 && entries <= K2B200_MAX_TOP, "a teacher has 1 to 128 entries per row");
    tokens = Classes(teacher_tokens, r, "teacher_tokens must be int32 or int64");
    Require(teacher_log_probs.sizes() == teacher_tokens.sizes() &&
                FloatType(teacher_log_probs) >= 0,
            "teacher_log_probs must be float32, float16 or bfloat16 of the shape of "
            "teacher_tokens");
    RequireCuda(teacher_log_probs, "teacher_log_probs");
    Require(teacher_log_probs.device() == device,
            "teacher_log_probs must be on the device of the logits");
    // (a silent zero is what a caller who wants that derivative would get)
    Require(!(at::GradMode::is_enabled() && teacher_log_probs.requires_grad()),
            "no gradient goes to teacher_log_probs: detach them");
    teacher_scores = Plain(teacher_log_probs);
    t.tokens = tokens.data_ptr();
    t.tokens_64 = tokens.scalar_type() == at::kLong;
    t.scores = teacher_scores.data_ptr();
    t.type = FloatType(teacher_scores);
    t.entries = (int32_t)entries;
    t.temperature = (float)temperature;
    t.weight = (float)weight;
    const int64_t num = r.rows.outer * r.rows.inner;
    // (rows' own losses need none)
    const size_t bytes = t.reduction == 0 ? 0 : k2b200_distillation_workspace_bytes(&r.rows);
    if (bytes > 0) workspace = NewOn({(int64_t)bytes}, at::kByte, device);
    void *const work = bytes > 0 ? workspace.data_ptr() : nullptr;
    if (graded) norm = NewOn({num, 4}, at::kFloat, device);
    int64_t outer = 0, inner = 0;
    // (whoever has hooks wants nothing large kept between the passes)
    if (graded && t.reduction != 0 && !at::SavedTensorDefaultHooks::get_hooks().has_value()) {
      ready = NewGrad(r);
      GradStrides(ready, r, &outer, &inner);
    }
    loss = t.reduction == 0 ? NewOn(scores.sizes().slice(0, scores.dim() - 1), at::kFloat, device)
                            : NewOn({}, at::kFloat, device);
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
    Check(k2b200_distillation(&r.rows, &t, loss.data_ptr<float>(),
                              graded ? norm.data_ptr<float>() : nullptr,
                              ready.defined() ? ready.data_ptr() : nullptr, outer, inner,
                              work, bytes, stream));
    if (ready.defined()) capture = CaptureOf(stream);
  }
  if (graded) {
    const std::shared_ptr<DistilNode> node(new DistilNode(), torch::autograd::deleteNode);
    node->scores.Keep(r.scores);
    if (r.lengths.defined()) node->lengths.Keep(r.lengths);
    node->tokens.Keep(tokens);
    node->teacher_scores.Keep(teacher_scores);
    node->norm.Keep(norm);
    node->teacher = t;
    node->workspace = workspace;
    node->ready = ready;
    node->capture = capture;
    node->set_next_edges(torch::autograd::collect_next_edges(scores));
    torch::autograd::set_history(loss, node);
  }
  return loss;
}

}  // namespace

void BindClassRows(py::module_ &m) {
  NameNode<TokenNode>("_TokenLogProbsBackward");
  NameNode<DistilNode>("_DistillationLossBackward");
  m.def("token_log_probs", &TokenLogProbs);
  m.def("distillation_loss", &DistillationLoss);
}
