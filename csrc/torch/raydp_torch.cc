// Torch front end of the optimizer and routed-expert kernels (raydp_amd/ops/adamw.py, raydp_amd/ops/expert_ops.py).
//
// A step over hundreds of tensors, or a routed batch of a few thousand samples, takes the GPU tens of microseconds; walking
// the tensors and running the autograd nodes from Python took the host hundreds. Here a tensor costs the host about 0.1 us
// and a node's backward runs without the interpreter. What the callers documented and checked holds here: tensors are on one
// GPU, launches go to its current stream, and every failure is a C++ exception that becomes the Python error it names.
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/engine.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <unordered_set>
#include <vector>

#include "hip/adamw.h"
#include "hip/experts.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// Bytes of the last-level cache: what touches more is streamed past it. Row moves, 64 experts of 1024 bf16, two a sample:
// 65536 samples (384 MB) combine 76 -> 66 us; 24576 (144 MB) dispatch 24 -> 29. The AdamW steps' figures are at the kernel.
int64_t g_last_level = 256ll << 20;

void* current_stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void check(int rc, const char* what) {
  if (rc != 0) throw std::runtime_error(std::string(what) + " failed with HIP error code " + std::to_string(rc));
}

template <class T>
T* ptr(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}

// a kernel wrote t: autograd, and the towers that keep images of weights, go by its version
void written(const Tensor& t) {
  if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

bool bf16(const Tensor& t) { return t.scalar_type() == at::kBFloat16; }

// A trace keeps torch's operators: of a call here it would keep the allocation of the results and not what fills them.
void check_trace(const char* what) {
  if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY))
    throw std::runtime_error(std::string(what) + " cannot be traced on the GPU: the trace would miss the kernel's launch");
}

// Wrappers say that they are on the GPU and have no memory there, or not the values that stand in it.
void check_memory(const Tensor& t, const char* what) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet odd({DispatchKey::Python, DispatchKey::Functionalize, DispatchKey::FuncTorchBatched,
                                     DispatchKey::FuncTorchGradWrapper, DispatchKey::Batched, DispatchKey::ZeroTensor,
                                     DispatchKey::Negative, DispatchKey::Conjugate});
  if (t.defined() && t.key_set().has_any(odd))
    throw py::type_error(std::string(what) + ": a kernel cannot read a wrapped tensor (a fake or functional one, a transform's, "
                         "a subclass that dispatches, a lazy negation)");
}

// Is anything differentiated in forward mode at all? (Asked once for a list: a tensor's own answer costs 20 ns.)
bool tangents() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }

// A launch computes no tangent: the result would have none, without a word.
void check_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), what,
                              ": forward-mode derivatives are not implemented on the GPU");
}

// A backward of ours is not differentiable itself: under create_graph its results carry a node that says so.
variable_list once(variable_list out) {
  if (!at::GradMode::is_enabled()) return out;
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "this gradient is computed by a fused kernel and cannot be differentiated again", out.size());
  variable_list wanted;
  for (auto& t : out) wanted.push_back(t.defined() ? t.detach().requires_grad_() : t);
  variable_list named = (*node)(std::move(wanted));
  for (size_t i = 0; i < out.size(); ++i)
    if (!out[i].defined()) named[i] = Variable();
  return named;
}

bool capturing(c10::DeviceIndex device) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  check((int)hipStreamIsCapturing(c10::hip::getCurrentHIPStream(device).stream(), &status), "hipStreamIsCapturing");
  return status != hipStreamCaptureStatusNone;
}

// Called by a backward of ours. A node of an eager call runs on that call's stream, and a leaf's gradient node is one of them
// as long as anything holds the call's graph. The default stream can have no part in a capture: trying to ends the process.
// What the pass would reach of that kind is found here first, and the call refused.
void check_capturable(const Tensor& t) {
  if (!capturing(t.get_device())) return;
  using torch::autograd::Node;
  const auto self = torch::autograd::get_current_node();
  if (!self) return;
  // (by number: torch's nodes name the same streams as of device type cuda, these as of type hip)
  const auto plain = c10::hip::getDefaultHIPStream(t.get_device()).id();
  const auto* wanted = torch::autograd::get_current_graph_task_exec_info();     // empty: all are
  std::vector<Node*> todo{self.get()};
  std::unordered_set<Node*> seen{self.get()};
  while (!todo.empty()) {
    Node* node = todo.back();
    todo.pop_back();
    for (const auto& edge : node->next_edges()) {
      Node* next = edge.function.get();
      if (next == nullptr || !seen.insert(next).second) continue;
      todo.push_back(next);
      if (wanted != nullptr && !wanted->empty()) {
        const auto at = wanted->find(next);
        if (at == wanted->end() || !at->second.should_execute()) continue;
      }
      const auto stream = next->stream();
      if (stream && stream->id() == plain)
        throw std::runtime_error("a backward pass cannot be captured when it reaches " + next->name() + " of an eager call on "
                                 "the default stream: drop what that call returned first, or run it on a side stream");
    }
  }
}

// ------------------------------------------------------------------------------------------------ gradient norm
struct NormPlan {
  std::vector<NormArgs> launches;
  std::vector<int> grids;
  int npart = 0;
  int64_t bytes = 0;
};

NormPlan norm_plan(const std::vector<Tensor>& grads) {
  NormPlan plan;
  for (size_t k = 0; k < grads.size(); k += kNormMax) {
    plan.launches.emplace_back();
    NormArgs& a = plan.launches.back();
    a.n = (int)std::min<size_t>(kNormMax, grads.size() - k);
    int64_t at = 0;
    for (int j = 0; j < a.n; ++j) {
      const Tensor& g = grads[k + j];
      a.g[j] = g.data_ptr();
      a.last[j] = (uint16_t)((g.numel() - 1) % kNormChunk + 1 + (bf16(g) ? kNormBf16 : 0));
      plan.bytes += g.numel() * g.element_size();
      a.start[j] = (unsigned)at;
      at += (g.numel() + kNormChunk - 1) / kNormChunk;
    }
    if (at > 0xFFFFFFFFll) throw py::value_error("gradient norm: too many elements for one launch");
    a.start[a.n] = a.chunks = (unsigned)at;
    plan.grids.push_back((int)std::min<int64_t>(at, kNormGrid));
    plan.npart += plan.grids.back();
  }
  return plan;
}

void launch_norm(NormPlan& plan, double* part, void* stream) {
  for (size_t k = 0; k < plan.launches.size(); ++k) {
    plan.launches[k].part = part;
    check(rx_norm_part(&plan.launches[k], plan.grids[k], plan.bytes > g_last_level, stream), "rx_norm_part");
    part += plan.grids[k];
  }
}

// [first, last) bytes of tensors that a launch writes: two workgroups on the same elements would race
void check_overlap(std::vector<std::pair<uintptr_t, uintptr_t>>& spans, const char* what) {
  if (!std::is_sorted(spans.begin(), spans.end())) std::sort(spans.begin(), spans.end());
  for (size_t k = 1; k < spans.size(); ++k)
    if (spans[k].first < spans[k - 1].second) throw py::value_error(std::string(what) + " share memory");
}

// grads: checked here, dense in any order of dimensions; returns the norm
Tensor clip_grad_norm(const std::vector<Tensor>& all, double max_norm) {
  check_trace("clip_grad_norm_");
  const bool forward = tangents();
  std::vector<Tensor> grads;
  const auto dev = all.at(0).device();
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  for (const Tensor& g : all) {
    check_memory(g, "clip_grad_norm_");
    if (forward) check_tangent(g, "clip_grad_norm_");
    if (g.layout() != at::kStrided) throw py::value_error("clip_grad_norm_: sparse gradients are not supported");
    if (g.device() != dev)
      throw py::value_error("clip_grad_norm_: gradients on " + dev.str() + " and " + g.device().str());
    if (g.scalar_type() != at::kFloat && !bf16(g))
      throw py::type_error(std::string("clip_grad_norm_: gradient dtype ") + c10::toString(g.scalar_type()) + " (fp32 or bf16)");
    if (!g.is_non_overlapping_and_dense())
      throw py::value_error("clip_grad_norm_: gradients must be dense (no gaps, no broadcast dimensions)");
    if (g.numel() == 0) continue;
    grads.push_back(g);
    spans.emplace_back((uintptr_t)g.data_ptr(), (uintptr_t)g.data_ptr() + g.numel() * g.element_size());
  }
  check_overlap(spans, "clip_grad_norm_: gradients");
  const auto f32 = all[0].options().dtype(at::kFloat).layout(at::kStrided);
  if (grads.empty()) return at::zeros({}, f32);
  c10::DeviceGuard guard(dev);
  void* stream = current_stream(grads[0]);
  NormPlan plan = norm_plan(grads);
  Tensor part = at::empty({plan.npart}, f32.dtype(at::kDouble)), norm = at::empty({}, f32);
  launch_norm(plan, ptr<double>(part), stream);
  for (size_t k = 0; k < plan.launches.size(); ++k) {
    ScaleArgs s;
    s.t = plan.launches[k];
    s.t.part = ptr<double>(part);
    s.npart = plan.npart;
    s.pad_ = 0;
    s.max_norm = max_norm;
    s.norm = k == 0 ? ptr<float>(norm) : nullptr;
    check(rx_norm_scale(&s, (int)std::min<unsigned>(s.t.chunks, 2 * kNormGrid), plan.bytes > g_last_level, stream),
          "rx_norm_scale");
  }
  for (const Tensor& g : grads) written(g);
  return norm;
}

// ------------------------------------------------------------------------------------------------ AdamW
struct Slot {            // one live parameter of a step
  Tensor p, g, step, m, v, sc;
  int place;
  uint16_t* img;
};

struct Group {
  std::vector<Slot> live;
  double lr, b1, b2, eps, wd;
  const float* lr_dev;
  int bits;
  bool maximize;
};

Tensor state_tensor(py::dict& st, const char* name, const Tensor& p) {
  PyObject* o = PyDict_GetItemString(st.ptr(), name);
  if (o == nullptr || !THPVariable_Check(o))
    throw py::value_error(std::string("FusedAdamW: a parameter's state lacks ") + name);
  Tensor t = THPVariable_Unpack(o);
  if (t.device() != p.device()) {      // state that was loaded before the model was moved
    t = t.to(p.device());
    st[name] = t;
  }
  if (!t.is_contiguous()) throw py::value_error(std::string("FusedAdamW: state ") + name + " must be contiguous");
  return t;
}

// groups: [(parameters, gradients, states, places, images, options)]; images: {index: bf16 tensor}. max_norm < 0: no
// clipping. Returns the norm, or None without clipping.
c10::optional<Tensor> adamw_step(const py::list& groups, double max_norm, int64_t seed) {
  check_trace("FusedAdamW.step");
  const bool forward = tangents();
  std::vector<Group> all;
  std::vector<Tensor> grads;
  c10::optional<c10::Device> dev;
  int64_t touched = 0;
  size_t count = 0;
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  for (const auto& item : groups) {
    const py::tuple t = item.cast<py::tuple>();
    const auto params = t[0].cast<std::vector<Tensor>>(), gs = t[1].cast<std::vector<Tensor>>();
    const py::list states = t[2].cast<py::list>();
    const auto places = t[3].cast<std::vector<int>>();
    const py::dict images = t[4].cast<py::dict>(), o = t[5].cast<py::dict>();
    const bool with_images = images.size() > 0;
    Group grp;
    grp.bits = o["state_bits"].cast<int>();
    const py::tuple betas = py::tuple(o["betas"]);
    grp.b1 = betas[0].cast<double>();
    grp.b2 = betas[1].cast<double>();
    grp.eps = o["eps"].cast<double>();
    grp.wd = o["weight_decay"].cast<double>();
    grp.maximize = o["maximize"].cast<bool>();
    grp.lr_dev = nullptr;
    grp.lr = 0.0;
    const py::object lr = o["lr"];
    if (THPVariable_Check(lr.ptr())) {
      const Tensor l = THPVariable_Unpack(lr.ptr());
      check_memory(l, "FusedAdamW");
      if (!l.is_cuda()) {
        if (capturing(params[0].get_device()))
          throw std::runtime_error("FusedAdamW: a tensor lr on the host cannot be captured into a graph, whose replays would "
                                   "keep its value: put it on the parameters' device");
        grp.lr = l.item<double>();
      } else if (l.scalar_type() != at::kFloat || l.device() != params[0].device() || l.numel() != 1)
        throw py::type_error("FusedAdamW: a tensor lr must be one fp32 value on the parameters' device");
      else
        grp.lr_dev = ptr<float>(l);
    } else {
      grp.lr = lr.cast<double>();
    }
    for (size_t i = 0; i < params.size(); ++i) {
      Slot s;
      s.p = params[i];
      s.g = gs[i];
      s.place = places[i];
      s.img = nullptr;
      if (s.g.layout() != at::kStrided) throw std::runtime_error("FusedAdamW does not support sparse gradients");
      if (s.p.numel() == 0) continue;
      check_memory(s.p, "FusedAdamW");
      check_memory(s.g, "FusedAdamW");
      if (forward) check_tangent(s.g, "FusedAdamW");
      if (!dev) dev = s.p.device();
      if (s.p.device() != *dev || s.g.device() != *dev)
        throw py::value_error("FusedAdamW: parameters with gradients on " + dev->str() + " and " +
                              (s.p.device() != *dev ? s.p : s.g).device().str());
      if ((s.p.scalar_type() != at::kFloat && !bf16(s.p)) || s.g.scalar_type() != s.p.scalar_type())
        throw py::type_error(std::string("FusedAdamW: parameter ") + c10::toString(s.p.scalar_type()) + " with gradient " +
                             c10::toString(s.g.scalar_type()) + " (both fp32 or both bf16)");
      if (!s.p.is_contiguous()) throw py::value_error("FusedAdamW: parameters must be contiguous");
      if (s.g.numel() != s.p.numel()) throw py::value_error("FusedAdamW: a gradient has another size than its parameter");
      s.g = s.g.contiguous();
      py::dict st = states[i].cast<py::dict>();
      s.step = state_tensor(st, "step", s.p);
      s.m = state_tensor(st, "exp_avg", s.p);
      s.v = state_tensor(st, "exp_avg_sq", s.p);
      const auto kind = grp.bits == 8 ? at::kByte : at::kFloat;
      if (s.m.scalar_type() != kind || s.v.scalar_type() != kind || s.m.numel() != s.p.numel() || s.v.numel() != s.p.numel())
        throw py::value_error("FusedAdamW: state_bits is " + std::to_string(grp.bits) + ", the moments of a parameter of " +
                              std::to_string(s.p.numel()) + " elements are " + c10::toString(s.m.scalar_type()) + " of " +
                              std::to_string(s.m.numel()) + " and " + c10::toString(s.v.scalar_type()) + " of " +
                              std::to_string(s.v.numel()));
      if (s.step.scalar_type() != at::kFloat || s.step.numel() != 1)
        throw py::value_error("FusedAdamW: a step count must be one fp32 value");
      const uintptr_t low = (uintptr_t)s.m.data_ptr() | (uintptr_t)s.v.data_ptr();
      if (low & (grp.bits == 8 ? 3 : 15))
        throw py::value_error("FusedAdamW: moments must start at a multiple of 4 (8 bits) or 16 bytes");
      if (grp.bits == 8) {
        s.sc = state_tensor(st, "scales", s.p);
        if (s.sc.scalar_type() != at::kByte || s.sc.numel() != 2 * ((s.p.numel() + kAwBlock - 1) / kAwBlock) ||
            ((uintptr_t)s.sc.data_ptr() & 1))
          throw py::value_error("FusedAdamW: scales must be two bytes for each 256 elements, at an even address");
      }
      if (with_images && !bf16(s.p) && images.contains(py::int_(i))) {   // (a bf16 parameter is its own image)
        const Tensor img = images[py::int_(i)].cast<Tensor>();
        if (!bf16(img) || !img.is_contiguous() || img.numel() != s.p.numel() || img.device() != *dev)
          throw py::value_error("FusedAdamW: a weight's image must be contiguous bf16 of its size");
        s.img = ptr<uint16_t>(img);
      }
      touched += s.p.numel() * (2 * s.p.element_size() + grp.bits / 4);
      grads.push_back(s.g);
      spans.emplace_back((uintptr_t)s.p.data_ptr(), (uintptr_t)s.p.data_ptr() + s.p.numel() * s.p.element_size());
      grp.live.push_back(std::move(s));
    }
    // fp32 parameters first: a launch takes one type
    std::stable_sort(grp.live.begin(), grp.live.end(), [](const Slot& a, const Slot& b) { return bf16(a.p) < bf16(b.p); });
    count += grp.live.size();
    all.push_back(std::move(grp));
  }
  if (count == 0) return c10::nullopt;
  check_overlap(spans, "FusedAdamW: parameters");
  c10::DeviceGuard guard(*dev);
  void* stream = current_stream(grads[0]);
  NormPlan plan;
  if (max_norm >= 0.0) plan = norm_plan(grads);
  const auto opts = grads[0].options();
  Tensor ws = at::empty({(int64_t)(sizeof(AwTensor) * count + sizeof(AwHead) * all.size() + 8 * plan.npart)}, opts.dtype(at::kByte));
  AwTensor* tensors = ptr<AwTensor>(ws);
  AwHead* heads = reinterpret_cast<AwHead*>(tensors + count);
  double* part = reinterpret_cast<double*>(heads + all.size());
  Tensor norm;
  if (max_norm >= 0.0) {
    norm = at::empty({}, opts.dtype(at::kFloat));
    launch_norm(plan, part, stream);
  }
  int first = 0;
  for (size_t k = 0; k < all.size(); ++k) {
    Group& grp = all[k];
    const size_t n = grp.live.size();
    for (size_t j = 0; j < n; j += kAwPrepMax) {
      AwPrep a;
      a.n = (int)std::min<size_t>(kAwPrepMax, n - j);
      a.maximize = grp.maximize;
      a.npart = plan.npart;
      a.first = first + (int)j;
      a.lr = grp.lr;
      a.lr_dev = grp.lr_dev;
      a.wd = grp.wd;
      a.b1 = grp.b1;
      a.b2 = grp.b2;
      a.max_norm = max_norm >= 0.0 ? max_norm : -1.0;
      a.part = part;
      a.head = heads + k;
      a.tensors = tensors;
      a.norm = norm.defined() && a.first == 0 ? ptr<float>(norm) : nullptr;
      a.seed = (uint32_t)seed;
      a.pad_ = 0;
      for (int i = 0; i < a.n; ++i) {
        a.step[i] = ptr<float>(grp.live[j + i].step);
        a.ordinal[i] = grp.live[j + i].place;
      }
      check(rx_aw_prep(&a, stream), "rx_aw_prep");
    }
    for (size_t j = 0; j < n;) {
      AwStep a;
      const bool low = bf16(grp.live[j].p);
      a.n = 0;
      a.pad_ = 0;
      a.pad2_ = 0.f;
      a.b1 = (float)grp.b1;
      a.omb1 = (float)(1.0 - grp.b1);
      a.b2 = (float)grp.b2;
      a.omb2 = (float)(1.0 - grp.b2);
      a.eps = (float)grp.eps;
      a.head = heads + k;
      a.tensors = tensors + first + j;
      int64_t at = 0;
      for (; j < n && a.n < kAwMax && bf16(grp.live[j].p) == low; ++j, ++a.n) {
        const Slot& s = grp.live[j];
        a.p[a.n] = s.p.data_ptr();
        a.g[a.n] = s.g.data_ptr();
        a.m[a.n] = s.m.data_ptr();
        a.v[a.n] = s.v.data_ptr();
        a.sc[a.n] = grp.bits == 8 ? ptr<uint8_t>(s.sc) : nullptr;
        a.img[a.n] = s.img;
        a.len[a.n] = s.p.numel();
        a.start[a.n] = (unsigned)at;
        at += (s.p.numel() + kAwChunk - 1) / kAwChunk;
        if (at > 0x7FFFFFFFll) throw py::value_error("FusedAdamW: too many elements for one launch");
      }
      a.start[a.n] = (unsigned)at;
      check(rx_aw_step(&a, grp.bits, low, touched > g_last_level, stream), "rx_aw_step");
    }
    first += (int)n;
  }
  for (const Group& grp : all)
    for (const Slot& s : grp.live) written(s.p);
  if (!norm.defined()) return c10::nullopt;
  return norm;
}

std::vector<Tensor> decode_moments(const Tensor& m, const Tensor& v, const Tensor& sc, bool to_bf16) {
  check_trace("decode_moments");
  for (const Tensor& t : {m, v, sc}) check_memory(t, "decode_moments");
  const auto kind = to_bf16 ? at::kBFloat16 : at::kFloat;
  Tensor mo = at::empty(m.sizes(), m.options().dtype(kind)), vo = at::empty(m.sizes(), m.options().dtype(kind));
  if (m.numel()) {
    c10::DeviceGuard guard(m.device());
    // (to bf16: 16 M, 96 MB, take 16 us through the caches and 18 streamed; 36 M, 216 MB, 42 and 38; 128 M 137 and 131)
    const bool past = 2 * m.numel() * (1 + mo.element_size()) > g_last_level / 2;
    check(rx_aw_decode(ptr<uint8_t>(m), ptr<uint8_t>(v), ptr<uint8_t>(sc), mo.data_ptr(), vo.data_ptr(), m.numel(), to_bf16,
                       past, current_stream(m)),
          "rx_aw_decode");
  }
  return {mo, vo};
}

// ------------------------------------------------------------------------------------------------ experts
int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: throw py::type_error(std::string("dtype ") + c10::toString(t.scalar_type()) + " (fp32, bf16 or fp16)");
  }
}

// contiguous rows, any distance between them
Tensor rows_of(const Tensor& t) { return t.stride(1) == 1 || t.size(1) == 1 ? t : t.contiguous(); }

variable_list route_forward(const Tensor& z, int64_t k, bool renorm, bool keep) {
  const int64_t T = z.size(0);
  const auto f32 = z.options().dtype(at::kFloat);
  Tensor w = at::empty({T, k}, f32), ids = at::empty({T, k}, z.options().dtype(at::kInt)), norm;
  if (keep) norm = at::empty({T, 2}, f32);
  c10::DeviceGuard guard(z.device());
  check(rx_route_fwd(z.data_ptr(), z.stride(0), dtype_code(z), T, (int)z.size(1), (int)k, renorm, ptr<float>(w),
                     ptr<int>(ids), keep ? ptr<float>(norm) : nullptr, current_stream(z)),
        "rx_route_fwd");
  return {w, ids, norm};
}

struct Route : torch::autograd::Function<Route> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t k, bool renorm) {
    const Tensor z = rows_of(logits);
    variable_list out = route_forward(z, k, renorm, !renorm);
    // the gradient of the renormalised weights needs no logits
    if (renorm) ctx->save_for_backward({out[0], out[1]});
    else ctx->save_for_backward({out[0], out[1], out[2], z});
    ctx->saved_data["E"] = logits.size(1);
    ctx->saved_data["dtype"] = (int64_t)logits.scalar_type();
    ctx->mark_non_differentiable({out[1]});
    ctx->set_materialize_grads(false);
    return {out[0], out[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {Variable(), Variable(), Variable()};
    check_memory(grads[0], "route");
    check_tangent(grads[0], "route");
    check_capturable(grads[0]);
    const auto saved = ctx->get_saved_variables();
    const Tensor &w = saved[0], &ids = saved[1], dw = grads[0].contiguous();
    const bool full = saved.size() == 4;
    const int64_t E = ctx->saved_data["E"].toInt();
    Tensor dz = at::empty({w.size(0), E}, w.options().dtype((at::ScalarType)ctx->saved_data["dtype"].toInt()));
    c10::DeviceGuard guard(w.device());
    check(rx_route_bwd(full ? saved[3].data_ptr() : nullptr, full ? saved[3].stride(0) : 0, dtype_code(dz),
                       full ? ptr<float>(saved[2]) : nullptr, ptr<float>(w), ptr<int>(ids), ptr<float>(dw), w.size(0), (int)E,
                       (int)w.size(1), dz.data_ptr(), current_stream(w)),
          "rx_route_bwd");
    return once({dz, Variable(), Variable()});
  }
};

std::tuple<Tensor, Tensor> route(const Tensor& logits, int64_t k, bool renorm) {
  check_trace("route");
  check_memory(logits, "route");
  check_tangent(logits, "route");
  variable_list out = logits.requires_grad() && at::GradMode::is_enabled() ? Route::apply(logits, k, renorm)
                                                                           : route_forward(rows_of(logits), k, renorm, false);
  return {out[0], out[1]};
}

// One workgroup up to 4096 choices, which needs one launch and not two; at most 256 workgroups beyond, as each of them sums
// the counts of all. (choices per workgroup, workgroups)
std::pair<int64_t, int64_t> plan_grid(int64_t n) {
  const auto up = [](int64_t v, int64_t m) { return (v + m - 1) / m * m; };
  if (n <= 4096) return {std::max<int64_t>(1024, up(n, 1024)), 1};
  const int64_t chunk = std::max<int64_t>(1024, up((n + 255) / 256, 1024));
  return {chunk, (n + chunk - 1) / chunk};
}

// (position, source, load, offsets); capacity 0: unlimited
std::vector<Tensor> expert_plan(const Tensor& experts, int64_t E, int64_t capacity) {
  check_trace("expert_plan");
  check_memory(experts, "expert_plan");
  const Tensor ids = experts.contiguous();
  const int64_t T = ids.size(0), k = ids.size(1), n = T * k, rows = capacity ? E * capacity : n;
  const auto [chunk, blocks] = plan_grid(n);
  // one allocation: position, source, load, offsets, scratch
  Tensor buf = at::empty({n + rows + 2 * E + 1 + (blocks > 1 ? blocks * E : 0)}, ids.options().dtype(at::kInt));
  int* at_ = ptr<int>(buf);
  PlanArgs a;
  a.ids = ids.data_ptr();
  a.wide = ids.scalar_type() == at::kLong;
  a.n = (int)n;
  a.E = (int)E;
  a.chunk = (int)chunk;
  a.blocks = (int)blocks;
  a.capacity = (int)capacity;
  a.rows = (int)rows;
  a.pad_ = 0;
  a.counts = nullptr;
  a.position = at_;
  a.source = at_ + n;
  a.load = at_ + n + rows;
  a.offsets = at_ + n + rows + E;
  c10::DeviceGuard guard(ids.device());
  check(rx_expert_plan(&a, blocks > 1 ? at_ + n + rows + 2 * E + 1 : nullptr, current_stream(ids)), "rx_expert_plan");
  std::vector<Tensor> out{buf.narrow(0, 0, n).view({T, k}), buf.narrow(0, n, rows), buf.narrow(0, n + rows, E),
                          buf.narrow(0, n + rows + E, E + 1)};
  // a version each: what the caller writes into load is no change of the positions that backward keeps
  for (const Tensor& t : out)
    if (!t.is_inference()) torch::autograd::impl::set_version_counter(t, c10::VariableVersion(0));
  return out;
}

RowArgs row_args(const Tensor& position, const Tensor& source, int64_t D, const Tensor& like, bool twice) {
  RowArgs a;
  a.T = position.size(0);
  a.k = (int)position.size(1);
  a.rows = source.size(0);
  a.D = (int)D;
  const int64_t units = (D * like.element_size() + 15) / 16;
  a.lg = 0;
  while (a.lg < 6 && (1ll << a.lg) < units) ++a.lg;
  // samples' rows and expert rows, these twice where products are taken
  a.stream = (a.T + a.rows * (twice ? 2 : 1)) * D * like.element_size() > g_last_level;
  a.position = ptr<int>(position);
  a.source = ptr<int>(source);
  a.ldx = 0;
  a.x = a.h = nullptr;
  a.w = nullptr;
  a.out = nullptr;
  a.dw = nullptr;
  return a;
}

// expert rows with x (times w) in them; with h also the inner products
std::pair<Tensor, Tensor> scatter(const Tensor& position, const Tensor& source, const Tensor& x_, const Tensor& w, const Tensor& h) {
  const Tensor x = rows_of(x_);
  Tensor out = at::empty({source.size(0), x.size(1)}, x.options()), dw;
  RowArgs a = row_args(position, source, x.size(1), x, h.defined());
  a.x = x.data_ptr();
  a.ldx = x.stride(0);
  a.out = out.data_ptr();
  if (w.defined()) a.w = ptr<float>(w);
  if (h.defined()) {
    dw = at::empty(position.sizes(), x.options().dtype(at::kFloat));
    a.h = h.data_ptr();
    a.dw = ptr<float>(dw);
  }
  c10::DeviceGuard guard(x.device());
  check(rx_rows_scatter(&a, dtype_code(x), current_stream(x)), "rx_rows_scatter");
  return {out, dw};
}

Tensor gather(const Tensor& position, const Tensor& source, const Tensor& h, const Tensor& w) {
  Tensor out = at::empty({position.size(0), h.size(1)}, h.options());
  RowArgs a = row_args(position, source, h.size(1), h, false);
  a.h = h.data_ptr();
  a.out = out.data_ptr();
  if (w.defined()) a.w = ptr<float>(w);
  c10::DeviceGuard guard(h.device());
  check(rx_rows_gather(&a, dtype_code(h), current_stream(h)), "rx_rows_gather");
  return out;
}

// What the row kernels take from a plan's tensors by address: a plan can be put together, or changed, by hand.
void check_plan(const Tensor& position, const Tensor& source, const Tensor& rows, bool samples, const char* what) {
  for (const Tensor& t : {position, source})
    if (t.scalar_type() != at::kInt || !t.is_contiguous() || t.device() != rows.device())
      throw py::value_error(std::string(what) + ": a plan's position and source must be contiguous int32 on the rows' device");
  if (position.dim() != 2 || position.size(1) < 1 || source.dim() != 1 || rows.size(0) != (samples ? position : source).size(0))
    throw py::value_error(std::string(what) + ": the plan's position must be [T, k] and its source [rows], with " +
                          (samples ? "T samples" : "that many expert rows") + " given");
}

struct Dispatch : torch::autograd::Function<Dispatch> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& position, const Tensor& source) {
    ctx->save_for_backward({position, source});
    return scatter(position, source, x, Tensor(), Tensor()).first;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_memory(grads[0], "dispatch");
    check_tangent(grads[0], "dispatch");
    check_capturable(grads[0]);
    const auto saved = ctx->get_saved_variables();
    return once({gather(saved[0], saved[1], grads[0].contiguous(), Tensor()), Variable(), Variable()});
  }
};

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const c10::optional<Tensor>& weights,
                        const Tensor& position, const Tensor& source) {
    const Tensor w = weights ? *weights : Tensor();
    // the rows are only kept for the weights' gradient
    ctx->save_for_backward({position, source, w, w.defined() && w.requires_grad() ? rows : Tensor()});
    return gather(position, source, rows, w);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    check_memory(grads[0], "combine");
    check_tangent(grads[0], "combine");
    check_capturable(grads[0]);
    const auto saved = ctx->get_saved_variables();
    auto [drows, dw] = scatter(saved[0], saved[1], grads[0], saved[2], saved[3]);
    return once({drows, dw, Variable(), Variable()});
  }
};

Tensor dispatch(const Tensor& x, const Tensor& position, const Tensor& source) {
  check_trace("dispatch");
  for (const Tensor& t : {x, position, source}) check_memory(t, "dispatch");
  check_plan(position, source, x, true, "dispatch");
  check_tangent(x, "dispatch");
  if (x.requires_grad() && at::GradMode::is_enabled()) return Dispatch::apply(x, position, source);
  return scatter(position, source, x, Tensor(), Tensor()).first;
}

Tensor combine(const Tensor& rows_, const c10::optional<Tensor>& weights, const Tensor& position, const Tensor& source) {
  check_trace("combine");
  for (const Tensor& t : {rows_, weights ? *weights : Tensor(), position, source}) check_memory(t, "combine");
  check_plan(position, source, rows_, false, "combine");
  if (weights && weights->sizes() != position.sizes()) throw py::value_error("combine: one weight for each place in the plan");
  check_tangent(rows_, "combine");
  if (weights) check_tangent(*weights, "combine");
  const Tensor rows = rows_.contiguous();
  c10::optional<Tensor> w;
  if (weights) w = weights->to(at::kFloat).contiguous();
  if (at::GradMode::is_enabled() && (rows.requires_grad() || (w && w->requires_grad())))
    return Combine::apply(rows, w, position, source);
  return gather(position, source, rows, w ? *w : Tensor());
}

}  // namespace

PYBIND11_MODULE(raydp_torch, m) {
  // its arguments are read by their layout in a library that is built by itself
  if (rx_aw_layout() != kAwLayout || rx_expert_layout() != kExpertLayout)
    throw py::import_error("raydp_torch.so and libhipkernels.so were built from different sources: build both again");
  py::register_local_exception_translator([](std::exception_ptr error) {
    try {
      if (error) std::rethrow_exception(error);
    } catch (const c10::NotImplementedError& e) {
      PyErr_SetString(PyExc_NotImplementedError, e.what_without_backtrace());
    }
  });
  m.def("clip_grad_norm", &clip_grad_norm);
  m.def("adamw_step", &adamw_step);
  m.def("decode_moments", &decode_moments);
  m.def("route", &route);
  m.def("plan_grid", &plan_grid);
  m.def("expert_plan", &expert_plan);
  m.def("dispatch", &dispatch);
  m.def("combine", &combine);
  m.def("set_last_level", [](int64_t bytes) { std::swap(g_last_level, bytes); return bytes; });   // (tests: returns the old)
  m.attr("layouts") = py::make_tuple(kAwLayout, kExpertLayout);
  m.attr("max_experts") = (int)kMaxExperts;
  m.attr("max_topk") = (int)kRouteMaxK;
  m.attr("block") = (int)kAwBlock;
}
