// Torch glue for the optimizer kernels (adamw_kernels.hip): the plan that an
// optimizer keeps for its tensors, its step, and the norm over many tensors.
// Like the GAR ops, all launches go to the current HIP stream of the tensors'
// device, nothing waits for the device, and everything can be captured into a
// graph.

#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <map>
#include <memory>
#include <optional>
#include <vector>

#include "adamw_kernels.h"

namespace {

using torch::Tensor;

int dtype_of(const Tensor& t, const char* what) {
  switch (t.scalar_type()) {
    case torch::kFloat32:
      return adamw::kF32;
    case torch::kBFloat16:
      return adamw::kBF16;
    case torch::kFloat16:
      return adamw::kF16;
    default:
      TORCH_CHECK(false, what, ": expected fp32, bf16 or fp16, got ",
                  t.scalar_type());
  }
}

// Bytes [lo, hi) that a tensor's elements lie in.
struct Range {
  uintptr_t lo, hi;
};

Range range_of(const Tensor& t) {
  const auto lo = reinterpret_cast<uintptr_t>(t.data_ptr());
  if (t.numel() == 0) return {lo, lo};
  uintptr_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d)
    last += (uintptr_t)(t.size(d) - 1) * t.stride(d);
  return {lo, lo + (last + 1) * t.element_size()};
}

// Whether equal places in memory hold equal elements of both.
bool same_layout(const Tensor& a, const Tensor& b) {
  if (a.sizes() != b.sizes()) return false;
  if (a.numel() < 2) return true;
  for (int64_t d = 0; d < a.dim(); ++d)
    if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0x9E3779B1u;
  x ^= x >> 15;
  x *= 0x85EBCA77u;
  return x ^ (x >> 16);
}

// The tensors of a Python list or tuple (the caller's, which holds them), null
// for None.
std::vector<const Tensor*> tensors_of(pybind11::handle given, bool none) {
  PyObject* const sequence = given.ptr();
  TORCH_CHECK(PyList_Check(sequence) || PyTuple_Check(sequence),
              "expected a list or tuple of tensors");
  const Py_ssize_t count = PySequence_Fast_GET_SIZE(sequence);
  PyObject** const items = PySequence_Fast_ITEMS(sequence);
  std::vector<const Tensor*> out((size_t)count, nullptr);
  for (Py_ssize_t i = 0; i < count; ++i) {
    if (none && items[i] == Py_None) continue;
    TORCH_CHECK(THPVariable_Check(items[i]), "expected a tensor at place ", i,
                " of the sequence");
    out[(size_t)i] = &THPVariable_Unpack(items[i]);
  }
  return out;
}

bool capturing() {
  return c10::hip::currentStreamCaptureStatusMayInitCtx() !=
         c10::hip::CaptureStatus::None;
}

// Tables that a captured graph reads stay for the process's life, and so do the
// step counts, which an optimizer makes for itself: a replay after the plan is
// gone would take addresses from memory that is something else by then, and
// count in it. 64 bytes for 1024 elements or 2048. Never destroyed.
std::vector<Tensor>& captured_tables() {
  static auto* kept = new std::vector<Tensor>();
  return *kept;
}

template <typename T>
Tensor upload(const std::vector<T>& host, const c10::Device& device) {
  auto bytes = torch::from_blob(const_cast<T*>(host.data()),
                                {(int64_t)(host.size() * sizeof(T))},
                                torch::kUInt8);
  return bytes.to(device);  // waits until `host` has been read
}

class Plan {
 public:
  Plan(int bits, std::vector<Tensor> params, std::vector<Tensor> m,
       std::vector<Tensor> ms, std::vector<Tensor> r, std::vector<Tensor> rs,
       Tensor steps, int64_t seed, std::vector<int64_t> places)
      : bits_(bits),
        params_(std::move(params)),
        m_(std::move(m)),
        ms_(std::move(ms)),
        r_(std::move(r)),
        rs_(std::move(rs)),
        steps_(std::move(steps)),
        seed_((uint32_t)seed),
        places_(std::move(places)) {
    TORCH_CHECK(bits_ == 8 || bits_ == 32, "adamw: states have 8 or 32 bits");
    TORCH_CHECK(!params_.empty(), "adamw: a plan needs a parameter");
    lay_out();
  }

  void step(pybind11::handle given, double lr, double beta1, double beta2,
            double eps, double weight_decay, const std::optional<Tensor>& norm,
            double max_norm) {
    const size_t count = params_.size();
    const auto grads = tensors_of(given, /*none=*/true);
    TORCH_CHECK(grads.size() == count, "adamw: ", count, " parameters, but ",
                grads.size(), " gradients");
    const c10::Device device = params_[0].device();
    c10::DeviceGuard guard(device);
    if (stale()) lay_out();

    adamw::Hyper hyper{lr, beta1, beta2, eps, weight_decay, nullptr, max_norm};
    if (norm) {
      TORCH_CHECK(norm->device() == device && norm->numel() == 1 &&
                      norm->scalar_type() == torch::kFloat32 &&
                      !norm->is_neg(),
                  "adamw: norm is one fp32 number on the parameters' device, "
                  "and no view that negates");
      check_apart(*norm, "adamw: norm");
      hyper.norm = norm->data_ptr<float>();
    }
    // Everything is checked before anything is launched.
    std::vector<int> types(count, 0);
    bool moved = false;
    for (size_t i = 0; i < count; ++i) {
      if (grads[i] == nullptr) continue;
      const Tensor& g = *grads[i];
      const Tensor& p = params_[i];
      TORCH_CHECK(g.layout() == torch::kStrided,
                  "adamw: gradient ", i, " is not dense");
      TORCH_CHECK(g.device() == device, "adamw: gradient ", i, " is on ",
                  g.device(), ", its parameter on ", device);
      TORCH_CHECK(g.sizes() == p.sizes(), "adamw: gradient ", i,
                  " has the shape ", g.sizes(), ", its parameter ", p.sizes());
      types[i] = dtype_of(g, "adamw: gradient");
      TORCH_CHECK(adamw::supported(table_[i].type, types[i]),
                  "adamw: gradient ", i, " is ", g.scalar_type(),
                  ", its parameter ", p.scalar_type(),
                  " (the same type, or fp32 parameters)");
      check_apart(g, "adamw: gradient");
      moved = moved || g.is_neg() || !same_layout(g, p);
    }
    // Gradients in another order than their parameters, laid out like them.
    std::vector<Tensor> copies(moved ? count : 0);
    std::vector<const void*> at(count, nullptr);
    for (size_t i = 0; i < count; ++i) {
      if (grads[i] == nullptr) continue;
      const Tensor& g = *grads[i];
      at[i] = g.data_ptr();
      if (g.is_neg() || !same_layout(g, params_[i])) {
        copies[i] = torch::empty_strided(params_[i].sizes(),
                                         params_[i].strides(), g.options());
        copies[i].copy_(g);
        at[i] = copies[i].data_ptr();
      }
    }

    const auto current = c10::hip::getCurrentHIPStream();
    const auto stream = current.stream();
    if (capturing()) {
      if (!captured_)
        for (const Tensor& t : {device_work_, tickets_, steps_})
          captured_tables().push_back(t.detach());
      captured_ = true;
    } else if (current != laid_out_on_) {
      // The allocator must not give these to others before this step is done.
      for (const Tensor& t : {device_work_, tickets_})
        t.record_stream(
            c10::hip::HIPStreamMasqueradingAsCUDA(current).unwrap());
    }
    const auto* work =
        reinterpret_cast<const adamw::Work*>(device_work_.data_ptr());
    auto* tickets = reinterpret_cast<unsigned*>(tickets_.data_ptr());
    int* steps = steps_.data_ptr<int>();
    for (size_t first = 0; first < count; first += adamw::kMaxTensors) {
      const size_t last = std::min(count, first + adamw::kMaxTensors);
      adamw::Grads g{};
      bool any = false;
      for (size_t i = first; i < last; ++i) {
        if (grads[i] == nullptr) continue;
        const size_t k = i - first;
        any = true;
        // A tensor of no elements has a gradient all the same: any address.
        g.g[k] = params_[i].numel() > 0 ? at[i] : (const void*)work;
        g.types[k / 16] |= (uint32_t)types[i] << (2 * (k % 16));
      }
      if (!any) continue;
      const int64_t begin = work_start_[first];
      adamw::update(bits_, chunk_, work + begin, work_start_[last] - begin,
                    (int)first, (int)(last - first), steps,
                    tickets + first / adamw::kMaxTensors * adamw::kTicketInts,
                    g, hyper, stream);
      C10_HIP_CHECK(hipGetLastError());
    }
    // What autograd has saved of the parameters is out of date.
    for (size_t i = 0; i < count; ++i)
      if (grads[i] != nullptr && !params_[i].is_inference())
        params_[i].unsafeGetTensorImpl()->bump_version();
  }

 private:
  // Whether a tensor of the plan has got other memory since it was laid out
  // (`param.data = ...`, or a module moved).
  bool stale() const {
    if (steps_.data_ptr() != steps_at_ ||
        steps_.numel() != (int64_t)params_.size())
      return true;
    for (size_t i = 0; i < params_.size(); ++i) {
      const auto& t = table_[i];
      if (params_[i].data_ptr() != t.p || m_[i].data_ptr() != t.m ||
          r_[i].data_ptr() != t.r || params_[i].numel() != numel_[i] ||
          params_[i].device() != steps_.device() ||
          dtype_of(params_[i], "adamw: parameter") != t.type ||
          !same_layout(params_[i], m_[i]) || !same_layout(params_[i], r_[i]))
        return true;
      if (bits_ == 8 &&
          (ms_[i].data_ptr() != t.ms || rs_[i].data_ptr() != t.rs ||
           ms_[i].numel() != rs_[i].numel() ||
           ms_[i].numel() != (numel_[i] + adamw::kGroup - 1) / adamw::kGroup))
        return true;
    }
    return false;
  }

  void check_state(const Tensor& s, const Tensor& p, torch::ScalarType type,
                   const char* what, size_t i) {
    TORCH_CHECK(s.scalar_type() == type, "adamw: ", what, " ", i, " is ",
                s.scalar_type(), ", expected ", type);
    TORCH_CHECK(s.device() == p.device(), "adamw: ", what, " ", i, " is on ",
                s.device(), ", its parameter on ", p.device());
    TORCH_CHECK(!s.is_neg(), "adamw: ", what, " ", i,
                " is a view that negates");
    TORCH_CHECK(same_layout(s, p), "adamw: ", what, " ", i,
                " has another shape or other strides than its parameter");
  }

  void lay_out() {
    TORCH_CHECK(!capturing(),
                "adamw: a plan cannot be laid out while a graph is captured "
                "(a parameter or state has other memory than before: run a "
                "step before the capture)");
    const size_t count = params_.size();
    const c10::Device device = params_[0].device();
    TORCH_CHECK(m_.size() == count && r_.size() == count &&
                    (bits_ == 32 ||
                     (ms_.size() == count && rs_.size() == count)),
                "adamw: as many states as parameters are needed");
    TORCH_CHECK(places_.size() == count,
                "adamw: as many places as parameters are needed");
    TORCH_CHECK(steps_.device() == device && steps_.dim() == 1 &&
                    steps_.size(0) == (int64_t)count &&
                    steps_.is_contiguous() &&
                    steps_.scalar_type() == torch::kInt32,
                "adamw: steps is a contiguous int32 tensor of one count for "
                "each parameter, on their device");
    const auto state_type =
        bits_ == 8 ? torch::kFloat8_e4m3fn : torch::kFloat32;
    std::vector<adamw::Work> table(count), work;
    std::vector<int64_t> work_start(count + 1, 0);
    int64_t total = 0;
    for (const Tensor& p : params_) total += p.numel();
    const int64_t chunk = adamw::chunk_of(bits_, total);
    std::vector<Range> written{range_of(steps_)};
    for (size_t i = 0; i < count; ++i) {
      const Tensor& p = params_[i];
      TORCH_CHECK(p.is_cuda() && p.layout() == torch::kStrided,
                  "adamw: expected dense GPU parameters");
      TORCH_CHECK(p.device() == device,
                  "adamw: the parameters of a plan are on one device");
      TORCH_CHECK(p.is_non_overlapping_and_dense(), "adamw: parameter ", i,
                  " of shape ", p.sizes(), " and strides ", p.strides(),
                  " does not fill its memory");
      TORCH_CHECK(!p.is_neg(), "adamw: parameter ", i,
                  " is a view that negates");
      check_state(m_[i], p, state_type, "exp_avg", i);
      check_state(r_[i], p, state_type,
                  bits_ == 8 ? "exp_avg_root" : "exp_avg_sq", i);
      const int64_t n = p.numel();
      auto& t = table[i];
      t.tensor = (int)i;
      t.p = p.data_ptr();
      t.m = m_[i].data_ptr();
      t.r = r_[i].data_ptr();
      t.key = mix(seed_ + 0x9E3779B9u * (uint32_t)(places_[i] + 1));
      t.type = dtype_of(p, "adamw: parameter");
      written.push_back(range_of(p));
      written.push_back(range_of(m_[i]));
      written.push_back(range_of(r_[i]));
      if (bits_ == 8) {
        const int64_t groups = (n + adamw::kGroup - 1) / adamw::kGroup;
        for (const Tensor* s : {&ms_[i], &rs_[i]}) {
          TORCH_CHECK(s->scalar_type() == torch::kFloat8_e8m0fnu &&
                          s->device() == device && s->dim() == 1 &&
                          s->size(0) == groups && s->is_contiguous(),
                      "adamw: the scales of state ", i,
                      " are a contiguous e8m0 tensor of ", groups,
                      " elements on its parameter's device");
          written.push_back(range_of(*s));
        }
        t.ms = reinterpret_cast<uint8_t*>(ms_[i].data_ptr());
        t.rs = reinterpret_cast<uint8_t*>(rs_[i].data_ptr());
      }
      for (int64_t start = 0; start < n; start += chunk) {
        adamw::Work w = t;
        const int64_t state = start * (bits_ / 8);
        w.p = (char*)t.p + start * p.element_size();
        w.m = (char*)t.m + state;
        w.r = (char*)t.r + state;
        if (bits_ == 8) {
          w.ms = t.ms + start / adamw::kGroup;
          w.rs = t.rs + start / adamw::kGroup;
        }
        w.start = start;
        w.left = (int)std::min(n - start, chunk);
        work.push_back(w);
      }
      work_start[i + 1] = (int64_t)work.size();
      TORCH_CHECK(work_start[i + 1] -
                          work_start[i - i % adamw::kMaxTensors] <=
                      adamw::kMaxWork,
                  "adamw: too many elements for one launch");
    }
    std::sort(written.begin(), written.end(),
              [](const Range& a, const Range& b) { return a.lo < b.lo; });
    written.erase(std::remove_if(written.begin(), written.end(),
                                 [](const Range& r) { return r.lo == r.hi; }),
                  written.end());
    for (size_t i = 1; i < written.size(); ++i)
      TORCH_CHECK(written[i - 1].hi <= written[i].lo,
                  "adamw: parameters, states and steps share memory");
    c10::DeviceGuard guard(device);
    const int64_t launches =
        (int64_t)(count + adamw::kMaxTensors - 1) / adamw::kMaxTensors;
    tickets_ = torch::zeros(
        {launches * adamw::kTicketInts},
        torch::TensorOptions().device(device).dtype(torch::kInt32));
    // The upload waits for the stream, so another may use all of these next.
    if (work.empty()) work.push_back(table[0]);
    device_work_ = upload(work, device);
    laid_out_on_ = c10::hip::getCurrentHIPStream();
    steps_at_ = steps_.data_ptr();
    numel_.clear();
    for (const Tensor& p : params_) numel_.push_back(p.numel());
    table_ = std::move(table);
    work_start_ = std::move(work_start);
    chunk_ = chunk;
    written_ = std::move(written);
    captured_ = false;
  }

  // What the step reads must not be what it writes.
  void check_apart(const Tensor& t, const char* what) const {
    const Range r = range_of(t);
    if (r.lo == r.hi) return;
    auto it = std::upper_bound(
        written_.begin(), written_.end(), r.lo,
        [](uintptr_t v, const Range& w) { return v < w.hi; });
    TORCH_CHECK(it == written_.end() || it->lo >= r.hi, what,
                " shares memory with a parameter or state");
  }

  int bits_;
  std::vector<Tensor> params_, m_, ms_, r_, rs_;
  Tensor steps_;
  uint32_t seed_;
  std::vector<int64_t> places_;  // what stands for a tensor in its random bits
  std::vector<adamw::Work> table_;  // each tensor's first
  std::vector<int64_t> work_start_;  // before each tensor's, in device_work_
  int64_t chunk_ = 0;
  std::vector<int64_t> numel_;
  std::vector<Range> written_;
  Tensor device_work_, tickets_;
  c10::hip::HIPStream laid_out_on_ = c10::hip::getDefaultHIPStream();
  const void* steps_at_ = nullptr;
  bool captured_ = false;
};

// Counters of the norm's arrivals, and room for its partial sums, for what a
// stream runs one after the other. (A captured graph may run beside its stream's
// later work: it has sums of its own, and adds them up in a launch of its own.)
// Never destroyed.
struct NormSpace {
  Tensor tickets, partials;
};

const NormSpace& norm_space(const c10::hip::HIPStream& stream,
                            const c10::Device& device) {
  static auto* all = new std::map<std::pair<int, hipStream_t>, NormSpace>();
  NormSpace& space = (*all)[{(int)device.index(), stream.stream()}];
  if (!space.partials.defined()) {
    const auto options = torch::TensorOptions().device(device);
    space.tickets =
        torch::zeros({adamw::kTicketInts}, options.dtype(torch::kInt32));
    space.partials =
        torch::empty({adamw::kNormBlocks}, options.dtype(torch::kFloat64));
  }
  return space;
}

Tensor grad_norm(pybind11::handle given_list) {
  const auto tensors = tensors_of(given_list, /*none=*/false);
  TORCH_CHECK(!tensors.empty(), "grad_norm: expected a tensor");
  const c10::Device device = tensors[0]->device();
  TORCH_CHECK(tensors[0]->is_cuda(), "grad_norm: expected GPU tensors");
  c10::DeviceGuard guard(device);
  const auto current = c10::hip::getCurrentHIPStream();
  const auto stream = current.stream();

  std::vector<std::unique_ptr<adamw::Spans>> launches;
  std::vector<Tensor> held;
  held.reserve(tensors.size());
  const char* end = nullptr;  // of the last span
  const bool differentiable = c10::GradMode::is_enabled();
  for (const Tensor* each : tensors) {
    const Tensor& given = *each;
    TORCH_CHECK(given.layout() == torch::kStrided && given.device() == device,
                "grad_norm: expected dense tensors on one device");
    const int type = dtype_of(given, "grad_norm");
    TORCH_CHECK(!differentiable || !given.requires_grad(),
                "grad_norm: has no gradient of its own; detach the tensors or "
                "call it under torch.no_grad()");
    int64_t n = given.numel();
    if (n == 0) continue;
    // The order of the elements does not matter, only that there are no gaps.
    if (!given.is_non_overlapping_and_dense())
      held.push_back(given.contiguous());
    const Tensor& t =
        given.is_non_overlapping_and_dense() ? given : held.back();
    const char* ptr = (const char*)t.data_ptr();
    if (!launches.empty()) {
      auto& s = *launches.back();
      const int last = s.count - 1;
      // Tensors that lie back to back, as views into a flat gradient do, are
      // one span: fewer partly filled chunks, and hardly any search.
      if (ptr == end && type == (int)(s.n4t[last] & 3)) {
        const int64_t all = (s.n4t[last] >> 2) + n;
        const int64_t chunks = (all * t.element_size() +
                                adamw::kNormChunkBytes - 1) /
                               adamw::kNormChunkBytes;
        TORCH_CHECK(s.start[last] + chunks <= INT32_MAX,
                    "grad_norm: too many elements");
        s.n4t[last] = 4 * all + type;
        s.start[last + 1] = (int)(s.start[last] + chunks);
        end = ptr + n * t.element_size();
        continue;
      }
    }
    if (launches.empty() || launches.back()->count == adamw::kMaxSpans) {
      launches.push_back(std::make_unique<adamw::Spans>());
      launches.back()->count = 0;
      launches.back()->start[0] = 0;
    }
    auto& s = *launches.back();
    const int i = s.count++;
    const int64_t chunks =
        (n * t.element_size() + adamw::kNormChunkBytes - 1) /
        adamw::kNormChunkBytes;
    TORCH_CHECK(s.start[i] + chunks <= INT32_MAX,
                "grad_norm: too many elements");
    s.ptr[i] = ptr;
    s.n4t[i] = 4 * n + type;
    s.start[i + 1] = (int)(s.start[i] + chunks);
    end = ptr + n * t.element_size();
  }
  auto options = torch::TensorOptions().device(device);
  auto out = torch::empty({}, options.dtype(torch::kFloat32));
  float* const result = out.data_ptr<float>();
  if (launches.size() == 1 && !capturing()) {
    const NormSpace& space = norm_space(current, device);
    adamw::norm_partials(*launches[0], space.partials.data_ptr<double>(),
                         reinterpret_cast<unsigned*>(space.tickets.data_ptr()),
                         result, stream);
    C10_HIP_CHECK(hipGetLastError());
    return out;
  }
  int count = 0;
  for (auto& s : launches) count += adamw::norm_blocks(*s);
  auto partials =
      torch::empty({std::max(count, 1)}, options.dtype(torch::kFloat64));
  double* at = partials.data_ptr<double>();
  for (auto& s : launches) {
    adamw::norm_partials(*s, at, nullptr, result, stream);
    C10_HIP_CHECK(hipGetLastError());
    at += adamw::norm_blocks(*s);
  }
  adamw::norm_finish(partials.data_ptr<double>(), count, result, stream);
  C10_HIP_CHECK(hipGetLastError());
  return out;
}

}  // namespace

void register_adamw(pybind11::module& mod) {
  namespace py = pybind11;
  py::class_<Plan>(mod, "AdamWPlan")
      .def(py::init<int, std::vector<Tensor>, std::vector<Tensor>,
                    std::vector<Tensor>, std::vector<Tensor>,
                    std::vector<Tensor>, Tensor, int64_t,
                    std::vector<int64_t>>())
      .def("step", &Plan::step);
  mod.def("grad_norm", &grad_norm,
          "L2 norm over all elements of many tensors (gfx950)");
}
