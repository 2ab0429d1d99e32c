// Marshalling of the AdamW kernels: what may be stepped is checked for all tensors before any count advances, tensors are sorted by
// element type, a launch takes as many as its table holds.
#include "adamw.hpp"

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>

namespace fsgs_host {
namespace {

int type_code(const std::string& what, const char* name, at::ScalarType type) {
  switch (type) {
    case at::kFloat: return FSGS_DTYPE_F32;
    case at::kHalf: return FSGS_DTYPE_F16;
    case at::kBFloat16: return FSGS_DTYPE_BF16;
    default: fail(what + ": " + name + " must have dtype torch.float32, torch.float16 or torch.bfloat16, got " + dtype_text(type));
  }
}

std::string number(size_t k) { return std::to_string(k); }

void require_device(const std::string& what, const char* name, const Tensor& t, const at::Device& device) {
  if (t.defined() && t.layout() != at::kStrided) fail(what + ": " + name + " must be dense, sparse tensors are not stepped");
  if (!t.defined() || !t.is_cuda()) fail(what + ": " + name + " must be a CUDA tensor");
  if (t.device() != device) fail(what + ": all tensors of a call must be on one device");
}

// Whether two tensors of one shape have their elements in the same order, without gaps.
bool alike(const Tensor& a, const Tensor& b) {
  return a.sizes() == b.sizes() &&
         ((a.is_contiguous() && b.is_contiguous()) || (a.strides() == b.strides() && a.is_non_overlapping_and_dense()));
}

struct Written {  // by the call: a tensor for each parameter
  const char* name;
  const std::vector<Tensor>& list;
};

// What a call writes, no other thread of it may read or write: a tensor that is there twice, or views that overlap, would be stepped in a race.
// Gradients may share their memory among themselves, or be the parameter that they belong to. Lists mostly rise in memory and are merged.
void refuse_shared(const std::string& what, std::initializer_list<Written> written, const std::vector<Tensor>& params, const std::vector<Tensor>& grads) {
  struct Range {
    const char *from, *to, *name;  // name: null for what is only read
  };
  const auto before = [](const Range& a, const Range& b) { return a.from < b.from; };
  std::vector<Range> all;
  all.reserve((written.size() + 1) * params.size());
  const auto add = [&](const char* name, const Tensor& t) {
    const char* from = (const char*) (name ? t.data_ptr() : t.const_data_ptr());  // what is written has memory of its own from here on
    if (t.numel() > 0) all.push_back({from, from + t.numel() * (int64_t) t.element_size(), name});
  };
  const auto merge = [&](size_t from) {
    if (!std::is_sorted(all.begin() + from, all.end(), before)) std::sort(all.begin() + from, all.end(), before);
    std::inplace_merge(all.begin(), all.begin() + from, all.end(), before);
  };
  for (const Written& w : written) {
    const size_t from = all.size();
    for (const Tensor& t : w.list) add(w.name, t);
    merge(from);
  }
  const size_t from = all.size();
  for (size_t k = 0; k < grads.size(); ++k)
    if (grads[k].const_data_ptr() != params[k].const_data_ptr()) add(nullptr, grads[k]);
  merge(from);
  Range none{nullptr, nullptr, nullptr}, last = none, last_written = none;  // of those so far, the ones that reach farthest
  for (const Range& r : all) {
    const Range& other = r.name ? last : last_written;
    if (r.from < other.to) {
      if (r.name == other.name && r.from == other.from) fail(what + ": a " + r.name + " is there twice");
      const auto named = [](const Range& x) { return std::string("a ") + (x.name ? x.name : "gradient"); };
      fail(what + ": " + named(other) + " and " + named(r) + " share memory");
    }
    if (last.to < r.to) last = r;
    if (r.name && last_written.to < r.to) last_written = r;
  }
}

void changed(const Tensor& t) {  // kernels write behind autograd's back: whoever saved or packed the tensor is told
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// The tensors of a call by element type, in launches of as many as a table holds.
struct Launches {
  std::vector<std::pair<int, std::vector<size_t>>> list;
  Launches(const std::string& what, const char* name, const std::vector<Tensor>& tensors) {
    const size_t most = (size_t) fsgs_adamw_max_tensors();
    for (const int code : {FSGS_DTYPE_F32, FSGS_DTYPE_F16, FSGS_DTYPE_BF16}) {
      bool open = false;
      for (size_t k = 0; k < tensors.size(); ++k) {
        if (type_code(what, name, tensors[k].scalar_type()) != code) continue;
        if (!open || list.back().second.size() == most) list.push_back({code, {}}), open = true;
        list.back().second.push_back(k);
      }
    }
  }
};

template <typename T, typename F>
std::vector<T> pick(const std::vector<size_t>& which, F of) {
  std::vector<T> out;
  out.reserve(which.size());
  for (const size_t k : which) out.push_back(of(k));
  return out;
}

struct Call {
  const char* what;
  std::vector<Tensor> grads;  // laid out as their parameters
  std::vector<double> count_of_steps;
  bool device_steps = false;

  Call(const char* name, const std::vector<Tensor>& params, const std::vector<Tensor>& given, const std::vector<Tensor>& steps,
       const AdamwSettings& set, const OptTensor& norm)
      : what(name) {
    const size_t n = params.size();
    const std::string w(what);
    if (given.size() != n || steps.size() != n || set.lr.size() != n || set.eps.size() != n || set.decay.size() != n)
      fail(w + ": a gradient, a step count and rates for each parameter tensor");
    if (!(set.b1 >= 0 && set.b1 < 1 && set.b2 >= 0 && set.b2 < 1)) fail(w + ": betas must be in [0, 1)");
    for (size_t k = 0; k < n; ++k)
      if (!(set.lr[k] >= 0 && set.eps[k] >= 0 && set.decay[k] >= 0)) fail(w + ": lr, eps and weight_decay must not be negative");
    if (n == 0) return;
    const at::Device device = params[0].device();
    device_steps = steps[0].is_cuda();
    int64_t elements = 0;
    for (size_t k = 0; k < n; ++k) {
      const Tensor &p = params[k], &g = given[k];
      require_device(w, "param", p, device), require_device(w, "grad", g, device);
      (void) type_code(w, "param", p.scalar_type());
      if (!p.is_contiguous() && !p.is_non_overlapping_and_dense()) fail(w + ": param " + number(k) + " has gaps or overlaps in memory");
      if (g.sizes() != p.sizes()) fail(w + ": tensor " + number(k) + "'s gradient differs from it in shape");
      if (g.scalar_type() != p.scalar_type())
        fail(w + ": tensor " + number(k) + "'s gradient must have dtype " + dtype_text(p.scalar_type()) + ", got " + dtype_text(g.scalar_type()));
      elements += p.numel() + 1024;  // the last block of a tensor is not always a whole one
      if (elements >= (int64_t) 1 << 34) fail(w + ": more elements than a launch takes (2^34)");
      const Tensor& s = steps[k];
      if (!s.defined() || s.numel() != 1) fail(w + ": a step count is one number");
      if (s.is_cuda() != device_steps) fail(w + ": step counts must all be on the host or all on the device");
      if (device_steps) {
        require_device(w, "step", s, device);
        if (s.scalar_type() != at::kFloat) fail(w + ": step counts on the device must have dtype torch.float32");
      } else {
        const auto type = s.scalar_type();  // 16 bits stop at 256 or 2048
        if (type != at::kFloat && type != at::kDouble && type != at::kInt && type != at::kLong)
          fail(w + ": step counts must have dtype torch.float32, torch.float64, torch.int32 or torch.int64, got " + dtype_text(type));
        if (!((type == at::kFloat ? (double) *s.const_data_ptr<float>() : s.item<double>()) >= 0)) fail(w + ": a step count must not be negative");
      }
    }
    if (has(norm)) {
      require(what, "norm", *norm, at::kFloat), require_device(w, "norm", *norm, device);
      const int64_t room = (int64_t) norm->storage().nbytes() - norm->storage_offset() * 4;
      if (norm->numel() != 2 || room < (int64_t) fsgs_grad_norm_bytes() || (uintptr_t) norm->data_ptr() % 8) fail(w + ": norm must be what grad_norm returned");
    }
    for (size_t k = 0; k < n; ++k)
      grads.push_back(alike(given[k], params[k]) ? given[k] : at::empty_like(params[k]).copy_(given[k]));
    if (!device_steps && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
      fail(w + ": a captured step needs its step counts on the device");
  }

  void advance(const std::vector<Tensor>& steps) {
    if (device_steps) return;
    for (const Tensor& s : steps)
      count_of_steps.push_back(s.scalar_type() == at::kFloat ? (double) (*s.data_ptr<float>() += 1.0f) : s.add_(1).item<double>());
  }

  // Rates of one launch's tensors by their counts on the device, which are advanced; undefined for counts on the host.
  Tensor rates(const std::vector<size_t>& which, const std::vector<Tensor>& steps, const AdamwSettings& set, uint32_t seed, void* stream) const {
    if (!device_steps) return Tensor();
    const Tensor out = empty({(int64_t) fsgs_adamw_rates_bytes((int) which.size())}, steps[0], at::kByte);
    const auto at = pick<float*>(which, [&](size_t k) { return f32(steps[k]); });
    const auto lr = pick<double>(which, [&](size_t k) { return set.lr[k]; });
    check(fsgs_adamw_rates((int) which.size(), at.data(), lr.data(), set.b1, set.b2, seed, out.data_ptr(), stream), what);
    return out;
  }
};

template <typename Launch>
void step_all(const Call& call, const std::vector<Tensor>& params, const std::vector<Tensor>& steps, const AdamwSettings& set,
              uint32_t seed, Launch launch) {
  void* stream = stream_of(params[0]);
  for (const auto& [code, which] : Launches(call.what, "param", params).list) {
    const Tensor rates = call.rates(which, steps, set, seed, stream);
    const auto count = pick<int64_t>(which, [&](size_t k) { return params[k].numel(); });
    const auto step = call.device_steps ? std::vector<double>() : pick<double>(which, [&](size_t k) { return call.count_of_steps[k]; });
    const auto lr = pick<double>(which, [&](size_t k) { return set.lr[k]; }), eps = pick<double>(which, [&](size_t k) { return set.eps[k]; });
    const auto decay = pick<double>(which, [&](size_t k) { return set.decay[k]; });
    const auto param = pick<void*>(which, [&](size_t k) { return params[k].data_ptr(); });
    const auto grad = pick<const void*>(which, [&](size_t k) { return (const void*) call.grads[k].data_ptr(); });
    check(launch(code, which, count.data(), step.empty() ? nullptr : step.data(), lr.data(), eps.data(), decay.data(), data<void>(rates),
                 param.data(), grad.data(), stream),
          call.what);
  }
}

}  // namespace

Tensor grad_norm(const std::vector<Tensor>& grads, double max_norm) {
  const std::string what = "grad_norm";
  if (grads.empty()) fail(what + ": no gradients");
  if (!(max_norm >= 0)) fail(what + ": max_norm must not be negative");
  const at::Device device = grads[0].device();
  std::vector<Tensor> dense;  // in any order of elements
  for (const Tensor& g : grads) {
    require_device(what, "grad", g, device);
    dense.push_back(g.is_contiguous() || g.is_non_overlapping_and_dense() ? g : g.contiguous());
  }
  const c10::DeviceGuard guard(device);
  const Launches launches(what, "grad", dense);
  const int each = std::max(64, fsgs_grad_square_sums_max() / (int) launches.list.size());
  const Tensor sums = empty({each * (int64_t) launches.list.size()}, dense[0], at::kDouble);
  const Tensor out = part_of(empty({(int64_t) fsgs_grad_norm_bytes()}, dense[0], at::kByte), 0, {2}, {1}, at::kFloat);
  void* stream = stream_of(dense[0]);
  double* at = data<double>(sums);
  for (const auto& [code, which] : launches.list) {
    const auto count = pick<int64_t>(which, [&](size_t k) { return dense[k].numel(); });
    const auto grad = pick<const void*>(which, [&](size_t k) { return (const void*) dense[k].data_ptr(); });
    check(fsgs_grad_square_sums((int) which.size(), code, count.data(), grad.data(), each, at, stream), "grad_norm");
    at += each;
  }
  check(fsgs_grad_norm_factor((int) sums.numel(), data<double>(sums), max_norm, f32(out), stream), "grad_norm");
  return out;
}

void adamw_step(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& m,
                const std::vector<Tensor>& v, const std::vector<Tensor>& steps, const AdamwSettings& set, const OptTensor& norm) {
  const std::string what = "adamw_step";
  const c10::OptionalDeviceGuard guard(params.empty() || !params[0].is_cuda() ? std::nullopt : std::optional<at::Device>(params[0].device()));
  Call call("adamw_step", params, grads, steps, set, norm);
  if (m.size() != params.size() || v.size() != params.size()) fail(what + ": two moments for each parameter tensor");
  if (params.empty()) return;
  for (size_t k = 0; k < params.size(); ++k)
    for (const Tensor* t : {&m[k], &v[k]}) {
      require_device(what, "moment", *t, params[k].device());
      if (t->scalar_type() != at::kFloat) fail(what + ": moments must have dtype torch.float32, got " + dtype_text(t->scalar_type()));
      if (!alike(*t, params[k])) fail(what + ": tensor " + number(k) + "'s moments differ from it in shape or layout");
    }
  refuse_shared(what, {{"parameter", params}, {"first moment", m}, {"second moment", v}, {"step count", steps}}, params, call.grads);
  call.advance(steps);
  const float* factor = f32(opt(norm));
  step_all(call, params, steps, set, 0,
           [&](int code, const std::vector<size_t>& which, const int64_t* count, const double* step, const double* lr, const double* eps,
               const double* decay, const void* rates, void* const* param, const void* const* grad, void* stream) {
             const auto first = pick<float*>(which, [&](size_t k) { return f32(m[k]); }), second = pick<float*>(which, [&](size_t k) { return f32(v[k]); });
             return fsgs_adamw_update_multi((int) which.size(), code, count, step, lr, set.b1, set.b2, eps, decay, rates, factor, param,
                                            grad, first.data(), second.data(), stream);
           });
  for (const auto* list : {&params, &m, &v})
    for (const Tensor& t : *list) changed(t);
}

void adamw8_step(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& states,
                 const std::vector<Tensor>& steps, const AdamwSettings& set, int64_t seed, const OptTensor& norm) {
  const std::string what = "adamw8_step";
  const c10::OptionalDeviceGuard guard(params.empty() || !params[0].is_cuda() ? std::nullopt : std::optional<at::Device>(params[0].device()));
  Call call("adamw8_step", params, grads, steps, set, norm);
  if (states.size() != params.size()) fail(what + ": a state for each parameter tensor");
  if (params.empty()) return;
  for (size_t k = 0; k < params.size(); ++k) {
    require(what.c_str(), "state", states[k], at::kByte), require_device(what, "state", states[k], params[k].device());
    if (states[k].numel() != adamw8_state_bytes(params[k].numel())) fail(what + ": state " + number(k) + " is that of another number of elements");
    if ((uintptr_t) states[k].data_ptr() % 16) fail(what + ": state " + number(k) + " must lie on a boundary of 16 bytes");
  }
  refuse_shared(what, {{"parameter", params}, {"state", states}, {"step count", steps}}, params, call.grads);
  call.advance(steps);
  const float* factor = f32(opt(norm));
  step_all(call, params, steps, set, (uint32_t) seed,
           [&](int code, const std::vector<size_t>& which, const int64_t* count, const double* step, const double* lr, const double* eps,
               const double* decay, const void* rates, void* const* param, const void* const* grad, void* stream) {
             const auto state = pick<void*>(which, [&](size_t k) { return states[k].data_ptr(); });
             return fsgs_adamw8_update_multi((int) which.size(), code, count, step, lr, set.b1, set.b2, eps, decay, (uint32_t) seed, rates,
                                             factor, param, grad, state.data(), stream);
           });
  for (const auto* list : {&params, &states})
    for (const Tensor& t : *list) changed(t);
}

int64_t adamw8_state_bytes(int64_t count) { return (int64_t) fsgs_adamw8_state_bytes(count); }

std::vector<std::pair<Tensor, Tensor>> adamw8_moments(const std::vector<Tensor>& states, const std::vector<Tensor>& like, at::ScalarType type) {
  const std::string what = "adamw8_moments";
  const int code = type_code(what, "the result", type);
  if (states.size() != like.size()) fail(what + ": a state for each tensor");
  std::vector<std::pair<Tensor, Tensor>> out;
  if (states.empty()) return out;
  const at::Device device = states[0].device();
  for (size_t k = 0; k < states.size(); ++k) {
    require(what.c_str(), "state", states[k], at::kByte), require_device(what, "state", states[k], device);
    if (!like[k].is_contiguous() && !like[k].is_non_overlapping_and_dense()) fail(what + ": tensor " + number(k) + " has gaps or overlaps in memory");
    if (states[k].numel() != adamw8_state_bytes(like[k].numel())) fail(what + ": state " + number(k) + " is that of another number of elements");
  }
  const c10::DeviceGuard guard(device);
  // parts of one allocation, each on a boundary of its own: an allocation for every one of 50 tensors took 40 us
  const int64_t size = type == at::kFloat ? 4 : 2;
  const auto room = [&](const Tensor& t) { return (t.numel() * size + 511) / 512 * 512; };
  int64_t total = 0;
  for (const Tensor& t : like) total += 2 * room(t);
  const Tensor all = empty({total}, states[0], at::kByte);
  int64_t at = 0;
  for (const Tensor& t : like) {
    const auto part = [&](int64_t from) { return part_of(all, from, t.sizes(), t.strides(), type); };
    out.push_back({part(at), part(at + room(t))}), at += 2 * room(t);
  }
  const size_t n = states.size(), most = (size_t) fsgs_adamw_max_tensors();
  for (size_t from = 0; from < n; from += most) {
    std::vector<size_t> which;
    for (size_t k = from; k < std::min(n, from + most); ++k) which.push_back(k);
    const auto count = pick<int64_t>(which, [&](size_t k) { return like[k].numel(); });
    const auto state = pick<const void*>(which, [&](size_t k) { return (const void*) states[k].data_ptr(); });
    const auto m = pick<void*>(which, [&](size_t k) { return out[k].first.data_ptr(); }), v = pick<void*>(which, [&](size_t k) { return out[k].second.data_ptr(); });
    check(fsgs_adamw8_unpack_multi((int) which.size(), code, count.data(), state.data(), m.data(), v.data(), stream_of(states[0])), what.c_str());
  }
  return out;
}

std::vector<Tensor> adamw8_pack(const std::vector<Tensor>& m, const std::vector<Tensor>& v) {
  const std::string what = "adamw8_pack";
  if (m.size() != v.size()) fail(what + ": a second moment for each first one");
  std::vector<Tensor> out;
  if (m.empty()) return out;
  const at::Device device = m[0].device();
  for (size_t k = 0; k < m.size(); ++k) {
    require_device(what, "moment", m[k], device), require_device(what, "moment", v[k], device);
    if (m[k].scalar_type() != at::kFloat || v[k].scalar_type() != at::kFloat) fail(what + ": moments must have dtype torch.float32");
    if (!m[k].is_contiguous() && !m[k].is_non_overlapping_and_dense()) fail(what + ": tensor " + number(k) + " has gaps or overlaps in memory");
    if (!alike(m[k], v[k])) fail(what + ": the moments of tensor " + number(k) + " differ in shape or layout");
  }
  const c10::DeviceGuard guard(device);
  for (const Tensor& t : m) out.push_back(empty({adamw8_state_bytes(t.numel())}, t, at::kByte));
  const size_t n = m.size(), most = (size_t) fsgs_adamw_max_tensors();
  for (size_t at = 0; at < n; at += most) {
    std::vector<size_t> which;
    for (size_t k = at; k < std::min(n, at + most); ++k) which.push_back(k);
    const auto count = pick<int64_t>(which, [&](size_t k) { return m[k].numel(); });
    const auto first = pick<const float*>(which, [&](size_t k) { return (const float*) f32(m[k]); }), second = pick<const float*>(which, [&](size_t k) { return (const float*) f32(v[k]); });
    const auto state = pick<void*>(which, [&](size_t k) { return out[k].data_ptr(); });
    check(fsgs_adamw8_pack_multi((int) which.size(), count.data(), first.data(), second.data(), state.data(), stream_of(m[0])), what.c_str());
  }
  return out;
}

}  // namespace fsgs_host
