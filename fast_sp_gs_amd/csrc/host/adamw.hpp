// AdamW steps over lists of tensors, each one C++ call.
#pragma once
#include "torch_util.hpp"

namespace fsgs_host {

struct AdamwSettings {  // one entry per tensor; betas shared by all
  std::vector<double> lr, eps, decay;
  double b1, b2;
};

// [2] float32: the 2-norm of all gradients together, and min(1, max_norm / (norm + 1e-6)).
Tensor grad_norm(const std::vector<Tensor>& grads, double max_norm);

// One step of every tensor; `steps` (one count per tensor, all on the host or all on the device) are advanced. `norm`: what grad_norm
// gave, its factor scales the gradients.
void adamw_step(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& m,
                const std::vector<Tensor>& v, const std::vector<Tensor>& steps, const AdamwSettings& set, const OptTensor& norm);
void adamw8_step(const std::vector<Tensor>& params, const std::vector<Tensor>& grads, const std::vector<Tensor>& states,
                 const std::vector<Tensor>& steps, const AdamwSettings& set, int64_t seed, const OptTensor& norm);

// 8-bit moments: bytes of a state, the values (m, v) of states in the shapes of `like`, and states of float32 values.
int64_t adamw8_state_bytes(int64_t count);
std::vector<std::pair<Tensor, Tensor>> adamw8_moments(const std::vector<Tensor>& states, const std::vector<Tensor>& like, at::ScalarType type);
std::vector<Tensor> adamw8_pack(const std::vector<Tensor>& m, const std::vector<Tensor>& v);

}  // namespace fsgs_host
