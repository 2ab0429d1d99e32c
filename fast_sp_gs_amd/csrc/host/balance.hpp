// Balance losses of an association, forward and backward, each one C++ call and one autograd node.
#pragma once
#include "torch_util.hpp"

namespace fsgs_host {

// (loss [], counts [M] int32, importance [M]) of logits [N,M]; `rows` [N] bool: the points that count.
std::tuple<Tensor, Tensor, Tensor> balance_loss(const Tensor& logits, int64_t K, const OptTensor& rows);
// The same of neighbour weights [N,K] with indices [N,K] of M superpoints.
std::tuple<Tensor, Tensor, Tensor> neighbour_balance(const Tensor& weights, const Tensor& indices, int64_t M, const OptTensor& rows);

}  // namespace fsgs_host
