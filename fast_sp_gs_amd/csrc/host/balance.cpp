#include "balance.hpp"

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/graph_task.h>

#include <climits>
#include <unordered_set>

namespace fsgs_host {
namespace {

// The results in one allocation, what the backward reads besides them in another: [2] totals, then `extra` bytes.
struct Outputs {
  Tensor loss, counts, importance, saved;
  Outputs(int64_t M, const Tensor& like, int64_t extra = 0) : saved(empty({16 + extra}, like, at::kByte)) {
    const Tensor all = empty({16 + 8 * M}, like, at::kByte);
    loss = part_of(all, 0, {}, {}, at::kFloat), importance = part_of(all, 16, {M}, {1}, at::kFloat);
    counts = part_of(all, 16 + 4 * M, {M}, {1}, at::kInt);
  }
  int64_t* totals() const { return data<int64_t>(saved); }
  float* stats() const { return (float*) (data<uint8_t>(saved) + 16); }
};

int logits_code(at::ScalarType type) {
  switch (type) {
    case at::kFloat: return FSGS_DTYPE_F32;
    case at::kHalf: return FSGS_DTYPE_F16;
    case at::kBFloat16: return FSGS_DTYPE_BF16;
    default: fail("balance_loss: logits must have dtype torch.float32, torch.float16 or torch.bfloat16, got " + dtype_text(type));
  }
}

void require_rows(const char* what, const Tensor& rows, const Tensor& like) {
  if (!rows.defined()) return;
  require(what, "rows", rows, at::kBool), require_shape(what, "rows", rows, {like.size(0)});
  if (rows.device() != like.device()) fail(std::string(what) + ": all tensors of a call must be on one device");
}

// Before anything is allocated, which for sizes beyond these takes gigabytes.
void require_sizes(const char* what, int64_t N, int64_t M) {
  if (N > INT_MAX - 1) fail(std::string(what) + ": more than 2^31 - 2 points");
  if (M > fsgs_balance_max_superpoints()) fail(std::string(what) + ": more than " + std::to_string(fsgs_balance_max_superpoints()) + " superpoints");
}

// A captured backward of a leaf whose accumulation node an eager graph on the default stream keeps alive would have that stream wait for
// the capture, which ends it and the process: refused while nothing is recorded.
void refuse_capture_beside_eager(const char* what, const char* name, const Tensor& t) {
  if (!t.is_leaf() || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!node) return;
  const auto stream = node->stream();
  if (stream && stream->id() == 0)
    fail(std::string(what) + ": " + name + " is part of an eager graph that is still alive: drop that graph before this call is captured");
}

// The same for everything that the backward under way has yet to reach: logits made from leaves while an eager graph of those leaves lives, or made
// eagerly themselves. The engine has the default stream wait for a node's results once the node returns: here is the last place to refuse.
void refuse_backward_into_eager(const char* what) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  const auto* run = torch::autograd::get_current_graph_task_exec_info();  // empty: all of the graph
  std::unordered_set<torch::autograd::Node*> seen;
  std::vector<torch::autograd::Node*> todo{node.get()};
  while (!todo.empty()) {
    const auto* at = todo.back();
    todo.pop_back();
    for (const auto& edge : at->next_edges()) {
      auto* next = edge.function.get();
      if (!next || !seen.insert(next).second) continue;
      if (run && !run->empty()) {
        const auto info = run->find(next);
        if (info == run->end() || !info->second.should_execute()) continue;
      }
      const auto stream = next->stream();
      if (stream && stream->id() == 0)
        fail(std::string(what) + ": " + next->name() + " is part of an eager graph that is still alive: drop that graph before this call is captured");
      todo.push_back(next);
    }
  }
}

OptTensor given(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// Rows one behind the other with a stride between them are read where they are.
Tensor rows_of(const Tensor& logits) {
  const bool whole = (logits.size(1) <= 1 || logits.stride(1) == 1) && (logits.size(0) <= 1 || logits.stride(0) >= logits.size(1));
  return whole ? logits : logits.contiguous();
}
int64_t stride_of(const Tensor& logits) { return logits.size(0) > 1 ? logits.stride(0) : logits.size(1); }

Outputs rows_forward(const Tensor& logits, int64_t K, const Tensor& rows, bool train) {
  const int64_t N = logits.size(0), M = logits.size(1);
  const int code = logits_code(logits.scalar_type());
  Outputs out(M, logits, train ? 8 * N : 0);
  const size_t bytes = fsgs_balance_loss_workspace_bytes(N, (int) M, code);
  const Tensor ws = empty({(int64_t) bytes}, logits, at::kByte);
  check(fsgs_balance_loss_forward(N, (int) M, stride_of(logits), (int) K, code, logits.data_ptr(), data<uint8_t>(rows), f32(out.loss),
                                  i32(out.counts), f32(out.importance), out.totals(), train ? out.stats() : nullptr, ws.data_ptr(), bytes, stream_of(logits)),
        "balance_loss");
  return out;
}

Outputs neighbours_forward(const Tensor& weights, const Tensor& indices, int64_t M, const Tensor& rows) {
  const int64_t N = weights.size(0), K = weights.size(1);
  Outputs out(M, weights);
  const size_t bytes = fsgs_neighbour_balance_workspace_bytes(N, (int) M);
  const Tensor ws = empty({(int64_t) bytes}, weights, at::kByte);
  check(fsgs_neighbour_balance_forward(N, (int) M, (int) K, f32(weights), i64(indices), data<uint8_t>(rows), f32(out.loss), i32(out.counts),
                                       f32(out.importance), out.totals(), ws.data_ptr(), bytes, stream_of(weights)),
        "neighbour_balance");
  return out;
}

// Upstream gradients of (loss, counts, importance): float32, dense; the counts have none.
struct Upstream {
  Tensor loss, importance;
  explicit Upstream(const variable_list& g) : loss(contiguous(g[0])), importance(contiguous(g[2])) {}
  bool any() const { return loss.defined() || importance.defined(); }
  void check_types(const char* what) const {
    if (loss.defined()) require(what, "grad of the loss", loss, at::kFloat);
    if (importance.defined()) require(what, "grad of the importance", importance, at::kFloat);
  }
};

struct RowsNode : public torch::autograd::Function<RowsNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, int64_t K, const OptTensor& rows) {
    const Outputs out = rows_forward(logits, K, opt(rows), true);
    ctx->save_for_backward({logits, out.saved, out.counts});
    ctx->mark_non_differentiable({out.counts});
    ctx->set_materialize_grads(false);
    return {out.loss, out.counts, out.importance};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const char* what = "balance_loss_backward";
    refuse_backward_into_eager(what);
    const Upstream up(g);
    if (!up.any()) return variable_list(3);
    const auto t = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView no_graph;
    const Tensor logits = rows_of(t[0]);  // a hook may hand it back in another layout
    const Tensor &saved = t[1], &counts = t[2];
    const c10::DeviceGuard guard(logits.device());
    up.check_types(what);
    const Tensor grad = at::empty(logits.sizes(), logits.options());
    if (grad.numel() > 0)
      check(fsgs_balance_loss_backward(logits.size(0), (int) logits.size(1), stride_of(logits), logits_code(logits.scalar_type()),
                                       logits.data_ptr(), (const float*) (data<uint8_t>(saved) + 16), i32(counts), data<int64_t>(saved), f32(up.loss), f32(up.importance),
                                       grad.data_ptr(), stream_of(logits)),
            what);
    return first_order_only(g, {t[0]}, {grad, Tensor(), Tensor()});
  }
};

struct NeighboursNode : public torch::autograd::Function<NeighboursNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& weights, const Tensor& indices, int64_t M, const OptTensor& rows) {
    const Outputs out = neighbours_forward(weights, indices, M, opt(rows));
    ctx->save_for_backward({indices, opt(rows), out.saved, out.counts});
    ctx->saved_data["M"] = M;
    ctx->mark_non_differentiable({out.counts});
    ctx->set_materialize_grads(false);
    return {out.loss, out.counts, out.importance};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const char* what = "neighbour_balance_backward";
    refuse_backward_into_eager(what);
    const Upstream up(g);
    if (!up.any()) return variable_list(4);
    const auto t = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView no_graph;
    const Tensor indices = t[0].contiguous(), rows = contiguous(t[1]);
    const Tensor &saved = t[2], &counts = t[3];
    const c10::DeviceGuard guard(indices.device());
    up.check_types(what);
    const Tensor grad = empty(indices.sizes(), saved);
    if (grad.numel() > 0)
      check(fsgs_neighbour_balance_backward(indices.size(0), (int) ctx->saved_data["M"].toInt(), (int) indices.size(1), i64(indices),
                                            data<uint8_t>(rows), i32(counts), data<int64_t>(saved), f32(up.loss), f32(up.importance), f32(grad),
                                            stream_of(indices)),
            what);
    return first_order_only(g, {}, {grad, Tensor(), Tensor(), Tensor()});
  }
};

}  // namespace

std::tuple<Tensor, Tensor, Tensor> balance_loss(const Tensor& logits, int64_t K, const OptTensor& rows) {
  const char* what = "balance_loss";
  refuse_duals(what, logits);
  if (!logits.defined() || !logits.is_cuda() || logits.layout() != at::kStrided) fail("balance_loss: logits must be a CUDA tensor");
  (void) logits_code(logits.scalar_type());
  if (logits.dim() != 2 || logits.size(1) < 1) fail("balance_loss: logits must be [N, M] with M >= 1");
  require_sizes(what, logits.size(0), logits.size(1));
  const Tensor on = contiguous(opt(rows));
  require_rows(what, on, logits);
  if (K < 1 || K > logits.size(1) || K > fsgs_balance_max_choices())
    fail("balance_loss: K must be in [1, min(M, " + std::to_string(fsgs_balance_max_choices()) + ")], got " + std::to_string(K));
  const c10::DeviceGuard guard(logits.device());
  const Tensor x = rows_of(logits);
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    refuse_capture_beside_eager(what, "logits", logits);
    const variable_list out = RowsNode::apply(x, K, given(on));
    return {out[0], out[1], out[2]};
  }
  const Outputs out = rows_forward(x, K, on, false);
  return {out.loss, out.counts, out.importance};
}

std::tuple<Tensor, Tensor, Tensor> neighbour_balance(const Tensor& weights, const Tensor& indices, int64_t M, const OptTensor& rows) {
  const char* what = "neighbour_balance";
  refuse_duals(what, weights);
  const Tensor w = contiguous(weights), index = contiguous(indices), on = contiguous(opt(rows));
  require(what, "weights", w, at::kFloat), require(what, "indices", index, at::kLong);
  if (w.dim() != 2 || w.size(1) < 1 || w.size(1) > INT_MAX) fail("neighbour_balance: weights must be [N, K] with K >= 1");
  require_shape(what, "indices", index, w.sizes());
  if (index.device() != w.device()) fail("neighbour_balance: all tensors of a call must be on one device");
  require_rows(what, on, w);
  if (M < 1) fail("neighbour_balance: M must be positive");
  require_sizes(what, w.size(0), M);
  const c10::DeviceGuard guard(w.device());
  if (at::GradMode::is_enabled() && w.requires_grad()) {
    refuse_capture_beside_eager(what, "weights", weights);
    const variable_list out = NeighboursNode::apply(w, index, M, given(on));
    return {out[0], out[1], out[2]};
  }
  const Outputs out = neighbours_forward(w, index, M, on);
  return {out.loss, out.counts, out.importance};
}

}  // namespace fsgs_host
