// What the source files of the pybind11 module table_batched_embeddings_cpp share.
#pragma once

#include <torch/extension.h>

#include <utility>

#include "tbe_hip.h"

namespace tbe_binding {

// Turns a non-zero return code into RuntimeError with the library's message.
void check(int rc);
// The current stream of the tensor's device.
void *stream_of(const at::Tensor &t);
// Address of the tensor's first element, null if there is no tensor.
const void *ptr(const c10::optional<at::Tensor> &t);

struct Shape {
  int32_t T, B, D;
  int64_t n, rows;
};
Shape check_common(const at::Tensor &weights, const at::Tensor &table_offsets, const at::Tensor &indices,
                   const at::Tensor &offsets);
at::Tensor check_grad(const at::Tensor &grad_output, const at::Tensor &weights, const Shape &s);
void check_weights_of_lookups(const c10::optional<at::Tensor> &indice_weights, const at::Tensor &weights,
                              const at::Tensor &indices);
void check_state(const at::Tensor &optimizer_state, const at::Tensor &weights);
int32_t dtype_code(const at::Tensor &t);
int64_t max_table_rows(const at::Tensor &starts_tensor, int64_t total_rows);
std::pair<uint64_t, uint64_t> rounding_stream(const at::Tensor &t);

// Expert routing, gradient clipping and the clipped table updates (table_batched_embeddings_training.cpp).
void bind_training(pybind11::module &m);

}  // namespace tbe_binding
