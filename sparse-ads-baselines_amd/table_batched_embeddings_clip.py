"""The global norm of gradients and clipping to it: for lists of dense gradients (what surrounds the tables),
and for the exact gradient of a batch's tables, which is never stored -- the fused updates apply it row by row.

Squares are added up in 64 bits and the norm is rounded once, to float32 (float64 if a gradient is float64); the
scale is min(1, max_norm / (norm + 1e-6)).  Nothing synchronises unless a caller asks for an error: the norm is
a tensor on the device.  Like torch.nn.utils.clip_grad_norm_, these functions take no part in autograd: norms carry
no graph.  Checks and outputs are those of the compiled module (table_batched_embeddings_cpp) over
the C-ABI library (include/tbe_hip.h).
"""
import torch

from tbe_native import compiled


def gradient_norm(gradients):
    """The norm over all elements of a list of GPU tensors (float16, bfloat16, float32, float64, mixed ones
    among them), as a 0-dim tensor."""
    return compiled().gradient_norm(gradients)


def clip_gradients(gradients, max_norm, out=None):
    """Scales the gradients so that their global norm is at most max_norm, in place or into the tensors of
    `out` (same shapes, strides and types); returns the norm they had.  The tensors are dense, in any order of
    their dimensions; two of a list may not share memory.  In place, nothing is written while the norm is
    within max_norm.  As for torch.nn.utils.clip_grad_norm_, a norm that is not a number makes every gradient one,
    and an infinite one makes finite gradients zero."""
    return compiled().clip_gradients(gradients, max_norm, out)


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ for models with embedding bags among their parameters: the bags' tables are
    updated inside backward and hand autograd an empty sparse gradient, which is passed over here (to clip the
    tables' own gradient see TableBatchedEmbeddingBags.clip_gradient).  error_if_nonfinite=True waits for the
    device and raises before anything is scaled."""
    if float(norm_type) != 2.0:
        raise RuntimeError("clip_grad_norm_ serves the 2-norm (got norm_type=%s)" % norm_type)
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    gradients = []
    for p in parameters:
        g = p.grad
        if g is None:
            continue
        if g.layout != torch.strided:
            if g.layout == torch.sparse_coo and g._nnz() == 0:
                continue
            raise RuntimeError("clip_grad_norm_ takes dense gradients (got %s)" % g.layout)
        gradients.append(g)
    if not gradients:
        return torch.tensor(0.0)
    if error_if_nonfinite and not bool(torch.isfinite(gradient_norm(gradients))):
        raise RuntimeError("the total norm of the gradients is not finite, so it cannot be clipped")
    return clip_gradients(gradients, float(max_norm))


def clip_table_gradient(grad_output, weights, table_offsets, indices, offsets, max_norm, indice_weights=None):
    """For a batch of TableBatchedEmbeddingBags: (grad_output scaled, norm).  The norm is that of the tables'
    exact gradient -- for every distinct (table, index) the sum over its lookups of (indice_weights *)
    grad_output of the lookup's bag -- and the scaled grad_output is the one whose gradient has a norm of at most
    max_norm, up to the rounding of its elements to their type.  For fp16 that rounding counts: an element may be off
    by half a step, 2**-11 of its value, and below 2**-14 by 2**-25 whatever its value, down to zero, so that a gradient
    scaled far down, and summed over many lookups of a row, may exceed max_norm or vanish (a module's clip_gradient
    does not go through such a copy)."""
    return compiled().clip_table_gradient(grad_output, weights, table_offsets, indices, offsets, max_norm,
                                          indice_weights)
