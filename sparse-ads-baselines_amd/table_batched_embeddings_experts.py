"""Expert routing: the rows of tokens in the order of the experts they chose, and back, with weights
applied, and the gradients of both -- the routed part of a mixture-of-experts layer, for example on top of
the embedding bags' outputs.  No counterpart in the reference.

    routing = ExpertRouting(expert_ids, num_experts)     # [tokens, choices] int32 or int64, as torch.topk gives them
    rows = routing.dispatch(x)                           # [tokens * choices, D], expert e's at
                                                         # expert_offsets[e] : expert_offsets[e + 1]
    rows = ...                                           # the experts, on their rows
    y = routing.combine(rows, gate_weights)              # [tokens, D]

A pair whose expert lies outside [0, num_experts) is dropped: it takes part in nothing.  All of it stays on
the device; nothing synchronises, so the calls can be captured in a graph.  Each call validates its tensors
and hands raw device pointers and the current stream to the C-ABI library (include/tbe_hip.h); the gradients
are the library's kernels too.
"""
import torch

import tbe_native as _native
from table_batched_embeddings import _ptr, _require, _stream

_DTYPE_CODES = {torch.float32: _native.DTYPE_F32, torch.float16: _native.DTYPE_F16, torch.float64: _native.DTYPE_F64,
                torch.bfloat16: _native.DTYPE_BF16}


def _check_rows(name, rows, num_rows=None):
    _require(rows.is_cuda, "%s must be a GPU tensor" % name)
    _require(rows.dim() == 2 and rows.size(1) > 0, "%s must be a [rows, D] tensor with D > 0" % name)
    _require(rows.dtype in _DTYPE_CODES, "%s must be float16, bfloat16, float32 or float64" % name)
    _require(num_rows is None or rows.size(0) == num_rows, "%s must have %s rows" % (name, num_rows))
    # rows at any distance from each other are read in place; anything else is laid out first
    return rows if rows.stride(1) == 1 and rows.stride(0) >= 0 else rows.contiguous()


def _check_plan(places, expert_offsets, device):
    for name, t, dim in (("places", places, 2), ("expert_offsets", expert_offsets, 1)):
        _require(t.dtype == torch.int32, "%s must be int32 (got %s)" % (name, t.dtype))
        _require(t.device == device, "%s must live on the rows' device" % name)
        _require(t.dim() == dim and t.is_contiguous(), "%s must be a contiguous %d-D tensor" % (name, dim))
    _require(places.size(1) > 0, "places must be [tokens, choices] with choices > 0")
    _require(expert_offsets.numel() > 1, "expert_offsets must hold num_experts + 1 entries")
    return places.size(0), places.size(1), expert_offsets.numel() - 1


def _check_weights(weights, rows, places):
    _require(weights.dtype in (rows.dtype, torch.float32), "weights must be float32 or have the rows' dtype")
    _require(weights.device == rows.device, "weights must live on the rows' device")
    _require(weights.shape == places.shape, "weights must be [tokens, choices]")
    return weights.contiguous()


def expert_plan(expert_ids, num_experts):
    """The stable order of the (token, choice) pairs by expert: (expert_offsets [num_experts + 1], order
    [tokens * choices], places [tokens, choices]), all int32.  expert_offsets[e] is the first row of expert e,
    expert_offsets[-1] the number of pairs kept; order[r] is the pair (token * choices + choice) of row r and
    places the row of every pair; the dropped pairs come last."""
    _require(expert_ids.is_cuda, "expert_ids must be a GPU tensor")
    _require(expert_ids.dtype in (torch.int32, torch.int64), "expert_ids must be int32 or int64 (got %s)" %
             expert_ids.dtype)
    _require(expert_ids.dim() == 2 and expert_ids.size(1) > 0, "expert_ids must be [tokens, choices] with choices > 0")
    expert_ids = expert_ids.contiguous()
    num_experts = int(num_experts)
    _require(0 < num_experts <= _native.MAX_EXPERTS, "num_experts must be 1 to %d (got %d)" %
             (_native.MAX_EXPERTS, num_experts))
    pairs = expert_ids.numel()
    _require(pairs < 2 ** 31 - 1, "tokens * choices must stay below 2^31 - 1")
    device = expert_ids.device
    lib = _native.load()
    nbytes = lib.tbe_expert_plan_workspace_bytes(pairs, num_experts)
    expert_offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=device)
    order = torch.empty(pairs, dtype=torch.int32, device=device)
    places = torch.empty(expert_ids.shape, dtype=torch.int32, device=device)
    # scratch of this call alone: two graphs captured on one stream do not share it
    scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
    with torch.cuda.device(device):
        _native.check(lib.tbe_expert_plan(
            _ptr(expert_ids), expert_ids.element_size(), pairs, num_experts, _ptr(expert_offsets), _ptr(order),
            _ptr(places), _ptr(scratch), nbytes, _stream(device)))
    return expert_offsets, order, places


def _dispatch(tokens, places, expert_offsets):
    tokens = _check_rows("tokens", tokens)
    n, choices, experts = _check_plan(places, expert_offsets, tokens.device)
    _require(tokens.size(0) == n, "tokens must have one row per row of places")
    D = tokens.size(1)
    rows = torch.empty((n * choices, D), dtype=tokens.dtype, device=tokens.device)
    with torch.cuda.device(tokens.device):
        _native.check(_native.load().tbe_expert_dispatch(
            _ptr(tokens), tokens.stride(0), _DTYPE_CODES[tokens.dtype], n, choices, experts, D, _ptr(places),
            _ptr(expert_offsets), _ptr(rows), _stream(tokens.device)))
    return rows


def _combine(rows, places, expert_offsets, weights):
    rows = _check_rows("rows", rows, places.numel())
    n, choices, experts = _check_plan(places, expert_offsets, rows.device)
    if weights is not None:
        weights = _check_weights(weights, rows, places)
    output = torch.empty((n, rows.size(1)), dtype=rows.dtype, device=rows.device)
    with torch.cuda.device(rows.device):
        _native.check(_native.load().tbe_expert_combine(
            _ptr(rows), rows.stride(0), _DTYPE_CODES[rows.dtype], n, choices, experts, rows.size(1), _ptr(places),
            _ptr(expert_offsets), _ptr(weights), _DTYPE_CODES[rows.dtype if weights is None else weights.dtype],
            _ptr(output), _stream(rows.device)))
    return output


def _combine_backward(grad_output, rows, places, expert_offsets, weights):
    rows = _check_rows("rows", rows, places.numel())
    n, choices, experts = _check_plan(places, expert_offsets, rows.device)
    weights = _check_weights(weights, rows, places)
    _require(grad_output.dtype == rows.dtype, "grad_output must have the rows' dtype")
    _require(grad_output.device == rows.device, "grad_output must live on the rows' device")
    _require(tuple(grad_output.shape) == (n, rows.size(1)), "grad_output must be [tokens, D]")
    grad_output = _check_rows("grad_output", grad_output)
    grad_rows = torch.empty((rows.size(0), rows.size(1)), dtype=rows.dtype, device=rows.device)
    grad_weights = torch.empty_like(weights)
    with torch.cuda.device(rows.device):
        _native.check(_native.load().tbe_expert_combine_backward(
            _ptr(grad_output), grad_output.stride(0), _ptr(rows), rows.stride(0), _DTYPE_CODES[rows.dtype], n, choices,
            experts, rows.size(1), _ptr(places), _ptr(expert_offsets), _ptr(weights), _DTYPE_CODES[weights.dtype],
            _ptr(grad_rows), _ptr(grad_weights), _stream(rows.device)))
    return grad_rows, grad_weights


class _DispatchFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, places, expert_offsets):
        ctx.save_for_backward(places, expert_offsets)
        return _dispatch(tokens, places, expert_offsets)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_rows):
        places, expert_offsets = ctx.saved_tensors
        return _combine(grad_rows, places, expert_offsets, None), None, None


class _CombineFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, places, expert_offsets, weights):
        ctx.weighted = weights is not None
        if ctx.weighted:
            ctx.save_for_backward(rows, places, expert_offsets, weights)
        else:
            ctx.save_for_backward(places, expert_offsets)
        return _combine(rows, places, expert_offsets, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        if not ctx.weighted:
            return _dispatch(grad_output, *ctx.saved_tensors), None, None, None
        rows, places, expert_offsets, weights = ctx.saved_tensors
        grad_rows, grad_weights = _combine_backward(grad_output, rows, places, expert_offsets, weights)
        return grad_rows, None, None, grad_weights


def expert_dispatch(tokens, places, expert_offsets):
    """The rows of `tokens` ([tokens, D]) in expert order: row places[t, j] is tokens[t]; zeros behind the
    last expert's rows.  Differentiable with respect to `tokens` (a token's gradient is the sum of its kept
    rows', added up in 32 bits, or 64 for float64)."""
    return _DispatchFunction.apply(tokens, places, expert_offsets)


def expert_combine(rows, places, expert_offsets, weights=None):
    """[tokens, D]: the sum over a token's kept pairs of weights[t, j] * rows[places[t, j]] (weights None:
    ones), added up in 32 bits (64 for float64) and rounded once.  Differentiable with respect to `rows` and
    `weights` (float32, or the rows' dtype)."""
    return _CombineFunction.apply(rows, places, expert_offsets, weights)


class ExpertRouting:
    """The plan of one batch -- expert_offsets, order and places of expert_plan() -- and the two row
    movements that follow it."""

    def __init__(self, expert_ids, num_experts):
        self.num_experts = int(num_experts)
        self.expert_offsets, self.order, self.places = expert_plan(expert_ids, num_experts)

    def dispatch(self, tokens):
        return expert_dispatch(tokens, self.places, self.expert_offsets)

    def combine(self, rows, weights=None):
        return expert_combine(rows, self.places, self.expert_offsets, weights)
