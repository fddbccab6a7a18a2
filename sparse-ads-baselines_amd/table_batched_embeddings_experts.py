"""Expert routing: the rows of tokens in the order of the experts they chose, and back, with weights
applied, and the gradients of both -- the routed part of a mixture-of-experts layer, for example on top of
the embedding bags' outputs.  No counterpart in the reference.

    routing = ExpertRouting(expert_ids, num_experts)     # [tokens, choices] int32 or int64, as torch.topk gives them
    rows = routing.dispatch(x)                           # [tokens * choices, D], expert e's at
                                                         # expert_offsets[e] : expert_offsets[e + 1]
    rows = ...                                           # the experts, on their rows
    y = routing.combine(rows, gate_weights)              # [tokens, D]

A pair whose expert lies outside [0, num_experts) is dropped: it takes part in nothing.  All of it stays on
the device; nothing synchronises, so the calls can be captured in a graph.  Checks, outputs and gradients are
those of the compiled module (table_batched_embeddings_cpp) over the C-ABI library (include/tbe_hip.h).
"""
from tbe_native import compiled


def expert_plan(expert_ids, num_experts):
    """The stable order of the (token, choice) pairs by expert: (expert_offsets [num_experts + 1], order
    [tokens * choices], places [tokens, choices]), all int32.  expert_offsets[e] is the first row of expert e,
    expert_offsets[-1] the number of pairs kept; order[r] is the pair (token * choices + choice) of row r and
    places the row of every pair; the dropped pairs come last."""
    return compiled().expert_plan(expert_ids, num_experts)


def expert_dispatch(tokens, places, expert_offsets):
    """The rows of `tokens` ([tokens, D]) in expert order: row places[t, j] is tokens[t]; zeros behind the
    last expert's rows.  `places` is a plan's: every row is named once (rows that a caller's own places leave out
    are not written, and of two pairs that name one row either may win).  Differentiable with respect to `tokens`, once (a token's gradient is the sum of its
    kept rows', added up in 32 bits, or 64 for float64)."""
    return compiled().expert_dispatch(tokens, places, expert_offsets)


def expert_combine(rows, places, expert_offsets, weights=None):
    """[tokens, D]: the sum over a token's kept pairs of weights[t, j] * rows[places[t, j]] (weights None:
    ones), added up in 32 bits (64 for float64) and rounded once.  Differentiable with respect to `rows` and
    `weights` (float32, or the rows' dtype), once; the gradient takes `places` for a plan's, as expert_dispatch does."""
    return compiled().expert_combine(rows, places, expert_offsets, weights)


class ExpertRouting:
    """The plan of one batch -- expert_offsets, order and places of expert_plan() -- and the two row
    movements that follow it."""

    def __init__(self, expert_ids, num_experts):
        self.num_experts = num_experts
        self.expert_offsets, self.order, self.places = compiled().expert_plan(expert_ids, num_experts)

    def dispatch(self, tokens):
        return compiled().expert_dispatch(tokens, self.places, self.expert_offsets)

    def combine(self, rows, weights=None):
        return compiled().expert_combine(rows, self.places, self.expert_offsets, weights)
