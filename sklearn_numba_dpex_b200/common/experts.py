"""Mixture of experts around the experts' own products: routing of tokens, the expert order of the
chosen rows, and the weighted sum back to the tokens.  The reference has none of these; routing keeps
the order rule of `topk` (descending, lowest index among equals).

A layer whose experts multiply in 8 bits reads::

    weights, experts = route_topk(logits, k)
    slots, rows, offsets = expert_slots(experts, n_experts)
    q, scales = quantize_rows(x.detach(), rows=rows)              # no gradient through 8 bits
    y = int8_matmul(q, scales, w, w_scales, offsets=offsets)      # w (n_experts, n, d) int8
    out = combine_experts(y, slots, weights)

All tensors live on one CUDA device; a call is enqueued on that device's current stream, waits for nothing
and can be captured into a CUDA graph.  `route_topk` and `combine_experts` are differentiable; a backward pass that
is to be captured calls `route_topk_grad` and `combine_experts_grad` itself, since autograd's own nodes belong to
the stream that first used their leaves.  Forward mode and the transforms of `torch.func` are refused with an error.
"""
import torch

from .._cabi import ROUTE_RENORMALIZE, ROUTE_SIGMOID
from . import _calls

_SCORINGS = {"softmax": 0, "sigmoid": ROUTE_SIGMOID}


def _flags(scoring, renormalize):
    if scoring not in _SCORINGS:
        raise ValueError(f"scoring must be one of {sorted(_SCORINGS)}, got {scoring!r}")
    return _SCORINGS[scoring] | (ROUTE_RENORMALIZE if renormalize else 0)


# ------------------------------------------------------------------------------- routing
class _RouteTopk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, bias, flags, n_groups, topk_groups, group_best, scale):
        weights, experts = _calls.route_topk(logits, k, bias, flags, n_groups, topk_groups, group_best, scale)
        ctx.save_for_backward(logits, experts)
        ctx.settings = (flags, scale)
        ctx.mark_non_differentiable(experts)
        return weights, experts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_weights, _):
        logits, experts = ctx.saved_tensors
        return (_calls.route_topk_grad(logits, experts, grad_weights, *ctx.settings),) + (None,) * 7


def route_topk(logits, k, bias=None, scoring="softmax", n_groups=1, topk_groups=None, group_best=1,
               renormalize=True, scale=1.0):
    """The `k` experts of each token and their weights.

    `logits` (n, n_experts) in float32, float16 or bfloat16; at most 1024 experts, `k` at most 32.
    Scores are the softmax over a token's logits or (``scoring="sigmoid"``) the sigmoid of each.  The choice
    goes by score + `bias` (n_experts float32; a bias for balance, which gets no gradient and does not enter
    the weights), greatest first, lowest index among equals, NaN greatest.  With `n_groups` > 1 the experts
    fall into consecutive groups; a group's score is the sum of its `group_best` (1 or 2) best, and the
    choice is made in the `topk_groups` best groups (None: in all).  Values that lie too near to each other
    for 32 bits are ordered in 64.

    Returns ``(weights (n, k) float32, experts (n, k) int32)``: weights are `scale` times the chosen scores,
    divided by their sum if `renormalize`.  An expert whose logit or key is -inf is never chosen (a way
    to mask experts, or whole padding tokens); a place without an expert holds expert -1 and weight 0.

    Differentiable in `logits`, the choice being held fixed.
    """
    flags = _flags(scoring, renormalize)
    topk_groups = n_groups if topk_groups is None else topk_groups
    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        return _RouteTopk.apply(logits, k, bias, flags, n_groups, topk_groups, group_best, scale)
    return _calls.route_topk(logits, k, bias, flags, n_groups, topk_groups, group_best, scale)


def route_topk_grad(logits, experts, grad_weights, scoring="softmax", renormalize=True, scale=1.0):
    """Gradient of the weights of `route_topk` to its logits (n, n_experts), in their dtype, for callers
    that keep their own backward pass; `experts` is what `route_topk` returned."""
    return _calls.route_topk_grad(logits, experts, grad_weights, _flags(scoring, renormalize), scale)


# --------------------------------------------------------------------------- expert order
def expert_slots(experts, n_experts):
    """Where the choices of `route_topk` go when they are sorted by expert, token order kept.

    `experts` (n, k) int32.  Returns int32 tensors ``(slots, rows, offsets)``: `slots` (n, k) is the place
    of each choice, `rows` (n * k) the token in each place, and expert e has the places
    ``offsets[e]:offsets[e + 1]``.  A choice that is no expert (-1) has slot -1 and takes no place; the
    places behind ``offsets[n_experts]`` then hold -1.  Nothing waits for the GPU.
    """
    return _calls.expert_slots(experts, n_experts)


# --------------------------------------------------------------------------- weighted sums
class _CombineExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, values, slots, weights):
        ctx.save_for_backward(values, slots, weights)
        return _calls.combine_experts(values, slots, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        grad_values, grad_weights = _calls.combine_experts_grad(*ctx.saved_tensors, grad_out)
        return grad_values, None, grad_weights


def combine_experts(values, slots, weights):
    """``out[t] = sum_j weights[t, j] * values[slots[t, j]]``: the experts' rows `values` (m, d), in expert
    order, back to the n tokens.

    `slots` (n, k) int32 and `weights` (n, k) float32 are those of `expert_slots` and `route_topk`; a
    slot outside ``[0, m)`` adds nothing.  Sums are held in 32 bits; the result has the dtype of `values`
    (float32, float16 or bfloat16).  Differentiable in `values` and `weights`.
    """
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (values, weights)):
        return _CombineExperts.apply(values, slots, weights)
    return _calls.combine_experts(values, slots, weights)


def combine_experts_grad(values, slots, weights, grad_out):
    """``(grad_values, grad_weights)`` of `combine_experts`, for callers that keep their own backward pass.
    Rows of `values` that several slots name get the sum of their gradients, in a fixed order; rows that
    none names get zeros."""
    return _calls.combine_experts_grad(values, slots, weights, grad_out)
