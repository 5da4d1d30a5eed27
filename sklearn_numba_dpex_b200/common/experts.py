"""Mixture of experts around the experts' own products: routing of tokens, the expert order of the
chosen rows, and the weighted sum back to the tokens.  The reference has none of these; routing keeps
the order rule of `topk` (descending, lowest index among equals).

A layer whose experts multiply in 8 bits reads::

    weights, experts = route_topk(logits, k)
    slots, rows, offsets = expert_slots(experts, n_experts)
    q, scales = quantize_rows(x, rows=rows)
    y = int8_matmul(q, scales, w, w_scales, offsets=offsets)      # w (n_experts, n, d) int8
    out = combine_experts(y, slots, weights)

All tensors live on one CUDA device; a call is enqueued on that device's current stream.
"""
import torch

from .._cabi import ROUTE_RENORMALIZE, ROUTE_SIGMOID, launch, lib, require_cuda_tensor, row_dtype_code

_SCORINGS = {"softmax": 0, "sigmoid": ROUTE_SIGMOID}


def _matrix(t, name, dtype=None):
    require_cuda_tensor(t, name, dtype, contiguous=False)
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, got {t.dim()}")
    return t if t.is_contiguous() else t.contiguous()


def _same_device(t, name, other):
    if t.device != other.device:
        raise ValueError(f"{name} must be on {other.device}, got {t.device}")


def _flags(scoring, renormalize):
    if scoring not in _SCORINGS:
        raise ValueError(f"scoring must be one of {sorted(_SCORINGS)}, got {scoring!r}")
    return _SCORINGS[scoring] | (ROUTE_RENORMALIZE if renormalize else 0)


# ------------------------------------------------------------------------------- routing
def _route(logits, k, bias, flags, n_groups, topk_groups, group_best, scale):
    n, e = logits.shape
    dev = logits.device
    weights = torch.empty((n, k), dtype=torch.float32, device=dev)
    experts = torch.empty((n, k), dtype=torch.int32, device=dev)
    launch("kmb_route_topk", dev, row_dtype_code(logits.dtype, "logits"), logits.data_ptr(),
           None if bias is None else bias.data_ptr(), n, e, k, flags, n_groups, topk_groups, group_best, scale,
           weights.data_ptr(), experts.data_ptr())
    return weights, experts


class _RouteTopk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, bias, scoring, n_groups, topk_groups, group_best, renormalize, scale):
        weights, experts = _route(logits, k, bias, _flags(scoring, renormalize), n_groups, topk_groups,
                                  group_best, scale)
        ctx.save_for_backward(logits, experts)
        ctx.settings = (scoring, renormalize, scale)
        ctx.mark_non_differentiable(experts)
        return weights, experts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_weights, _):
        logits, experts = ctx.saved_tensors
        scoring, renormalize, scale = ctx.settings
        grad = route_topk_grad(logits, experts, grad_weights, scoring, renormalize, scale)
        return (grad,) + (None,) * 8


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
    logits = _matrix(logits, "logits")
    if bias is not None:
        require_cuda_tensor(bias, "bias", torch.float32)
        _same_device(bias, "bias", logits)
        if bias.shape != (logits.shape[1],):
            raise ValueError(f"bias must have shape ({logits.shape[1]},), got {tuple(bias.shape)}")
    k, n_groups = int(k), int(n_groups)
    topk_groups = n_groups if topk_groups is None else int(topk_groups)
    if k < 1:
        raise ValueError(f"k must be at least 1, got {k}")
    if torch.is_grad_enabled() and logits.requires_grad:
        return _RouteTopk.apply(logits, k, bias, scoring, n_groups, topk_groups, int(group_best),
                                bool(renormalize), float(scale))
    return _route(logits, k, bias, _flags(scoring, renormalize), n_groups, topk_groups, int(group_best),
                  float(scale))


def route_topk_grad(logits, experts, grad_weights, scoring="softmax", renormalize=True, scale=1.0):
    """Gradient of the weights of `route_topk` to its logits (n, n_experts), in their dtype, for callers
    that keep their own backward pass; `experts` is what `route_topk` returned."""
    logits = _matrix(logits, "logits")
    experts = _matrix(experts, "experts", torch.int32)
    grad_weights = _matrix(grad_weights, "grad_weights", torch.float32)
    n, e = logits.shape
    if experts.shape[0] != n or grad_weights.shape != experts.shape:
        raise ValueError(f"experts and grad_weights must both have shape ({n}, k), got {tuple(experts.shape)} "
                         f"and {tuple(grad_weights.shape)}")
    _same_device(experts, "experts", logits)
    _same_device(grad_weights, "grad_weights", logits)
    grad = torch.empty_like(logits)
    launch("kmb_route_topk_grad", logits.device, row_dtype_code(logits.dtype, "logits"), logits.data_ptr(),
           experts.data_ptr(), grad_weights.data_ptr(), n, e, experts.shape[1], _flags(scoring, renormalize),
           float(scale), grad.data_ptr())
    return grad


# --------------------------------------------------------------------------- expert order
def expert_slots(experts, n_experts):
    """Where the choices of `route_topk` go when they are sorted by expert, token order kept.

    `experts` (n, k) int32.  Returns int32 tensors ``(slots, rows, offsets)``: `slots` (n, k) is the place
    of each choice, `rows` (n * k) the token in each place, and expert e has the places
    ``offsets[e]:offsets[e + 1]``.  A choice that is no expert (-1) has slot -1 and takes no place; the
    places behind ``offsets[n_experts]`` then hold -1.  Nothing waits for the GPU.
    """
    experts = _matrix(experts, "experts", torch.int32)
    n, k = experts.shape
    n_experts = int(n_experts)
    if k < 1:
        raise ValueError("experts must have at least one column")
    dev = experts.device
    slots = torch.empty_like(experts)
    rows = torch.empty(n * k, dtype=torch.int32, device=dev)
    offsets = torch.empty(max(n_experts, 0) + 1, dtype=torch.int32, device=dev)
    nbytes = lib.kmb_expert_slots_workspace_bytes(n, k, n_experts)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    launch("kmb_expert_slots", dev, experts.data_ptr(), n, k, n_experts, slots.data_ptr(), rows.data_ptr(),
           offsets.data_ptr(), ws.data_ptr() if nbytes else None, nbytes)
    return slots, rows, offsets


# --------------------------------------------------------------------------- weighted sums
def _combine_args(values, slots, weights):
    values = _matrix(values, "values")
    slots = _matrix(slots, "slots", torch.int32)
    weights = _matrix(weights, "weights", torch.float32)
    if weights.shape != slots.shape:
        raise ValueError(f"weights must have the shape of slots {tuple(slots.shape)}, got {tuple(weights.shape)}")
    _same_device(slots, "slots", values)
    _same_device(weights, "weights", values)
    return values, slots, weights


def _combine(values, slots, weights):
    n, k = slots.shape
    dev = values.device
    out = torch.empty((n, values.shape[1]), dtype=values.dtype, device=dev)
    launch("kmb_combine_experts", dev, row_dtype_code(values.dtype, "values"), values.data_ptr(), values.shape[0],
           slots.data_ptr(), weights.data_ptr(), n, k, values.shape[1], out.data_ptr())
    return out


class _CombineExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, values, slots, weights):
        ctx.save_for_backward(values, slots, weights)
        return _combine(values, slots, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_out):
        grad_values, grad_weights = combine_experts_grad(*ctx.saved_tensors, grad_out)
        return grad_values, None, grad_weights


def combine_experts(values, slots, weights):
    """``out[t] = sum_j weights[t, j] * values[slots[t, j]]``: the experts' rows `values` (m, d), in expert
    order, back to the n tokens.

    `slots` (n, k) int32 and `weights` (n, k) float32 are those of `expert_slots` and `route_topk`; a
    slot outside ``[0, m)`` adds nothing.  Sums are held in 32 bits; the result has the dtype of `values`
    (float32, float16 or bfloat16).  Differentiable in `values` and `weights`.
    """
    values, slots, weights = _combine_args(values, slots, weights)
    if torch.is_grad_enabled() and (values.requires_grad or weights.requires_grad):
        return _CombineExperts.apply(values, slots, weights)
    return _combine(values, slots, weights)


def combine_experts_grad(values, slots, weights, grad_out):
    """``(grad_values, grad_weights)`` of `combine_experts`, for callers that keep their own backward pass.
    Rows of `values` that several slots name get the sum of their gradients, in a fixed order; rows that
    none names get zeros."""
    values, slots, weights = _combine_args(values, slots, weights)
    grad_out = _matrix(grad_out, "grad_out", values.dtype)
    n, k = slots.shape
    if grad_out.shape != (n, values.shape[1]):
        raise ValueError(f"grad_out must have shape ({n}, {values.shape[1]}), got {tuple(grad_out.shape)}")
    _same_device(grad_out, "grad_out", values)
    dev = values.device
    grad_values, grad_weights = torch.empty_like(values), torch.empty_like(weights)
    nbytes = lib.kmb_combine_experts_grad_workspace_bytes(values.shape[0])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    launch("kmb_combine_experts_grad", dev, row_dtype_code(values.dtype, "values"), values.data_ptr(),
           values.shape[0], slots.data_ptr(), weights.data_ptr(), grad_out.data_ptr(), n, k, values.shape[1],
           grad_values.data_ptr(), grad_weights.data_ptr(), ws.data_ptr(), nbytes)
    return grad_values, grad_weights
