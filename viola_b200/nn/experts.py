"""Routing around the expert linear: choose experts, sort the tokens by expert, bring the results back.

:class:`viola_b200.nn.GroupedLinear` takes rows sorted by expert.  The four functions here lead to it and back::

    routing = route_tokens(router(x), top_k)                 # weights, indices, counts, balance_loss, z_loss
    plan = plan_experts(routing.indices, num_experts)        # offsets, positions
    rows = dispatch_tokens(x, plan)                          # [tokens * top_k, width], sorted by expert
    rows = experts(rows, plan.offsets)                       # GroupedLinear layers
    x = combine_tokens(rows, routing.weights, plan)          # [..., width]

The four functions and their gradients never wait for the GPU, and neither does the forward pass of ``GroupedLinear``: the
row count is ``tokens * top_k`` whatever was chosen, and rows that no choice fills (tokens of a padded batch) are zero and lie
behind the last expert's.  (``GroupedLinear``'s weight gradient does wait: it reads the offsets on the host, so a training step
through expert layers cannot be captured into a CUDA graph.)  Results do not depend on the order in which the GPU runs
its blocks.  CPU tensors take the same path through the PyTorch restatements.  On the GPU the gradients cannot be
differentiated again, and inputs with forward-mode tangents are refused.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import ops

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


class Routing(NamedTuple):
    """Result of :func:`route_tokens`."""

    weights: torch.Tensor        # fp32 [..., top_k]
    indices: torch.Tensor        # int32 [..., top_k], -1 where there was nothing to choose
    counts: torch.Tensor         # int32 [experts], choices per expert
    balance_loss: torch.Tensor   # fp32 scalar, 1 for an even load
    z_loss: torch.Tensor         # fp32 scalar


class ExpertPlan(NamedTuple):
    """Result of :func:`plan_experts`: where the rows of the experts lie.

    The two belong together: every row below ``offsets[-1]`` is the row of exactly one choice, and on the GPU nothing checks
    that.  A row that no position names is left unwritten there, in :func:`dispatch_tokens` and in the gradient of
    :func:`combine_tokens`; to drop a choice, set its index to -1 before planning."""

    offsets: torch.Tensor        # int32 [experts + 1]: expert e has the rows offsets[e] .. offsets[e + 1] - 1
    positions: torch.Tensor      # int32 [tokens, top_k]: the row of every choice, -1 for none


def _float(tensor, name):
    if tensor.dtype not in _DTYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {tensor.dtype}")


def _same_device(tensor, name, other):
    if tensor.device != other.device:
        raise ValueError(f"{name} is on {tensor.device}, not on {other.device}")


def route_tokens(logits, top_k, *, bias=None, mask=None, normalize=True):
    """Chooses ``top_k`` experts for every token of ``logits`` [..., experts] (up to 1024 experts, ``top_k`` up to 32).

    With p the softmax of a token's logits and S its chosen experts, the weights are ``p_e / sum_S p`` (``normalize``) or
    ``p_e``, in fp32 whatever the logits' dtype.  S holds the largest ``fp32(logit) + bias`` (``bias``: optional fp32
    [experts], it moves the choice and nothing else; +inf counts as the largest number), the lowest index among equals; an
    expert whose logit is -inf is never chosen, and slots left over get index -1 and weight 0.  The bias is added to the
    logits, which multiplies an expert's p by ``exp(bias)``: one that was trained to be added to p, or to a sigmoid of the
    logit, chooses other experts here.  ``mask`` (bool, the leading shape) is False for padding:
    those tokens, like tokens with no logit above -inf, choose nothing and enter no sum whatever their logits hold.

    ``balance_loss = experts * sum_e f_e P_e`` with f_e the expert's share of all choices (``counts``) and P_e the mean of
    its p; ``z_loss`` is the mean squared log-sum-exp.  Gradients of the weights and of both losses reach ``logits``."""
    if logits.is_cuda:                       # checked by the operator
        return Routing(*ops.route(logits, top_k, bias=bias, mask=mask, normalize=normalize))
    if logits.dim() < 1:
        raise ValueError("logits must have an experts dimension")
    _float(logits, "logits")
    experts = logits.shape[-1]
    if not 1 <= experts <= ops.MAX_EXPERTS:
        raise ValueError(f"the number of experts must be between 1 and {ops.MAX_EXPERTS}, got {experts}")
    if not 1 <= top_k <= min(experts, ops.MAX_TOP_K):
        raise ValueError(f"top_k must be between 1 and min(experts, {ops.MAX_TOP_K}), got {top_k} for {experts} experts")
    if bias is not None:
        if bias.shape != (experts,):
            raise ValueError(f"bias must have shape ({experts},), got {tuple(bias.shape)}")
        _same_device(bias, "bias", logits)
        bias = bias.detach().float().contiguous()
    if mask is not None:
        if mask.dtype != torch.bool or mask.shape != logits.shape[:-1]:
            raise ValueError(f"mask must be bool of shape {tuple(logits.shape[:-1])}, got {mask.dtype} {tuple(mask.shape)}")
        _same_device(mask, "mask", logits)
        mask = mask.contiguous()
    return Routing(*ops.route(logits, top_k, bias=bias, mask=mask, normalize=normalize))


def plan_experts(indices, num_experts):
    """Where the choices ``indices`` (int32 or int64 [..., top_k]) go when sorted by expert, tokens in order within an
    expert.  Values outside ``0 .. num_experts - 1`` are dropped: they take no row."""
    if indices.is_cuda:
        return ExpertPlan(*ops.expert_plan(indices, num_experts))
    if indices.dim() < 1 or indices.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"indices must be int32 or int64 [..., top_k], got {indices.dtype} {tuple(indices.shape)}")
    if not 1 <= num_experts <= ops.MAX_EXPERTS:
        raise ValueError(f"the number of experts must be between 1 and {ops.MAX_EXPERTS}, got {num_experts}")
    if not 1 <= indices.shape[-1] <= ops.MAX_TOP_K:
        raise ValueError(f"indices must hold between 1 and {ops.MAX_TOP_K} choices per token, got {indices.shape[-1]}")
    return ExpertPlan(*ops.expert_plan(indices, num_experts))


def _check_plan(plan, tensor, name):
    offsets, positions = plan
    if (positions.dtype != torch.int32 or positions.dim() != 2 or not 1 <= positions.shape[1] <= ops.MAX_TOP_K
            or offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.numel() < 2):
        raise ValueError("plan must hold int32 offsets [experts + 1] and int32 positions [tokens, top_k]")
    _same_device(positions, "plan.positions", tensor)
    _same_device(offsets, "plan.offsets", tensor)
    if tensor.dim() < 1:
        raise ValueError(f"{name} must have a width dimension")
    return offsets.contiguous(), positions.contiguous()


def dispatch_tokens(x, plan):
    """The rows of ``x`` [..., width] sorted by expert: [tokens * top_k, width], one row per choice, zeros behind the last
    expert's rows (``plan.offsets[-1]``)."""
    if x.is_cuda:
        return ops.expert_dispatch(x, plan[1], plan[0])
    offsets, positions = _check_plan(plan, x, "x")
    _float(x, "x")
    width = x.shape[-1]
    if not 1 <= width <= ops.MAX_DISPATCH_WIDTH or x.numel() != positions.shape[0] * width:
        raise ValueError(f"x of shape {tuple(x.shape)} does not hold the plan's {positions.shape[0]} tokens")
    return ops.expert_dispatch(x, positions, offsets)


def combine_tokens(rows, weights, plan):
    """``sum_j weights[..., j] * rows[positions[..., j]]``: the experts' results back in token order, [..., width].

    ``rows`` [tokens * top_k, width] as :func:`dispatch_tokens` lays them out, ``weights`` [..., top_k] (float32, bfloat16
    or float16).  A choice without a row adds nothing; rows behind the last expert's are not read, and their gradient is
    zero.  Sums are taken in fp32 and rounded once to the rows' dtype."""
    if rows.is_cuda:
        return ops.expert_combine(rows, weights, plan[1], plan[0])
    offsets, positions = _check_plan(plan, rows, "rows")
    _float(rows, "rows")
    _float(weights, "weights")
    _same_device(weights, "weights", rows)
    tokens, top_k = positions.shape
    if rows.dim() != 2 or rows.shape[0] != tokens * top_k or not 1 <= rows.shape[1] <= ops.MAX_DISPATCH_WIDTH:
        raise ValueError(f"rows must be [{tokens * top_k}, width], got {tuple(rows.shape)}")
    if weights.dim() < 1 or weights.shape[-1] != top_k or weights.numel() != tokens * top_k:
        raise ValueError(f"weights of shape {tuple(weights.shape)} do not match the plan's {tokens} tokens x {top_k} choices")
    return ops.expert_combine(rows, weights, positions, offsets)
