"""Gated experts (csrc/experts_ops.hip): a learned gate in the place of the
KiloNeRF grid's rule (``kilonerf_cuda``: a sample's network follows from its
position). ``route`` chooses each row's k experts, ``plan`` sorts the choices by
expert (what ``sort_by_key_int16_*`` does for the grid), ``expert_linear`` runs
the experts' 8-bit layers on the sorted rows, ``combine`` joins their outputs.
``route`` and ``combine`` are differentiable; a trained expert may be any torch
function of the sorted rows.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import _lib, fp8
from ._lib import enqueue, ptr
from .fp8 import TYPES

MAX_EXPERTS, MAX_CHOICES, MAX_GROUPS = 1024, 32, 64


class _Route(ctypes.Structure):
    """NerfRoute (include/nerfhip.h)."""
    _fields_ = [("logits", ctypes.c_void_p), ("ld", ctypes.c_int64), ("T", ctypes.c_int64),
                ("type", ctypes.c_int), ("E", ctypes.c_int), ("k", ctypes.c_int),
                ("sigmoid", ctypes.c_int), ("groups", ctypes.c_int), ("top_groups", ctypes.c_int),
                ("group_top2", ctypes.c_int), ("renorm", ctypes.c_int), ("bias", ctypes.c_void_p),
                ("scale", ctypes.c_float), ("weights", ctypes.c_void_p), ("experts", ctypes.c_void_p)]


def _route_desc(logits, opts, weights, experts):
    k, sigmoid, bias, groups, top_groups, top2, renorm, scale = opts
    return _Route(ptr(logits), logits.stride(0), logits.shape[0], TYPES[logits.dtype], logits.shape[1], k, sigmoid,
                  groups, top_groups, top2, renorm, ptr(bias), scale, ptr(weights), ptr(experts))


def _route(logits, opts):
    T, k = logits.shape[0], opts[0]
    weights = torch.empty((T, k), device=logits.device, dtype=torch.float32)
    experts = torch.empty((T, k), device=logits.device, dtype=torch.int32)
    if T:
        d = _route_desc(logits, opts, weights, experts)
        enqueue("nerf_route", logits, ctypes.addressof(d))
    return weights, experts


class _RouteFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, opts):
        weights, experts = _route(logits, opts)
        ctx.save_for_backward(logits, experts)
        ctx.opts = opts
        ctx.mark_non_differentiable(experts)
        return weights, experts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dweights, _):
        logits, experts = ctx.saved_tensors
        d = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
        if d.numel():
            dweights = dweights.contiguous()
            r = _route_desc(logits, ctx.opts, None, experts)
            enqueue("nerf_route_backward", logits, ctypes.addressof(r), ptr(dweights), ptr(d))
        return d, None


def route(logits, k, score="softmax", bias=None, groups=1, top_groups=1, group_score="max", renormalise=True,
          scale=1.0):
    """(weights float32 [T, k], experts int32 [T, k]) of logits [T, E] (float32, bfloat16, float16).

    s = softmax or sigmoid (``score``) of a row; the k experts with the highest s + ``bias`` ([E] float32; it
    only chooses, and has no gradient) in falling order of the 64-bit keys, ties to the lowest index.
    ``groups`` > 1: only experts of the ``top_groups`` groups of E / groups neighbours with the highest
    ``group_score`` ("max": their highest s + bias, "top2": the sum of their two highest).
    weights = ``scale`` * s, with ``renormalise`` divided by the sum of the row's chosen s. Keys of NaN and -inf
    are the lowest, below every number (masks of the type's lowest value go before them); a row that holds one (or +inf under softmax) has NaN weights, one whose chosen logits are all
    -inf zeros. E <= 1024, k <= 32, groups <= 64."""
    if logits.dim() != 2 or logits.dtype not in TYPES:
        raise ValueError("route: logits must be [T, E] float32, bfloat16 or float16")
    T, E = logits.shape
    k, groups, top_groups = int(k), int(groups), int(top_groups)
    if not 1 <= E <= MAX_EXPERTS or not 1 <= k <= min(E, MAX_CHOICES):
        raise ValueError(f"route: needs 1 to {MAX_EXPERTS} experts and k of 1 to {MAX_CHOICES}, at most E "
                         f"(E = {E}, k = {k})")
    if not 1 <= groups <= MAX_GROUPS or E % groups or not 1 <= top_groups <= groups or \
            top_groups * (E // groups) < k:
        raise ValueError(f"route: {groups} groups must divide E = {E}, and top_groups = {top_groups} of them hold "
                         f"k = {k} experts")
    if score not in ("softmax", "sigmoid") or group_score not in ("max", "top2"):
        raise ValueError("route: score must be 'softmax' or 'sigmoid', group_score 'max' or 'top2'")
    scale = float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError("route: scale must be positive and finite")
    if bias is not None:
        if bias.dtype != torch.float32 or tuple(bias.shape) != (E,) or bias.device != logits.device:
            raise ValueError(f"route: bias must be float32 [{E}] on {logits.device}")
        bias = bias.detach().contiguous()
    fp8.refuse_dual("route", logits)
    _lib.require_gpu(logits)
    if logits.stride(1) != 1 and E > 1:
        logits = logits.contiguous()
    opts = (k, int(score == "sigmoid"), bias, groups, top_groups, int(group_score == "top2"), int(bool(renormalise)),
            scale)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _RouteFn.apply(logits, opts)
    return _route(logits.detach(), opts)


class Plan(NamedTuple):
    """The n = T * k slots (t * k + j) sorted by expert: ``order`` int32 [n], the slot of each sorted row (-1
    behind the last expert's); ``position`` int32 [T, k], the sorted row of each slot (-1: no expert);
    ``offsets`` int32 [E + 1], where each expert's rows begin (from 0 on, never falling)."""
    order: torch.Tensor
    position: torch.Tensor
    offsets: torch.Tensor


def plan(experts, num_experts):
    """``Plan`` of experts int32 [T, k]; slots of one expert keep their order. Numbers outside of
    [0, num_experts) take part in nothing (a dropped choice, a padded row: -1)."""
    E = int(num_experts)
    if experts.dim() != 2 or experts.dtype != torch.int32 or experts.shape[1] < 1:
        raise ValueError("plan: experts must be int32 [T, k]")
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"plan: num_experts must be 1 to {MAX_EXPERTS}")
    _lib.require_gpu(experts)
    experts = experts.contiguous()
    n, dev = experts.numel(), experts.device
    order = torch.empty((n,), device=dev, dtype=torch.int32)
    position = torch.empty(experts.shape, device=dev, dtype=torch.int32)
    if n == 0:
        return Plan(order, position, torch.zeros((E + 1,), device=dev, dtype=torch.int32))
    offsets = torch.empty((E + 1,), device=dev, dtype=torch.int32)
    need = _lib.lib().nerf_expert_plan_workspace(n, E)
    ws = torch.empty((need,), device=dev, dtype=torch.uint8) if need else None
    enqueue("nerf_expert_plan", experts, ptr(experts), n, E, ptr(order), ptr(position), ptr(offsets), ptr(ws), need)
    return Plan(order, position, offsets)


def _check_plan(p, device, who):
    if not isinstance(p, Plan) or p.order.dim() != 1 or p.position.dim() != 2 or p.offsets.dim() != 1 or \
            p.order.numel() != p.position.numel():
        raise ValueError(f"{who}: plan must be a Plan (order [T * k], position [T, k], offsets [E + 1])")
    for t in p:
        if t.dtype != torch.int32 or not t.is_contiguous() or t.device != device:
            raise ValueError(f"{who}: the plan's tensors must be contiguous int32 on {device}")


def expert_linear(x, weight, plan, gather=False, bias=None, relu=False, out_dtype=None):
    """The experts' layers on sorted rows: y [n, N], row i by the matrix of the expert that ``plan`` sorted it
    to (``fp8.linear``'s arithmetic; ``weight`` an ``Fp8Weight`` stack [E, N, K], ``bias`` [E, N] float32).
    ``gather``: x [T, K] holds the unsorted rows, each taken k times; else x [n, K] is sorted already.
    Rows behind the last expert's become zeros."""
    if not isinstance(weight, fp8.Fp8Weight) or weight.q.dim() != 3:
        raise ValueError("expert_linear: weight must be an Fp8Weight of a stack [E, N, K]")
    _check_plan(plan, x.device, "expert_linear")
    if plan.offsets.numel() != weight.q.shape[0] + 1:
        raise ValueError(f"expert_linear: the plan is for {plan.offsets.numel() - 1} experts, the weights for "
                         f"{weight.q.shape[0]}")
    T, k = plan.position.shape
    n = plan.order.numel()
    if x.dim() != 2 or x.shape[0] != (T if gather else n):
        raise ValueError(f"expert_linear: activations must be [{T if gather else n}, K]")
    return fp8.launch(x, weight, n, plan.order if gather else None, k, plan.offsets, bias, relu, out_dtype,
                      "expert_linear")


def _combine(y, weights, p):
    T, k = p.position.shape
    out = torch.empty((T, y.shape[1]), device=y.device, dtype=y.dtype)
    if out.numel():
        enqueue("nerf_expert_combine", y, ptr(y), TYPES[y.dtype], y.shape[0], y.shape[1], ptr(weights),
                ptr(p.position), T, k, ptr(out))
    return out


class _CombineFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, order, position, offsets):
        ctx.save_for_backward(y, weights, order, position)
        return _combine(y, weights, Plan(order, position, offsets))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        y, weights, order, position = ctx.saved_tensors
        dy = torch.empty_like(y) if ctx.needs_input_grad[0] else None
        dw = torch.empty_like(weights) if ctx.needs_input_grad[1] else None
        if y.numel() and weights.numel():
            dout = dout.contiguous()
            enqueue("nerf_expert_combine_backward", y, ptr(y), TYPES[y.dtype], y.shape[0], y.shape[1], ptr(weights),
                    ptr(position), ptr(order), ptr(dout), *position.shape, ptr(dy), ptr(dw))
        elif dw is not None:
            dw.zero_()   # (rows without columns)
        return dy, dw, None, None, None


def combine(y, weights, plan):
    """out [T, N] in y's type: out[t] = sum_j weights[t, j] * y[plan.position[t, j]], added in float32 in the
    order of j. y [n, N] float32, bfloat16 or float16, weights float32 [T, k]; differentiable in both. A slot
    whose position was set to -1 since (over a capacity, say) has no part; no two slots may have one position."""
    if y.dim() != 2 or y.dtype not in TYPES:
        raise ValueError("combine: y must be [n, N] float32, bfloat16 or float16")
    _check_plan(plan, y.device, "combine")
    if y.shape[0] != plan.order.numel():
        raise ValueError(f"combine: y must have the plan's {plan.order.numel()} rows")
    if weights.dtype != torch.float32 or weights.shape != plan.position.shape or weights.device != y.device:
        raise ValueError(f"combine: weights must be float32 {list(plan.position.shape)} on {y.device}")
    fp8.refuse_dual("combine", y, weights)
    _lib.require_gpu(y)
    y, weights = y.contiguous(), weights.contiguous()
    if torch.is_grad_enabled() and (y.requires_grad or weights.requires_grad):
        return _CombineFn.apply(y, weights, *plan)
    return _combine(y.detach(), weights.detach(), plan)
