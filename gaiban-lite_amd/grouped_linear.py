"""Linears grouped by expert over experts kept in bf16 or int8.

The framework's expert layers (``ops.experts_*_into``) fuse both products of
a layer over int4 and MXFP4 weights.  These are the products by themselves,
over unpacked weights [experts, N, K] as a checkpoint stores them: each slot
``token * topk + j`` takes the weights of the expert it was routed to, with
ragged numbers of slots per expert given by the alignment
(``deterministic_moe_align_block_size``) of the route.

* rows of ``x``: one per token (serving its ``topk`` slots), or with
  ``per_slot`` one per slot;
* ``swiglu``: N = 2 I channels, gate rows first; the output is
  ``silu(min(g, L)) * clamp(u, -L, L)`` of both halves [slots, I];
* ``route_weights`` [tokens, topk]: each slot's output times its weight.

So a layer's experts are ``up = grouped_linear_into(x, w13, swiglu)``,
``down = grouped_linear_into(up, w2, per_slot, route_weights)`` and the sum of
``down`` over ``topk``.  int8 weights carry one bf16 scale per expert and
channel; their activations are quantised per row as in ``int8_linear.py``.

Outputs are written for aligned slots only: a padding slot, a block whose
expert id is out of range and, where the alignment reported an id out of
range (``num_tokens_post_padded`` = -1), every slot keep what ``out`` held.
Tensors are contiguous and 16-byte aligned (views that start elsewhere are
refused), N a multiple of 16 (32 with ``swiglu``), K of 8 (bf16) or 16
(int8, up to 65536).  The entry points look at metadata only, allocate
nothing and never synchronise, so they can be captured in a graph.
"""

from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache
from typing import Final

import torch

from . import contracts as C
from . import ops
from .deterministic_moe_align import max_padded_tokens

WEIGHT_DTYPES: Final = (torch.bfloat16, torch.int8)
OUTPUT_DTYPE: Final = torch.bfloat16
BLOCK_SIZES: Final = (8, 16, 32, 48, 64)


@dataclass(frozen=True)
class GroupedPlan:
    """One geometry of a product by expert and the shapes of its tensors."""

    tokens: int
    topk: int
    experts: int
    n: int
    k: int
    block_size: int
    swiglu: bool = False
    per_slot: bool = False
    capacity: int = 0  # of the alignment's sorted_token_ids

    slots = property(lambda self: self.tokens * self.topk)
    rows = property(lambda self: self.slots if self.per_slot else self.tokens)
    activation_shape = property(lambda self: (self.rows, self.k))
    activation_scale_shape = property(lambda self: (self.rows,))
    weight_shape = property(lambda self: (self.experts, self.n, self.k))
    weight_scale_shape = property(lambda self: (self.experts, self.n))
    output_shape = property(lambda self: (self.slots, self.n // 2 if self.swiglu else self.n))


@lru_cache(maxsize=4096, typed=True)
def make_grouped_plan(tokens: int, topk: int, experts: int, n: int, k: int, *, block_size: int | None = None,
                      swiglu: bool = False, per_slot: bool = False) -> GroupedPlan:
    """A validated plan.  ``block_size`` is the alignment's; None takes the
    framework's rule (``ops.block_size_m``).  ValueError for a bad value,
    TypeError for a flag that is no bool."""

    tokens, topk, experts, n, k = (C.positive_int(name, v) for name, v in (
        ("tokens", tokens), ("topk", topk), ("experts", experts), ("n", n), ("k", k)))
    C.boolean("swiglu", swiglu)
    C.boolean("per_slot", per_slot)
    if block_size is None:
        block_size = ops.block_size_m(tokens, topk, experts)
    if isinstance(block_size, bool) or block_size not in BLOCK_SIZES:
        raise ValueError(f"block_size={block_size!r} is not one of {BLOCK_SIZES}")
    multiple = 32 if swiglu else 16
    if n % multiple:
        raise ValueError(f"n={n} is not a multiple of {multiple}")
    if k % 8:
        raise ValueError(f"k={k} is not a multiple of 8")
    return GroupedPlan(tokens=tokens, topk=topk, experts=experts, n=n, k=k, block_size=block_size, swiglu=swiglu,
                       per_slot=per_slot, capacity=max_padded_tokens(tokens * topk, experts, block_size))


def _check_plan(plan: GroupedPlan, x, weight, sorted_token_ids, dtype: torch.dtype) -> None:
    if not isinstance(plan, GroupedPlan):
        raise TypeError(f"plan: expected GroupedPlan, got {type(plan).__name__}")
    for name, value, shape in (("activation", x, plan.activation_shape), ("weight", weight, plan.weight_shape),
                               ("sorted_token_ids", sorted_token_ids, (plan.capacity,))):
        if not isinstance(value, torch.Tensor) or value.shape != shape:
            C.tensor(name, value, shape=shape)
    if weight.dtype is not dtype:
        C.tensor("weight", weight, dtype=dtype)


def grouped_linear_into(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor, *, plan: GroupedPlan,
                        sorted_token_ids: torch.Tensor, expert_ids: torch.Tensor,
                        num_tokens_post_padded: torch.Tensor, route_weights: torch.Tensor | None = None,
                        clamp_limit: float = 0.0) -> None:
    """The product over bf16 weights [experts, n, k]: ``x`` bf16
    ``plan.activation_shape``, ``out`` bf16 ``plan.output_shape``."""

    _check_plan(plan, x, weight, sorted_token_ids, torch.bfloat16)
    ops.grouped_gemm_into(x, weight, out, tokens=plan.tokens, topk=plan.topk, sorted_token_ids=sorted_token_ids,
                          expert_ids=expert_ids, num_tokens_post_padded=num_tokens_post_padded,
                          block_size=plan.block_size, per_slot=plan.per_slot, swiglu=plan.swiglu,
                          clamp_limit=clamp_limit, route_weights=route_weights)


def grouped_int8_gemm_into(activation: torch.Tensor, activation_scale: torch.Tensor, weight: torch.Tensor,
                           weight_scale: torch.Tensor, out: torch.Tensor, *, plan: GroupedPlan,
                           sorted_token_ids: torch.Tensor, expert_ids: torch.Tensor,
                           num_tokens_post_padded: torch.Tensor, route_weights: torch.Tensor | None = None,
                           clamp_limit: float = 0.0) -> None:
    """The product over int8 weights [experts, n, k] with bf16 scales
    [experts, n], of activations quantised before (int8 codes with one fp32
    scale per row: ``int8_linear.activation_quant_into``)."""

    _check_plan(plan, activation, weight, sorted_token_ids, torch.int8)
    ops.grouped_gemm_into(activation, weight, out, tokens=plan.tokens, topk=plan.topk,
                          sorted_token_ids=sorted_token_ids, expert_ids=expert_ids,
                          num_tokens_post_padded=num_tokens_post_padded, block_size=plan.block_size,
                          per_slot=plan.per_slot, swiglu=plan.swiglu, clamp_limit=clamp_limit,
                          route_weights=route_weights, x_scale=activation_scale, ws=weight_scale)


def grouped_int8_linear_into(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, out: torch.Tensor,
                             quantized: torch.Tensor, scale: torch.Tensor, *, plan: GroupedPlan,
                             sorted_token_ids: torch.Tensor, expert_ids: torch.Tensor,
                             num_tokens_post_padded: torch.Tensor, route_weights: torch.Tensor | None = None,
                             clamp_limit: float = 0.0) -> None:
    """The quantiser over ``x`` (bf16, fp16 or fp32) into ``quantized`` int8
    and ``scale`` fp32 (one per row), then ``grouped_int8_gemm_into``."""

    _check_plan(plan, x, weight, sorted_token_ids, torch.int8)
    ops.grouped_gemm_into(x, weight, out, tokens=plan.tokens, topk=plan.topk, sorted_token_ids=sorted_token_ids,
                          expert_ids=expert_ids, num_tokens_post_padded=num_tokens_post_padded,
                          block_size=plan.block_size, per_slot=plan.per_slot, swiglu=plan.swiglu,
                          clamp_limit=clamp_limit, route_weights=route_weights, x_scale=scale, ws=weight_scale,
                          quantized=C.tensor("quantized", quantized))


__all__ = [
    "BLOCK_SIZES",
    "GroupedPlan",
    "OUTPUT_DTYPE",
    "WEIGHT_DTYPES",
    "grouped_int8_gemm_into",
    "grouped_int8_linear_into",
    "grouped_linear_into",
    "make_grouped_plan",
]
