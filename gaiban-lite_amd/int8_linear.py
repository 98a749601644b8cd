"""W8A8 dense linear in 8-bit integers, beside the block-FP8 W8A8 linear of
``fp8_linear.py``.

``out = bf16((Q . Wq^T) * s[m] * ws[n])``: int8 weights [N, K] with one bf16
scale per output channel, the format of ``weight_only_linear``'s
``w8a16_int8_gemm_into``, against activations quantised per token to int8
(``s = max(amax, 1e-12) / 127``, round half to even).  The product runs on
the int8 MFMA, at twice the bf16 rate, and is exact: sums in int32, scaled in
fp32 and rounded once to bf16.

Three entry points with caller-owned storage: ``activation_quant_into``,
``int8_gemm_into`` over its outputs, and ``int8_linear_into``, both in one
call (which for few tokens need not write the codes).  They look at metadata
only, allocate nothing and never synchronise, so they can be captured in a
graph.  Tensors are contiguous and 16-byte aligned, N a multiple of 16, K a
multiple of 16 up to 65536.

A row of x that holds a NaN or an infinity gives a row of NaN.  No
counterpart in the reference (its W8A8 linear is block-FP8,
``runtime/dsv4_direct/fp8_linear.py``).
"""

from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache
from typing import Final

import torch

from . import contracts as C
from . import ops

ACTIVATION_DTYPES: Final = (torch.bfloat16, torch.float16, torch.float32)
QUANTIZED_DTYPE: Final = torch.int8
SCALE_DTYPE: Final = torch.float32
WEIGHT_SCALE_DTYPE: Final = torch.bfloat16
OUTPUT_DTYPE: Final = torch.bfloat16
K_MULTIPLE: Final = 16
N_MULTIPLE: Final = 16
MAX_K: Final = 65536


@dataclass(frozen=True)
class Int8GemmPlan:
    """One geometry and the shapes of its caller-owned tensors."""

    m: int
    n: int
    k: int

    activation_shape = property(lambda self: (self.m, self.k))
    activation_scale_shape = property(lambda self: (self.m,))
    weight_shape = property(lambda self: (self.n, self.k))
    weight_scale_shape = property(lambda self: (self.n,))
    output_shape = property(lambda self: (self.m, self.n))


@lru_cache(maxsize=4096, typed=True)
def make_gemm_plan(m: int, n: int, k: int) -> Int8GemmPlan:
    """A validated plan; ValueError for any bad dimension."""

    m, n, k = (C.positive_int(name, v) for name, v in (("m", m), ("n", n), ("k", k)))
    if n % N_MULTIPLE:
        raise ValueError(f"n={n} is not a multiple of {N_MULTIPLE}: the kernels store 16-channel strips")
    if k % K_MULTIPLE or k > MAX_K:
        raise ValueError(f"k={k} is not a multiple of {K_MULTIPLE} up to {MAX_K}")
    return Int8GemmPlan(m=m, n=n, k=k)


def _check_plan(plan: Int8GemmPlan, activation, weight=None) -> None:
    if not isinstance(plan, Int8GemmPlan):
        raise TypeError(f"plan: expected Int8GemmPlan, got {type(plan).__name__}")
    if not isinstance(activation, torch.Tensor) or activation.shape != (plan.m, plan.k):
        C.tensor("activation", activation, shape=plan.activation_shape)
    if weight is not None and (not isinstance(weight, torch.Tensor) or weight.shape != (plan.n, plan.k)):
        C.tensor("weight", weight, shape=plan.weight_shape)


def activation_quant_into(x: torch.Tensor, quantized_out: torch.Tensor, scale_out: torch.Tensor, *,
                          plan: Int8GemmPlan) -> None:
    """int8 codes [m, k] and fp32 scales [m] of ``x`` (bf16, fp16 or fp32)
    into caller-owned tensors."""

    _check_plan(plan, x)
    ops.act_quant_int8_into(x, quantized_out, scale_out)


def int8_gemm_into(activation: torch.Tensor, activation_scale: torch.Tensor, weight: torch.Tensor,
                   weight_scale: torch.Tensor, out: torch.Tensor, *, plan: Int8GemmPlan) -> None:
    """``out = bf16((activation . weight^T) * activation_scale * weight_scale)``
    over int8 operands."""

    _check_plan(plan, activation, weight)
    ops.int8_gemm_into(activation, activation_scale, weight, weight_scale, out)


def int8_linear_into(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, out: torch.Tensor,
                     quantized: torch.Tensor, scale: torch.Tensor, *, plan: Int8GemmPlan) -> None:
    """``activation_quant_into`` and ``int8_gemm_into`` in one call, the same
    bits.  ``quantized`` int8 [m, k] and ``scale`` fp32 [m] are storage of the
    call, their contents afterwards unspecified."""

    _check_plan(plan, x, weight)
    ops.int8_linear_into(x, weight, weight_scale, out, quantized, scale)


def int8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor) -> torch.Tensor:
    """Allocating convenience call for cold paths and tests."""

    plan = make_gemm_plan(x.shape[0], weight.shape[0], x.shape[1])
    out = torch.empty(plan.output_shape, dtype=OUTPUT_DTYPE, device=x.device)
    q = torch.empty(plan.activation_shape, dtype=QUANTIZED_DTYPE, device=x.device)
    s = torch.empty(plan.activation_scale_shape, dtype=SCALE_DTYPE, device=x.device)
    int8_linear_into(x, weight, weight_scale, out, q, s, plan=plan)
    return out


__all__ = [
    "ACTIVATION_DTYPES",
    "Int8GemmPlan",
    "K_MULTIPLE",
    "MAX_K",
    "N_MULTIPLE",
    "OUTPUT_DTYPE",
    "QUANTIZED_DTYPE",
    "SCALE_DTYPE",
    "WEIGHT_SCALE_DTYPE",
    "activation_quant_into",
    "int8_gemm_into",
    "int8_linear",
    "int8_linear_into",
    "make_gemm_plan",
]
