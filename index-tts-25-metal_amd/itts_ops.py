"""Operators on 4-bit weights and 8-bit activations, on torch tensors (include/itts_ops.h).

    rmsnorm_q8(x, weight, eps, residual=, group=)  h = x + residual; its RMS norm as 8-bit codes
    q8_quantize(x, group)                          rows as 8-bit codes
    q4_pack(w, group) -> Q4Weight                  float weights to 4 bits with group scales
    q4_unpack(weight, dtype)                       what a Q4Weight stands for
    q4_matmul(q, scales, weight, ...)              8-bit rows times 4-bit weights
    q4_linear(x, weight, norm_weight=, ...)        norm, 8-bit codes and product in one call

QwenDecoder(weights, weight_bits=4) runs on the same kernels.  Matrices are float32, bfloat16 or
float16 with unit column stride; `group` is 32, 64 or 128 columns.  Calls run on the current stream of
the tensors' device and return without waiting for it; none keeps anything between calls, and all
may be captured into a graph.  Outputs that are not given are made.  Arguments that do not fit
raise InvalidArgument.  There are no gradients (tensors that require them are refused unless under
no_grad, and so are forward mode's dual tensors) and there is no CPU path.

The library has to run on the HIP runtime that torch brings, whose streams it is given: import torch (or
this module) before itts_gpt, else two runtimes are loaded and this import fails.
"""
from __future__ import annotations

from pathlib import Path
from typing import NamedTuple, Optional

import torch

import itts_gpt
from itts_gpt import GptRuntimeError, InvalidArgument, LogicError


def _load():
    with open("/proc/self/maps") as f:
        runtimes = {line.split()[-1] for line in f if "/libamdhip64.so" in line}
    if len(runtimes) > 1:
        raise ImportError("two HIP runtimes are loaded (" + ", ".join(sorted(runtimes)) + "): import torch before itts_gpt")
    at = Path(itts_gpt.LIB_PATH).with_name("_itts_ops.so")
    if not at.exists():
        raise ImportError(f"torch binding not built: {at} is missing (run index-tts-25-metal_amd/build.py)")
    import _itts_ops

    _itts_ops.errors(InvalidArgument, GptRuntimeError, LogicError)
    return _itts_ops


_ops = _load()
_KINDS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class Q4Weight(NamedTuple):
    """An [n][k] matrix in 4 bits: packed uint8 [n/16][k/128][1024] and bfloat16 scales
    [n/16][k/128][16][128/group] (sizes rounded up), laid out as include/itts_ops.h says."""

    packed: torch.Tensor
    scales: torch.Tensor
    n: int
    k: int
    group: int


class Q8(NamedTuple):
    """Rows in 8 bits: int8 codes [rows][k rounded up to 128], float32 scales [rows][that / group], and
    what they stand for in the rows' type (None unless asked for)."""

    q: torch.Tensor
    scales: torch.Tensor
    values: Optional[torch.Tensor]


class NormQ8(NamedTuple):
    """As Q8, with the rows that were normed: x + residual, or x itself."""

    h: torch.Tensor
    q: torch.Tensor
    scales: torch.Tensor
    values: Optional[torch.Tensor]


def rmsnorm_q8(x, weight, eps=1e-6, *, residual=None, group=128, h=None, q=None, scales=None, values=None) -> NormQ8:
    """The RMS norm of h = x + residual, times weight ([cols], x's type or float32), as 8-bit codes.
    h, q, scales: where to write them (h may be x or residual); values: True, or where to write what the codes
    stand for.  Without a residual h is x, and is written only where a place is given."""
    return tuple.__new__(NormQ8, _ops.rmsnorm_q8(x, weight, eps, residual, group, h, q, scales, values))


def q8_quantize(x, group=128, *, q=None, scales=None, values=None) -> Q8:
    """The rows of x as 8-bit codes with a scale per `group` columns."""
    return tuple.__new__(Q8, _ops.q8_quantize(x, None, 0.0, None, group, None, q, scales, values))


def q4_pack(w, group=128) -> Q4Weight:
    """The float matrix w [n][k] in 4 bits."""
    return tuple.__new__(Q4Weight, _ops.q4_pack(w, group))


def _kind(dtype, name):
    kind = _KINDS.get(dtype)
    if kind is None:
        raise InvalidArgument(f"{name}: float32, bfloat16 or float16 is wanted, not {dtype}")
    return kind


def q4_unpack(weight, dtype=torch.float32, *, out=None):
    """The [n][k] matrix that a Q4Weight stands for, rounded to dtype."""
    return _ops.q4_unpack(weight, _kind(dtype, "dtype"), out)


def q4_matmul(q, scales, weight, *, bias=None, residual=None, swiglu=False, out_dtype=torch.float32, out=None):
    """Rows in 8 bits (q, scales of a Q8) times weight's rows: [rows][n], + bias (float32 [n]).  With
    swiglu, columns 2i and 2i + 1 become silu(column 2i) * column 2i + 1.  + residual (of out_dtype);
    out may be residual."""
    return _ops.q4_matmul(q, scales, weight, bias, residual, swiglu, _kind(out_dtype, "out_dtype"), out)


def q4_linear(x, weight, *, norm_weight=None, eps=1e-6, bias=None, residual=None, swiglu=False, out_dtype=None, out=None):
    """q4_matmul of x's rows in 8 bits, after the RMS norm with norm_weight where one is given, with the
    same result as the two calls.  out_dtype: x's type unless given."""
    return _ops.q4_linear(x, weight, norm_weight, eps, bias, residual, swiglu, _kind(out_dtype or x.dtype, "out_dtype"), out)
