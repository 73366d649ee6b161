"""Operators on 4-bit weights and 8-bit activations, on torch tensors (include/itts_ops.h).

    rmsnorm_q8(x, weight, eps, residual=, group=)  h = x + residual; its RMS norm as 8-bit codes
    q8_quantize(x, group)                          rows as 8-bit codes
    q4_pack(w, group) -> Q4Weight                  float weights to 4 bits with group scales
    q4_unpack(weight, dtype)                       what a Q4Weight stands for
    q4_matmul(q, scales, weight, ...)              8-bit rows times 4-bit weights
    q4_linear(x, weight, norm_weight=, ...)        norm, 8-bit codes and product in one call

QwenDecoder(weights, weight_bits=4) runs on the same kernels.  Calls run on the current stream of
the tensors' device and return without waiting for it; none keeps anything between calls.
Arguments that do not fit raise InvalidArgument.  Kernels exist for gfx950 only: there is no CPU
path.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from itts_gpt import InvalidArgument, _lib, _raise

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_GROUPS = (32, 64, 128)
SWIGLU = 1


def _bind():
    p, i64, i32, u32, f32, z = C.c_void_p, C.c_int64, C.c_int32, C.c_uint32, C.c_float, C.c_size_t
    sig = {
        "itts_ops_last_error": (C.c_char_p, []),
        "itts_rmsnorm_q8": (i32, [p, i64, p, i64, p, i32, i32, i64, i64, f32, i32, p, i64, p, i64, p, p, p]),
        "itts_q8_quantize": (i32, [p, i64, i32, i64, i64, i32, p, i64, p, p, p]),
        "itts_q4_packed_bytes": (z, [i64, i64]),
        "itts_q4_scale_count": (z, [i64, i64, i32]),
        "itts_q4_pack": (i32, [p, i64, i32, i64, i64, i32, p, p, p]),
        "itts_q4_unpack": (i32, [p, p, i64, i64, i32, i32, p, i64, p]),
        "itts_q4_matmul": (i32, [p, p, i64, p, p, i64, i64, i32, p, p, i64, u32, i32, p, i64, p]),
        "itts_q4_linear_workspace": (z, [i64, i64, i64, i32]),
        "itts_q4_linear": (i32, [p, i64, i32, i64, p, i32, f32, p, p, i64, i64, i32, p, p, i64, u32, i32, p, i64, p, z, p]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(_lib, name)
        fn.restype = res
        fn.argtypes = args


_bind()


class Q4Weight(NamedTuple):
    """An [n][k] matrix in 4 bits: packed uint8 [n/16][k/128][1024] and BF16 scales
    [n/16][k/128][16][128/group] (sizes rounded up), laid out as include/itts_ops.h says."""

    packed: torch.Tensor
    scales: torch.Tensor
    n: int
    k: int
    group: int


class Q8(NamedTuple):
    """Rows in 8 bits: int8 codes [rows][k rounded up to 128], float scales [rows][that / group], and
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


def _no(message):
    raise InvalidArgument(message)


def _rows(t, name):
    """A float matrix with unit column stride: (type, rows, columns, row stride)."""
    kind = _TYPES.get(t.dtype)
    if kind is None:
        _no(f"{name}: float32, bfloat16 or float16 is wanted, not {t.dtype}")
    if t.dim() != 2:
        _no(f"{name}: a matrix is wanted, not {t.dim()} dimensions")
    rows, cols = t.shape
    stride = t.stride()
    if cols > 1 and stride[1] != 1:
        _no(f"{name}: columns have to lie next to each other")
    # the stride of a single row says nothing
    return kind, rows, cols, stride[0] if rows > 1 else max(cols, 1)


def _like(t, x, shape, name):
    if t.dtype != x.dtype or tuple(t.shape) != tuple(shape):
        _no(f"{name}: {x.dtype} {tuple(shape)} is wanted, not {t.dtype} {tuple(t.shape)}")
    return _rows(t, name)[3]


def _vector(t, n, name):
    if t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        _no(f"{name}: {n} contiguous values are wanted, not {tuple(t.shape)}")


def _group(group):
    if group not in _GROUPS:
        _no(f"group: 32, 64 or 128 is wanted, not {group}")


def _weight(w):
    if not isinstance(w, Q4Weight):
        _no("weight: a Q4Weight is wanted")
    _group(w.group)
    nt, kb = -(-w.n // 16), -(-w.k // 128)
    if w.n < 1 or w.k < 1 or w.packed.dtype != torch.uint8 or w.packed.numel() != nt * kb * 1024 or not w.packed.is_contiguous():
        _no(f"weight: packed codes of {w.n} x {w.k} are {nt * kb * 1024} contiguous bytes")
    if w.scales.dtype != torch.bfloat16 or w.scales.numel() != nt * kb * (2048 // w.group) or not w.scales.is_contiguous():
        _no(f"weight: the scales of {w.n} x {w.k} are {nt * kb * (2048 // w.group)} contiguous bfloat16 values")


def _call(fn, tensors, *args):
    """fn(*args, stream) on the tensors' device and its current stream."""
    device = None
    for t in tensors:
        if t is not None:
            if not t.is_cuda:
                _no("tensors have to be on the GPU")
            if device is None:
                device = t.device
            elif t.device != device:
                _no(f"tensors on {device} and {t.device}")
            if t.requires_grad and torch.is_grad_enabled():
                _no("these operators have no gradients: detach the tensors, or call under torch.no_grad()")
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            st = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        st = fn(*args, torch.cuda.current_stream(device).cuda_stream)
    if st != 0:
        _raise(st, _lib.itts_ops_last_error().decode())


def _ptr(t):
    return None if t is None else t.data_ptr()


def _codes(x, rows, cols, group, q, scales):
    kp = -(-cols // 128) * 128
    if q is None:
        q = torch.empty((rows, kp), dtype=torch.int8, device=x.device)
    elif q.dtype != torch.int8 or tuple(q.shape) != (rows, kp) or not q.is_contiguous():
        _no(f"q: contiguous int8 {(rows, kp)} is wanted")
    if scales is None:
        scales = torch.empty((rows, kp // group), dtype=torch.float32, device=x.device)
    elif scales.dtype != torch.float32 or tuple(scales.shape) != (rows, kp // group) or not scales.is_contiguous():
        _no(f"scales: contiguous float32 {(rows, kp // group)} is wanted")
    return q, scales


def _values(x, rows, cols, values):
    if values is None or values is False:
        return None, 0
    if values is True:
        values = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
        return values, cols
    return values, _like(values, x, (rows, cols), "values")


def rmsnorm_q8(x, weight, eps=1e-6, *, residual=None, group=128, h=None, q=None, scales=None, values=None) -> NormQ8:
    """The RMS norm of h = x + residual, times weight ([cols], x's type or float32), as 8-bit codes.
    h, q, scales: where to write them (made if absent; h may be x or residual); values: True or where
    to write what the codes stand for.  Without a residual h is x, unless it is to be written."""
    kind, rows, cols, xs = _rows(x, "x")
    _group(group)
    _vector(weight, cols, "weight")
    wkind = _TYPES.get(weight.dtype)
    if weight.dtype != x.dtype and wkind != 0:
        _no(f"weight: {x.dtype} or float32 is wanted, not {weight.dtype}")
    rs = hs = 0
    if residual is not None:
        rs = _like(residual, x, (rows, cols), "residual")
        if h is None:
            h = torch.empty((rows, cols), dtype=x.dtype, device=x.device)
            hs = cols
    if h is not None and not hs:
        hs = _like(h, x, (rows, cols), "h")
    q, scales = _codes(x, rows, cols, group, q, scales)
    values, vs = _values(x, rows, cols, values)
    _call(_lib.itts_rmsnorm_q8, (x, weight, residual, h, q, scales, values), x.data_ptr(), xs, _ptr(residual), rs, weight.data_ptr(), wkind,
          kind, rows, cols, eps, group, _ptr(h), hs, _ptr(values), vs, q.data_ptr(), scales.data_ptr())
    return NormQ8(x if h is None else h, q, scales, values)


def q8_quantize(x, group=128, *, q=None, scales=None, values=None) -> Q8:
    """The rows of x as 8-bit codes with a scale per `group` columns."""
    kind, rows, cols, xs = _rows(x, "x")
    _group(group)
    q, scales = _codes(x, rows, cols, group, q, scales)
    values, vs = _values(x, rows, cols, values)
    _call(_lib.itts_q8_quantize, (x, q, scales, values), x.data_ptr(), xs, kind, rows, cols, group, _ptr(values), vs, q.data_ptr(),
          scales.data_ptr())
    return Q8(q, scales, values)


def q4_pack(w, group=128) -> Q4Weight:
    """The float matrix w [n][k] in 4 bits."""
    kind, n, k, ws = _rows(w, "w")
    _group(group)
    if n < 1 or k < 1:
        _no("w: a matrix without rows or columns")
    nt, kb = -(-n // 16), -(-k // 128)
    packed = torch.empty((nt, kb, 1024), dtype=torch.uint8, device=w.device)
    scales = torch.empty((nt, kb, 16, 128 // group), dtype=torch.bfloat16, device=w.device)
    _call(_lib.itts_q4_pack, (w, packed, scales), w.data_ptr(), ws, kind, n, k, group, packed.data_ptr(), scales.data_ptr())
    return Q4Weight(packed, scales, n, k, group)


def q4_unpack(weight, dtype=torch.float32, *, out=None):
    """The [n][k] matrix that a Q4Weight stands for, rounded to dtype."""
    _weight(weight)
    if dtype not in _TYPES:
        _no(f"dtype: float32, bfloat16 or float16 is wanted, not {dtype}")
    if out is None:
        out = torch.empty((weight.n, weight.k), dtype=dtype, device=weight.packed.device)
    elif out.dtype != dtype or tuple(out.shape) != (weight.n, weight.k):
        _no(f"out: {dtype} {(weight.n, weight.k)} is wanted")
    os = _rows(out, "out")[3]
    _call(_lib.itts_q4_unpack, (weight.packed, weight.scales, out), weight.packed.data_ptr(), weight.scales.data_ptr(), weight.n, weight.k,
          weight.group, _TYPES[dtype], out.data_ptr(), os)
    return out


def _product(rows, weight, bias, residual, swiglu, out_dtype, out, device):
    """Checks what a product adds and where it goes: (out, its stride, residual's stride)."""
    n = weight.n
    if out_dtype not in _TYPES:
        _no(f"out_dtype: float32, bfloat16 or float16 is wanted, not {out_dtype}")
    if swiglu and n % 2:
        _no(f"swiglu: pairs of columns are wanted, not {n} columns")
    cols = n // 2 if swiglu else n
    if bias is not None:
        _vector(bias, n, "bias")
        if bias.dtype != torch.float32:
            _no(f"bias: float32 is wanted, not {bias.dtype}")
    if out is None:
        out, os = torch.empty((rows, cols), dtype=out_dtype, device=device), cols
    elif out.dtype != out_dtype or tuple(out.shape) != (rows, cols):
        _no(f"out: {out_dtype} {(rows, cols)} is wanted, not {out.dtype} {tuple(out.shape)}")
    else:
        os = _rows(out, "out")[3]
    return out, os, 0 if residual is None else _like(residual, out, (rows, cols), "residual")


def q4_matmul(q, scales, weight, *, bias=None, residual=None, swiglu=False, out_dtype=torch.float32, out=None):
    """Rows in 8 bits (q, scales of a Q8) times weight's rows: [rows][n], + bias (float32 [n]).  With
    swiglu, columns 2i and 2i + 1 become silu(column 2i) * column 2i + 1.  + residual (out_dtype);
    out may be residual."""
    _weight(weight)
    kp = -(-weight.k // 128) * 128
    if q.dtype != torch.int8 or q.dim() != 2 or q.shape[1] != kp or not q.is_contiguous():
        _no(f"q: contiguous int8 rows of {kp} codes are wanted, not {q.dtype} {tuple(q.shape)}")
    rows = q.shape[0]
    if scales.dtype != torch.float32 or tuple(scales.shape) != (rows, kp // weight.group) or not scales.is_contiguous():
        _no(f"scales: contiguous float32 {(rows, kp // weight.group)} is wanted, not {scales.dtype} {tuple(scales.shape)}")
    out, os, rs = _product(rows, weight, bias, residual, swiglu, out_dtype, out, q.device)
    _call(_lib.itts_q4_matmul, (q, scales, weight.packed, weight.scales, bias, residual, out), q.data_ptr(), scales.data_ptr(), rows,
          weight.packed.data_ptr(), weight.scales.data_ptr(), weight.n, weight.k, weight.group, _ptr(bias), _ptr(residual), rs,
          SWIGLU if swiglu else 0, _TYPES[out_dtype], out.data_ptr(), os)
    return out


def q4_linear(x, weight, *, norm_weight=None, eps=1e-6, bias=None, residual=None, swiglu=False, out_dtype=None, out=None):
    """q4_matmul of x's rows in 8 bits, after the RMS norm with norm_weight where one is given.
    out_dtype: x's type unless given."""
    kind, rows, cols, xs = _rows(x, "x")
    _weight(weight)
    if cols != weight.k:
        _no(f"x: rows of {weight.k} are wanted, not {cols}")
    wkind = 0
    if norm_weight is not None:
        _vector(norm_weight, cols, "norm_weight")
        wkind = _TYPES.get(norm_weight.dtype)
        if norm_weight.dtype != x.dtype and wkind != 0:
            _no(f"norm_weight: {x.dtype} or float32 is wanted, not {norm_weight.dtype}")
    out_dtype = out_dtype or x.dtype
    out, os, rs = _product(rows, weight, bias, residual, swiglu, out_dtype, out, x.device)
    need = _lib.itts_q4_linear_workspace(rows, weight.n, weight.k, weight.group)
    work = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _call(_lib.itts_q4_linear, (x, weight.packed, weight.scales, norm_weight, bias, residual, out), x.data_ptr(), xs, kind, rows,
          _ptr(norm_weight), wkind, eps, weight.packed.data_ptr(), weight.scales.data_ptr(), weight.n, weight.k, weight.group, _ptr(bias),
          _ptr(residual), rs, SWIGLU if swiglu else 0, _TYPES[out_dtype], out.data_ptr(), os, _ptr(work), need)
    return out
