"""Root-mean-square norms that end in 8- or 4-bit rows: the step between a model's last layer, or an embedding, and a product of such rows.

One pass reads a row, adds the residual, norms, weighs and quantises it; the normed values themselves never go to memory.  Everything is a torch
tensor on the GPU; calls run on the current stream of the tensors' device and do not wait.  Results carry no gradient.
"""
import torch

from . import _lib as T
from .fp4 import Fp4Rows
from .fp8 import _MAX_DIM, _ROW_ALIGN, _SCALES, _VALUES, Fp8Rows, _blocks, _call, _gpu, _same_device

_INF = float("inf")


def _like(name, t, x):
    """What is wrong with a tensor that has to be like x."""
    _gpu(name, t, (x.dtype,))
    if t.shape != x.shape:
        raise ValueError(f"{name} must be {tuple(x.shape)}, as x, got {tuple(t.shape)}")
    _same_device(x.device, name, t)
    return t


def _made(x, residual, summed, weight, eps, to, scale):
    rows, dim = x.shape
    if not 1 <= dim <= _MAX_DIM:
        raise ValueError(f"dim must be 1 to {_MAX_DIM}, got {dim}")
    device = x.device
    weight_ptr, weight_type = None, 0
    if weight is not None:
        _gpu("weight", weight, _VALUES, ndim=1)
        if weight.shape[0] != dim:
            raise ValueError(f"weight must have {dim} values, got {len(weight)}")
        _same_device(device, "weight", weight)
        weight_ptr, weight_type = weight.data_ptr(), _VALUES[weight.dtype]
    if not 0 <= eps < _INF:
        raise ValueError(f"eps must be finite and not below 0, got {eps}")
    if to == "fp8":
        if scale not in _SCALES:
            raise ValueError(f"scale must be 'e8m0' or 'f32', got {scale!r}")
        kind, dtype = _SCALES[scale]
        stride, blocks = -(-dim // _ROW_ALIGN) * _ROW_ALIGN, _blocks(dim)
        codes = torch.empty_strided((rows, dim), (stride, 1), dtype=torch.float8_e4m3fn, device=device)
        scales = torch.empty_strided((rows, blocks), (blocks, 1), dtype=dtype, device=device)
        made, row_kind = Fp8Rows.__new__(Fp8Rows)._set(codes, scales, 1, kind), T.ROWS_FP8
        out = codes.data_ptr(), stride, scales.data_ptr(), blocks
    elif to == "fp4":
        if scale != "e8m0":
            raise ValueError(f"4-bit rows have 'e8m0' scales, got {scale!r}")
        made, row_kind, kind = Fp4Rows._new(rows, dim, device), T.ROWS_FP4, T.SCALE_E8M0
        out = made._args()[:4]
    else:
        raise ValueError(f"to must be 'fp8' or 'fp4', got {to!r}")
    residual_ptr, residual_stride, sum_ptr, sum_stride = None, 0, None, 0
    if residual is not None:
        residual_ptr, residual_stride, sum_ptr, sum_stride = residual.data_ptr(), residual.stride(0), summed.data_ptr(), summed.stride(0)
    _call(T.lib().tv_rms_norm_dev, device, x.data_ptr(), _VALUES[x.dtype], x.stride(0), residual_ptr, residual_stride, sum_ptr, sum_stride, weight_ptr, weight_type, eps,
          rows, dim, row_kind, kind, *out)
    return made


def rms_norm(x, weight=None, *, eps=1e-6, to="fp8", scale="e8m0"):
    """Rows x / sqrt(mean(x^2) + eps) * weight as `Fp8Rows` (`to` "fp8"; scales "e8m0" or "f32") or `Fp4Rows` ("fp4") (tv_rms_norm_dev).  `x`: float32,
    float16 or bfloat16 [rows, dim]; `weight`: [dim] of any of these, or none.  All of it is taken in 32 bits (long sums in 64) and rounded once, to the codes."""
    return _made(_gpu("x", x, _VALUES), None, None, weight, eps, to, scale)


def add_rms_norm(x, residual, weight=None, *, eps=1e-6, to="fp8", scale="e8m0", out=None):
    """(the norm of x + residual as rows, x + residual): `rms_norm` of the sum before it is rounded, and the sum as a tensor of x's type, which is the next
    residual.  `out`: where the sum goes, a tensor like x; `x` or `residual` itself may be given, and overlaps no other way."""
    if residual is None:
        raise TypeError("residual must be a 2-D tensor like x; rms_norm takes none")
    _gpu("x", x, _VALUES)
    _like("residual", residual, x)
    out = torch.empty_strided(x.shape, (x.shape[1], 1), dtype=x.dtype, device=x.device) if out is None else _like("out", out, x)
    return _made(x, residual, out, weight, eps, to, scale), out
