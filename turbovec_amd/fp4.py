"""Rows in 4 bits beside an index: making them, reading them back, and their products with queries.

Half the memory of 8-bit rows, and products at the matrix units' highest rate, for collections and weights whose scores may be coarse: e2m1 codes, two a byte,
with a power of two for every block of 32 coordinates (the microscaling format MXFP4).  Everything is a torch tensor on the GPU; calls run on the
current stream of the tensors' device and do not wait.  Results carry no gradient.
"""
import torch

from . import _lib as T
from .fp8 import _MAX_DIM, _VALUES, _call, _gpu, _same_device

BLOCK = 32                      # coordinates that share a scale
_CODES = (torch.uint8,)
_SCALES = (torch.float8_e8m0fnu,)
_ROW_ALIGN = 16                 # bytes: rows of codes made here start at multiples of it


def _blocks(dim):
    return -(-dim // BLOCK)


class Fp4Rows:
    """`codes` uint8 [rows, ceil(dim / 2)], coordinate 2i in the low half of byte i, and `scales` float8_e8m0fnu [rows, ceil(dim / 32)]; a coordinate
    is code * scale.  `dim`: 2 for each byte of a row, or 1 less where the last byte holds one coordinate.

    Beside an index row i is its slot i, which is the caller's to keep so, as with 8-bit rows."""

    __slots__ = ("_codes", "_scales", "_dim")

    def __init__(self, codes, scales, dim=None):
        _gpu("codes", codes, _CODES)
        _gpu("scales", scales, _SCALES)
        rows, row_bytes = codes.shape
        dim = 2 * row_bytes if dim is None else int(dim)
        if not 1 <= dim <= _MAX_DIM:
            raise ValueError(f"dim must be 1 to {_MAX_DIM}, got {dim}")
        if row_bytes != (dim + 1) // 2:
            raise ValueError(f"codes of dim {dim} must be {(rows, (dim + 1) // 2)}, got {tuple(codes.shape)}")
        if scales.shape != (rows, _blocks(dim)):
            raise ValueError(f"scales of {rows} rows of dim {dim} must be {(rows, _blocks(dim))}, got {tuple(scales.shape)}")
        _same_device(codes.device, "scales", scales)
        self._codes, self._scales, self._dim = codes, scales, dim

    @classmethod
    def _new(cls, rows, dim, device):
        self = cls.__new__(cls)
        self._codes = torch.empty_strided((rows, (dim + 1) // 2), (-(-dim // (2 * _ROW_ALIGN)) * _ROW_ALIGN, 1), dtype=torch.uint8, device=device)
        self._scales = torch.empty((rows, _blocks(dim)), dtype=torch.float8_e8m0fnu, device=device)
        self._dim = dim
        return self

    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)
    dim = property(lambda self: self._dim)

    def __len__(self):
        return self._codes.shape[0]

    def _args(self):
        c, s = self._codes, self._scales
        return c.data_ptr(), c.stride(0), s.data_ptr(), s.stride(0), c.shape[0]

    def values(self, dtype=torch.float32):
        """The coordinates, code * scale, as float32, float16 or bfloat16 [rows, dim] (tv_fp4_values_dev)."""
        if dtype not in _VALUES:
            raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        device = self._codes.device
        out = torch.empty((len(self), self._dim), dtype=dtype, device=device)
        _call(T.lib().tv_fp4_values_dev, device, *self._args(), self._dim, out.data_ptr(), _VALUES[dtype], self._dim)
        return out

    def __repr__(self):
        return f"Fp4Rows({len(self)} x {self.dim}, {self.codes.device})"


def quantize(x):
    """4-bit rows of `x` (float32, float16 or bfloat16 [rows, dim]; tv_fp4_quantize_dev).  A block with an infinity or a NaN is NaN.

    A block's scale is the smallest power of two that its largest magnitude is below 7 times of, which rounds that one as all others.  The format's usual conversion takes
    half of it where the largest is 1.75 times a power of two or more, and cuts at 6: rows made so can be given to `Fp4Rows`, but have other bytes."""
    _gpu("x", x, _VALUES)
    rows, dim = x.shape
    if not 1 <= dim <= _MAX_DIM:
        raise ValueError(f"dim must be 1 to {_MAX_DIM}, got {dim}")
    device = x.device
    made = Fp4Rows._new(rows, dim, device)
    _call(T.lib().tv_fp4_quantize_dev, device, x.data_ptr(), _VALUES[x.dtype], x.stride(0), rows, dim, *made._args()[:4])
    return made


def matmul(a, b, *, dtype=torch.float32, out=None):
    """Inner products of every row of `a` with every row of `b` (tv_fp4_matmul_dev): [len(a), len(b)] of `dtype`, as good as sums in 32 bits
    rounded once, whatever `dtype`."""
    if not isinstance(a, Fp4Rows) or not isinstance(b, Fp4Rows):
        raise TypeError(f"a and b must be Fp4Rows, got {type(a).__name__} and {type(b).__name__}")
    if a._dim != b._dim:
        raise ValueError(f"dim {a._dim} of a does not match dim {b._dim} of b")
    device = a._codes.device
    _same_device(device, "b", b._codes)
    m, n = len(a), len(b)
    if out is None:
        if dtype not in _VALUES:
            raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        out = torch.empty((m, n), dtype=dtype, device=device)
    else:
        _gpu("out", out, _VALUES)
        if out.shape != (m, n):
            raise ValueError(f"out must be {(m, n)}, got {tuple(out.shape)}")
        _same_device(device, "out", out)
    _call(T.lib().tv_fp4_matmul_dev, device, *a._args(), *b._args(), a._dim, out.data_ptr(), _VALUES[out.dtype], out.stride(0))
    return out
