"""Rows in 8 bits beside an index: making them, their products with queries, and re-scoring of what a search returned.

An index holds 2 to 4 bits a coordinate.  These rows hold 8 (e4m3, with a scale for every block of 128 coordinates) and
answer what the index's codes are too coarse for: exact-to-8-bits scores of every row (`matmul`), and of the candidates
of a search (`rescore`).  Everything is a torch tensor on the GPU; calls run on the current stream of the tensors' device
and do not wait.
"""
from dataclasses import dataclass

import torch

from . import _lib as T

_VALUES = {torch.float32: T.F32, torch.float16: T.F16, torch.bfloat16: T.BF16}
_SCALES = {"e8m0": (T.SCALE_E8M0, torch.float8_e8m0fnu), "f32": (T.SCALE_F32, torch.float32)}
_SCALE_TYPES = {torch.float8_e8m0fnu: T.SCALE_E8M0, torch.float32: T.SCALE_F32}
BLOCK = 128                     # coordinates that share a scale
_MAX_DIM = 16384
_ROW_ALIGN = 16                 # bytes: rows of codes made here start at multiples of it


def _blocks(dim):
    return -(-dim // BLOCK)


def _desc(obj):
    return f"{obj.dim()}-D {obj.dtype} on {obj.device}" if isinstance(obj, torch.Tensor) else type(obj).__name__


def _gpu(name, t, dtypes, ndim=2):
    """`t`, or an error that names the argument: a GPU tensor of one of the types whose last axis is dense."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.dim() != ndim:
        wanted = " or ".join(str(d).replace("torch.", "") for d in dtypes)
        raise TypeError(f"{name} must be a {ndim}-D {wanted} tensor, got {_desc(t)}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU, got {t.device}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: elements of a row must lie next to each other; call contiguous() first")
    return t


def _same_device(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")


def _call(fn, device, *args):
    T.check(fn(device.index, torch.cuda.current_stream(device).cuda_stream, *args))


@dataclass(frozen=True)
class Fp8Rows:
    """`codes` float8_e4m3fn [rows, dim], `scales` [ceil(rows / group), ceil(dim / 128)] of float8_e8m0fnu or float32; a
    coordinate is code * scale.  `group`: rows that share a scale, 1 or 128."""
    codes: torch.Tensor
    scales: torch.Tensor
    group: int = 1

    def __post_init__(self):
        _gpu("codes", self.codes, (torch.float8_e4m3fn,))
        _gpu("scales", self.scales, tuple(_SCALE_TYPES))
        if self.group not in (1, BLOCK):
            raise ValueError(f"group must be 1 or {BLOCK}, got {self.group}")
        rows, dim = self.codes.shape
        if not 1 <= dim <= _MAX_DIM:
            raise ValueError(f"dim must be 1 to {_MAX_DIM}, got {dim}")
        if tuple(self.scales.shape) != (-(-rows // self.group), _blocks(dim)):
            raise ValueError(f"scales of {rows} x {dim} codes in groups of {self.group} rows must be "
                             f"{(-(-rows // self.group), _blocks(dim))}, got {tuple(self.scales.shape)}")
        _same_device(self.codes.device, scales=self.scales)

    def __len__(self):
        return self.codes.shape[0]

    @property
    def dim(self):
        return self.codes.shape[1]

    @property
    def _scale_type(self):
        return _SCALE_TYPES[self.scales.dtype]

    def _args(self):
        return self.codes.data_ptr(), self.codes.stride(0), self.scales.data_ptr(), self.scales.stride(0), len(self)


def quantize(x, *, scale="e8m0", group=1):
    """8-bit rows of `x` (float32, float16 or bfloat16 [rows, dim]; tv_fp8_quantize_dev).  `scale`: "e8m0", powers of two, which
    the matrix units apply at no cost, or "f32"; `group`: rows that share a scale, 1 or 128."""
    _gpu("x", x, tuple(_VALUES))
    if scale not in _SCALES:
        raise ValueError(f"scale must be 'e8m0' or 'f32', got {scale!r}")
    if group not in (1, BLOCK):
        raise ValueError(f"group must be 1 or {BLOCK}, got {group}")
    rows, dim = x.shape
    if not 1 <= dim <= _MAX_DIM:
        raise ValueError(f"dim must be 1 to {_MAX_DIM}, got {dim}")
    kind, dtype = _SCALES[scale]
    codes = torch.empty(rows, -(-dim // _ROW_ALIGN) * _ROW_ALIGN, dtype=torch.float8_e4m3fn, device=x.device)[:, :dim]
    scales = torch.empty(-(-rows // group), _blocks(dim), dtype=dtype, device=x.device)
    _call(T.lib().tv_fp8_quantize_dev, x.device, x.data_ptr(), _VALUES[x.dtype], x.stride(0), rows, dim, kind, group,
          codes.data_ptr(), codes.stride(0), scales.data_ptr(), scales.stride(0))
    return Fp8Rows(codes, scales, group)


def matmul(a, b, *, dtype=torch.float32, out=None):
    """Inner products of every row of `a` with every row of `b` (tv_fp8_matmul_dev): [len(a), len(b)] of `dtype`.  The
    rows of `a` have scales of their own, `b` may share them; both have the same type of scales."""
    if not isinstance(a, Fp8Rows) or not isinstance(b, Fp8Rows):
        raise TypeError(f"a and b must be Fp8Rows, got {type(a).__name__} and {type(b).__name__}")
    if a.group != 1:
        raise ValueError("rows of a must have scales of their own (group 1)")
    if a.dim != b.dim:
        raise ValueError(f"dim {a.dim} of a does not match dim {b.dim} of b")
    if a.scales.dtype != b.scales.dtype:
        raise ValueError(f"scales of a are {a.scales.dtype}, of b {b.scales.dtype}")
    _same_device(a.codes.device, b=b.codes)
    if out is None:
        if dtype not in _VALUES:
            raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        out = torch.empty(len(a), len(b), dtype=dtype, device=a.codes.device)
    else:
        _gpu("out", out, tuple(_VALUES))
        if tuple(out.shape) != (len(a), len(b)):
            raise ValueError(f"out must be {(len(a), len(b))}, got {tuple(out.shape)}")
        _same_device(a.codes.device, out=out)
    _call(T.lib().tv_fp8_matmul_dev, a.codes.device, *a._args(), *b._args(), b.group, a.dim, a._scale_type,
          out.data_ptr(), _VALUES[out.dtype], out.stride(0))
    return out


def rescore(queries, rows, slots, k):
    """The `k` best of each query's own candidate `slots` (int64 [queries, candidates], as a search returns them), scored against
    their 8-bit rows (tv_fp8_rescore_dev): (scores float32, slots int64), sorted (score desc, slot asc).  Slots outside the
    rows count as absent; a query with fewer than `k` present ends in (-inf, -1)."""
    if not isinstance(rows, Fp8Rows):
        raise TypeError(f"rows must be Fp8Rows, got {type(rows).__name__}")
    _gpu("queries", queries, tuple(_VALUES))
    _gpu("slots", slots, (torch.int64,))
    nq, m = slots.shape
    if tuple(queries.shape) != (nq, rows.dim):
        raise ValueError(f"queries must be {(nq, rows.dim)}, got {tuple(queries.shape)}")
    k = int(k)
    if not 0 <= k <= m:
        raise ValueError(f"k must be 0 to {m}, the number of candidates, got {k}")
    device = queries.device
    _same_device(device, rows=rows.codes, slots=slots)
    scores = torch.empty(nq, k, dtype=torch.float32, device=device)
    best = torch.empty(nq, k, dtype=torch.int64, device=device)
    ws = torch.empty(T.lib().tv_fp8_rescore_workspace(nq, m), dtype=torch.uint8, device=device)
    _call(T.lib().tv_fp8_rescore_dev, device, queries.data_ptr(), _VALUES[queries.dtype], queries.stride(0), nq,
          *rows._args(), rows.group, rows.dim, rows._scale_type, slots.data_ptr(), slots.stride(0), m, k,
          scores.data_ptr(), best.data_ptr(), ws.data_ptr(), ws.numel())
    return scores, best
