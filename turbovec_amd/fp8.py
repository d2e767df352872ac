"""Rows in 8 bits beside an index: making them, their products with queries, and re-scoring of what a search returned.

An index holds 2 to 4 bits a coordinate.  These rows hold 8 (e4m3, with a scale for every block of 128 coordinates) and
answer what the index's codes are too coarse for: exact-to-8-bits scores of every row (`matmul`), and of the candidates
of a search (`rescore`).  Everything is a torch tensor on the GPU; calls run on the current stream of the tensors' device
and do not wait.  Results carry no gradient.
"""
import torch

from . import _lib as T

_VALUES = {torch.float32: T.F32, torch.float16: T.F16, torch.bfloat16: T.BF16}
_SCALES = {"e8m0": (T.SCALE_E8M0, torch.float8_e8m0fnu), "f32": (T.SCALE_F32, torch.float32)}
_CODES = (torch.float8_e4m3fn,)
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
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name}: elements of a row must lie next to each other; call contiguous() first")
    return t


def _same_device(device, name, t):
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")


def _call(fn, device, *args):
    at = device.index
    status = fn(at, _stream_of(at), *args)
    if status != T.OK:
        T.check(status)


# (the pointer itself, where this torch hands it out: a Stream object takes a fifth of a short call's time)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream_of(index):
    return _raw_stream(index) if _raw_stream is not None else torch.cuda.current_stream(index).cuda_stream


def _workspace(size, device):
    """(tensor, address, bytes) of a call's workspace.  It is given back when the call has been made: what the stream runs
    later may take it over, and comes later."""
    if size == 0:
        return None, None, 0
    t = torch.empty(size, dtype=torch.uint8, device=device)
    return t, t.data_ptr(), size


class Fp8Rows:
    """`codes` float8_e4m3fn [rows, dim], `scales` [ceil(rows / group), ceil(dim / 128)] of float8_e8m0fnu or float32; a
    coordinate is code * scale.  `group`: rows that share a scale, 1 or 128.

    Beside an index row i is its slot i, which is the caller's to keep so: an index's `add` puts new rows at the end, its `swap_remove(i)` the last
    one in place of row i (with `group` 1 the same move of a row of `codes` and one of `scales`)."""

    __slots__ = ("_codes", "_scales", "_group", "_scale_type")

    def __init__(self, codes, scales, group=1):
        _gpu("codes", codes, _CODES)
        _gpu("scales", scales, _SCALE_TYPES)
        if group not in (1, BLOCK):
            raise ValueError(f"group must be 1 or {BLOCK}, got {group}")
        rows, dim = codes.shape
        if not 1 <= dim <= _MAX_DIM:
            raise ValueError(f"dim must be 1 to {_MAX_DIM}, got {dim}")
        if scales.shape != (-(-rows // group), -(-dim // BLOCK)):
            raise ValueError(f"scales of {rows} x {dim} codes in groups of {group} rows must be "
                             f"{(-(-rows // group), _blocks(dim))}, got {tuple(scales.shape)}")
        _same_device(codes.device, "scales", scales)
        self._codes, self._scales, self._group, self._scale_type = codes, scales, group, _SCALE_TYPES[scales.dtype]

    def _set(self, codes, scales, group, scale_type):
        self._codes, self._scales, self._group, self._scale_type = codes, scales, group, scale_type
        return self

    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)
    group = property(lambda self: self._group)
    dim = property(lambda self: self._codes.shape[1])

    def __len__(self):
        return self._codes.shape[0]

    def _args(self):
        c, s = self._codes, self._scales
        return c.data_ptr(), c.stride(0), s.data_ptr(), s.stride(0), c.shape[0]

    def __repr__(self):
        return f"Fp8Rows({len(self)} x {self.dim}, scales {self.scales.dtype} of {self.group} rows, {self.codes.device})"


def quantize(x, *, scale="e8m0", group=1):
    """8-bit rows of `x` (float32, float16 or bfloat16 [rows, dim]; tv_fp8_quantize_dev).  `scale`: "e8m0", powers of two, which
    the matrix units apply at no cost, or "f32"; `group`: rows that share a scale, 1 or 128."""
    _gpu("x", x, _VALUES)
    if scale not in _SCALES:
        raise ValueError(f"scale must be 'e8m0' or 'f32', got {scale!r}")
    if group not in (1, BLOCK):
        raise ValueError(f"group must be 1 or {BLOCK}, got {group}")
    rows, dim = x.shape
    if not 1 <= dim <= _MAX_DIM:
        raise ValueError(f"dim must be 1 to {_MAX_DIM}, got {dim}")
    kind, dtype = _SCALES[scale]
    device = x.device
    codes = torch.empty_strided((rows, dim), (-(-dim // _ROW_ALIGN) * _ROW_ALIGN, 1), dtype=torch.float8_e4m3fn, device=device)
    scales = torch.empty((-(-rows // group), _blocks(dim)), dtype=dtype, device=device)
    made = Fp8Rows.__new__(Fp8Rows)._set(codes, scales, group, kind)
    _call(T.lib().tv_fp8_quantize_dev, device, x.data_ptr(), _VALUES[x.dtype], x.stride(0), rows, dim, kind, group, *made._args()[:4])
    return made


def matmul(a, b, *, dtype=torch.float32, out=None):
    """Inner products of every row of `a` with every row of `b` (tv_fp8_matmul_dev): [len(a), len(b)] of `dtype`.  The
    rows of `a` have scales of their own, `b` may share them; both have the same type of scales.  float32 results are as good as sums in 32
    bits; float16 and bfloat16 ones come from 8-bit matrix instructions, which lose 1.4e-5 of the usual result of random rows, more of one close to 0."""
    if not isinstance(a, Fp8Rows) or not isinstance(b, Fp8Rows):
        raise TypeError(f"a and b must be Fp8Rows, got {type(a).__name__} and {type(b).__name__}")
    if a._group != 1:
        raise ValueError("rows of a must have scales of their own (group 1)")
    (m, dim), (n, b_dim) = a._codes.shape, b._codes.shape
    if dim != b_dim:
        raise ValueError(f"dim {dim} of a does not match dim {b_dim} of b")
    if a._scale_type != b._scale_type:
        raise ValueError(f"scales of a are {a.scales.dtype}, of b {b.scales.dtype}")
    device = a._codes.device
    _same_device(device, "b", b._codes)
    if out is None:
        if dtype not in _VALUES:
            raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
        out = torch.empty((m, n), dtype=dtype, device=device)
    else:
        _gpu("out", out, _VALUES)
        if out.shape != (m, n):
            raise ValueError(f"out must be {(m, n)}, got {tuple(out.shape)}")
        _same_device(device, "out", out)
    _call(T.lib().tv_fp8_matmul_dev, device, *a._args(), *b._args(), b._group, dim, a._scale_type,
          out.data_ptr(), _VALUES[out.dtype], out.stride(0))
    return out


def rescore(queries, rows, slots, k):
    """The `k` best of each query's own candidate `slots` (int64 [queries, candidates] on their device: `torch.from_numpy` of
    those that `TurboQuantIndex.search` returns, or what tv_search_dev wrote there), scored against their 8-bit rows (tv_fp8_rescore_dev): (scores float32, slots int64), sorted (score desc, slot asc).  Slots outside the
    rows count as absent; a query with fewer than `k` present ends in (-inf, -1)."""
    if not isinstance(rows, Fp8Rows):
        raise TypeError(f"rows must be Fp8Rows, got {type(rows).__name__}")
    _gpu("queries", queries, _VALUES)
    _gpu("slots", slots, (torch.int64,))
    nq, m = slots.shape
    dim = rows._codes.shape[1]
    if queries.shape != (nq, dim):
        raise ValueError(f"queries must be {(nq, dim)}, got {tuple(queries.shape)}")
    k = int(k)
    if not 0 <= k <= m:
        raise ValueError(f"k must be 0 to {m}, the number of candidates, got {k}")
    device = queries.device
    _same_device(device, "rows", rows._codes)
    _same_device(device, "slots", slots)
    scores = torch.empty((nq, k), dtype=torch.float32, device=device)
    best = torch.empty((nq, k), dtype=torch.int64, device=device)
    ws = _workspace(T.lib().tv_fp8_rescore_workspace(nq, m, dim), device)
    _call(T.lib().tv_fp8_rescore_dev, device, queries.data_ptr(), _VALUES[queries.dtype], queries.stride(0), nq,
          *rows._args(), rows._group, dim, rows._scale_type, slots.data_ptr(), slots.stride(0), m, k,
          scores.data_ptr(), best.data_ptr(), *ws[1:])
    return scores, best
