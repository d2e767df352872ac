"""Drawing a slot from rows of scores: temperature, top-k, top-p and min-p, from given random numbers.

Where a search returns the best rows, a draw returns each row with its probability under a softmax of the scores: hard
negatives for training, varied retrieval, the next token where the rows are an output embedding.  Everything is a torch
tensor on the GPU; calls run on the current stream of the tensors' device and do not wait.  Results carry no gradient.
"""
import torch

from . import _lib as T
from .fp8 import _VALUES, _call, _gpu, _same_device, _workspace


def _a_row(name, value, rows, dtype, device):
    """A value a row: a tensor as it is, or a number for all of them."""
    if value is None:
        return None
    if not isinstance(value, torch.Tensor):
        return torch.full((rows,), value, dtype=dtype, device=device)
    if value.dtype is dtype and value.shape == (rows,) and value.device == device and value.is_contiguous():
        return value
    # (what is wrong with it)
    _gpu(name, value, (dtype,), ndim=1)
    if len(value) != rows:
        raise ValueError(f"{name} must have a value a row, {rows}, got {len(value)}")
    _same_device(device, name, value)
    return value


def sample(scores, u, *, temperature=None, top_k=None, top_p=None, min_p=None, mask=None):
    """One slot from each row of `scores` (float32, float16 or bfloat16 [rows, n]; tv_sample_dev): (slots int64, probabilities
    float32).  `u` (float32 [rows], in [0, 1)) are the random numbers.  Each parameter is a number or a tensor of a value a row
    (float32, `top_k` int32); None: temperature 1, no limit.  `mask`: int64 words of 64 slots, slot i in bit
    i % 64 of word i // 64 (`torch.from_numpy(_lib.pack_mask(allowed)[0].view(numpy.int64))`, moved to the scores' device), [ceil(n / 64)] for all rows or
    [rows, ceil(n / 64)].  Slots are limited by top-k, then top-p, then min-p, and drawn in
    the order of slots; a row that allows nothing gives (-1, 0).  A slot whose weight is less than 2^-(63 - ceil(log2 n)) of the best one's
    is never drawn (less than 2e-5 of a draw in all at ten million slots, a third at most at 2^31 - 1)."""
    _gpu("scores", scores, _VALUES)
    rows, n = scores.shape
    if n == 0:
        raise ValueError("rows without scores")
    device = scores.device
    if not isinstance(u, torch.Tensor):
        raise TypeError(f"u must be a 1-D float32 tensor, got {type(u).__name__}")
    u = _a_row("u", u, rows, torch.float32, device)
    params = [_a_row(name, value, rows, dtype, device) for name, value, dtype in (
        ("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32))]
    mask_ptr, mask_stride = None, 0
    if mask is not None:
        words = -(-n // 64)
        _gpu("mask", mask, (torch.int64,), ndim=2 if isinstance(mask, torch.Tensor) and mask.dim() == 2 else 1)
        if tuple(mask.shape) not in ((words,), (rows, words)):
            raise ValueError(f"mask must be {(words,)} or {(rows, words)}, got {tuple(mask.shape)}")
        _same_device(device, "mask", mask)
        mask_ptr, mask_stride = mask.data_ptr(), mask.stride(0) if mask.dim() == 2 else 0
    slots = torch.empty(rows, dtype=torch.int64, device=device)
    probs = torch.empty(rows, dtype=torch.float32, device=device)
    ws = _workspace(T.lib().tv_sample_workspace(rows, n), device)
    _call(T.lib().tv_sample_dev, device, scores.data_ptr(), _VALUES[scores.dtype], scores.stride(0), rows, n, mask_ptr, mask_stride,
          u.data_ptr(), *(None if p is None else p.data_ptr() for p in params), slots.data_ptr(), probs.data_ptr(), *ws[1:])
    return slots, probs
