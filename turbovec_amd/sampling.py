"""Drawing a slot from rows of scores -- temperature, top-k, top-p and min-p, from given random numbers -- and log probabilities of slots.

Where a search returns the best rows, a draw returns each row with its probability under a softmax of the scores: hard
negatives for training, varied retrieval, the next token where the rows are an output embedding.  `log_probs` is what training and serving ask
of the same softmax.  Everything is a torch tensor on the GPU; calls run on the current stream of the tensors' device and do not wait.  A draw carries
no gradient; log probabilities and entropies carry one to the scores.
"""
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

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


def _mask(mask, rows, n, device):
    """(address, words from one row's mask to the next's) of a mask of one row of words for all, or one for each."""
    if mask is None:
        return None, 0
    words = -(-n // 64)
    _gpu("mask", mask, (torch.int64,), ndim=2 if isinstance(mask, torch.Tensor) and mask.dim() == 2 else 1)
    if tuple(mask.shape) not in ((words,), (rows, words)):
        raise ValueError(f"mask must be {(words,)} or {(rows, words)}, got {tuple(mask.shape)}")
    _same_device(device, "mask", mask)
    return mask.data_ptr(), mask.stride(0) if mask.dim() == 2 else 0


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
    mask_ptr, mask_stride = _mask(mask, rows, n, device)
    slots = torch.empty(rows, dtype=torch.int64, device=device)
    probs = torch.empty(rows, dtype=torch.float32, device=device)
    ws = _workspace(T.lib().tv_sample_workspace(rows, n), device)
    _call(T.lib().tv_sample_dev, device, scores.data_ptr(), _VALUES[scores.dtype], scores.stride(0), rows, n, mask_ptr, mask_stride,
          u.data_ptr(), *(None if p is None else p.data_ptr() for p in params), slots.data_ptr(), probs.data_ptr(), *ws[1:])
    return slots, probs


_MOST_GIVEN = _MOST_TOP = 128


class LogProbs(NamedTuple):
    """`log_probs` float32 [rows] or [rows, given], as the slots were; `entropy` float32 [rows]; `top_slots` int64 and `top_log_probs` float32 [rows, top]."""

    log_probs: torch.Tensor
    entropy: torch.Tensor
    top_slots: torch.Tensor
    top_log_probs: torch.Tensor


def _forward(scores, slots, temperature, mask, top, stats):
    rows, n = scores.shape
    device, new = scores.device, torch.empty_strided
    shape = slots.shape
    given = shape[1] if len(shape) == 2 else 1
    log_p = new(shape, (given, 1)[-len(shape):], dtype=torch.float32, device=device)
    entropy = new((rows,), (1,), dtype=torch.float32, device=device)
    top_slots = new((rows, top), (top, 1), dtype=torch.int64, device=device)
    top_log_p = new((rows, top), (top, 1), dtype=torch.float32, device=device)
    L = T.lib()
    ws, ws_ptr, ws_bytes = _workspace(L.tv_log_probs_workspace(rows, n, top), device)
    _call(L.tv_log_probs_dev, device, scores.data_ptr(), _VALUES[scores.dtype], scores.stride(0), rows, n, *_mask(mask, rows, n, device),
          None if temperature is None else temperature.data_ptr(), slots.data_ptr(), slots.stride(0), given, top, log_p.data_ptr(), entropy.data_ptr(),
          top_slots.data_ptr(), top_log_p.data_ptr(), None if stats is None else stats.data_ptr(), ws_ptr, ws_bytes)
    return LogProbs(log_p, entropy, top_slots, top_log_p)


def _no_tangent(**tensors):
    """There is no derivative forward: a tangent that is dropped would read as zero."""
    if getattr(forward_ad, "_current_level", 0) < 0:          # (outside of every level, where this torch says so: no tensor has one)
        return
    for name, t in tensors.items():
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"{name}: log_probs has no forward-mode derivative")


class _WithGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, slots, temperature, mask, top, alternatives):
        stats = torch.empty((scores.shape[0], 4), dtype=torch.float32, device=scores.device)
        log_p, entropy, *alternatives[:] = _forward(scores, slots, temperature, mask, top, stats)
        ctx.save_for_backward(scores, slots, temperature, mask, stats)
        ctx.set_materialize_grads(False)
        return log_p, entropy

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g_log_probs, g_entropy):
        scores, slots, temperature, mask, stats = ctx.saved_tensors
        rows, n = scores.shape
        device = scores.device
        g_log_probs, g_entropy = (None if g is None else g.contiguous() for g in (g_log_probs, g_entropy))       # (a sum's is one number, spread)
        grad = torch.empty((rows, n), dtype=scores.dtype, device=device)
        _call(T.lib().tv_log_probs_grad_dev, device, scores.data_ptr(), _VALUES[scores.dtype], scores.stride(0), rows, n, *_mask(mask, rows, n, device),
              None if temperature is None else temperature.data_ptr(), slots.data_ptr(), slots.stride(0), slots.shape[1] if slots.dim() == 2 else 1, stats.data_ptr(),
              None if g_log_probs is None else g_log_probs.data_ptr(), None if g_entropy is None else g_entropy.data_ptr(), grad.data_ptr(), n)
        return grad, None, None, None, None, None


def log_probs(scores, slots, *, temperature=None, mask=None, top=0):
    """Log probabilities of given `slots` under a softmax of each row of `scores` / temperature, its entropy, and its `top` best slots (tv_log_probs_dev): a
    `LogProbs`.  `scores`: float32, float16 or bfloat16 [rows, n]; `slots`: int64 [rows] or [rows, given], at most 128 a row; `temperature` (a number, or float32 [rows]) and
    `mask` as `sample` takes them; `top`: 0 to 128, sorted (score desc, slot asc).

    A slot that the mask leaves out, one outside the row (-1, a draw from a row that allows nothing) and one of score -infinity have log probability -infinity, and what
    stands in a masked place never counts; a row that allows nothing has entropy 0, and where fewer than `top` slots have a probability the alternatives end in (-1, -infinity).
    An allowed NaN or +infinity makes its row NaN.  A temperature below 2^-126, 0 and negative ones among them, is the limit: the best slots share the mass, and the row has no gradient.  An infinite
    one gives every slot that has a probability the same, and the row's gradient is 0.

    `log_probs` and `entropy` carry a gradient to the scores (tv_log_probs_grad_dev; in the scores' type, rounded once, once differentiable); the alternatives carry none: give
    them as `slots` for that.  A temperature that requires a gradient is refused, and so are scores or a temperature with a forward-mode tangent."""
    _no_tangent(scores=scores, temperature=temperature)
    _gpu("scores", scores, _VALUES)
    rows, n = scores.shape
    if n == 0:
        raise ValueError("rows without scores")
    device = scores.device
    _gpu("slots", slots, (torch.int64,), ndim=2 if isinstance(slots, torch.Tensor) and slots.dim() == 2 else 1)
    if len(slots) != rows:
        raise ValueError(f"slots must be of {rows} rows, as scores, got {tuple(slots.shape)}")
    if slots.dim() == 2 and slots.shape[1] > _MOST_GIVEN:
        raise ValueError(f"at most {_MOST_GIVEN} slots a row, got {slots.shape[1]}")
    _same_device(device, "slots", slots)
    top = int(top)
    if not 0 <= top <= _MOST_TOP:
        raise ValueError(f"top must be 0 to {_MOST_TOP}, got {top}")
    temperature = _a_row("temperature", temperature, rows, torch.float32, device)
    if torch.is_grad_enabled() and temperature is not None and temperature.requires_grad:
        raise ValueError("a temperature has no gradient here: detach it, or divide the scores by it")
    if scores.requires_grad and torch.is_grad_enabled():
        alternatives = []          # (they carry no gradient, and need no place in its graph)
        return LogProbs(*_WithGradient.apply(scores, slots, temperature, mask, top, alternatives), *alternatives)
    return _forward(scores, slots, temperature, mask, top, None)
