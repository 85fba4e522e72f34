"""Logits adjusted before a token is drawn: penalties for tokens that occurred, biases, grammar masks.

One launch of st_logits_adjust (include/st_b200.h) for a batch of rows, each with a history, penalties, bias
entries and a mask of its own.  There is no counterpart in the reference.
"""
import torch

from . import _native as N
from .device import handle, ptr

_DTYPES = {torch.float32: N.ST_F32, torch.float16: N.ST_F16, torch.bfloat16: N.ST_BF16}


def _of(t, dtype, like, name, shape=None):
    if t is None:
        return None
    if t.dtype != dtype or not t.is_contiguous() or t.device != like.device:
        raise ValueError("%s must be a contiguous %s tensor on %s" % (name, str(dtype)[6:], like.device))
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError("%s has shape %s, not %s" % (name, tuple(t.shape), tuple(shape)))
    return t


def adjust(logits: torch.Tensor, tokens=None, starts=None, prompt=None, repetition=None, presence=None,
           frequency=None, bias=None, mask=None, out=None):
    """-> adjusted logits [rows, vocab] of the same type, in float32 arithmetic (``out`` may be ``logits``).

    Row r's history is tokens[starts[r]:starts[r + 1]] (int32; negative ones are padding), its first prompt[r]
    tokens the prompt.  For each token: x / repetition[r] (x > 0) or x * repetition[r] if it occurs in the history;
    - frequency[r] * n - presence[r] if it occurs n > 0 times after the prompt; + the row's entries of ``bias``
    = (tokens int32, values float32, starts int32 [rows + 1]); -inf where the row's mask has a 0 for it, ``mask``
    being (words int32 [masks, ceil(vocab / 32)], rows int32 [rows] or None): row r uses mask rows[r], none if
    negative; None: mask r.  Penalties are float32 [rows] or None."""
    if logits.dim() != 2 or not logits.is_cuda or logits.dtype not in _DTYPES:
        raise ValueError("logits are a float32, float16 or bfloat16 CUDA matrix")
    rows, vocab = logits.shape
    if logits.stride(1) != 1 or logits.stride(0) < vocab:
        logits = logits.contiguous()
    out = torch.empty((rows, vocab), dtype=logits.dtype, device=logits.device) if out is None else out
    if out.dtype != logits.dtype or tuple(out.shape) != (rows, vocab) or out.device != logits.device or \
            (rows and (out.stride(1) != 1 or out.stride(0) < vocab)):
        raise ValueError("out must be like logits, its rows contiguous")
    if (tokens is None) != (starts is None):
        raise ValueError("a history is tokens and starts")
    _of(tokens, torch.int32, logits, "tokens"), _of(starts, torch.int32, logits, "starts", (rows + 1,))
    _of(prompt, torch.int32, logits, "prompt", (rows,))
    for t, name in ((repetition, "repetition"), (presence, "presence"), (frequency, "frequency")):
        _of(t, torch.float32, logits, name, (rows,))
    ids, values, at = bias if bias is not None else (None, None, None)
    if bias is not None:
        _of(ids, torch.int32, logits, "bias tokens"), _of(values, torch.float32, logits, "bias values", ids.shape)
        _of(at, torch.int32, logits, "bias starts", (rows + 1,))
    words, which = mask if mask is not None else (None, None)
    if mask is not None:
        _of(words, torch.int32, logits, "mask", (words.shape[0], (vocab + 31) // 32))
        _of(which, torch.int32, logits, "mask rows", (rows,))
    handle(logits.device).call("st_logits_adjust", ptr(logits), max(vocab, logits.stride(0)), ptr(out),
                               max(vocab, out.stride(0)), rows, vocab, ptr(tokens),
                               0 if tokens is None else tokens.numel(), ptr(starts), ptr(prompt), ptr(repetition),
                               ptr(presence), ptr(frequency), ptr(ids), ptr(values),
                               0 if ids is None else ids.numel(), ptr(at),
                               ptr(words), 0 if words is None else words.shape[0], ptr(which), _DTYPES[logits.dtype])
    return out
