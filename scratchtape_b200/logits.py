"""Logits adjusted before a token is drawn: penalties for tokens that occurred, biases, grammar masks.

One launch of st_logits_adjust (include/st_b200.h) for a batch of rows, each with a history, penalties, bias
entries and a mask of its own.  There is no counterpart in the reference.
"""
import torch

from . import _native as N
from .device import handle

_DTYPES = {torch.float32: N.ST_F32, torch.float16: N.ST_F16, torch.bfloat16: N.ST_BF16}


def _of(t, dtype, device, name, shape=None):
    """t's pointer (None: NULL), t being a contiguous tensor of that type."""
    if t is None:
        return None
    if t.dtype is not dtype or t.device != device or not t.is_contiguous():
        raise ValueError("%s must be a contiguous %s tensor on %s" % (name, str(dtype)[6:], device))
    if shape is not None and t.shape != shape:
        raise ValueError("%s has shape %s, not %s" % (name, tuple(t.shape), tuple(shape)))
    return t.data_ptr()


def adjust(logits: torch.Tensor, tokens=None, starts=None, prompt=None, repetition=None, presence=None,
           frequency=None, bias=None, mask=None, out=None):
    """-> adjusted logits [rows, vocab] of the same type, in float32 arithmetic (``out`` may be ``logits``).

    Row r's history is tokens[starts[r]:starts[r + 1]] (int32; negative ones are padding), its first prompt[r]
    tokens the prompt.  For each token: x / repetition[r] (x > 0) or x * repetition[r] if it occurs in the history;
    - frequency[r] * n - presence[r] if it occurs n > 0 times after the prompt; + the row's entries of ``bias``
    = (tokens int32, values float32, starts int32 [rows + 1]); -inf where the row's mask has a 0 for it, ``mask``
    being (words int32 [masks, ceil(vocab / 32)], rows int32 [rows] or None): row r uses mask rows[r], none if
    negative; None: mask r.  Penalties are float32 [rows] or None."""
    code = _DTYPES.get(logits.dtype)
    if code is None or logits.dim() != 2 or not logits.is_cuda:
        raise ValueError("logits are a float32, float16 or bfloat16 CUDA matrix")
    rows, vocab = logits.shape
    ld, one = logits.stride()
    if one != 1 or ld < vocab:
        logits = logits.contiguous()
        ld = max(vocab, 1)
    device = logits.device
    if out is None:
        out = torch.empty((rows, vocab), dtype=logits.dtype, device=device)
        out_ld = vocab
    else:
        out_ld, one = out.stride()
        if out.dtype is not logits.dtype or out.shape != (rows, vocab) or out.device != device or \
                (rows and (one != 1 or out_ld < vocab)):
            raise ValueError("out must be like logits, its rows contiguous")
    if (tokens is None) != (starts is None):
        raise ValueError("a history is tokens and starts")
    f32, i32 = torch.float32, torch.int32
    ids = values = at = words = which = None
    n_bias = masks = 0
    if bias is not None:
        n_bias = bias[0].numel()
        ids, values = _of(bias[0], i32, device, "bias tokens"), _of(bias[1], f32, device, "bias values", bias[0].shape)
        at = _of(bias[2], i32, device, "bias starts", (rows + 1,))
    if mask is not None:
        masks = mask[0].shape[0]
        words = _of(mask[0], i32, device, "mask", (masks, (vocab + 31) // 32))
        which = _of(mask[1], i32, device, "mask rows", (rows,))
    handle(device).call("st_logits_adjust", logits.data_ptr(), max(vocab, ld), out.data_ptr(), max(vocab, out_ld), rows,
                        vocab, _of(tokens, i32, device, "tokens"), 0 if tokens is None else tokens.numel(),
                        _of(starts, i32, device, "starts", (rows + 1,)), _of(prompt, i32, device, "prompt", (rows,)),
                        _of(repetition, f32, device, "repetition", (rows,)),
                        _of(presence, f32, device, "presence", (rows,)),
                        _of(frequency, f32, device, "frequency", (rows,)), ids, values, n_bias, at, words, masks, which,
                        code)
    return out
