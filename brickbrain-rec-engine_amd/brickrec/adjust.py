"""Penalties, biases and masks on dense scores (or logits) before they are picked from: the face of
``bb_adjust_scores`` (include/brickrec.h).  Torch CUDA tensors in and out, on torch's current stream or
the ``stream`` given, no synchronisation.  No gradient flows through the call."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Union

import torch

from . import _lib as L
from .fp8 import _CODE, _On, _check_out, _ld, _refuse_grad, _rows_of

Number = Union[float, torch.Tensor]


def mask_words(mask: torch.Tensor) -> torch.Tensor:
    """bool [..., n] on a GPU -> int32 words [..., ⌈n/32⌉], bit i of word w = entry 32w + i: the layout of
    ``ItemIndex.eval_mask_bits`` and ``engine.bits_from_bool``, packed on the device."""
    n = mask.shape[-1]
    pad = torch.nn.functional.pad(mask, (0, -n % 32)).view(*mask.shape[:-1], -1, 32)
    bit = torch.arange(32, device=mask.device)
    return (pad.to(torch.int64) << bit).sum(-1).to(torch.int32)


def _list(t, name, dtypes, B, dev):
    """A list for each row [B, m], or one for all [m] -> (tensor, entries, elements between rows)."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.device != dev:
        raise TypeError(f"{name} is a tensor of {' or '.join(str(d) for d in dtypes)} on {dev}")
    if t.dim() == 1:
        return t.contiguous(), t.shape[0], 0
    if t.dim() != 2 or t.shape[0] != B:
        raise ValueError(f"{name} is [{B}, m] or [m]: got {tuple(t.shape)}")
    if t.stride(0) == 0 and t.stride(1) == 1:  # one list expanded over the rows
        return t, t.shape[1], 0
    t = _rows_of(t)
    return t, t.shape[1], _ld(t)


def _per_row(v: Number, name, B, dev):
    """A value for all rows, or a tensor of one for each -> (pointer or None, value, tensor)."""
    if isinstance(v, torch.Tensor):
        if v.dtype != torch.float32 or v.device != dev or tuple(v.shape) != (B,):
            raise TypeError(f"{name} is a number or a float32 tensor [{B}] on {dev}")
        v = v.contiguous()
        return v.data_ptr(), 0.0, v
    return None, float(v), None


def adjust_scores(scores: torch.Tensor, *, seen: Optional[torch.Tensor] = None,
                  seen_len: Optional[torch.Tensor] = None, repetition: Number = 1.0, presence: Number = 0.0,
                  frequency: Number = 0.0, bias_ids: Optional[torch.Tensor] = None,
                  bias: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Adjusted scores of [B, n] (f32, bf16 or f16; computed in f32, rounded once), in this order:

    * an id that stands c > 0 times among the first ``seen_len`` entries of the row's ``seen`` list: the
      score is divided by ``repetition`` if it is positive, multiplied if not, and loses ``frequency`` · c
      + ``presence``;
    * an id in the row's ``bias_ids`` gains the ``bias`` beside it (the last one, where it stands twice);
    * a 0 bit of ``mask`` makes the score -inf, whatever it was.

    seen, bias_ids: int32 or int64, [B, m] or [m] for all rows; ids outside [0, n) are skipped (pad with
    -1).  seen_len: int32 [B].  repetition (> 0), presence, frequency: numbers, or f32 [B].  bias: f32, as
    bias_ids.  mask: words [⌈n/32⌉] or [B, ⌈n/32⌉] (``ItemIndex.eval_mask_bits``), or bool [n] or [B, n],
    which costs a few launches more.  out: where to write; may be ``scores`` itself."""
    if not isinstance(scores, torch.Tensor) or scores.device.type != "cuda" or scores.dtype not in _CODE:
        raise TypeError("scores are a float32, bfloat16 or float16 tensor on a GPU")
    if scores.dim() != 2:
        raise ValueError(f"scores are [B, n]: got {tuple(scores.shape)}")
    params = (repetition, presence, frequency)
    tensors = [t for t in (scores, seen, seen_len, bias_ids, bias, mask, out, *params) if isinstance(t, torch.Tensor)]
    _refuse_grad(*tensors)
    if not isinstance(repetition, torch.Tensor) and not float(repetition) > 0.0:
        raise ValueError(f"repetition is above 0: got {repetition}")
    B, n = scores.shape
    dev = scores.device
    a = L.bb_adjust()
    with _On(stream, dev, tensors) as handle:
        keep = []
        if out is None:
            scores = _rows_of(scores)
            out = torch.empty((B, n), dtype=scores.dtype, device=dev)
        else:
            _check_out(out, (B, n), scores.dtype, dev)
            scores = _rows_of(scores)
        a.scores, a.out, a.B, a.n, a.ld_scores, a.ld_out = scores.data_ptr(), out.data_ptr(), B, n, _ld(scores), _ld(out)
        a.dtype = _CODE[scores.dtype]
        if seen is not None:
            t, a.n_seen, a.ld_seen = _list(seen, "seen", (torch.int32, torch.int64), B, dev)
            a.seen = t.data_ptr()
            a.ids64 |= int(t.dtype == torch.int64)
            keep.append(t)
            if seen_len is not None:
                if seen_len.dtype != torch.int32 or seen_len.device != dev or tuple(seen_len.shape) != (B,):
                    raise TypeError(f"seen_len is an int32 tensor [{B}] on {dev}")
                seen_len = seen_len.contiguous()
                a.seen_len = seen_len.data_ptr()
            a.repetition, a.repetition_all, t0 = _per_row(repetition, "repetition", B, dev)
            a.presence, a.presence_all, t1 = _per_row(presence, "presence", B, dev)
            a.frequency, a.frequency_all, t2 = _per_row(frequency, "frequency", B, dev)
            keep += [t0, t1, t2]
        elif seen_len is not None:
            raise ValueError("seen_len without seen")
        if (bias_ids is None) != (bias is None):
            raise ValueError("bias_ids and bias come together")
        if bias_ids is not None:
            if bias.shape != bias_ids.shape:
                raise ValueError(f"bias is as bias_ids: got {tuple(bias.shape)} and {tuple(bias_ids.shape)}")
            t, a.n_bias, a.ld_bias = _list(bias_ids, "bias_ids", (torch.int32, torch.int64), B, dev)
            v, _, ld = _list(bias, "bias", (torch.float32,), B, dev)
            if ld != a.ld_bias:  # (the two lists share one distance between rows)
                t, v = t.contiguous(), v.contiguous()
                a.ld_bias = 0 if t.dim() == 1 else _ld(t)
            a.bias_ids, a.bias = t.data_ptr(), v.data_ptr()
            a.ids64 |= 2 * int(t.dtype == torch.int64)
            keep += [t, v]
        if mask is not None:
            if mask.dtype == torch.bool:
                if mask.shape[-1] != n:
                    raise ValueError(f"a bool mask is [{n}] or [{B}, {n}]: got {tuple(mask.shape)}")
                mask = mask_words(mask)
            t, w, a.ld_mask = _list(mask, "mask", (torch.int32, torch.uint32), B, dev)
            if w != (n + 31) // 32:
                raise ValueError(f"the mask of {n} scores has {(n + 31) // 32} words: got {w}")
            a.mask = t.data_ptr()
            keep.append(t)
        L.check(L.load().bb_adjust_scores(dev.index, C.byref(a), handle), "bb_adjust_scores")
    return out
