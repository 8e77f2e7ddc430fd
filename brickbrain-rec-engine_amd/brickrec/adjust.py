"""Penalties, biases and masks on dense scores (or logits) before they are picked from: the face of
``bb_adjust_scores`` (include/brickrec.h).  Torch CUDA tensors in and out, on torch's current stream or
the ``stream`` given, no synchronisation.  No gradient flows through the call."""
from __future__ import annotations

import struct
from typing import Optional, Union

import torch

from . import _lib as L
from .fp8 import _CODE, _On, _check_out, _empty, _forward, _ld, _raw_stream, _refuse_grad, _rows_of, _wrote

Number = Union[float, torch.Tensor]


def mask_words(mask: torch.Tensor) -> torch.Tensor:
    """bool [..., n] on a GPU -> int32 words [..., ⌈n/32⌉], bit i of word w = entry 32w + i: the layout of
    ``ItemIndex.eval_mask_bits`` and ``engine.bits_from_bool``, packed on the device."""
    n = mask.shape[-1]
    pad = torch.nn.functional.pad(mask.bool(), (0, -n % 32)).contiguous().view(torch.uint8)
    bit = torch.arange(8, dtype=torch.uint8, device=mask.device)
    # (8 bits to a byte, 4 bytes to a word: two bytes a score besides the words)
    return (pad.view(*mask.shape[:-1], (n + 31) // 32, 4, 8) << bit).sum(-1, dtype=torch.uint8).view(torch.int32).squeeze(-1)


# bb_adjust packed into bytes (a third of the time of a ctypes structure); its fields in order
_PACK = struct.Struct("@PPqqqqiiPqqPPPPfffPPqqPq").pack
_IDS = {torch.int32: 0, torch.int64: 1}
_F32 = {torch.float32: 0}
_FLOAT, _BOOL = torch.float32, torch.bool
_WORDS = {torch.int32: 0, torch.uint32: 0}


def _list(t, name, dtypes, B, dev):
    """A list for each row [B, m], or one for all [m] -> (tensor, entries, elements between rows)."""
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes or t.get_device() != dev:
        raise TypeError(f"{name} is a tensor of {' or '.join(str(d) for d in dtypes)} on cuda:{dev}")
    shape = t.shape
    flat = t.is_contiguous()
    if len(shape) == 2 and shape[0] == B:
        m = shape[1]
        if flat:
            return t, m, m or 1
        if t.stride(0) == 0 and t.stride(1) == 1:  # one list expanded over the rows
            return t, m, 0
        t = _rows_of(t)
        return t, m, _ld(t)
    if len(shape) != 1:
        raise ValueError(f"{name} is [{B}, m] or [m]: got {tuple(shape)}")
    return t if flat else t.contiguous(), shape[0], 0


def _per_row(v: Number, name, B, dev):
    """A value for all rows, or a tensor of one for each -> (pointer or 0, value, tensor)."""
    if not isinstance(v, torch.Tensor):
        return 0, float(v), None
    if v.dtype is not _FLOAT or v.get_device() != dev or v.dim() != 1 or v.numel() != B:
        raise TypeError(f"{name} is a number or a float32 tensor [{B}] on cuda:{dev}")
    if v.requires_grad or _forward._current_level >= 0:
        _refuse_grad(v)
    if not v.is_contiguous():
        v = v.contiguous()
    return v.data_ptr(), 0.0, v


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
    which costs a few launches and two bytes of memory a score more.  out: where to write; may be ``scores`` itself."""
    if not isinstance(scores, torch.Tensor) or not scores.is_cuda or scores.dtype not in _CODE:
        raise TypeError("scores are a float32, bfloat16 or float16 tensor on a GPU")
    if scores.dim() != 2:
        raise ValueError(f"scores are [B, n]: got {tuple(scores.shape)}")
    if stream is not None:
        with _On(stream, scores.device, (scores, seen, seen_len, repetition, presence, frequency, bias_ids, bias, mask, out)):
            return adjust_scores(scores, seen=seen, seen_len=seen_len, repetition=repetition, presence=presence,
                                 frequency=frequency, bias_ids=bias_ids, bias=bias, mask=mask, out=out)
    if scores.requires_grad or _forward._current_level >= 0:
        _refuse_grad(scores)
    shape, dtype, dev = scores.shape, scores.dtype, scores.get_device()
    B, n = shape
    ld_scores = ld = n or 1
    if not scores.is_contiguous():
        scores = _rows_of(scores)
        ld_scores = _ld(scores)
    given = out is not None
    if not given:
        out = _empty(B, n, dtype, scores.device)
    else:
        ld = _check_out(out, shape, dtype, dev)
    # every tensor that the launch reads has a name here until it is out
    seen_p = seen_len_p = rep_p = pre_p = fre_p = bias_ids_p = bias_p = mask_p = 0
    n_seen = ld_seen = n_bias = ld_bias = ld_mask = ids64 = 0
    rep, pre, fre = 1.0, 0.0, 0.0
    if not isinstance(repetition, torch.Tensor) and not repetition > 0.0:
        raise ValueError(f"repetition is above 0: got {repetition}")
    if isinstance(seen, torch.Tensor) and isinstance(bias_ids, torch.Tensor) and {seen.dtype, bias_ids.dtype} == _IDS.keys():
        seen, bias_ids = seen.to(torch.int64), bias_ids.to(torch.int64)  # (the lists of one call have ids of one size)
    if seen is not None:
        seen, n_seen, ld_seen = _list(seen, "seen", _IDS, B, dev)
        seen_p, ids64 = seen.data_ptr(), int(seen.dtype is torch.int64)
        if seen_len is not None:
            if (not isinstance(seen_len, torch.Tensor) or seen_len.dtype is not torch.int32 or seen_len.get_device() != dev
                    or seen_len.dim() != 1 or seen_len.numel() != B):
                raise TypeError(f"seen_len is an int32 tensor [{B}] on cuda:{dev}")
            if not seen_len.is_contiguous():
                seen_len = seen_len.contiguous()
            seen_len_p = seen_len.data_ptr()
        rep_p, rep, repetition = _per_row(repetition, "repetition", B, dev)
        pre_p, pre, presence = _per_row(presence, "presence", B, dev)
        fre_p, fre, frequency = _per_row(frequency, "frequency", B, dev)
    elif seen_len is not None:
        raise ValueError("seen_len without seen")
    if (bias_ids is None) != (bias is None):
        raise ValueError("bias_ids and bias come together")
    if bias_ids is not None:
        bias_ids, n_bias, ld_bias = _list(bias_ids, "bias_ids", _IDS, B, dev)
        bias, m, ld_v = _list(bias, "bias", _F32, B, dev)
        if m != n_bias or bias.dim() != bias_ids.dim():
            raise ValueError(f"bias is as bias_ids: got {tuple(bias.shape)} and {tuple(bias_ids.shape)}")
        if bias.requires_grad or _forward._current_level >= 0:
            _refuse_grad(bias)
        if ld_v != ld_bias:  # (the two lists share one distance between rows)
            bias_ids, bias = bias_ids.contiguous(), bias.contiguous()
            ld_bias = _ld(bias_ids)
        bias_ids_p, bias_p = bias_ids.data_ptr(), bias.data_ptr()
        ids64 = int(bias_ids.dtype is torch.int64)
    if mask is not None:
        if isinstance(mask, torch.Tensor) and mask.dtype is _BOOL:
            if mask.dim() == 0 or mask.shape[-1] != n:
                raise ValueError(f"a bool mask is [{n}] or [{B}, {n}]: got {tuple(mask.shape)}")
            mask = mask_words(mask)
        mask, w, ld_mask = _list(mask, "mask", _WORDS, B, dev)
        if w != (n + 31) // 32:
            raise ValueError(f"the mask of {n} scores has {(n + 31) // 32} words: got {w}")
        mask_p = mask.data_ptr()
    rc = L.load().bb_adjust_scores(
        dev, _PACK(scores.data_ptr(), out.data_ptr(), B, n, ld_scores, ld, _CODE[dtype], ids64, seen_p, n_seen, ld_seen,
                   seen_len_p, rep_p, pre_p, fre_p, rep, pre, fre, bias_ids_p, bias_p, n_bias, ld_bias, mask_p, ld_mask),
        _raw_stream(dev))
    if rc:
        L.check(rc, "bb_adjust_scores")
    if given:
        _wrote(out)
    return out
