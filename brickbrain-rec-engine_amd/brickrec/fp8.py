"""Rows of 8-bit floating point with an f32 scale for each block of 128, and dense scores of them.

``quantize_rows`` turns embedding rows, activations or weights into :class:`Fp8Rows`;
``scores_fp8`` gives the dense products of two sets of them (every query against every item) and
``adjust.adjust_scores`` changes those before they are picked from.  A thin face of
``bb_quantize_fp8`` and ``bb_scores_fp8`` (include/brickrec.h), which say what is computed: torch CUDA
tensors in and out, on torch's current stream or the ``stream`` given, no synchronisation, no state
kept between calls.  No gradient or tangent flows through these calls, so inputs that ask for one are refused.
"""
from __future__ import annotations

import operator
import struct
from typing import Optional

import torch
from torch.autograd import forward_ad as _forward

from . import _lib as L

BLOCK = 128
_E4M3, _F32 = torch.float8_e4m3fn, torch.float32
# bb_fp8_rows packed into bytes (a third of the time of a ctypes structure); its fields in order
_PACK = struct.Struct("@PPqqqqi4x").pack
_CODE = {torch.float32: L.BB_F32, torch.bfloat16: L.BB_BF16, torch.float16: L.BB_F16}


def blocks_of(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _refuse_grad(*tensors):
    """(Called where a tensor requires a gradient, or within a forward-mode level: _forward._current_level >= 0.)"""
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError("no gradient flows through this call: detach the inputs or call it under torch.no_grad()")
    if any(_forward.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError("no tangent flows through this call: unpack the inputs first")


def _wrote(*outs):
    """Tells autograd of a write into a caller's tensors, as torch's own calls do."""
    for t in outs:
        if not t.is_inference():  # (inference tensors have no version)
            torch.autograd.graph.increment_version(t)


_raw_stream = torch._C._cuda_getCurrentRawStream  # current_stream(device).cuda_stream, without the object (2 us a call)


class _On:
    """A stream of the caller's for one call: outputs are made for it, and the inputs' memory is kept
    from reuse until it has passed the call."""

    __slots__ = ("handle", "_ctx")

    def __init__(self, stream, device, inputs):
        if stream.device != device:
            raise ValueError(f"stream of {stream.device} for tensors of {device}")
        self.handle, self._ctx = stream.cuda_stream, torch.cuda.stream(stream)
        if self.handle != _raw_stream(device.index):
            for t in inputs:
                if isinstance(t, torch.Tensor):
                    t.record_stream(stream)

    def __enter__(self):
        self._ctx.__enter__()
        return self.handle

    def __exit__(self, *exc):
        self._ctx.__exit__(*exc)


def _empty(n, m, dtype, device):
    return torch.empty_strided((n, m), (m or 1, 1), dtype=dtype, device=device)  # (a third off torch.empty's time)


def _rows_of(x: torch.Tensor) -> torch.Tensor:
    """x with its columns next to each other and its rows apart (copied where they are not)."""
    if x.is_contiguous():
        return x
    n, d = x.shape
    if (d > 1 and x.stride(1) != 1) or (n > 1 and x.stride(0) < d):
        return x.contiguous()
    return x


def _ld(x: torch.Tensor) -> int:
    """Elements between the rows of x."""
    return x.stride(0) if x.shape[0] > 1 else max(1, x.shape[1])


class Fp8Rows:
    """``codes`` float8_e4m3fn [n, 128·⌈d/128⌉] (columns from d on zero) and ``scales`` f32
    [⌈d/128⌉, n], or [⌈d/128⌉, ⌈n/128⌉] with ``tile`` (one scale for 128 × 128): element (i, j) is
    codes[i, j] · scales[j // 128, i or i // 128].  The calls use the tensors' memory as it is when the
    rows are made: their contents may change after that, their storage may not be resized or replaced."""

    __slots__ = ("_codes", "_scales", "_d", "_tile", "_c", "_cut")  # (_cut: other rows share the last tile's scale)
    codes = property(operator.attrgetter("_codes"), doc="float8_e4m3fn [n, 128·⌈d/128⌉]")
    scales = property(operator.attrgetter("_scales"), doc="f32 [⌈d/128⌉, n], or [⌈d/128⌉, ⌈n/128⌉] with tile")
    d = property(operator.attrgetter("_d"), doc="columns of a row")
    tile = property(operator.attrgetter("_tile"), doc="whether a scale covers 128 rows")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, d: int, tile: bool = False):
        if not isinstance(codes, torch.Tensor) or not isinstance(scales, torch.Tensor):
            raise TypeError("codes and scales are tensors")
        if codes.dtype is not _E4M3 or scales.dtype is not _F32:
            raise TypeError(f"codes are float8_e4m3fn and scales float32: got {codes.dtype} and {scales.dtype}")
        if not codes.is_cuda or scales.get_device() != codes.get_device():
            raise TypeError("codes and scales are tensors of one GPU")
        if d < 0 or codes.dim() != 2 or scales.dim() != 2:
            raise ValueError("codes and scales are matrices")
        (n, w), (sk, sn), kb = codes.shape, scales.shape, (d + 127) // 128
        if w != kb * BLOCK:
            raise ValueError(f"codes of rows {d} wide are [n, {kb * BLOCK}]: got {tuple(codes.shape)}")
        want = (n + 127) // 128 if tile else n
        if sk != kb or sn != want:
            raise ValueError(f"scales of {n} rows {d} wide are [{kb}, {want}]: got {tuple(scales.shape)}")
        ld, sld = w, sn
        if not (codes.is_contiguous() and scales.is_contiguous()):
            if n > 0 and kb > 0 and (codes.stride(1) != 1 or (sn > 1 and scales.stride(1) != 1)):
                raise ValueError("codes and scales are contiguous along their rows")
            ld, sld = _ld(codes), _ld(scales)
        if codes.requires_grad or scales.requires_grad or _forward._current_level >= 0:
            _refuse_grad(codes, scales)
        self._codes, self._scales, self._d, self._tile, self._cut = codes, scales, d, bool(tile), False
        self._c = _PACK(codes.data_ptr(), scales.data_ptr(), n, d, ld, sld, self._tile)

    @classmethod
    def empty(cls, n: int, d: int, tile: bool = False, device=None) -> "Fp8Rows":
        """Rows to be written (``quantize_rows(..., out=...)``)."""
        dev = torch.device("cuda" if device is None else device)
        if dev.type != "cuda":
            raise TypeError(f"rows are on a GPU: not on {dev}")
        kb = (d + 127) // 128
        sn = (n + 127) // 128 if tile else n
        new = cls.__new__(cls)
        new._codes = _empty(n, kb * BLOCK, _E4M3, dev)
        new._scales = _empty(kb, sn, _F32, dev)
        new._d, new._tile, new._cut = d, bool(tile), False
        new._c = _PACK(new._codes.data_ptr(), new._scales.data_ptr(), n, d, kb * BLOCK or 1, sn or 1, new._tile)
        return new

    def __reduce__(self):
        return Fp8Rows, (self._codes, self._scales, self._d, self._tile)

    def __len__(self) -> int:
        return self._codes.shape[0]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def part(self, start: int, stop: int) -> "Fp8Rows":
        """Rows [start, stop) as a view; with ``tile`` a start that is a multiple of 128, and a view that ends inside
        a tile is for reading."""
        if not 0 <= start <= stop <= len(self) or (self.tile and start % BLOCK):
            raise ValueError(f"no part [{start}, {stop}) of {len(self)} rows")
        a, b = (start // BLOCK, blocks_of(stop)) if self.tile else (start, stop)
        new = Fp8Rows(self.codes[start:stop], self.scales[:, a:b], self.d, self.tile)
        new._cut = self.tile and stop % BLOCK > 0 and (stop < len(self) or self._cut)
        return new

    def dequantize(self) -> torch.Tensor:
        """The rows as f32 [n, d] (for inspection: the scores are computed from the codes)."""
        n, kb = len(self), blocks_of(self.d)
        s = self.scales.repeat_interleave(BLOCK, dim=1)[:, :n] if self.tile else self.scales
        x = self.codes.float().view(n, kb, BLOCK) * s.t().unsqueeze(2)
        return x.reshape(n, kb * BLOCK)[:, : self.d]


def quantize_rows(x: torch.Tensor, *, tile: bool = False, out: Optional[Fp8Rows] = None, stream=None) -> Fp8Rows:
    """8-bit rows of x ([n, d] f32, bf16 or f16; rows may be strided).

    One scale for each block of 128 columns of a row, or with ``tile`` for each 128 × 128 block; a
    block with an infinity or a NaN gets scale NaN and codes 0.  ``out``: rows of the same shape to
    write into."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _CODE:
        raise TypeError("rows are a float32, bfloat16 or float16 tensor on a GPU")
    if out is not None and not isinstance(out, Fp8Rows):
        raise TypeError(f"out is Fp8Rows: got {type(out).__name__}")
    if x.dim() != 2:
        raise ValueError(f"rows are [n, d]: got {tuple(x.shape)}")
    if x.requires_grad or _forward._current_level >= 0:
        _refuse_grad(x)
    if stream is not None:
        with _On(stream, x.device, (x,) if out is None else (x, out.codes, out.scales)):
            return quantize_rows(x, tile=tile, out=out)
    x = _rows_of(x)
    n, d = x.shape
    dev, given = x.get_device(), out is not None
    if not given:
        out = Fp8Rows.empty(n, d, tile, x.device)
    elif (len(out), out._d, out._tile, out._codes.get_device()) != (n, d, bool(tile), dev):
        raise ValueError(f"out is {len(out)} rows {out.d} wide (tile={out.tile}) on {out.device}, not as x and tile ask")
    elif out._cut:
        raise ValueError(f"out ends inside a tile of 128 rows, whose scale the rows behind it share: {len(out)} rows")
    elif out._scales.requires_grad:
        _refuse_grad(out._scales)
    rc = L.load().bb_quantize_fp8(dev, x.data_ptr(), _CODE[x.dtype], _ld(x), out._c, _raw_stream(dev))
    if rc:
        L.check(rc, "bb_quantize_fp8")
    if given:
        _wrote(out._codes, out._scales)
    return out


def scores_fp8(queries: Fp8Rows, items: Fp8Rows, *, dtype: torch.dtype = torch.float32,
               out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Dense scores [queries, items] of 8-bit rows: the inner product of every pair, accumulated in f32 and
    rounded once to ``dtype`` (f32, bf16 or f16).  bf16 scores come from the 8-bit matrix instruction, at up to
    twice the rate: it cuts each product at 2^-13 of the largest of its group of 8 columns, at most 2^-10 of
    the sum of the products' magnitudes in all; f32 and f16 scores lose nothing there.  The queries' scales are
    per row; the items' per row or per tile.  ``out``: a tensor of that shape (its dtype is then the scores') to
    write into; its rows may be strided, columns behind them stay as they were."""
    if not isinstance(queries, Fp8Rows) or not isinstance(items, Fp8Rows):
        raise TypeError(f"queries and items are Fp8Rows: got {type(queries).__name__} and {type(items).__name__}")
    q, x = queries._codes, items._codes
    dev = q.get_device()
    if dev < 0:
        raise TypeError(f"rows are on a GPU: not on {q.device}")
    if x.get_device() != dev:
        raise ValueError("queries and items are on one device")
    if queries._scales.requires_grad or items._scales.requires_grad:  # (asked for after the rows were made)
        _refuse_grad(queries._scales, items._scales)
    if stream is not None:
        with _On(stream, q.device, (q, queries.scales, x, items.scales, out)):
            return scores_fp8(queries, items, dtype=dtype, out=out)
    given = out is not None
    if not given:
        if dtype not in _CODE:
            raise TypeError(f"scores are float32, bfloat16 or float16: not {dtype}")
        out = _empty(q.shape[0], x.shape[0], dtype, q.device)
        ld = x.shape[0] or 1
    else:
        ld = _check_out(out, (q.shape[0], x.shape[0]), None, dev)
    rc = L.load().bb_scores_fp8(dev, queries._c, items._c, out.data_ptr(), _CODE[out.dtype], ld,
                                _raw_stream(dev))
    if rc:
        L.check(rc, "bb_scores_fp8")
    if given:
        _wrote(out)
    return out


def _check_out(out, shape, dtype, dev):
    """The elements between the rows of a tensor to write into."""
    if not isinstance(out, torch.Tensor):
        raise TypeError(f"out is a tensor: got {type(out).__name__}")
    if out.requires_grad or _forward._current_level >= 0:
        _refuse_grad(out)
    if out.dtype not in _CODE or (dtype is not None and out.dtype is not dtype):
        raise TypeError(f"out has dtype {out.dtype}")
    if out.get_device() != dev or out.shape != shape:
        raise ValueError(f"out is {tuple(shape)} on cuda:{dev}: got {tuple(out.shape)} on {out.device}")
    if out.is_contiguous():
        return shape[1] or 1
    if (shape[1] > 1 and out.stride(1) != 1) or (shape[0] > 1 and out.stride(0) < shape[1]):
        raise ValueError("out is contiguous along its rows, and its rows do not overlap")
    return _ld(out)
