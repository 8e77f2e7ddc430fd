"""Rows of 8-bit floating point with an f32 scale for each block of 128, and dense scores of them.

``quantize_rows`` turns embedding rows, activations or weights into :class:`Fp8Rows`;
``scores_fp8`` gives the dense products of two sets of them (every query against every item) and
``adjust.adjust_scores`` changes those before they are picked from.  A thin face of
``bb_quantize_fp8`` and ``bb_scores_fp8`` (include/brickrec.h), which say what is computed: torch CUDA
tensors in and out, on torch's current stream or the ``stream`` given, no synchronisation, no state
kept between calls.  No gradient flows through these calls, so inputs that ask for one are refused.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib as L

BLOCK = 128
_CODE = {torch.float32: L.BB_F32, torch.bfloat16: L.BB_BF16, torch.float16: L.BB_F16}


def blocks_of(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _refuse_grad(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("no gradient flows through this call: detach the inputs or call it under torch.no_grad()")


class _On:
    """The stream of a call (``handle``).  With a stream of the caller's, outputs are made for it and
    the inputs' memory is kept from reuse until it has passed this call."""

    __slots__ = ("stream", "device", "handle", "_ctx")

    def __init__(self, stream, device, inputs):
        self.stream, self.device, self._ctx = stream, device, None
        if stream is None:
            self.handle = torch.cuda.current_stream(device).cuda_stream
            return
        if stream.device != device:
            raise ValueError(f"stream of {stream.device} for tensors of {device}")
        self.handle = stream.cuda_stream
        if stream != torch.cuda.current_stream(device):
            for t in inputs:
                if t is not None:
                    t.record_stream(stream)
            self._ctx = torch.cuda.stream(stream)

    def __enter__(self):
        if self._ctx is not None:
            self._ctx.__enter__()
        return self.handle

    def __exit__(self, *exc):
        if self._ctx is not None:
            self._ctx.__exit__(*exc)


def _rows_of(x: torch.Tensor) -> torch.Tensor:
    """x with its columns next to each other and its rows apart (copied where they are not)."""
    n, d = x.shape
    if (d > 1 and x.stride(1) != 1) or (n > 1 and x.stride(0) < d):
        return x.contiguous()
    return x


def _ld(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else max(1, x.shape[1])


class Fp8Rows:
    """``codes`` float8_e4m3fn [n, 128·⌈d/128⌉] (columns from d on zero) and ``scales`` f32
    [⌈d/128⌉, n], or [⌈d/128⌉, ⌈n/128⌉] with ``tile`` (one scale for 128 × 128): element (i, j) is
    codes[i, j] · scales[j // 128, i or i // 128]."""

    __slots__ = ("codes", "scales", "d", "tile", "_c")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, d: int, tile: bool = False):
        if codes.dtype != torch.float8_e4m3fn or scales.dtype != torch.float32:
            raise TypeError(f"codes are float8_e4m3fn and scales float32: got {codes.dtype} and {scales.dtype}")
        if codes.device.type != "cuda" or scales.device != codes.device:
            raise TypeError("codes and scales are tensors of one GPU")
        n, kb = codes.shape[0], blocks_of(d)
        if d < 0 or codes.dim() != 2 or codes.shape[1] != kb * BLOCK:
            raise ValueError(f"codes of rows {d} wide are [n, {kb * BLOCK}]: got {tuple(codes.shape)}")
        if tuple(scales.shape) != (kb, blocks_of(n) if tile else n):
            raise ValueError(f"scales of {n} rows {d} wide are [{kb}, {blocks_of(n) if tile else n}]: got {tuple(scales.shape)}")
        if (n > 0 and kb > 0) and (codes.stride(1) != 1 or (scales.shape[1] > 1 and scales.stride(1) != 1)):
            raise ValueError("codes and scales are contiguous along their rows")
        self.codes, self.scales, self.d, self.tile = codes, scales, d, bool(tile)
        self._c = L.bb_fp8_rows(codes.data_ptr(), scales.data_ptr(), n, d, _ld(codes), _ld(scales), int(self.tile))

    @classmethod
    def empty(cls, n: int, d: int, tile: bool = False, device=None) -> "Fp8Rows":
        dev = torch.device("cuda" if device is None else device)
        kb = blocks_of(d)
        return cls(torch.empty((n, kb * BLOCK), dtype=torch.float8_e4m3fn, device=dev),
                   torch.empty((kb, blocks_of(n) if tile else n), dtype=torch.float32, device=dev), d, tile)

    def __len__(self) -> int:
        return self.codes.shape[0]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def part(self, start: int, stop: int) -> "Fp8Rows":
        """Rows [start, stop) as a view; with ``tile`` a start that is a multiple of 128."""
        if not 0 <= start <= stop <= len(self) or (self.tile and start % BLOCK):
            raise ValueError(f"no part [{start}, {stop}) of {len(self)} rows")
        a, b = (start // BLOCK, blocks_of(stop)) if self.tile else (start, stop)
        return Fp8Rows(self.codes[start:stop], self.scales[:, a:b], self.d, self.tile)

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
    if not isinstance(x, torch.Tensor) or x.device.type != "cuda" or x.dtype not in _CODE:
        raise TypeError("rows are a float32, bfloat16 or float16 tensor on a GPU")
    if x.dim() != 2:
        raise ValueError(f"rows are [n, d]: got {tuple(x.shape)}")
    _refuse_grad(x)
    with _On(stream, x.device, (x,) if out is None else (x, out.codes, out.scales)) as handle:
        x = _rows_of(x)
        n, d = x.shape
        if out is None:
            out = Fp8Rows.empty(n, d, tile, x.device)
        elif (len(out), out.d, out.tile, out.device) != (n, d, bool(tile), x.device):
            raise ValueError(f"out is {len(out)} rows {out.d} wide (tile={out.tile}) on {out.device}, not as x and tile ask")
        L.check(L.load().bb_quantize_fp8(x.device.index, x.data_ptr(), _CODE[x.dtype], _ld(x), C.byref(out._c), handle),
                "bb_quantize_fp8")
    return out


def scores_fp8(queries: Fp8Rows, items: Fp8Rows, *, dtype: torch.dtype = torch.float32,
               out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Dense scores [queries, items] of 8-bit rows: the inner product of every pair, accumulated in f32 and
    rounded once to ``dtype`` (f32, bf16 or f16).  The queries' scales are per row; the items' per
    row or per tile.  ``out``: a tensor of that shape (its dtype is then the scores') to write into; its
    rows may be strided, columns behind them stay as they were."""
    dev = queries.codes.device
    if items.codes.device != dev:
        raise ValueError("queries and items are on one device")
    inputs = () if stream is None else (queries.codes, queries.scales, items.codes, items.scales, out)
    with _On(stream, dev, inputs) as handle:
        if out is None:
            if dtype not in _CODE:
                raise TypeError(f"scores are float32, bfloat16 or float16: not {dtype}")
            out = torch.empty((queries.codes.shape[0], items.codes.shape[0]), dtype=dtype, device=dev)
        else:
            _check_out(out, (queries.codes.shape[0], items.codes.shape[0]), None, dev)
        L.check(L.load().bb_scores_fp8(dev.index, C.byref(queries._c), C.byref(items._c), out.data_ptr(),
                                       _CODE[out.dtype], _ld(out), handle), "bb_scores_fp8")
    return out


def _check_out(out, shape, dtype, dev):
    _refuse_grad(out)
    if out.dtype not in _CODE or (dtype is not None and out.dtype != dtype):
        raise TypeError(f"out has dtype {out.dtype}")
    if tuple(out.shape) != tuple(shape) or out.device != dev:
        raise ValueError(f"out is {tuple(shape)} on {dev}: got {tuple(out.shape)} on {out.device}")
    if (shape[1] > 1 and out.stride(1) != 1) or (shape[0] > 1 and out.stride(0) < shape[1]):
        raise ValueError("out is contiguous along its rows, and its rows do not overlap")
