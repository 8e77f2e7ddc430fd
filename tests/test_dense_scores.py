"""The host side of the dense scores, without a GPU."""
import contextlib
import threading
import types

import numpy as np
import pytest
import torch

from brickrec import _lib as L
from brickrec import engine, fp8


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_rows_of_any_magnitude_are_normalised(dtype):
    g = torch.Generator().manual_seed(1)
    q = (torch.randn((50, 384), generator=g) * torch.exp(torch.randn((50, 1), generator=g))).to(dtype)
    want = torch.nn.functional.normalize(q, dim=1)
    assert torch.equal(engine._unit_rows(q), want)            # ordinary rows: bit for bit
    far = (66, 120, -66, -100) if dtype == torch.float32 else (600, 1000, -600, -900)
    for e in far:
        assert torch.equal(engine._unit_rows(q * 2.0 ** e), want), e
    f = torch.finfo(dtype)
    s = torch.zeros((5, 4), dtype=dtype)
    s[0, 1], s[1], s[3, 0], s[4, 2] = f.smallest_normal * f.eps, f.max, float("inf"), float("nan")
    got = engine._unit_rows(s)
    assert got[0].tolist() == [0, 1, 0, 0] and got[2].tolist() == [0, 0, 0, 0]
    # 4 equal numbers: squares below 4, their sum, its root and the quotient each off by at most half a step
    assert bool(((got[1] - 0.5).abs() <= 4 * f.eps).all())
    assert bool(torch.isnan(got[3:]).any(1).all())


class _Lib:
    """What the index's calls reach here, with the library's status codes."""

    def __init__(self, rc=0):
        self.rc = rc

    def bb_upload_items(self, *a):
        return self.rc

    def bb_last_error(self):
        return b"stub"


def _index(monkeypatch, n=10, d=8):
    """An index whose rows are host tensors, and whose 8-bit copies are made by nothing."""
    from brickrec import fp8

    class Rows:
        def __init__(self, n=n, d=d, **kw):
            self.got = []

        def part(self, a, b):
            return self.got

    idx = engine.ItemIndex.__new__(engine.ItemIndex)
    idx._lib, idx._h, idx._mu = _Lib(), None, threading.RLock()
    idx.dtype, idx.device, idx.id_offset, idx.n_items, idx.d = "f32", 0, 0, n, d
    real = torch.arange
    monkeypatch.setattr(torch, "arange", lambda *a, device=None: real(*a))
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: types.SimpleNamespace(synchronize=lambda: None))
    monkeypatch.setattr(fp8.Fp8Rows, "empty", staticmethod(Rows))
    monkeypatch.setattr(fp8, "quantize_rows", lambda x, out: out.append(x))
    idx.get_rows = lambda ids: ids
    return idx


@pytest.mark.parametrize("through_view", [False, True])
@pytest.mark.parametrize("at", [0, 8])
def test_an_upload_waits_for_the_copy_and_drops_it(monkeypatch, at, through_view):
    idx = _index(monkeypatch)
    other = None

    def get_rows(ids):
        nonlocal other
        if int(ids[0]) == at:   # another thread uploads while this chunk is read
            other = threading.Thread(target=idx.upload_items, args=(np.zeros((10, 8), np.float32),))
            other.start()
            other.join(0.3)
        return ids
    idx.get_rows = get_rows
    who = idx
    if through_view:
        who = engine.ItemIndex.__new__(engine.ItemIndex)
        who.__dict__.update(idx.__dict__, _mu=threading.RLock(), _base=idx)
    rows = who.quantize_items(chunk=4)
    assert [r.tolist() for r in rows.got] == [[0, 1, 2, 3], [4, 5, 6, 7], [8, 9]]
    other.join()
    assert idx.quantized is None
    who._mu = None   # (nothing to close)


@pytest.mark.parametrize("rc, kept", [(L.BB_E_ARG, True), (L.BB_E_STATE, True), (L.BB_E_HIP, False), (L.BB_E_NOMEM, False)])
def test_a_failed_upload_drops_the_copy_and_a_refused_one_keeps_it(monkeypatch, rc, kept):
    idx = _index(monkeypatch)
    rows = idx.quantize_items()
    assert idx.quantized is rows
    idx._lib.rc = rc
    monkeypatch.setattr(L, "load", lambda: idx._lib)
    with pytest.raises(L.BrickrecError):
        idx.upload_items(np.zeros((10, 8), np.float32))
    assert (idx.quantized is rows) == kept


def _launches_nothing(monkeypatch):
    """A library in which every launch is recorded instead: none may be reached with host memory."""
    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: calls.append(name) or 0
    monkeypatch.setattr(L, "load", lambda: Lib())
    monkeypatch.setattr(fp8, "_raw_stream", lambda dev: 0)
    return calls


@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_rows_are_made_on_a_gpu_only(monkeypatch, device):
    calls = _launches_nothing(monkeypatch)
    with pytest.raises(TypeError):
        fp8.Fp8Rows.empty(3, 128, device=device)
    # rows that came by other means: neither side may reach a launch
    rows = fp8.Fp8Rows.__new__(fp8.Fp8Rows)
    rows._codes = torch.empty((3, 128), dtype=torch.float8_e4m3fn, device=device)
    rows._scales = torch.empty((1, 3), device=device)
    rows._d, rows._tile = 128, False
    rows._c = fp8._PACK(0, 0, 3, 128, 128, 3, False)
    with pytest.raises(TypeError):
        fp8.scores_fp8(rows, rows)
    with pytest.raises(TypeError):
        fp8.scores_fp8(rows, rows, out=torch.empty((3, 3), device=device))
    assert calls == []


def test_semantic_scores_need_an_index_that_has_them():
    from _oracle_index import OracleIndex
    from brickrec.semantic import SemanticIndex
    sem = SemanticIndex(["a", "b"], np.eye(2, 4), index_factory=OracleIndex)
    with pytest.raises(L.BrickrecError, match="OracleIndex"):
        sem.scores(np.ones(4))


def test_dtype_and_out_agree(monkeypatch):
    idx = _index(monkeypatch)
    idx.quantize_items()
    for q in (np.zeros((2, 8), np.float32), types.SimpleNamespace()):
        with pytest.raises(TypeError, match="out"):
            idx.scores(q, dtype=torch.float32, out=torch.empty((2, 10), dtype=torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8, torch.int32, torch.float32])
def test_mask_words_of_any_type(dtype):
    from brickrec.adjust import mask_words
    m = torch.rand((2, 70), generator=torch.Generator().manual_seed(1)) < 0.5
    assert np.array_equal(mask_words(m.to(dtype)).numpy().view(np.uint32), engine.bits_from_bool(m.numpy()))
