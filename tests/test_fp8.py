"""The 8-bit rows' and the adjustment's refusals, without a GPU: every bad argument is an error before
any device call, and a good one fails loudly where there is no device."""
import ctypes as C

import pytest
import torch

from brickrec import _lib as L

GOOD = dict(codes=1 << 20, scales=1 << 30, rows=10, d=200, ld=256, scales_ld=10, tile=0)


def rows(**kw):
    return L.bb_fp8_rows(**{**GOOD, **kw})


def err(rc, word):
    assert rc == L.BB_E_ARG, rc
    msg = L.load().bb_last_error().decode()
    assert word in msg, msg


@pytest.mark.parametrize("kw, word", [
    (dict(codes=None), "null"), (dict(scales=None), "null"), (dict(codes=(1 << 20) + 8), "16-byte"),
    (dict(ld=264), "16-byte"), (dict(ld=128), "rounded up"), (dict(scales=(1 << 30) + 2), "not aligned"),
    (dict(scales_ld=9), "scales_ld"), (dict(rows=-1), "negative"), (dict(d=-1), "negative"),
    (dict(rows=1 << 31, scales_ld=1 << 31), "2^31"), (dict(d=(1 << 24) + 1), "2^24"),
])
def test_rows_are_checked(kw, word):
    lib = L.load()
    bad, good, x = rows(**kw), rows(), C.c_void_p(1 << 40)
    err(lib.bb_quantize_fp8(0, x, L.BB_F32, 200, C.byref(bad), None), word)
    err(lib.bb_scores_fp8(0, C.byref(bad), C.byref(good), x, L.BB_F32, 10, None), word)
    err(lib.bb_scores_fp8(0, C.byref(good), C.byref(bad), x, L.BB_F32, 10, None), word)


def test_quantize_and_scores_arguments():
    lib = L.load()
    g, x = rows(), C.c_void_p(1 << 40)
    err(lib.bb_quantize_fp8(0, x, L.BB_F64, 200, C.byref(g), None), "dtype")
    err(lib.bb_quantize_fp8(0, None, L.BB_F32, 200, C.byref(g), None), "null")
    err(lib.bb_quantize_fp8(0, C.c_void_p((1 << 40) + 2), L.BB_F32, 200, C.byref(g), None), "aligned")
    err(lib.bb_quantize_fp8(0, x, L.BB_F32, 199, C.byref(g), None), "ldx")
    err(lib.bb_quantize_fp8(0, x, L.BB_F32, 200, None, None), "null")
    err(lib.bb_quantize_fp8(0, C.c_void_p((1 << 20) + 256), L.BB_BF16, 200, C.byref(g), None), "overlap")
    err(lib.bb_scores_fp8(0, C.byref(g), C.byref(rows(d=201)), x, L.BB_F32, 10, None), "width")
    err(lib.bb_scores_fp8(0, C.byref(rows(tile=1)), C.byref(g), x, L.BB_F32, 10, None), "queries")
    err(lib.bb_scores_fp8(0, C.byref(rows(d=0)), C.byref(rows(d=0)), x, L.BB_F32, 10, None), "width 0")
    err(lib.bb_scores_fp8(0, C.byref(g), C.byref(g), None, L.BB_F32, 10, None), "null out")
    err(lib.bb_scores_fp8(0, C.byref(g), C.byref(g), x, L.BB_F32, 9, None), "ldo")
    err(lib.bb_scores_fp8(0, C.byref(g), C.byref(g), x, 7, 10, None), "dtype")
    err(lib.bb_scores_fp8(0, C.byref(g), C.byref(g), C.c_void_p((1 << 40) + 1), L.BB_F16, 10, None), "aligned")
    err(lib.bb_scores_fp8(0, C.byref(g), C.byref(g), C.c_void_p(1 << 20), L.BB_F32, 10, None), "overlap")


def adj(**kw):
    base = dict(scores=1 << 20, out=1 << 30, B=3, n=100, ld_scores=100, ld_out=100, dtype=L.BB_F32)
    return L.bb_adjust(**{**base, **kw})


@pytest.mark.parametrize("kw, word", [
    (dict(scores=None), "null"), (dict(out=None), "null"), (dict(B=-1), "negative"), (dict(n=1 << 31), "2^31"),
    (dict(ld_scores=99), "ld < n"), (dict(ld_out=99), "ld < n"), (dict(dtype=L.BB_F64), "dtype"),
    (dict(scores=(1 << 20) + 2), "aligned"), (dict(out=(1 << 20) + 4), "overlaps"),
    (dict(out=1 << 20, ld_out=101), "overlaps"), (dict(n_seen=4), "without seen"),
    (dict(seen=1 << 12, n_seen=4, ld_seen=3), "ld_seen"), (dict(seen=(1 << 12) + 4, n_seen=4, ids64=1), "aligned"),
    (dict(n_bias=2, bias_ids=1 << 12), "n_bias"), (dict(n_bias=2, bias_ids=1 << 12, bias=1 << 13, ld_bias=1), "ld_bias"),
    (dict(mask=1 << 12, ld_mask=3), "ld_mask"), (dict(mask=(1 << 12) + 1), "aligned"), (dict(n_seen=-1), "negative"),
    (dict(B=1 << 40, out=1 << 62), "too many"),
])
def test_adjust_is_checked(kw, word):
    a = adj(**kw)
    err(L.load().bb_adjust_scores(0, C.byref(a), None), word)


def test_nothing_to_do_needs_no_device():
    lib = L.load()
    assert lib.bb_adjust_scores(0, C.byref(adj(B=0)), None) == L.BB_OK
    assert lib.bb_adjust_scores(0, C.byref(adj(n=0)), None) == L.BB_OK
    assert lib.bb_quantize_fp8(0, None, L.BB_F32, 0, C.byref(rows(rows=0)), None) == L.BB_OK
    assert lib.bb_scores_fp8(0, C.byref(rows(rows=0)), C.byref(rows()), None, L.BB_F32, 10, None) == L.BB_OK


def test_no_device_is_an_error():
    if torch.cuda.is_available():
        pytest.skip("there is a device")
    lib = L.load()
    assert lib.bb_adjust_scores(0, C.byref(adj()), None) == L.BB_E_HIP
    assert lib.bb_quantize_fp8(0, C.c_void_p(1 << 40), L.BB_F32, 200, C.byref(rows()), None) == L.BB_E_HIP
    assert lib.bb_scores_fp8(0, C.byref(rows()), C.byref(rows()), C.c_void_p(1 << 40), L.BB_F32, 10, None) == L.BB_E_HIP


def test_host_tensors_are_refused():
    import brickrec as br
    with pytest.raises(TypeError):
        br.quantize_rows(torch.zeros(3, 5))
    with pytest.raises(TypeError):
        br.adjust_scores(torch.zeros(3, 5))
    with pytest.raises(TypeError):
        br.Fp8Rows(torch.zeros(3, 128, dtype=torch.float8_e4m3fn), torch.zeros(1, 3), 5)


def test_layouts_match_the_header():
    from test_abi import _c_layout
    structs = {n: [f[0] for f in getattr(L, n)._fields_] for n in ("bb_fp8_rows", "bb_adjust")}
    lay = _c_layout(structs)
    for n, fields in structs.items():
        assert C.sizeof(getattr(L, n)) == lay[n], n
        for f in fields:
            assert getattr(getattr(L, n), f).offset == lay[f"{n}.{f}"], f"{n}.{f}"


def test_codes_and_scales_apart():
    g = rows(scales=(1 << 20) + 2048)
    err(L.load().bb_quantize_fp8(0, C.c_void_p(1 << 40), L.BB_F32, 200, C.byref(g), None), "codes and scales")


@pytest.mark.parametrize("kw", [
    dict(seen=(1 << 30) + 1024, n_seen=4), dict(seen=(1 << 30) - 4, n_seen=2), dict(mask=1 << 30),
    dict(bias_ids=1 << 12, bias=(1 << 30) + 8, n_bias=1), dict(bias_ids=(1 << 30) + 8, bias=1 << 12, n_bias=1),
    dict(seen=1 << 12, n_seen=1, seen_len=(1 << 30) - 8), dict(repetition=1 << 30), dict(presence=1 << 30),
    dict(frequency=1 << 30), dict(seen=(1 << 30) - 200, n_seen=1, ld_seen=25),
])
def test_adjust_out_apart_from_what_is_read(kw):
    a = adj(**kw)
    err(L.load().bb_adjust_scores(0, C.byref(a), None), "overlaps a list")


def test_rows_packed_as_the_structure():
    from brickrec import fp8
    b = fp8._PACK(1 << 20, 1 << 30, 10, 200, 256, 11, True)
    r = L.bb_fp8_rows.from_buffer_copy(b)
    assert len(b) == C.sizeof(r)
    assert [getattr(r, f[0]) for f in r._fields_] == [1 << 20, 1 << 30, 10, 200, 256, 11, 1]
