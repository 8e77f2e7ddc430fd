"""Penalties, biases and masks on dense scores, on the device, against f64 (tests/_fp8_ref.py adjust)."""
import pytest
import torch

import _fp8_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")


@pytest.fixture(scope="module")
def br():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a ROCm device")
    import brickrec
    return brickrec


def make(B, n, dtype, H=0, nb=0, ids=torch.int32, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = {"scores": (3 * torch.randn((B, n), generator=g)).to(dtype)}
    if H:
        a["seen"] = torch.randint(-2, n + 2, (B, H), generator=g).to(ids)
        a["seen"][:, ::3] = a["seen"][:, :1].clone()           # one id again and again
        a["seen_len"] = torch.randint(-1, H + 3, (B,), generator=g).to(torch.int32)
        a["repetition"], a["presence"], a["frequency"] = (torch.rand(B, generator=g) + o for o in (1.0, -0.5, 0.0))
    if nb:
        a["bias_ids"] = torch.randint(-1, n + 1, (B, nb), generator=g).to(ids)
        a["bias_ids"][:, nb // 2:] = a["bias_ids"][:, :nb - nb // 2].clone()   # ids that stand twice: the last one counts
        a["bias"] = 5 * torch.randn((B, nb), generator=g)
    return a


def run(br, a, mask=None, **kw):
    dev = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    return br.adjust_scores(dev.pop("scores"), mask=None if mask is None else mask.to(DEV), **dev, **kw)


def check(a, got, mask=None):
    y, tol = R.adjust(a["scores"], a.get("seen"), a.get("seen_len"), a.get("repetition", 1.0), a.get("presence", 0.0),
                      a.get("frequency", 0.0), a.get("bias_ids"), a.get("bias"), mask)
    g = got.cpu().double()
    same = (g == y) | (torch.isnan(g) & torch.isnan(y))
    ok = same | ((g - y).abs() <= tol)
    assert bool(ok.all()), ((g - y).abs() / tol)[~ok]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B, n, H, nb", [(1, 1, 1, 1), (1, 7, 0, 2), (2, 31, 5, 0), (3, 33, 1, 1), (5, 1000, 300, 17), (4, 4096, 64, 8),
                                         (3, 4097, 700, 300), (2, 25216, 64, 8), (1, 50001, 5000, 600), (7, 8191, 2, 4),
                                         (300, 129, 20, 5)])
def test_adjust(br, B, n, H, nb, dtype):
    a = make(B, n, dtype, H, nb, seed=B + n)
    check(a, run(br, a))
    m = torch.rand((B, n), generator=torch.Generator().manual_seed(1)) < 0.5
    m[0] = False                                     # a row that the mask leaves empty
    check(a, run(br, a, m), m)
    one = m[-1]
    check(a, run(br, a, one), one.expand(B, n))


def test_plain_copy_and_mask_alone(br):
    a = make(3, 500, torch.bfloat16)
    assert torch.equal(run(br, a).cpu(), a["scores"])
    m = torch.zeros(500, dtype=torch.bool)
    assert bool((run(br, a, m) == -INF).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_special_scores(br, dtype):
    a = make(2, 100, dtype)
    s = a["scores"]
    s[:, 0], s[:, 1], s[:, 2] = INF, -INF, float("nan")
    s[:, 3], s[:, 4], s[:, 5] = torch.finfo(dtype).min, torch.finfo(dtype).max, 0.0
    s[:, 10:16] = s[:, 0:6]
    m = torch.ones(100, dtype=torch.bool)
    m[10:16] = False                                 # the same values in masked places
    a["seen"] = torch.tensor([[0, 1, 2, 3, 4, 5, 5, 10, 12]] * 2, dtype=torch.int32)
    a["repetition"], a["presence"], a["frequency"] = 2.0, 0.5, 0.25
    got = run(br, a, m).cpu().float()
    assert bool((got[:, 10:16] == -INF).all())
    assert bool((got[:, 0] == INF).all()) and bool((got[:, 1] == -INF).all()) and bool(torch.isnan(got[:, 2]).all())
    assert bool((got[:, 5] == -1.0).all())
    lowest = torch.tensor(torch.finfo(dtype).min * 2 - 0.75, dtype=torch.float64).to(torch.float32).to(dtype).float()
    assert bool((got[:, 3] == lowest).all())


@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
def test_id_types_and_shared_lists(br, ids):
    a = make(4, 3001, torch.float32, 50, 10, ids)
    check(a, run(br, a))
    far = a["seen"].clone().to(torch.int64)
    far[:, 0], far[:, 1] = 2 ** 40, -2 ** 40         # far outside [0, n): skipped
    check({**a, "seen": far}, run(br, {**a, "seen": far}))
    mixed = {**a, "seen": a["seen"].to(torch.int32), "bias_ids": a["bias_ids"].to(torch.int64)}
    check(mixed, run(br, mixed))
    b = {**a, "seen": a["seen"][0], "bias_ids": a["bias_ids"][1], "bias": a["bias"][1], "repetition": 1.5, "presence": 0.0}
    check(b, run(br, b))
    c = {**b, "seen": b["seen"].expand(4, 50)}
    check(c, run(br, c))
    d = {**a, "bias": a["bias"][:1].expand(4, 10)}   # ids by row, one set of values
    check(d, run(br, d))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1000, 4099])
def test_in_place_strided_and_misaligned(br, dtype, n):
    a = make(5, n, dtype, 30, 6, seed=3)
    m = torch.rand((5, n), generator=torch.Generator().manual_seed(2)) < 0.8
    want = run(br, a, m)
    buf = torch.full((7, n + 11), 9.0, dtype=dtype, device=DEV)
    view = buf[1:6, 3:n + 3]
    view.copy_(a["scores"])
    dev = {k: v.to(DEV) for k, v in a.items() if k != "scores"}
    assert br.adjust_scores(view, mask=m.to(DEV), out=view, **dev) is view
    assert torch.equal(view, want)
    view.fill_(9.0)
    assert bool((buf == 9.0).all())
    # lists with room behind their rows, scores whose columns lie apart
    wide = torch.full((5, 45), 1, dtype=torch.int32, device=DEV)
    wide[:, :30] = dev["seen"]
    wb = torch.full((5, 20), 1, dtype=torch.int32, device=DEV)
    wb[:, 4:10] = dev["bias_ids"]
    words = torch.full((5, (n + 31) // 32 + 3), -1, dtype=torch.int32, device=DEV)
    words[:, 1:-2] = br.mask_words(m.to(DEV))
    got = br.adjust_scores(a["scores"].t().contiguous().to(DEV).t(), mask=words[:, 1:-2],
                           **{**dev, "seen": wide[:, :30], "bias_ids": wb[:, 4:10]})
    assert torch.equal(got, want)


@pytest.mark.parametrize("H, nb", [(70000, 3), (5, 70000), (65535, 65535), (0, 65536), (65536, 0)])
def test_lists_at_and_past_16_bits(br, H, nb):
    n = 9000
    a = make(2, n, torch.float32, H, nb, seed=H + nb)
    if H:
        a["seen"][0] = 7                              # one id in every entry
        a["seen_len"] = torch.tensor([H, H - 1], dtype=torch.int32)
        a["frequency"] = torch.tensor([0.5, 0.25])
    if nb:
        a["bias_ids"][1] = 8                          # the last of all entries counts
    check(a, run(br, a))


def test_mask_words_layout(br):
    from brickrec.engine import bits_from_bool
    import numpy as np
    m = torch.rand((3, 77), generator=torch.Generator().manual_seed(1)) < 0.5
    w = br.mask_words(m.to(DEV)).cpu().numpy().view(np.uint32)
    assert np.array_equal(w, bits_from_bool(m.numpy()))


def test_replayed_with_new_inputs(br):
    a = make(6, 9000, torch.float32, 40, 5)
    dev = {k: v.to(DEV) for k, v in a.items()}
    scores = dev.pop("scores")
    out = torch.zeros_like(scores)
    br.adjust_scores(scores, out=out, **dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        br.adjust_scores(scores, out=out, **dev)
    for s in range(4):
        b = make(6, 9000, torch.float32, 40, 5, seed=50 + s)
        scores.copy_(b["scores"])
        for k, v in dev.items():
            v.copy_(b[k])
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run(br, b)), s
        out.sum().item()


def test_on_another_stream(br):
    a = make(6, 9000, torch.float32, 40, 5)
    want = run(br, a)
    dev = {k: v.to(DEV) for k, v in a.items()}
    scores = dev.pop("scores")
    s = torch.cuda.Stream(DEV)
    torch.cuda.synchronize()
    got = br.adjust_scores(scores, stream=s, **dev)
    s.synchronize()
    assert torch.equal(got, want)


def test_rows_further_apart_than_32_bits(br):
    ld = (1 << 31) + 4096
    buf = torch.empty(2 * ld + 1024, dtype=torch.float16, device=DEV)
    far = torch.as_strided(buf, (3, 600), (ld, 1))
    a = make(3, 600, torch.float16, 20, 3)
    far.copy_(a["scores"])
    dev = {k: v.to(DEV) for k, v in a.items() if k != "scores"}
    br.adjust_scores(far, out=far, **dev)
    assert torch.equal(far, run(br, a))


def test_refusals(br):
    s = torch.zeros((3, 64), device=DEV)
    i32 = torch.zeros((3, 4), dtype=torch.int32, device=DEV)
    f = torch.zeros((3, 4), device=DEV)
    for kw, e in (({"seen": i32.float()}, TypeError), ({"seen": i32[:2]}, ValueError), ({"seen": i32.cpu()}, TypeError),
                  ({"seen_len": i32[:, 0]}, ValueError), ({"seen": i32, "seen_len": i32[:, 0].long()}, TypeError),
                  ({"seen": i32, "repetition": 0.0}, ValueError), ({"seen": i32, "repetition": -1.0}, ValueError),
                  ({"seen": i32, "repetition": float("nan")}, ValueError), ({"seen": i32, "presence": f}, TypeError),
                  ({"bias_ids": i32}, ValueError), ({"bias": f}, ValueError), ({"bias_ids": i32, "bias": f[:, :3]}, ValueError),
                  ({"bias_ids": i32, "bias": f.double()}, TypeError), ({"mask": i32}, ValueError),
                  ({"mask": torch.ones((3, 63), dtype=torch.bool, device=DEV)}, ValueError),
                  ({"mask": torch.ones((3, 2), device=DEV)}, TypeError), ({"out": s.bfloat16()}, TypeError),
                  ({"out": s[:2]}, ValueError)):
        with pytest.raises(e):
            br.adjust_scores(s, **kw)
    with pytest.raises(br.BrickrecError):
        buf = torch.zeros((4, 64), device=DEV)
        br.adjust_scores(buf[:3], out=buf[1:])          # out overlaps scores
    with pytest.raises(ValueError):
        br.adjust_scores(torch.zeros((3, 64), device=DEV, requires_grad=True))
    with pytest.raises(TypeError):
        br.adjust_scores(torch.zeros((3, 64), device=DEV, dtype=torch.float64))
    with pytest.raises(ValueError):
        br.adjust_scores(torch.zeros(64, device=DEV))
    assert br.adjust_scores(s[:0]).shape == (0, 64) and br.adjust_scores(s[:, :0]).shape == (3, 0)


def test_no_rows_with_every_argument(br):
    for B, n in ((0, 64), (3, 0), (0, 0)):
        s = torch.zeros((B, n), device=DEV)
        y = br.adjust_scores(s, seen=torch.zeros((B, 4), dtype=torch.int32, device=DEV),
                             seen_len=torch.zeros(B, dtype=torch.int32, device=DEV),
                             bias_ids=torch.zeros((B, 2), dtype=torch.int32, device=DEV), bias=torch.zeros((B, 2), device=DEV),
                             mask=torch.ones((B, n), dtype=torch.bool, device=DEV))
        assert y.shape == (B, n)
    with pytest.raises(ValueError):
        br.adjust_scores(s, mask=torch.ones((), dtype=torch.bool, device=DEV))


def test_ids_at_the_ends_of_their_type(br):
    n = 9000
    a = make(2, n, torch.float32, 8, 4, torch.int64)
    lo, hi = torch.iinfo(torch.int64).min, torch.iinfo(torch.int64).max
    a["seen"][:] = torch.tensor([lo, hi, lo + n, -n, n, n - 1, 0, 2 ** 32])
    a["bias_ids"][:] = torch.tensor([lo, hi, 8192, 2 ** 32 + 1])
    a["seen_len"][:] = 8
    check(a, run(br, a))


def test_out_over_what_is_read(br):
    buf = torch.zeros(4 * 64, dtype=torch.int32, device=DEV)
    out = buf.view(torch.float32).view(4, 64)
    s = torch.zeros((4, 64), device=DEV)
    for kw in ({"seen": buf[:8]}, {"seen": buf[-4:]}, {"mask": buf[4:6]}, {"seen": torch.zeros_like(buf[:8]), "seen_len": buf[:4]},
               {"bias_ids": torch.zeros_like(buf[:8]), "bias": out.view(-1)[8:16]}, {"bias_ids": buf[:8], "bias": s.view(-1)[:8]},
               {"seen": torch.zeros_like(buf[:8]), "repetition": out.view(-1)[:4]}):
        with pytest.raises(br.BrickrecError):
            br.adjust_scores(s, out=out, **kw)


@pytest.mark.parametrize("B, n", [(1, 33), (6, 9000), (64, 131072)])
def test_replayed_with_a_bool_mask(br, B, n):
    """The words of a bool mask are made by a few more launches: captured with the call, replayed with other masks."""
    scores = torch.randn((B, n), device=DEV)
    mask = torch.ones((B, n), dtype=torch.bool, device=DEV)
    out = torch.zeros_like(scores)
    br.adjust_scores(scores, out=out, mask=mask)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        br.adjust_scores(scores, out=out, mask=mask)
    for s in range(4):
        m = torch.rand((B, n), generator=torch.Generator().manual_seed(s)) < 0.5
        mask.copy_(m)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, scores.masked_fill(~mask, -INF)), s
        out.clamp(min=0).sum().item()


def test_what_is_no_tensor_is_a_type_error(br):
    s = torch.zeros((2, 64), device=DEV)
    ids = torch.zeros((2, 3), dtype=torch.int32, device=DEV)
    one = torch.ones((2, 3), device=DEV)
    for kw in ({"seen": [1, 2]}, {"seen": [[1], [2]], "bias_ids": ids, "bias": one}, {"seen": ids, "bias_ids": [1, 2, 3], "bias": one},
               {"seen": ids, "seen_len": [3, 3]}, {"bias_ids": ids, "bias": [1.0, 2.0, 3.0]}, {"mask": [True] * 64},
               {"mask": bytes(8)}, {"seen": ids, "repetition": [1.0, 2.0]}, {"seen": ids, "presence": "much"}, {"out": [0.0]}):
        with pytest.raises((TypeError, ValueError)):
            br.adjust_scores(s, **kw)


def test_mask_words_take_little_memory(br):
    """One byte a score for the padded copy, one for its shifted bits, an eighth for the words, and room for the allocator's
    rounding of each."""
    m = torch.ones((64, 131001), dtype=torch.bool, device=DEV)
    br.mask_words(m)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    w = br.mask_words(m)
    assert torch.cuda.max_memory_allocated() - before <= 2.25 * m.numel() + (1 << 20)
    assert w.shape == (64, 4094) and w.dtype == torch.int32
    assert bool((w[:, :-1] == -1).all()) and bool((w[:, -1] == (1 << 131001 % 32) - 1).all())


@pytest.mark.parametrize("shape", [(1,), (31,), (32,), (33,), (2, 3, 70), (0, 5), (4, 0)])
def test_mask_words_of_any_shape(br, shape):
    from brickrec.engine import bits_from_bool
    import numpy as np
    m = torch.rand(shape, generator=torch.Generator().manual_seed(2)) < 0.5
    for t in (m.to(DEV), torch.stack((m, m), -1).to(DEV)[..., 0]):      # (and one whose scores lie apart)
        assert np.array_equal(br.mask_words(t).cpu().numpy().view(np.uint32), bits_from_bool(m.numpy()))
