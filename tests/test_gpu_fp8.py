"""8-bit rows on the device: codes and scales bit for bit as the f32 rule gives them, scores within a
derived bound of the f64 product (tests/_fp8_ref.py), the layouts, streams and captures that the calls
allow, and the index's own dense scores."""
import threading

import numpy as np
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


def make(n, d, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, d), generator=g) * torch.exp(torch.randn((n, 1), generator=g))
    return x.to(dtype)


def quantized(br, n, d, tile=False, seed=0):
    return br.quantize_rows(make(n, d, seed=seed).to(DEV), tile=tile)


def check_scores(q, x, got, dev="cpu"):
    y, tol = R.scores_bound(*(R.values(r.codes.to(dev), r.scales.to(dev), r.tile) for r in (q, x)), got.dtype)
    got, most = got.double().to(dev), torch.finfo(got.dtype).max
    off = (got - y).abs()
    # a sum that the bound lets reach the type's largest value (f16: 65504) rounds to the infinity of its sign
    past = torch.isinf(got) & (y.abs() + tol >= most) & (torch.sign(got) == torch.sign(y))
    assert bool(((off <= tol) | past).all()), float((off / tol)[~past].max())


# ---- quantising -----------------------------------------------------------------------------
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, d", [(1, 1), (1, 128), (3, 127), (33, 129), (128, 384), (129, 50), (200, 1000), (257, 4097)])
def test_quantize(br, n, d, dtype, tile):
    x = make(n, d, dtype, seed=n + d)
    codes, scales = R.quantize(x, tile)
    got = br.quantize_rows(x.to(DEV), tile=tile)
    assert torch.equal(got.codes.cpu().float(), codes.float())
    assert torch.equal(got.scales.cpu(), scales)
    # the values are within half a step: 2^-4 of the value, or half of 2^-9 of the scale below 2^-6,
    # with the f32 roundings of the scale, the inverse and the product
    off = (got.dequantize().cpu().double() - x.double()).abs()
    s = scales.double().t().repeat_interleave(128, 1)[:, :d]
    s = s.repeat_interleave(128, 0)[:n] if tile else s
    assert bool((off <= (x.double().abs() * 2.0 ** -4 + s * 2.0 ** -10) * (1 + 2.0 ** -20)).all())


@pytest.mark.parametrize("tile", [False, True])
def test_quantize_special_values(br, tile):
    x = make(300, 400, seed=5)
    x[0] = 0.0                      # a block of zeros
    x[1] *= 1e-38                   # denormal after scaling, below the floor
    x[2] = 3e38
    x[130, 5] = float("inf")
    x[131, 200] = float("nan")
    x[290, 399] = -float("inf")
    codes, scales = R.quantize(x, tile)
    got = br.quantize_rows(x.to(DEV), tile=tile)
    assert torch.equal(got.codes.cpu().float(), codes.float())
    assert torch.equal(torch.nan_to_num(got.scales.cpu(), nan=-1.0), torch.nan_to_num(scales, nan=-1.0))
    assert torch.isnan(scales).any()
    # a score that reads such a block is NaN, every other one is not; but for row 2, whose blocks' sums
    # are 3e38 times the sum of 128 query values: past f32's 3.4e38 as soon as those sum to 1.14, with either
    # sign, so that infinities of both signs may meet in any order of the blocks
    q = br.quantize_rows(make(4, 400).to(DEV))
    nan = torch.isnan(br.scores_fp8(q, got)).cpu()
    bad = torch.isnan(scales).any(0)
    bad = bad.repeat_interleave(128)[:300] if tile else bad
    nan[:, 2] = False
    assert torch.equal(nan, bad[None, :].expand(4, 300))


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_strided_and_misaligned(br, dtype):
    big = make(40, 700, dtype, seed=9).to(DEV)
    for x in (big[:, 3:390], big[::2, 1:], big.t()[5:300], big[:1].expand(7, 700), big[7:8, 5:6]):
        codes, scales = R.quantize(x.cpu())
        got = br.quantize_rows(x)
        assert torch.equal(got.codes.cpu().float(), codes.float()) and torch.equal(got.scales.cpu(), scales)


def test_quantize_into_parts(br):
    x = make(500, 300, seed=3).to(DEV)
    for tile in (False, True):
        whole = br.quantize_rows(x, tile=tile)
        out = br.Fp8Rows.empty(500, 300, tile, DEV)
        for a, b in ((0, 128), (128, 384), (384, 500)):
            br.quantize_rows(x[a:b], tile=tile, out=out.part(a, b))
        assert torch.equal(out.codes.view(torch.uint8), whole.codes.view(torch.uint8))
        assert torch.equal(out.scales, whole.scales)


# ---- the product ----------------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 64, 128), (1, 25216, 384), (2, 65, 129), (15, 257, 640), (16, 1000, 2048), (17, 127, 4096),
         (33, 513, 384), (64, 300, 256), (65, 4100, 128), (100, 129, 1000), (128, 128, 4224), (129, 255, 96), (250, 777, 777),
         (256, 256, 512), (257, 1025, 384), (512, 2050, 1280), (700, 515, 2100)]


@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", SIZES)
def test_scores(br, m, n, k, dtype, tile):
    q, x = quantized(br, m, k, seed=1), quantized(br, n, k, tile, seed=2)
    out = torch.full((m, n), float("nan"), dtype=dtype, device=DEV)
    check_scores(q, x, br.scores_fp8(q, x, out=out))


# enough tiles that a workgroup takes several, one after the other: rows of one block and more, edges inside the tiles,
# score rows that begin at lines (ld) and anywhere
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k, ld", [(2040, 8190, 100, 8190), (2040, 8190, 300, 8192), (4090, 8100, 384, 8128), (4096, 8001, 130, 8001),
                                         (1800, 20000, 200, 20000), (70, 60000, 128, 60000)])
def test_scores_of_many_rows(br, m, n, k, ld, dtype, tile):
    q, x = quantized(br, m, k, seed=1), quantized(br, n, k, tile, seed=2)
    buf = torch.full((m, ld), float("nan"), dtype=dtype, device=DEV)
    check_scores(q, x, br.scores_fp8(q, x, out=buf[:, :n]), DEV)
    assert bool(torch.isnan(buf[:, n:]).all())


@pytest.mark.parametrize("m, n, k", [(1, 70, 128), (20, 130, 300), (300, 270, 256)])
@pytest.mark.parametrize("dtype", TYPES)
def test_scores_into_strided_rows(br, m, n, k, dtype):
    q, x = quantized(br, m, k, seed=1), quantized(br, n, k, seed=2)
    want = br.scores_fp8(q, x, dtype=dtype)
    buf = torch.full((m + 2, n + 9), 7.0, dtype=dtype, device=DEV)
    out = buf[1:m + 1, 3:n + 3]
    assert br.scores_fp8(q, x, out=out) is out
    assert torch.equal(out, want)
    buf[1:m + 1, 3:n + 3] = 7.0
    assert bool((buf == 7.0).all())


def test_scores_of_parts(br):
    q, x = quantized(br, 50, 500, seed=1), quantized(br, 700, 500, seed=2)
    whole = br.scores_fp8(q, x)
    assert torch.equal(br.scores_fp8(q, x.part(100, 300)), whole[:, 100:300])
    y = quantized(br, 700, 500, True, seed=2)
    assert torch.equal(br.scores_fp8(q, y.part(128, 700)), br.scores_fp8(q, y)[:, 128:])


def test_rows_further_apart_than_32_bits(br):
    # codes and scores whose offsets pass 2^32: three rows, 2^31 + 4096 bytes apart
    ld = (1 << 31) + 4096
    store = torch.empty(2 * ld + 1024, dtype=torch.uint8, device=DEV)
    far = torch.as_strided(store, (3, 256), (ld, 1)).view(torch.float8_e4m3fn)
    near = quantized(br, 3, 200, seed=4)
    out = br.Fp8Rows(far, torch.empty_like(near.scales), 200)
    br.quantize_rows(make(3, 200, seed=4).to(DEV), out=out)
    assert torch.equal(far.float(), near.codes.float())
    q = quantized(br, 5, 200, seed=5)
    assert torch.equal(br.scores_fp8(q, out), br.scores_fp8(q, near))
    assert torch.equal(br.scores_fp8(out, q), br.scores_fp8(near, q))
    # 20 rows 2^24 bytes apart: past what the tiles address, so read as a few rows are
    wide = torch.as_strided(store, (20, 256), (1 << 24, 1)).view(torch.float8_e4m3fn)
    rows = quantized(br, 20, 200, seed=6)
    wide.copy_(rows.codes)
    assert torch.equal(br.scores_fp8(br.Fp8Rows(wide, rows.scales, 200), rows, dtype=torch.bfloat16),
                       br.scores_fp8(rows.part(0, 20), rows, dtype=torch.bfloat16))
    del far, out, wide, store
    buf = torch.empty(2 * ld + 1024, dtype=torch.float16, device=DEV)
    y = torch.as_strided(buf, (3, 5), (ld, 1))
    br.scores_fp8(near, q, out=y)
    assert torch.equal(y, br.scores_fp8(near, q, dtype=torch.float16))


def test_scores_span_many_items(br):
    # more than 2^32 bytes of scores, checked at both ends against the parts
    q, x = quantized(br, 600, 128, seed=1), quantized(br, 2000, 128, seed=2)
    reps = 1000
    big = br.Fp8Rows(x.codes.view(torch.uint8).repeat(reps, 1).view(torch.float8_e4m3fn), x.scales.repeat(1, reps), 128)
    y = br.scores_fp8(q, big, dtype=torch.float32)
    want = br.scores_fp8(q, x)
    assert torch.equal(y[:, :2000], want) and torch.equal(y[:, -2000:], want) and torch.equal(y[:, 10 ** 6:10 ** 6 + 2000], want)


@pytest.mark.parametrize("m, n, k, dtype", [(8, 4096, 1024, torch.bfloat16), (300, 600, 512, torch.float32)])
def test_scores_replayed(br, m, n, k, dtype):
    q, x = quantized(br, m, k, seed=1), quantized(br, n, k, seed=2)
    raw = make(m, k, seed=1).to(DEV)
    out = torch.zeros((m, n), dtype=dtype, device=DEV)
    br.scores_fp8(q, x, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        br.scores_fp8(br.quantize_rows(raw, out=q), x, out=out)
    for s in range(4):
        raw.copy_(make(m, k, seed=10 + s))
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        want = br.scores_fp8(br.quantize_rows(raw), x, dtype=dtype)
        assert torch.equal(out, want), s
        want.sum().item()


def test_scores_on_streams_and_threads(br):
    x = quantized(br, 5000, 384, seed=2)
    qs = [quantized(br, 40, 384, seed=20 + i) for i in range(4)]
    want = [br.scores_fp8(q, x) for q in qs]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        s = torch.cuda.Stream(DEV)
        for _ in range(10):
            got[i] = br.scores_fp8(qs[i], x, stream=s)
        s.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_refusals(br):
    q, x = quantized(br, 3, 200), quantized(br, 5, 200, True)
    with pytest.raises(br.BrickrecError):
        br.scores_fp8(x, q)                              # tiles as queries
    with pytest.raises(br.BrickrecError):
        br.scores_fp8(q, quantized(br, 5, 201))
    with pytest.raises(TypeError):
        br.scores_fp8(q, x, dtype=torch.float64)
    with pytest.raises(ValueError):
        br.scores_fp8(q, x, out=torch.empty((3, 6), device=DEV))
    with pytest.raises(ValueError):
        br.scores_fp8(q, x, out=torch.empty((5, 3), device=DEV).t())
    with pytest.raises(TypeError):
        br.scores_fp8(q, x, out=torch.empty((3, 5), dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        br.Fp8Rows(q.codes, q.scales, 300)
    with pytest.raises(ValueError):
        br.Fp8Rows(q.codes, q.scales[:, :2], 200)
    with pytest.raises(TypeError):
        br.Fp8Rows(q.codes.view(torch.uint8), q.scales, 200)
    with pytest.raises(TypeError):
        br.quantize_rows(torch.zeros((3, 5), dtype=torch.float64, device=DEV))
    with pytest.raises(ValueError):
        br.quantize_rows(torch.zeros(5, device=DEV))
    with pytest.raises(ValueError):
        br.quantize_rows(torch.zeros((3, 200), device=DEV, requires_grad=True))
    with pytest.raises(ValueError):
        br.quantize_rows(torch.zeros((3, 200), device=DEV), out=x)
    with pytest.raises(ValueError):
        x.part(1, 3)
    assert br.scores_fp8(quantized(br, 0, 200), x).shape == (0, 5)
    assert br.quantize_rows(torch.zeros((4, 0), device=DEV)).codes.shape == (4, 0)


# ---- a run of them together -------------------------------------------------------------------
def test_weights_activations_scores_adjusted(br):
    """Quantised activations against quantised weights, the logits adjusted in place: against f64 from the
    unquantised inputs, by e4m3's half step 2^-4 on each factor (and 2^-10 of the block's scale)."""
    m, n, k = 12, 1500, 640
    a, w = make(m, k, torch.bfloat16, seed=1), make(n, k, torch.bfloat16, seed=2)
    qa, qw = br.quantize_rows(a.to(DEV)), br.quantize_rows(w.to(DEV), tile=True)
    logits = br.scores_fp8(qa, qw, dtype=torch.float32)
    g = torch.Generator().manual_seed(3)
    seen = torch.randint(-1, n, (m, 40), generator=g, dtype=torch.int32)
    allowed = torch.rand((m, n), generator=g) < 0.7
    y = br.adjust_scores(logits, seen=seen.to(DEV), repetition=1.3, presence=0.2, frequency=0.1, mask=allowed.to(DEV),
                         out=logits).cpu().double()
    va, vw = a.double(), w.double()
    ea, ew = (R.values(q.codes.cpu(), q.scales.cpu(), q.tile)[:, :k] - v for q, v in ((qa, va), (qw, vw)))
    plain, _ = R.adjust((va @ vw.t()).float(), seen, None, 1.3, 0.2, 0.1, mask=allowed)
    tol = 1.3 * (va.abs() @ ew.abs().t() + ea.abs() @ (vw.abs() + ew.abs()).t()) + 1e-3 * (va.abs() @ vw.abs().t())
    assert torch.equal(torch.isinf(y), ~allowed)
    assert bool(((y - plain).abs()[allowed] <= tol[allowed]).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_index_scores(br, dtype):
    n, d, B = 3001, 384, 9
    x, q = make(n, d, seed=1), make(B, d, seed=2)
    idx = br.ItemIndex(device=0, dtype=dtype, id_offset=100)
    with pytest.raises(br.BrickrecError):
        idx.quantize_items()
    idx.upload_items(x.numpy())
    with pytest.raises(br.BrickrecError):
        idx.scores(q.to(DEV))
    rows = idx.quantize_items(chunk=1000)
    stored = torch.from_numpy(np.asarray(idx.get_rows(np.arange(100, 100 + n))))
    codes, scales = R.quantize(stored)
    assert torch.equal(rows.codes.cpu().float(), codes.float()) and torch.equal(rows.scales.cpu(), scales)
    got = idx.scores(q.to(DEV))
    assert torch.equal(torch.from_numpy(idx.scores(q.numpy())), got.cpu())
    unit = torch.nn.functional.normalize(q.to(DEV), dim=1, eps=1e-30)
    assert torch.equal(got, br.scores_fp8(br.quantize_rows(unit), rows))
    # within e4m3's half steps of the exact cosine: 2^-4 of each factor, and their product
    cos = torch.nn.functional.normalize(q.double(), dim=1) @ torch.nn.functional.normalize(x.double(), dim=1).t()
    assert float((got.cpu().double() - cos).abs().max()) < 2 * 2.0 ** -4 + 2.0 ** -7
    idx.upload_attrs(np.arange(n), np.full(n, 2015), np.zeros(n, np.int32))
    bits = idx.eval_mask_bits(br.Predicate(parts_min=100, parts_max=2000))
    view = idx.view()
    s = torch.cuda.Stream(DEV)
    seen = torch.tensor([[5, 7, 7, -1]] * B, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    y = view.scores(q.to(DEV), stream=s, mask=bits, seen=seen, frequency=0.5, presence=0.25)
    s.synchronize()
    want = got.clone()
    want[:, 5] -= 0.75
    want[:, 7] -= 1.25
    want[:, :100] = -float("inf")
    want[:, 2001:] = -float("inf")
    assert torch.equal(y, want)
    view.close()
    idx.upload_items(x.numpy())
    with pytest.raises(br.BrickrecError):
        idx.scores(q.to(DEV))
    idx.close()


def test_semantic_scores(br):
    from brickrec.semantic import SemanticIndex
    x = make(500, 64, seed=1)
    sem = SemanticIndex([f"s{i}" for i in range(500)], x.numpy())
    one = sem.scores(x[7].numpy())
    assert one.shape == (1, 500) and int(one[0].argmax()) == 7
    assert np.array_equal(sem.scores([x[7].tolist(), x[8].tolist()])[:1], one)


def test_index_scores_refusals_and_streams(br):
    n, d, B = 70000, 256, 64
    x, q = make(n, d, seed=1), make(B, d, seed=2)
    idx = br.ItemIndex()
    idx.upload_items(x.numpy())
    assert idx.quantized is None
    with pytest.raises(ValueError):
        idx.quantize_items(chunk=0)
    with pytest.raises(ValueError):
        idx.quantize_items(chunk=-5)
    rows = idx.quantize_items()
    assert idx.quantized is rows
    with pytest.raises(TypeError):
        idx.scores(q)                                    # a host tensor
    with pytest.raises(TypeError):
        idx.scores(q.numpy(), dtype=torch.bfloat16)      # numpy has no such type
    with pytest.raises(ValueError):
        idx.scores(q[:, :100].to(DEV))
    with pytest.raises(ValueError):
        idx.scores(q.numpy()[0])
    want = idx.scores(q.to(DEV)).cpu()
    assert idx.scores(q[:0].numpy()).shape == (0, n)
    # numpy rows through another stream that is busy: the copy to the host waits for that one
    s = torch.cuda.Stream(DEV)
    a = torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(20):
            a = torch.tanh(a @ a)
    assert torch.equal(torch.from_numpy(idx.scores(q.numpy(), stream=s)), want)
    # captured and replayed with other queries
    raw, out = q.to(DEV), torch.zeros((B, n), device=DEV)
    idx.scores(raw, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        idx.scores(raw, out=out)
    for i in range(3):
        raw.copy_(make(B, d, seed=30 + i))
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, idx.scores(raw)), i
        out.sum().item()
    del g
    idx.close()
    with pytest.raises(br.BrickrecError):
        idx.scores(raw)


def test_rows_keep_their_tensors(br):
    import copy
    import io
    q = quantized(br, 5, 200)
    for name in ("codes", "scales", "d", "tile"):
        with pytest.raises(AttributeError):
            setattr(q, name, None)
    want = br.scores_fp8(q, q)                           # one set of rows on both sides
    assert torch.equal(br.scores_fp8(copy.deepcopy(q), q), want)
    f = io.BytesIO()
    torch.save(q, f)
    f.seek(0)
    with torch.serialization.safe_globals([br.Fp8Rows]):
        assert torch.equal(br.scores_fp8(q, torch.load(f, weights_only=True)), want)
    with pytest.raises(ValueError):
        br.Fp8Rows(q.codes, q.scales.clone().requires_grad_(), 200)
    with torch.no_grad():
        br.Fp8Rows(q.codes, q.scales.clone().requires_grad_(), 200)


@pytest.mark.parametrize("m, n", [(3, 40), (100, 300), (2100, 8200)])
def test_two_graphs_at_once(br, m, n):
    """Two captured calls replayed side by side, each with its own tensors: neither sees the other."""
    sets = [[quantized(br, m, 384, seed=2 * i), quantized(br, n, 384, seed=2 * i + 1)] for i in range(2)]
    want = [br.scores_fp8(q, x, dtype=torch.bfloat16) for q, x in sets]
    outs = [torch.zeros((m, n), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    graphs = []
    torch.cuda.synchronize()
    for (q, x), o in zip(sets, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            br.scores_fp8(q, x, out=o)
            br.adjust_scores(o, out=o, seen=torch.zeros(1, dtype=torch.int32, device=DEV), presence=1.0)
        graphs.append(g)
    want = [br.adjust_scores(w, seen=torch.zeros(1, dtype=torch.int32, device=DEV), presence=1.0) for w in want]
    for _ in range(3):
        [o.zero_() for o in outs]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
        outs[0].float().sum().item()


# sizes on both sides of the rules that choose how the product is cut up
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k, ld", [(4090, 8100, 100, 8100), (4090, 8100, 100, 8192), (2040, 8190, 1600, 8190), (2040, 8190, 1500, 8192),
                                         (333, 10007, 1000, 10007), (256, 20001, 260, 20032), (130, 14900, 2100, 14900),
                                         (64, 20001, 2048, 20001), (100, 16300, 2200, 16300), (1000, 7100, 770, 7100)])
def test_scores_cut_up(br, m, n, k, ld, dtype, tile):
    q, x = quantized(br, m, k, seed=3), quantized(br, n, k, tile, seed=4)
    buf = torch.full((m, ld), float("nan"), dtype=dtype, device=DEV)
    check_scores(q, x, br.scores_fp8(q, x, out=buf[:, :n]), DEV)
    assert bool(torch.isnan(buf[:, n:]).all())


@pytest.mark.parametrize("far_side", ["items", "queries"])
def test_offsets_within_a_tile_past_31_bits(br, far_side):
    # 256 rows just under 2^24 bytes apart, in one tile of 256: offsets up to nearly 2^32
    ld = (1 << 24) - 16
    store = torch.empty(255 * ld + 128, dtype=torch.uint8, device=DEV)
    far = torch.as_strided(store, (256, 128), (ld, 1)).view(torch.float8_e4m3fn)
    near, many = quantized(br, 256, 128, seed=4), quantized(br, 131072, 128, seed=5)
    far.copy_(near.codes)
    rows = br.Fp8Rows(far, near.scales, 128)
    a, b = ((many, rows), (many, near)) if far_side == "items" else ((rows, many), (near, many))
    assert torch.equal(br.scores_fp8(*a, dtype=torch.bfloat16), br.scores_fp8(*b, dtype=torch.bfloat16))


# one size for each way the product is cut up, in bf16 and in the wider types
WAYS = [(1, 300, 384), (16, 40, 2304), (20, 6000, 128), (64, 4100, 1024), (60, 20100, 2048), (250, 8100, 384), (1000, 7100, 384),
        (2040, 8190, 300)]


def small_codes(n, k, seed):
    """Codes of 0, +-1 and +-2."""
    return torch.randint(-2, 3, (n, -(-k // 128) * 128), generator=torch.Generator().manual_seed(seed)).float()


def rows_of_codes(br, codes, exponents=0.0):
    n, k = codes.shape
    scales = torch.full((k // 128, n), 2.0) ** exponents
    return br.Fp8Rows(codes.to(torch.float8_e4m3fn).to(DEV), scales.float().to(DEV), k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("m, n, k", WAYS)
def test_small_products_beside_large_ones_that_cancel(br, m, n, k, dtype):
    """In every 8 columns two products of 448 x 448 cancel and six of at most 4 are left.  Every product is a whole number
    and every partial sum of a block is below 2^24, so f32 sums are exact; the result is at most 4 * 6 * 16 a block, over at
    most 18 blocks.  f32 holds it; f16 rounds it once."""
    q, x = small_codes(m, k, 1), small_codes(n, k, 2)
    q[:, ::8], q[:, 1::8], x[:, ::8], x[:, 1::8] = 448.0, 448.0, 448.0, -448.0
    want = (q.double().to(DEV) @ x.double().to(DEV).t().contiguous()).to(dtype)
    assert torch.equal(br.scores_fp8(rows_of_codes(br, q), rows_of_codes(br, x), dtype=dtype), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m, n, k", WAYS)
def test_exact_sums_are_rounded_once(br, m, n, k, dtype):
    """Products of 0, 1, 2 and 4 lie within 2^-2 of each other, so that no type's way cuts any of them: blocks are whole
    numbers of at most 512, scaled by 2^-3 to 2^3, so that every sum has at most 20 bits and the one rounding is left."""
    q, x = small_codes(m, k, 3), small_codes(n, k, 4)
    g = torch.Generator().manual_seed(5)
    eq = torch.randint(-1, 2, (q.shape[1] // 128, m), generator=g)
    ex = torch.randint(-2, 3, (x.shape[1] // 128, n), generator=g)
    a, b = rows_of_codes(br, q, eq), rows_of_codes(br, x, ex)
    want = R.values(a.codes, a.scales).to(DEV) @ R.values(b.codes, b.scales).to(DEV).t().contiguous()
    assert torch.equal(br.scores_fp8(a, b, dtype=dtype), want.to(dtype))


def test_index_scores_of_any_magnitude(br):
    """Queries are normalised whatever their magnitude: a power of two in front changes nothing, in f32 up to where
    squares leave its range on either side, in f64 beyond f32's range altogether."""
    n, d, B = 700, 384, 5
    idx = br.ItemIndex()
    idx.upload_items(make(n, d, seed=1).numpy())
    idx.quantize_items()
    q = make(B, d, seed=2)
    want = idx.scores(q.to(DEV))
    for e in (66, 120, -66, -83, -110):
        assert torch.equal(idx.scores((q * 2.0 ** e).to(DEV)), want), e
    wide = idx.scores(q.double().to(DEV))
    cos = torch.nn.functional.normalize(q.double(), dim=1) @ torch.from_numpy(idx.get_rows(np.arange(n))).double().t()
    for got in (want, wide):  # (the bound of test_index_scores)
        assert float((got.cpu().double() - cos).abs().max()) < 2 * 2.0 ** -4 + 2.0 ** -7
    for e in (600, -600, 1010, -1000):
        assert torch.equal(idx.scores((q.double() * 2.0 ** e).to(DEV)), wide), e
        assert np.array_equal(idx.scores((q.double() * 2.0 ** e).numpy()), wide.cpu().numpy()), e
    # the smallest power of two and the largest, zeros, infinities and NaN
    q = torch.zeros((6, d))
    q[0], q[1, 3], q[2] = 2.0 ** -149, 2.0 ** -149, 2.0 ** 127
    q[4, 7], q[5, 9] = INF, float("nan")
    got = idx.scores(q.to(DEV))
    one = torch.zeros((2, d))
    one[0], one[1, 3] = 1.0, 1.0
    assert torch.equal(got[[0, 2]], idx.scores(one[[0, 0]].to(DEV)))
    assert torch.equal(got[1], idx.scores(one[1:].to(DEV))[0])
    assert bool((got[3] == 0).all()) and bool(torch.isnan(got[4:]).all())
    idx.close()


def test_tangents_are_refused(br):
    from torch.autograd import forward_ad
    q = quantized(br, 3, 200)
    x, one = torch.randn((3, 200), device=DEV), torch.ones(3, device=DEV)
    ids, bias = torch.zeros((3, 2), dtype=torch.int32, device=DEV), torch.ones((3, 2), device=DEV)
    want = br.adjust_scores(x, seen=ids, repetition=one, presence=one, frequency=one, bias_ids=ids, bias=bias)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: br.quantize_rows(dual(x)), lambda: br.Fp8Rows(q.codes, dual(q.scales), 200),
                     lambda: br.scores_fp8(q, q, out=dual(torch.empty((3, 3), device=DEV))),
                     lambda: br.adjust_scores(dual(x)), lambda: br.adjust_scores(x, out=dual(torch.empty_like(x))),
                     lambda: br.adjust_scores(x, seen=ids, repetition=dual(one)),
                     lambda: br.adjust_scores(x, seen=ids, presence=dual(one)),
                     lambda: br.adjust_scores(x, seen=ids, frequency=dual(one)),
                     lambda: br.adjust_scores(x, bias_ids=ids, bias=dual(bias))):
            with pytest.raises(ValueError):
                call()
            with torch.no_grad(), pytest.raises(ValueError):     # (no_grad stops gradients, not tangents)
                call()
        got = br.adjust_scores(x, seen=ids, repetition=one, presence=one, frequency=one, bias_ids=ids, bias=bias)
        assert torch.equal(got, want)                            # plain tensors within a level
    with pytest.raises(ValueError):
        torch.func.jvp(br.adjust_scores, (x,), (x,))


def test_scales_that_come_to_ask_for_a_gradient(br):
    q = quantized(br, 3, 200)
    q.scales.requires_grad_()
    with pytest.raises(ValueError):
        br.scores_fp8(q, quantized(br, 4, 200))
    with pytest.raises(ValueError):
        br.scores_fp8(quantized(br, 4, 200), q)
    with pytest.raises(ValueError):
        br.quantize_rows(make(3, 200).to(DEV), out=q)
    with torch.no_grad():
        assert br.scores_fp8(q, q).shape == (3, 3)


def test_writes_into_out_are_seen_by_autograd(br):
    """A tensor that a backward pass has saved and that a call overwrites is torch's own error, not a wrong gradient."""
    q = quantized(br, 4, 64)

    def saved(shape):
        y = torch.sigmoid(torch.randn(shape, device=DEV, requires_grad=True))   # (its backward reads y)
        return y, y.detach()
    y, out = saved((4, 4))
    br.scores_fp8(q, q, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y, out = saved((4, 4))
    br.adjust_scores(torch.zeros((4, 4), device=DEV), out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y, out = saved((4, 4))
    br.adjust_scores(out, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y, out = saved((1, 4))
    rows = br.Fp8Rows(q.codes, out, 64)
    br.quantize_rows(make(2, 64).to(DEV), out=rows.part(1, 3))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    before = q.codes._version
    br.quantize_rows(make(4, 64).to(DEV), out=q)
    assert q.codes._version > before
    with torch.inference_mode():                     # (such tensors have no version to advance)
        o = torch.empty((4, 4), device=DEV)
        want = br.scores_fp8(q, q)
        assert torch.equal(br.scores_fp8(q, q, out=o), want)
        assert torch.equal(br.adjust_scores(o, out=o), want)
        assert br.quantize_rows(make(4, 64).to(DEV), out=br.Fp8Rows.empty(4, 64, device=DEV)).codes.shape == (4, 128)


def test_index_scores_with_numpy_lists(br):
    n, d, B = 1000, 64, 3
    idx = br.ItemIndex()
    idx.upload_items(make(n, d, seed=1).numpy())
    idx.quantize_items()
    q = make(B, d, seed=2).numpy()
    kw = {"seen": np.array([[5, 7, 7, -1]] * B, np.int32), "seen_len": np.array([4, 3, 0], np.int32), "repetition": np.full(B, 1.5, np.float32),
          "presence": 0.25, "frequency": 0.5, "bias_ids": np.array([3, 9], np.int32), "bias": np.array([1.0, -2.0], np.float32)}
    allowed = np.random.default_rng(1).random((B, n)) < 0.5
    dev = {k: torch.from_numpy(v).to(DEV) if isinstance(v, np.ndarray) else v for k, v in kw.items()}
    want = idx.scores(torch.from_numpy(q).to(DEV), mask=torch.from_numpy(allowed).to(DEV), **dev).cpu().numpy()
    for mask in (allowed, br.bits_from_bool(allowed)):
        assert np.array_equal(idx.scores(q, mask=mask, **kw), want)
    assert np.array_equal(idx.scores(q, mask=torch.from_numpy(allowed).to(DEV), **{**kw, "seen": dev["seen"]}), want)
    with pytest.raises(TypeError):
        idx.scores(q, bias_ids=kw["bias_ids"], bias=kw["bias"].astype(np.float64))
    with pytest.raises(TypeError):
        idx.scores(torch.from_numpy(q).to(DEV), seen=kw["seen"])    # torch rows take torch lists
    idx.close()


def test_what_are_no_rows_is_a_type_error(br):
    q = quantized(br, 3, 200)
    for call in (lambda: br.scores_fp8(q.codes, q), lambda: br.scores_fp8(q, None), lambda: br.scores_fp8(q, q, out=[0.0]),
                 lambda: br.quantize_rows(make(3, 200).to(DEV), out=q.codes), lambda: br.quantize_rows([[1.0]]),
                 lambda: br.Fp8Rows([1], q.scales, 200), lambda: br.Fp8Rows(q.codes, None, 200)):
        with pytest.raises(TypeError):
            call()


def test_no_quantizing_into_part_of_a_tile(br):
    """A tile has one scale: writing some of its rows would change the values of the others."""
    x = make(300, 200, seed=1).to(DEV)
    rows = br.quantize_rows(x, tile=True)
    want = rows.dequantize()
    for part in (rows.part(0, 100), rows.part(128, 299), rows.part(0, 256).part(128, 130), rows.part(0, 140).part(128, 140)):
        with pytest.raises(ValueError):
            br.quantize_rows(100 * x[:len(part)], tile=True, out=part)
    assert torch.equal(rows.dequantize(), want)
    assert torch.equal(rows.part(0, 100).dequantize(), want[:100])      # reading is another matter
    for a, b in ((0, 128), (128, 256), (256, 300), (128, 300), (0, 300)):
        br.quantize_rows(x[a:b], tile=True, out=rows.part(a, b))
    assert torch.equal(rows.dequantize(), want)
    plain = br.quantize_rows(x)
    br.quantize_rows(x[5:9], out=plain.part(5, 9))                      # a row has its own scales
