"""The host side of the dense scores, without a GPU."""
import pytest
import torch

from brickrec import engine


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
