"""Plain restatements, on the CPU, of the 8-bit rows' operators for the tests: the quantising rule in
f32 (which the device follows bit for bit), the scores and the adjustments in f64."""
import numpy as np
import torch

BLOCK = 128


def quantize(x, tile=False):
    """Codes [n, 128 kb] (float8) and scales of x (CPU, any float type), by the rule's own f32 steps."""
    n, d = x.shape
    kb, nb = -(-d // BLOCK), -(-n // BLOCK)
    codes = torch.zeros((n, kb * BLOCK), dtype=torch.float8_e4m3fn)
    scales = torch.zeros((kb, nb if tile else n), dtype=torch.float32)
    step = BLOCK if tile else 1
    for b in range(kb):
        for r in range(0, n, step):
            part = x[r:r + step, b * BLOCK:(b + 1) * BLOCK].float().numpy()
            top = np.float32(max(np.abs(part).max(), np.float32(2.0 ** -100))) if np.isfinite(part).all() else np.float32(np.nan)
            i = r // step
            if np.isnan(top):
                scales[b, i] = float("nan")
                continue
            scales[b, i] = float(top / np.float32(448))
            y = torch.from_numpy(part * (np.float32(448) / top))
            codes[r:r + step, b * BLOCK:b * BLOCK + part.shape[1]] = y.to(torch.float8_e4m3fn)
    return codes, scales


def values(codes, scales, tile=False):
    """The rows in f64 (exact: a code times its scale fits)."""
    n = codes.shape[0]
    s = scales.double().t()
    s = s.repeat_interleave(BLOCK, 0)[:n] if tile else s
    return (codes.float().double().view(n, -1, BLOCK) * s[:, :, None]).reshape(n, -1)


def scores_bound(q, x, dtype):
    """f64 scores and how far the kernels' sums and one rounding may leave them.  In a block 128 exact
    products are summed, each step off by at most 2^-23 of the partial sums' bound (a truncating
    adder included); the scales' product, the fused multiply-add of each block and the join of at
    most 16 parts add a half step of 2^-23 each; the result is rounded once.  Scores of 16 bits
    come from the 8-bit matrix instruction, which first cuts each product of a group of 8 at 2^-13 of
    the group's largest: 8 cuts lose at most 8 * 2^-13 = 2^-10 of that product, so at most 2^-10 of the sum
    of magnitudes over all groups."""
    xt = x.t().contiguous()
    y = q @ xt
    mag = q.abs() @ xt.abs()
    kb = q.shape[1] // BLOCK
    cut = 0.0 if dtype == torch.float32 else 2.0 ** -10
    tol = (cut + BLOCK * 2.0 ** -23 + (kb + 18) * 2.0 ** -24) * mag
    half = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    sub = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}[dtype]
    return y, tol * (1 + half) + half * y.abs() + sub


def adjust(scores, seen=None, seen_len=None, rep=1.0, pre=0.0, fre=0.0, bias_ids=None, bias=None, mask=None):
    """f64 adjusted scores, and the bound of the f32 steps: up to six half steps of 2^-23 on the
    magnitudes that enter, and one rounding to the type."""
    B, n = scores.shape
    y = scores.double().clone()
    mag = torch.zeros_like(y)
    for i in range(B):
        r, p, f = (float(v[i]) if isinstance(v, torch.Tensor) else float(np.float32(v)) for v in (rep, pre, fre))
        if seen is not None:
            ids = (seen[i] if seen.dim() == 2 else seen).tolist()
            if seen_len is not None:
                ids = ids[:min(max(int(seen_len[i]), 0), len(ids))]
            count = {}
            for v in ids:
                if 0 <= v < n:
                    count[v] = count.get(v, 0) + 1
            for v, c in count.items():
                s = y[i, v].item()
                s = s / r if s > 0 else s * r
                y[i, v] = s - (f * c + p)
                mag[i, v] = abs(s) + abs(f * c) + abs(p)
        if bias_ids is not None:
            ids = (bias_ids[i] if bias_ids.dim() == 2 else bias_ids).tolist()
            bs = (bias[i] if bias.dim() == 2 else bias).tolist()
            last = {v: b for v, b in zip(ids, bs) if 0 <= v < n}
            for v, b in last.items():
                mag[i, v] = mag[i, v] + y[i, v].abs() + abs(b)
                y[i, v] += b
        if mask is not None:
            m = mask[i] if mask.dim() == 2 else mask
            y[i, ~m] = -float("inf")
            mag[i, ~m] = 0
    half = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[scores.dtype]
    tol = 6 * 2.0 ** -24 * mag
    touched = mag > 0
    return y, torch.where(touched, tol * (1 + half) + half * y.abs() + 2.0 ** -25, torch.zeros_like(y))
