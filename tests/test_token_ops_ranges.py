"""The transformer operators over the whole range of their inputs: scores of any size, non-finite values, far positions,
scales at both ends, the longest launches, and every way a call can be traced, differentiated or intercepted.

Values are compared with the formulas in 64 bits; tolerances count roundings as in test_token_ops.py.
"""
import math

import pytest
import torch

from test_token_ops import HALF, TINY, close, cu_of, gen

DT = {"f16": torch.float16, "bf16": torch.bfloat16}


# ---- attention_packed: scores of any size ------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dt,val", [("f16", 1e4), ("f16", 6e4), ("bf16", 1e4), ("bf16", 1e15)])
@pytest.mark.parametrize("d", [40, 64, 128])
def test_attention_equal_scores_of_any_size(d, dt, val):
    """Every key of a row scores the same, far beyond what exp takes: the row is the mean of the values it sees (one key:
    that value, bit for bit)."""
    from sesa import ops
    lens = [1, 1, 5, 70, 200]
    cu, cut = cu_of(lens)
    k = torch.full((cu[-1], 2, d), val, device="cuda", dtype=DT[dt])
    v = torch.randn(cu[-1], 2, d, generator=gen(d), device="cuda").to(DT[dt])
    for q in (k, -k):
        for causal in (True, False):
            got = ops.attention_packed(q, k, v, cut, causal=causal)
            assert torch.equal(got[:2], v[:2])
            for a, b in zip(cu[:-1], cu[1:]):
                n = torch.arange(1, b - a + 1, device="cuda").double()[:, None, None]
                x = v[a:b].double()
                ref, mag = ((y.cumsum(0) / n if causal else y.mean(0, keepdim=True).expand_as(y)) for y in (x, x.abs()))
                # every probability is the same number: sums of up to 200 terms, a quotient, the result's rounding
                close(got[a:b], ref, 210 * 2.0 ** -24 * mag + HALF[v.dtype] * ref.abs() * (1 + 1e-6) + TINY[v.dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("base", [2.0 ** 21, -2.0 ** 21, 2.0 ** 23, -2.0 ** 23])
@pytest.mark.parametrize("d,dt", [(64, "f16"), (128, "bf16"), (40, "f16")])
def test_attention_scores_around_a_far_value(d, dt, base):
    """Scores that differ by a few around a large common value, all of them exact in fp32: what counts is the difference,
    also between key blocks on either side of a move of the running maximum."""
    from sesa import ops
    step = 0.25 if abs(base) < 2 ** 22 else 1.0
    lens = [200] * 8
    cu, cut = cu_of(lens)
    level = torch.full((8, 200), -40.0)
    level[:, :64] = 0
    for i in range(8):
        level[i, 70 + i] = 6 + step * (i % 3)        # one key outweighs the first block, and moves the maximum
        level[i, 130:150] = 3                        # ... and a later block counts against it
    q = torch.zeros(1600, 2, d, device="cuda", dtype=DT[dt])
    k = torch.zeros_like(q)
    q[..., 0], q[..., 9] = 1024.0, 1.0
    k[..., 0], k[..., 9] = base / 1024, level.flatten()[:, None].to("cuda", DT[dt])
    v = torch.randn(1600, 2, d, generator=gen(d), device="cuda").to(DT[dt])
    p = torch.softmax(level.double(), -1).to("cuda")
    x = v.double().view(8, 200, 2, d)
    ref, mag = ((p[:, :, None, None] * y).sum(1, keepdim=True).expand_as(y).reshape(v.shape) for y in (x, x.abs()))
    got = ops.attention_packed(q, k, v, cut, causal=False, scale=1.0)
    u = HALF[v.dtype]
    # each probability rounded once to the type; exp2 of a difference of at most 70 (2^-24 of it) and the sums: 2^-17
    tol = (u + 2.0 ** -17) * mag + (2.0 ** -25 * 200 * float(v.abs().max()) if dt == "f16" else 0)
    close(got, ref, tol + u * (ref.abs() + tol) + TINY[v.dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("d,dt,val", [(64, "f16", 3e3), (64, "bf16", 1e9), (128, "bf16", 1e15), (96, "f16", 2e4)])
def test_attention_random_far_scores(d, dt, val):
    """Random scores so far apart that one key takes a row: that key's value, and never anything but finite."""
    from sesa import ops
    cu, cut = cu_of([300, 77])
    g = gen(d)
    q, k = ((torch.randn(377, 2, d, generator=g, device="cuda") * val).clamp(-6.5e4, 6.5e4) if dt == "f16" else
            torch.randn(377, 2, d, generator=g, device="cuda") * val for _ in range(2))
    q, k = q.to(DT[dt]), k.to(DT[dt])
    v = torch.randn(377, 2, d, generator=g, device="cuda").to(DT[dt])
    got = ops.attention_packed(q, k, v, cut)
    assert bool(torch.isfinite(got).all()) and float(got.abs().max()) <= float(v.abs().max())
    clear = 0
    for a, b in zip(cu[:-1], cu[1:]):
        for h in range(2):
            Q, K = q[a:b, h].double(), k[a:b, h].double()
            hide = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").triu(1)
            s = (Q @ K.t().contiguous() * d ** -0.5).masked_fill(hide, -math.inf)
            err = (d + 8) * 2.0 ** -24 * (Q.abs() @ K.abs().t().contiguous() * d ** -0.5).amax(-1)
            top, at = s.topk(2, -1)
            sure = top[:, 0] - top[:, 1] > 2 * err + 20      # (the rest of the row: below e^-20 a key)
            sure[0] = True                                   # one key only
            clear += int(sure.sum())
            want = v[a:b, h][at[:, 0]]
            assert bool(((got[a:b, h] - want).double().abs() <= 2 * HALF[v.dtype] * (want.double().abs() + 0.01))[sure].all())
    assert clear > 377
