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


# ---- attention_packed: infinite and NaN values ---------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("gap", [10.0, 14.0, 60.0, 95.0, 400.0])
@pytest.mark.parametrize("d,dt", [(64, "f16"), (128, "f16"), (40, "f16"), (64, "bf16"), (128, "bf16")])
def test_attention_infinite_values_at_small_probabilities(d, dt, gap):
    """A visible infinity counts however small its probability is (e^-gap of the largest), wherever its key lies in its
    block, also when the maximum moves behind it; a key that a row does not see counts for nothing."""
    from sesa import ops
    cu, cut = cu_of([300, 140])
    g = gen(d)
    q = torch.zeros(440, 2, d, device="cuda", dtype=DT[dt])
    k = torch.zeros_like(q)
    q[..., 0] = 1.0
    level = torch.rand(440, generator=g, device="cuda")
    level[[5, 70, 299, 303]] -= gap            # in whole and in masked blocks, at the ends of the sequences
    level[200] += gap / 2                       # the maximum moves far behind the first infinities
    k[..., 0] = level[:, None].to(DT[dt])
    v = torch.randn(440, 2, d, generator=g, device="cuda").to(DT[dt])
    clean = {c: ops.attention_packed(q, k, v, cut, causal=c, scale=1.0) for c in (True, False)}
    v[5, :, 3], v[70, :, 4], v[299, :, 5], v[303, :, 6] = math.inf, -math.inf, math.inf, -math.inf
    for causal in (True, False):
        got = ops.attention_packed(q, k, v, cut, causal=causal, scale=1.0)
        want = clean[causal].double()
        for key, end, col, val in ((5, 300, 3, math.inf), (70, 300, 4, -math.inf), (299, 300, 5, math.inf), (303, 440, 6, -math.inf)):
            want[key if causal else 300 * (key >= 300):end, :, col] = val
        # finite columns: two results of the same rows, each a rounding of P and of itself off
        x = torch.where(torch.isfinite(v), v, 0).double().abs().amax()
        close(got, want, 4 * HALF[v.dtype] * x)


@pytest.mark.gpu
@pytest.mark.parametrize("d,dt", [(64, "f16"), (128, "bf16"), (96, "f16")])
def test_attention_rows_beside_non_finite_ones_keep_their_bits(d, dt):
    """Of the rows of one tile, those that see no NaN and whose masked keys hold none are what they are without it."""
    from sesa import ops
    cu, cut = cu_of([400])
    g = gen(d)
    q, k, v = (torch.randn(400, 2, d, generator=g, device="cuda").to(DT[dt]) for _ in range(3))
    clean = ops.attention_packed(q, k, v, cut)
    v[200, 0, 1] = math.nan
    got = ops.attention_packed(q, k, v, cut)
    assert torch.equal(got[:, 1], clean[:, 1]) and torch.equal(got[:128], clean[:128])   # another head, earlier blocks
    assert bool(torch.isnan(got[200:, 0, 1]).all()) and int(torch.isnan(got).sum()) == 200
    off = (got[:, 0].double() - clean[:, 0].double()).abs()
    off[:, 1] = torch.where(torch.arange(400, device="cuda") < 200, off[:, 1], 0)
    assert float(off.max()) <= 4 * HALF[v.dtype] * float(torch.nan_to_num(v).abs().max())
    q[300, 0] = math.nan                                                  # a NaN query: its row and no other
    got2 = ops.attention_packed(q, k, v, cut)
    assert bool(torch.isnan(got2[300, 0]).all())
    keep = torch.arange(400, device="cuda") != 300
    assert torch.equal(torch.nan_to_num(got2[keep]), torch.nan_to_num(got[keep]))


# ---- attention_packed: many small probabilities --------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("d,dt,n", [(64, "f16", 100_000), (128, "f16", 60_001), (64, "bf16", 100_000), (48, "f16", 100_000)])
def test_attention_one_large_score_over_many_small_ones(d, dt, n):
    """One key takes most of a row and a long sequence of small probabilities the rest: about 2^-23.4 each, which fp16 (and
    an fp32 sum that adds them one by one) would round by a third."""
    from sesa import ops
    q = torch.zeros(n, 1, d, device="cuda", dtype=DT[dt])
    k = torch.zeros_like(q)
    q[..., 0], k[3, 0, 0] = 1.0, 16.234375
    gap = float(k[3, 0, 0])
    v = torch.ones_like(q)
    v[3] = -1.0
    m = (n - 1) * math.exp(-gap)
    ref = (m - 1) / (m + 1)
    got = ops.attention_packed(q, k, v, causal=False, scale=1.0).double()
    u = HALF[DT[dt]]
    # small weights rounded to the type, exp2, n / 64 block sums and n / 16 products added in fp32, the result's rounding
    tol = m * (u + 2.0 ** -20) + (n / 64 + n / 16) * 2.0 ** -24 + u * 1.01
    assert float((got - ref).abs().max()) <= tol, (float((got - ref).abs().max()), tol, ref)


# ---- quantize_i8 -----------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dt,rows,dim", [(torch.float32, 40_000, 512), (torch.float32, 3000, 1537), (torch.float16, 20_000, 1024),
                                         (torch.bfloat16, 500, 9000)])
@pytest.mark.parametrize("size", [1.0, 1e-35, 1e-30, 1e30, 5e37])
def test_quantize_i8_is_the_rounded_quotient(dt, rows, dim, size):
    """q = round(x / q_scale) to even for every element, the quotient rounded once to fp32 (here: in 64 bits, which holds it
    well enough that rounding it again is the same)."""
    from sesa import ops
    if dt == torch.float16:
        size = min(max(size, 1e-3), 1e3)
    x = (torch.randn(rows, dim, generator=gen(dim), device="cuda") * size).to(dt)
    x[:, 0] = x.abs().amax(-1)                              # (a positive largest value ...)
    step = (x[:, 0].double() / 127).float().double()         # ... and values at and beside half steps
    for i in range(1, 100):
        x[:, i] = ((i - 50 + 0.5) * step * (1 + (i % 3 - 1) * 2.0 ** -24)).to(dt)
    q, s = ops.quantize_i8(x)
    assert torch.equal(s, step.float())
    assert torch.equal(q.double(), torch.round((x.double() / s.double()[:, None]).float().double()))


# ---- linear_i8 -------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("xe,we", [(-120, -20), (-20, -120), (-100, 60), (90, -90), (95, 20), (20, 110)])
@pytest.mark.parametrize("m", [3, 40, 300])
def test_linear_i8_scales_at_both_ends(m, xe, we):
    """Scales whose own product would be subnormal, or past the largest fp32 number under a sum of 0: the result is what
    the formula gives."""
    from sesa import ops
    g = gen(m)
    x, w = (torch.randint(-127, 128, (r, 200), generator=g, device="cuda", dtype=torch.int8) for r in (m, 70))
    w[5] = 0                                                 # sums of 0
    if xe + we > 100:                                        # ... and small ones, in range times scales as large as these
        x[:, 1:], w[:, 1:] = 0, 0
        x[:, 0], w[:, 0] = x[:, 0].clamp(-1, 1), w[:, 0].clamp(-1, 1)
    xs, ws = (2.0 ** e * (1 + torch.rand(r, generator=g, device="cuda")) for r, e in ((m, xe), (70, we)))
    for bias in (None, torch.randn(70, generator=g, device="cuda")):
        want = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
        tol = 4 * 2.0 ** -24 * want.abs()
        if bias is not None:
            want = want + bias.double()
        tol = tol + 2.0 ** -24 * want.abs() + 2.0 ** -149
        got = ops.linear_i8(x, xs, w, ws, bias, out_dtype=torch.float32)
        big = want.abs() > 3.4e38
        assert bool(torch.isinf(got)[big].all()) and not bool(torch.isnan(got).any())
        assert bool(((got.double() - want).abs() <= tol)[~big].all())


@pytest.mark.gpu
def test_linear_i8_longest_rows_of_workgroups():
    """As many channels, and as many tokens, as the entry takes: more threads than one grid dimension holds."""
    from sesa import ops
    n = 2 ** 27 - 1
    w = torch.randint(-127, 128, (n, 1), generator=gen(1), device="cuda", dtype=torch.int8)
    ones = torch.ones(n, device="cuda")
    x = torch.tensor([[3], [-2]], dtype=torch.int8, device="cuda")
    got = ops.linear_i8(x, ones[:2], w, ones)
    assert torch.equal(got[0], (w[:, 0] * 3.0).half()) and torch.equal(got[1], (w[:, 0] * -2.0).half())
    del got
    m = 2 ** 27 + 1000                                       # tokens: tiles of 128 with one channel each
    x = torch.cat([w, w[:1001]])
    got = ops.linear_i8(x, torch.ones(m, device="cuda"), torch.full((1, 1), 5, dtype=torch.int8, device="cuda"), ones[:1])
    assert torch.equal(got[:, 0], (x[:, 0] * 5.0).half())


# ---- rope_axes -------------------------------------------------------------------------------------------------
TURNS_2_200 = 255752132986241185678408580023709873616295664310550962376831   # floor(2^200 / (2 pi)), from pi to 110 digits


def far_angles(pos, freqs):
    """position * freq modulo one turn in whole numbers, as angles in 64 bits."""
    rows = []
    for p in pos:
        row = []
        for f in freqs:
            num, den = float(f).as_integer_ratio()            # (an fp32 number: den a power of two)
            row.append((p * num * TURNS_2_200 // den) % 2 ** 200 / 2 ** 200 * 2 * math.pi)
        rows.append(row)
    return torch.tensor(rows, dtype=torch.double)


def test_turns_literal():
    """pi from Machin's formula in whole numbers."""
    one = 10 ** 110

    def arctan_inverse(x):
        t, s, k = one // x, one // x, 3
        while t:
            t //= -x * x
            s += t // k
            k += 2
        return s
    pi = 4 * (4 * arctan_inverse(5) - arctan_inverse(239))
    assert abs(2 ** 200 * one // (2 * pi) - TURNS_2_200) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("freq", [1e-4, 1.0, 10.0, 100.0, 1000.0, 1e6, 1e11])
def test_rope_axes_far_positions_at_any_frequency(freq):
    from sesa import ops
    g = gen(5)
    pos = [0, 1, -1, 4095, 10 ** 6, 2 ** 31 - 1, -2 ** 31, 2 ** 37 + 1, -2 ** 40, 2 ** 45 + 7]
    freqs = freq * (1 + torch.rand(8, generator=g, device="cuda"))
    x = torch.randn(len(pos), 2, 16, generator=g, device="cuda")
    ang = far_angles(pos, freqs.cpu()).to("cuda")[:, None]
    c, s, u, v = torch.cos(ang), torch.sin(ang), x[..., :8].double(), x[..., 8:].double()
    p = torch.tensor(pos, device="cuda")[:, None]
    ref, mag = torch.cat([u * c - v * s, u * s + v * c], -1), torch.cat([u.abs() + v.abs()] * 2, -1)
    # angle 2^-25 half-turns off and the position's share, sine and cosine two steps, two products and a sum
    tol = (16 * 2.0 ** -24 + 2 * math.pi * 2.0 ** -63 * p.double().abs()[:, None]) * mag + 2.0 ** -24 * ref.abs()
    close(ops.rope_axes(x, None, p, freqs, [8]), ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_rope_axes_non_finite_frequencies(layout):
    """A NaN or infinite frequency makes its own pair NaN, at every position, and nothing else."""
    from sesa import ops
    x = torch.randn(3, 2, 24, generator=gen(6), device="cuda")
    pos = torch.tensor([[0], [1], [-7]], device="cuda")
    freqs = torch.rand(10, generator=gen(7), device="cuda")
    want = ops.rope_axes(x, None, pos, freqs, [10], layout=layout)
    bad = [1, 4, 9]
    freqs[bad] = torch.tensor([math.nan, math.inf, -math.inf], device="cuda")
    at = [e for i in bad for e in ((i, 10 + i) if layout == "halves" else (2 * i, 2 * i + 1))]
    got = ops.rope_axes(x, None, pos, freqs, [10], layout=layout)
    assert bool(torch.isnan(got[..., at]).all())
    rest = [e for e in range(24) if e not in at]
    assert torch.equal(got[..., rest], want[..., rest])


# ---- traced, transformed and intercepted calls ----------------------------------------------------------------
def test_the_direct_path_is_for_plain_calls_only():
    """What sends a call through the registered op instead of straight to its kernel."""
    from torch.autograd import forward_ad
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode
    from sesa.token_ops import _plain
    x = torch.zeros(2, 4)
    assert _plain(x, None, torch.nn.Parameter(x))
    assert not _plain(x, x.as_subclass(type("Mine", (torch.Tensor,), {})))

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    class Function(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    for mode in (Dispatch(), Function(), forward_ad.dual_level()):
        with mode:
            assert not _plain(x)
    seen = []

    def look(t):
        seen.append(_plain(t))
        return t * 2
    torch.jit.trace(look, (x,), check_trace=False)   # (the check is a plain call)
    torch.func.vmap(look)(x)
    torch.func.grad(lambda t: look(t).sum())(x)
    torch.func.jvp(look, (x,), (x,))
    assert len(seen) >= 4 and not any(seen)
    assert _plain(x)


def test_fx_records_the_ops():
    from sesa import ops

    def f(x, xs, w, ws, q, k, pos, freqs, cu):
        a, b = ops.rope_axes(q, k, pos, freqs, [8])
        ops.rope_axes_(a, b, pos, freqs, [8])
        y, n = ops.norm_residual(x)
        y, q8, s = ops.norm_residual_i8(n, y)
        return ops.linear_i8(x, xs, w, ws), ops.attention_packed(a, b, b, cu), ops.quantize_i8(y)
    graph = torch.fx.symbolic_trace(f).graph
    names = [str(n.target) for n in graph.nodes if n.op == "call_function"]
    for op in ("linear_i8", "norm_residual", "norm_residual_i8", "quantize_i8", "rope_axes", "rope_axes_", "attention_packed"):
        assert any(n.split(".")[-1] == op or n.endswith(f"sesa.{op}") for n in names), (op, names)


@pytest.fixture
def some():
    """Small inputs of every operator, by seed."""
    def make(seed):
        g = gen(seed)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        return dict(x=r(6, 32).half(), res=r(6, 32), w=r(24, 32), qkv=r(6, 4, 16).half(),
                    pos=torch.randint(0, 99, (6, 1), generator=g, device="cuda"), freqs=r(8))
    return make


def all_ops(x, res, w, qkv, pos, freqs):
    from sesa import ops
    y, n = ops.norm_residual(x, res)
    y8, q8, s = ops.norm_residual_i8(x, res, pre="layer")
    out = ops.linear_i8(q8, s, *ops.quantize_i8(w), act="gelu")
    a, b = ops.rope_axes(qkv[:, :2], qkv[:, 2:3], pos, freqs, [8])
    return y, n, y8, q8, s, out, a, b, ops.attention_packed(a, b, qkv[:, 3:])


@pytest.mark.gpu
def test_jit_trace(some):
    """A traced function computes: new inputs give what the eager call gives."""
    names = list(some(0))
    traced = torch.jit.trace(lambda *a: all_ops(*a), tuple(some(1)[n] for n in names), check_trace=False)
    assert "sesa::linear_i8" in str(traced.graph) and "sesa::attention_packed" in str(traced.graph)
    for seed in (2, 3):
        args = [some(seed)[n] for n in names]
        junk = [torch.full((1 << 18,), math.nan, device="cuda") for _ in range(8)]   # (what an unwritten result would hold)
        del junk
        for a, b in zip(traced(*args), all_ops(*args)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_vmap_and_function_modes(some):
    from torch.overrides import TorchFunctionMode
    from sesa import ops
    sets = [some(s) for s in (4, 5, 6)]
    x, res, w = (torch.stack([s[n] for s in sets]) for n in ("x", "res", "w"))
    want = [ops.norm_residual_i8(s["x"], s["res"]) for s in sets]
    for a, b in zip(torch.func.vmap(lambda x, r: ops.norm_residual_i8(x, r))(x, res), zip(*want)):
        assert torch.equal(a, torch.stack(b))
    w8, ws = ops.quantize_i8(w)
    y = torch.func.vmap(lambda x, w, ws: ops.linear_i8(*ops.quantize_i8(x), w, ws))(x, w8, ws)
    assert all(torch.equal(y[i], ops.linear_i8(*ops.quantize_i8(x[i]), w8[i], ws[i])) for i in range(3))
    seen = []

    class Watch(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))
    with Watch():
        got = all_ops(**sets[0])
    assert all(torch.equal(a, b) for a, b in zip(got, all_ops(**sets[0])))
    for op in ("linear_i8", "norm_residual", "norm_residual_i8", "quantize_i8", "rope_axes", "attention_packed"):
        assert any(s.endswith(f"sesa.{op}") for s in seen), (op, seen)


# ---- gradients: refused, however the call is made --------------------------------------------------------------
def op_calls(dev):
    """(name, call of the op with one of its tensors in place of x) for every operator; the rest on ``dev``."""
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device=dev)  # noqa: E731
    i8 = torch.int8
    O = torch.ops.sesa  # noqa: N806
    rest = (None, "none", "none", None, None, None, "rms", None, None, 1e-6)
    pos = z(2, 1, dt=torch.int32)
    return [
        ("linear_i8", z(2, dt=torch.float32), lambda x: O.linear_i8(z(2, 16, dt=i8), x, z(4, 16, dt=i8), z(4, dt=torch.float32), None,
                                                                   "none", torch.float32)),
        ("norm_residual", z(2, 8), lambda x: O.norm_residual(x, None, *rest)[0]),
        ("norm_residual", z(2, 8), lambda x: O.norm_residual(z(2, 8), x, *rest)[0]),
        ("norm_residual_i8", z(2, 8), lambda x: O.norm_residual_i8(x, None, *rest)[0]),
        ("quantize_i8", z(2, 8), lambda x: O.quantize_i8(x)[1]),
        ("rope_axes", z(2, 1, 8), lambda x: O.rope_axes([z(2, 1, 8), x], pos, z(4, dt=torch.float32), [4], "halves")[0]),
        ("rope_axes", z(4, dt=torch.float32), lambda x: O.rope_axes([z(2, 1, 8)], pos, x, [4], "halves")[0]),
        ("rope_axes_", z(4, dt=torch.float32), lambda x: O.rope_axes_([z(2, 1, 8)], pos, x, [4], "halves")),
        ("attention_packed", z(2, 1, 8), lambda x: O.attention_packed(x, x, x, None, True, None, None)),
        ("attention_packed", z(2, 1), lambda x: O.attention_packed(z(2, 1, 8), z(2, 1, 8), z(2, 1, 8), None, True, None, x)),
        ("attention_packed_into", z(2, 1, 8), lambda x: O.attention_packed_into(x, x, x, None, True, None, None, z(2, 1, 8))),
    ]


def refuse_gradients(dev):
    from torch.autograd import forward_ad
    from sesa import ops  # noqa: F401
    from sesa._native import SesaError
    for name, t, call in op_calls(dev):
        with pytest.raises(SesaError, match=f"{name}: .* requires a gradient"):
            call(t.clone().requires_grad_())
        for grad_of in (lambda x: torch.func.grad(lambda y: call(y).float().sum())(x), lambda x: torch.func.jvp(call, (x,), (x,))):
            with pytest.raises(SesaError, match=f"{name}: .* requires a gradient"):
                grad_of(t)
        with forward_ad.dual_level(), pytest.raises(SesaError, match=f"{name}: .* requires a gradient"):
            call(forward_ad.make_dual(t, torch.ones_like(t)))


def test_gradients_are_refused_by_every_op():
    refuse_gradients("cpu")


def test_gradients_are_refused_while_compiling():
    from sesa import ops  # noqa: F401
    for backend in ("eager", "aot_eager"):
        for name, t, call in op_calls("cpu"):
            torch._dynamo.reset()
            out = []

            def f(x):
                y = call(x * 2)
                return x if y is None else y * 1.0
            with pytest.raises(Exception, match=f"{name}: .* requires a gradient"):
                out.append(torch.compile(f, backend=backend, fullgraph=True)(t.clone().requires_grad_()))
            assert not out


@pytest.mark.gpu
def test_gradients_are_refused_on_the_device(some):
    from torch.autograd import forward_ad
    from sesa import ops
    from sesa._native import SesaError
    refuse_gradients("cuda")
    x = torch.randn(4, 32, device="cuda")
    with forward_ad.dual_level(), pytest.raises(SesaError, match="requires a gradient"):
        ops.norm_residual(forward_ad.make_dual(x, x))
    w = torch.nn.Parameter(torch.ones(32, device="cuda"))
    f = torch.compile(lambda x: ops.norm_residual(x, pre_weight=w)[1] * 2, backend="aot_eager", fullgraph=True)
    with pytest.raises(Exception, match="requires a gradient"):
        f(x)
    with torch.no_grad():                       # ... and with gradients off the same call runs
        torch._dynamo.reset()
        assert torch.equal(f(x), ops.norm_residual(x, pre_weight=w)[1] * 2)
    with torch.inference_mode():
        assert torch.equal(ops.norm_residual(x.clone(), pre_weight=w)[1], f(x) / 2)


@pytest.mark.gpu
def test_tensors_written_in_place_count_a_version(some):
    """An op that saved the tensor for its backward notices that it changed, also under no_grad and through the op."""
    from sesa import ops
    s = some(8)
    for call in (ops.rope_axes_, lambda q, k, *a: torch.ops.sesa.rope_axes_([q, k], *a, "halves")):
        leaf = torch.ones(6, 2, 16, device="cuda", requires_grad=True)
        q, k = torch.randn(6, 2, 16, device="cuda"), torch.randn(6, 1, 16, device="cuda")
        y = (leaf * q).sum()
        with torch.no_grad():
            call(q, k, s["pos"], s["freqs"], [8])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        assert k._version == 1
    q, k, v = s["qkv"].split([2, 1, 1], 1)
    for call in (lambda o: ops.attention_packed(q, k, v, out=o),
                 lambda o: torch.ops.sesa.attention_packed_into(q, k, v, None, True, None, None, o)):
        out = torch.zeros(6, 2, 16, device="cuda", dtype=torch.float16)
        call(out)
        assert out._version == 1 and torch.equal(out, ops.attention_packed(q, k, v))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [512, 520, 640, 648, 656, 1000])
@pytest.mark.parametrize("m,n", [(8200, 2064), (40_000, 520)])
def test_linear_i8_either_side_of_the_short_k_rule(m, n, k):
    from sesa import ops
    from test_token_ops import linear_case, linear_check
    x, xs, w, ws, b = linear_case(m + k, m, k, n)
    linear_check(ops.linear_i8(x, xs, w, ws, b, act="gelu", out_dtype=torch.float32), x, xs, w, ws, b, "gelu")


# ---- the build -----------------------------------------------------------------------------------------------------
def test_makefile_builds_every_declared_symbol():
    """The one Makefile names every source, and the library it links has every entry that the bindings declare."""
    import glob
    import os
    import subprocess
    import sesa
    from sesa import _native
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(sesa.__file__))), "csrc")
    dry = subprocess.run(["make", "-f", "Makefile", "-n", "-B"], cwd=csrc, capture_output=True, text=True, check=True).stdout
    sources = [os.path.basename(f) for f in glob.glob(os.path.join(csrc, "*.hip")) + glob.glob(os.path.join(csrc, "*.cpp"))]
    assert len(sources) >= 16
    for src in sources:
        assert f"-c {src} " in dry, src
        assert f"build/{src}.o" in dry.split("-shared")[1], src
    lib = _native.lib()
    assert all(hasattr(lib, name) for name in _native.SIGNATURES)


# ---- rows without elements ---------------------------------------------------------------------------------------
def test_rows_without_elements():
    from sesa.token_ops import _rows
    for shape, rows in (((2, 3, 0), 6), ((0, 5, 4), 0), ((4,), 1), ((3, 1, 7), 3), ((0,), 1)):
        assert _rows(torch.zeros(*shape)).shape == (rows, shape[-1])


@pytest.mark.gpu
def test_rows_without_elements_are_refused():
    from sesa import ops
    from sesa._native import SesaError
    i8 = lambda *s: torch.zeros(*s, dtype=torch.int8, device="cuda")  # noqa: E731
    for bad in (lambda: ops.linear_i8(i8(2, 3, 0), torch.ones(2, 3, device="cuda"), i8(4, 0), torch.ones(4, device="cuda")),
                lambda: ops.norm_residual(torch.zeros(2, 3, 0, device="cuda")), lambda: ops.quantize_i8(torch.zeros(2, 3, 0, device="cuda"))):
        with pytest.raises(SesaError):
            bad()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 300])
def test_linear_i8_gelu_in_fp32(m):
    """fp32 results carry GELU to fp32, down its negative tail (the argument exact: one product by powers of two)."""
    from sesa import ops
    x = torch.arange(-128, 128, device="cuda").to(torch.int8)[:, None]
    ws = torch.tensor([2.0 ** -4, 2.0 ** -5, 2.0 ** -9, 2.0 ** 3], device="cuda")
    w = torch.ones(4, 1, dtype=torch.int8, device="cuda")
    for at in range(0, 256, m):
        rows = x[at:at + m]
        got = ops.linear_i8(rows, torch.ones(len(rows), device="cuda"), w, ws, act="gelu", out_dtype=torch.float32).double()
        v = rows.double() * ws.double()
        ref = 0.5 * v * torch.erfc(-v / math.sqrt(2.0))
        # erfc to 4 half-steps and two products; its argument half a step off counts |v|^2 times where erfc falls
        tol = (8 + v * v) * 2.0 ** -23 * ref.abs() + 2.0 ** -140
        assert bool(((got - ref).abs() <= tol).all()), float(((got - ref).abs() / tol).max())
    big = torch.tensor([[-128], [127]], dtype=torch.int8, device="cuda")
    y = ops.linear_i8(big, torch.full((2,), 3e38, device="cuda"), w[:1], torch.ones(1, device="cuda"), act="gelu", out_dtype=torch.float32)
    assert float(y[0]) == 0 and float(y[1]) == math.inf


@pytest.mark.gpu
def test_jit_trace_of_calls_in_place(some):
    """In-place rotation and attention into a given tensor, traced: the traced function does the same to new inputs."""
    from sesa import ops

    def f(qkv, pos, freqs):
        rows = qkv * 1
        q, k, v = rows.split([2, 1, 1], 1)
        ops.rope_axes_(q, k, pos, freqs, [8])
        out = torch.zeros_like(q)
        ops.attention_packed(q, k, v, out=out)
        return rows, out
    names = ("qkv", "pos", "freqs")
    traced = torch.jit.trace(f, tuple(some(1)[n] for n in names), check_trace=False)
    for seed in (2, 3):
        args = [some(seed)[n] for n in names]
        for a, b in zip(traced(*args), f(*args)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_calls_from_several_threads(some):
    """Two threads, each with its own stream and inputs, at once."""
    import threading
    sets = [some(s) for s in (11, 12)]
    want = [[t.clone() for t in all_ops(**s)] for s in sets]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                got = all_ops(**sets[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_calls_in_place(some, backend):
    """In-place rotation and attention into a given tensor in a compiled function, inputs of two sizes."""
    from sesa import ops

    def f(qkv, pos, freqs):
        rows = qkv * 1
        q, k, v = rows[:, :2], rows[:, 2:3], rows[:, 3:]
        ops.rope_axes_(q, k, pos, freqs, [8])
        out = torch.zeros(rows.shape[0], 2, 16, device="cuda", dtype=torch.float16)
        ops.attention_packed(q, k, v, out=out)
        return rows, out
    torch._dynamo.reset()
    compiled = torch.compile(f, backend=backend, fullgraph=True)
    for seed, n in ((2, 6), (3, 6), (4, 5)):
        s = some(seed)
        args = (s["qkv"][:n], s["pos"][:n], s["freqs"])
        for a, b in zip(compiled(*args), f(*args)):
            assert torch.equal(a, b)


# ---- attention_packed: the second pass -------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,dt", [(64, "f16"), (64, "bf16"), (128, "f16"), (128, "bf16"), (40, "f16"), (96, "bf16")])
@pytest.mark.parametrize("odd", [False, True])
def test_attention_second_pass_leaves_finite_columns_alone(d, dt, causal, odd):
    """A tile that goes through its keys twice: the columns without non-finite values, and the rows that did not ask for it,
    bit for bit what they are without; infinities of both signs and NaN meet in a column as in the formula."""
    from sesa import ops
    cu, cut = cu_of([700, 333])
    g = gen(d)
    pad = (lambda x: torch.nn.functional.pad(x, (1, 2))[..., 1:d + 1]) if odd else (lambda x: x)
    q, k, v = (torch.randn(1033, n, d, generator=g, device="cuda").to(DT[dt]) for n in (4, 2, 2))
    bad = {2: (7, math.inf), 5: (7, -math.inf), 11: (40, math.nan), 17: (699, math.inf), 19: (1032, math.nan), 23: (700, -math.inf)}
    zero = v.clone()
    for col, (key, val) in bad.items():
        zero[key, 0, col], v[key, 0, col] = 0, val
    zero[20:300, 0, 30], v[20:300, 0, 30] = 0, math.inf          # many at once, one sign ...
    zero[50, 0, 31], v[50, 0, 31] = 0, math.inf                  # ... and both in one column
    zero[90, 0, 31], v[90, 0, 31] = 0, -math.inf
    want = ops.attention_packed(*map(pad, (q, k, zero)), cut, causal=causal)
    got = ops.attention_packed(*map(pad, (q, k, v)), cut, causal=causal)
    assert torch.equal(got[:, 2:], want[:, 2:])                  # the other key head's
    keep = [c for c in range(d) if c not in bad and c not in (30, 31)]
    assert torch.equal(got[..., keep], want[..., keep])
    row = torch.arange(1033, device="cuda")
    for col, (key, val) in list(bad.items()) + [(30, (20, math.inf)), (31, (50, math.inf))]:
        first = key < 700
        sees = (row >= key if causal else row >= 0) & ((row < 700) == first)
        seen, rest = got[:, :2, col][sees].float(), got[:, :2, col][~sees]
        if col == 31:
            both = got[:, :2, col][(row >= 90 if causal else row >= 0) & (row < 700)]
            assert bool(torch.isnan(both).all())
            if causal:
                assert bool((got[50:90, :2, col] == math.inf).all())
        else:
            assert bool((torch.isnan(seen) if math.isnan(val) else seen == val).all())
        assert torch.equal(rest, want[:, :2, col][~sees])


@pytest.mark.gpu
@pytest.mark.parametrize("d,dt", [(64, "f16"), (128, "bf16"), (48, "bf16")])
def test_attention_far_rows_leave_the_others_alone(d, dt):
    """One query of a tile with scores far out: its own row is done over, the tile's others keep their bits."""
    from sesa import ops
    q, k, v = (torch.randn(300, 1, d, generator=gen(d), device="cuda").to(DT[dt]) for _ in range(3))
    want = ops.attention_packed(q, k, v)
    q2 = q.clone()
    q2[[131, 200]] = (q2[[131, 200]].float() * 6e3).to(DT[dt])
    k2 = k.clone()
    k2[:, :, 0] = (k2[:, :, 0].float() * 6e3).to(DT[dt])
    q[:, :, 0], q2[:, :, 0] = 0, torch.where(torch.isin(torch.arange(300, device="cuda"), torch.tensor([131, 200], device="cuda"))[:, None], 6e3, 0.0)
    want, got = ops.attention_packed(q, k2, v), ops.attention_packed(q2, k2, v)
    near = [i for i in range(300) if i not in (131, 200)]
    assert torch.equal(got[near], want[near])
    for i in (131, 200):
        s = (q2[i, 0].double() * k2[:i + 1, 0].double()).sum(-1)
        top, at = s.topk(2)
        # the two scores' sums of d products in fp32, d + 8 half-steps each, and e^-100 between them
        assert float(top[0] - top[1]) > 2 * (d + 8) * 2.0 ** -24 * float(s.abs().max()) + 100 * d ** 0.5
        assert torch.equal(got[i, 0], v[at[0], 0])


@pytest.mark.gpu
@pytest.mark.parametrize("d,dt", [(64, "f16"), (128, "bf16")])
def test_attention_keys_with_a_score_of_minus_infinity(d, dt):
    """A key whose score is -inf contributes nothing, whatever its value; a row of such keys alone is NaN."""
    from sesa import ops
    cu, cut = cu_of([150])
    q, k, v = (torch.randn(150, 1, d, generator=gen(d), device="cuda").to(DT[dt]) for _ in range(3))
    q[..., 0] = q[..., 0].abs() + 0.1
    k[[0, 40, 100], :, 0] = -math.inf
    rest = [i for i in range(150) if i not in (0, 40, 100)]
    want = ops.attention_packed(q[rest], k[rest], v[rest])
    for val in (1.0, math.inf, math.nan):
        v[[0, 40, 100]] = val
        got = ops.attention_packed(q, k, v, cut)
        assert bool(torch.isnan(got[0]).all())
        close(got[rest], want.double(), 4 * HALF[v.dtype] * v[rest].double().abs().amax())
