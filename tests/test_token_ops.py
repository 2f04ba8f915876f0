"""The transformer operators (sesa.ops.linear_i8, norm_residual, rope_axes, attention_packed; csrc/sesa_linear_i8.hip,
sesa_norm.hip, sesa_rope.hip, sesa_attn_packed.hip).

CPU: the C entries refuse bad arguments before any device work, schemas and fake shapes, no CPU fallback.
GPU: every operator against its formula in 64 bits.  Tolerances count roundings: a result is rounded once to its type
(half a step, eps / 2 of the value), and what lies before is fp32, some number of 2^-24 of the largest value that
enters the sum; each check names its count.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}   # half the smallest fp16 subnormal
E = 2.0 ** -24


def close(got, ref, tol):
    got = got.double()
    assert got.shape == ref.shape
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    both = torch.isfinite(ref)
    assert torch.equal(got[~both & ~torch.isnan(ref)], ref[~both & ~torch.isnan(ref)])
    off = (got - ref).abs()[both]
    lim = tol.expand_as(ref)[both]
    assert bool((off <= lim).all()), f"off by {float((off / lim.clamp_min(1e-300)).max()):.3g} of the tolerance"


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- CPU ------------------------------------------------------------------------------------------------
def _lib():
    from sesa import _native
    return _native, _native.lib()


def test_linear_i8_refuses():
    N, L = _lib()
    ok = [16, 16, 16, 16, 16, 16, None, 0, 4, 4, 16, 16, 1, 4, None]   # pointers are never read: every call is refused

    def rc(**bad):
        a = list(ok)
        for i, v in bad.items():
            a[int(i[1:])] = v
        return L.sesa_linear_i8(*a)
    for bad in ({"_8": -1}, {"_9": 0}, {"_10": 0}, {"_10": 131072}, {"_7": 4}, {"_7": -1}, {"_12": 3}, {"_0": None},
                {"_2": None}, {"_3": None}, {"_5": None}, {"_11": None}, {"_13": 3}, {"_8": 2 ** 31}):
        assert rc(**bad) == -1, bad
        assert b"linear_i8" in L.sesa_last_error()
    assert rc(_8=0) == 0   # no rows: nothing to do


def _norm_args(N, **kw):
    a = dict(rows=4, dim=8, x_dtype=1, r_dtype=0, x=16, x_ld=8, residual=16, r_ld=8, post=1, pre=1, eps=1e-6, y=16, y_ld=8,
             n=16, n_ld=8)
    a.update(kw)
    return N.SesaNormArgs(**a)


def test_norm_residual_refuses():
    N, L = _lib()
    assert L.sesa_norm_residual(None, None) == -1
    for bad in (dict(rows=-1), dict(rows=2 ** 31), dict(dim=0), dict(dim=32769), dict(x_dtype=3), dict(r_dtype=2), dict(post=3),
                dict(pre=-1), dict(gate_act=4), dict(eps=-1.0), dict(eps=math.inf), dict(eps=math.nan), dict(x=None),
                dict(q=16, q_ld=8, q_scale=16), dict(n=None, q=16, q_ld=8), dict(y=None, n=None),
                dict(gate=16, rows_per_gate=0), dict(y_ld=7), dict(n_ld=0), dict(n=None, q=16, q_ld=7, q_scale=16)):
        assert L.sesa_norm_residual(ctypes.byref(_norm_args(N, **bad)), None) == -1, bad
        assert b"norm_residual" in L.sesa_last_error()
    assert L.sesa_norm_residual(ctypes.byref(_norm_args(N, rows=0)), None) == 0


def _rope_args(N, **kw):
    a = dict(tokens=4, head_dim=16, dtype=1, layout=0, n_axes=2, sections=(ctypes.c_int * 4)(4, 4), positions=16,
             positions_ld=2, freqs=16, n_tensors=1)
    t = N.SesaRopeTensor(16, 32, 16, 16, 32, 16, 2)
    a.update(kw)
    t = a.pop("t0", t)
    r = N.SesaRopeArgs(**a)
    r.t[0] = t
    return r


def test_rope_axes_refuses():
    N, L = _lib()
    assert L.sesa_rope_axes(None, None) == -1
    s4 = lambda *v: (ctypes.c_int * 4)(*v)  # noqa: E731
    for bad in (dict(tokens=-1), dict(head_dim=1), dict(head_dim=4097), dict(dtype=3), dict(layout=2), dict(n_axes=0), dict(n_axes=5),
                dict(sections=s4(8, 1)), dict(sections=s4(0, 0)), dict(sections=s4(-1, 4)), dict(n_tensors=3), dict(n_tensors=0),
                dict(positions=None), dict(freqs=None), dict(t0=N.SesaRopeTensor(None, 1, 1, 16, 1, 1, 2)),
                dict(t0=N.SesaRopeTensor(16, 1, 1, 16, 1, 1, 0)), dict(n_tensors=2)):
        assert L.sesa_rope_axes(ctypes.byref(_rope_args(N, **bad)), None) == -1, bad
        assert b"rope_axes" in L.sesa_last_error()
    assert L.sesa_rope_axes(ctypes.byref(_rope_args(N, tokens=0)), None) == 0


def _attn_args(N, **kw):
    a = dict(tokens=8, lanes=1, heads=4, kv_heads=2, head_dim=64, dtype=1, q=16, k=16, v=16, cu_seqlens=16, n_seq=2, causal=1,
             scale=0.125, out=16)
    a.update(kw)
    return N.SesaAttnArgs(**a)


def test_attention_packed_refuses():
    N, L = _lib()
    assert L.sesa_attention_packed(None, None) == -1
    for bad in (dict(tokens=-1), dict(tokens=2 ** 31), dict(lanes=0), dict(heads=3), dict(kv_heads=0), dict(head_dim=12),
                dict(head_dim=136), dict(head_dim=0), dict(dtype=0), dict(n_seq=0), dict(cu_seqlens=None, n_seq=3),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(q=None), dict(k=None),
                dict(v=None), dict(out=None), dict(tokens=2 ** 30, heads=2 ** 20, kv_heads=1)):
        assert L.sesa_attention_packed(ctypes.byref(_attn_args(N, **bad)), None) == -1, bad
        assert b"attention_packed" in L.sesa_last_error()
    assert L.sesa_attention_packed(ctypes.byref(_attn_args(N, tokens=0)), None) == 0


def test_schemas_and_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from sesa import ops  # noqa: F401
    assert "Tensor(a!) out" in str(torch.ops.sesa.attention_packed_into.default._schema)
    assert "Tensor(a!)[] xs" in str(torch.ops.sesa.rope_axes_.default._schema)
    with FakeTensorMode():
        i8 = torch.int8
        o = torch.ops.sesa.linear_i8(torch.empty(3, 5, 64, dtype=i8), torch.empty(3, 5), torch.empty(7, 64, dtype=i8),
                                     torch.empty(7), None, "none", torch.bfloat16)
        assert o.shape == (3, 5, 7) and o.dtype == torch.bfloat16
        x = torch.empty(6, 32, dtype=torch.float16)
        rest = (None, "none", "none", None, None, None, "rms", None, None, 1e-6)
        y, n = torch.ops.sesa.norm_residual(x, torch.empty(6, 32), *rest)
        assert y.dtype == torch.float32 and n.dtype == torch.float16
        y, q, s = torch.ops.sesa.norm_residual_i8(x, None, *rest)
        assert y.dtype == torch.float16 and q.dtype == i8 and s.shape == (6,) and s.dtype == torch.float32
        q, s = torch.ops.sesa.quantize_i8(x)
        assert q.shape == x.shape and s.shape == (6,)
        h = torch.empty(6, 2, 16)
        a, b = torch.ops.sesa.rope_axes([h, h[:, :1]], torch.zeros(6, 2, dtype=torch.int32), torch.empty(8), [4, 4], "pairs")
        assert a.shape == (6, 2, 16) and b.shape == (6, 1, 16)
        assert torch.ops.sesa.attention_packed(x.view(6, 4, 8), x.view(6, 4, 8), x.view(6, 4, 8), None, True, None,
                                               None).shape == (6, 4, 8)


def test_no_cpu_fallback():
    from sesa import ops
    from sesa._native import SesaError
    x = torch.zeros(2, 16, dtype=torch.int8)
    for call in (lambda: ops.linear_i8(x, torch.ones(2), x, torch.ones(2)), lambda: ops.norm_residual(torch.ones(2, 4)),
                 lambda: ops.norm_residual_i8(torch.ones(2, 4)), lambda: ops.quantize_i8(torch.ones(2, 4)),
                 lambda: ops.rope_axes(torch.ones(2, 1, 4), None, torch.zeros(2, 1, dtype=torch.int32), torch.ones(2), [2]),
                 lambda: ops.rope_axes_(torch.ones(2, 1, 4), None, torch.zeros(2, 1, dtype=torch.int32), torch.ones(2), [2]),
                 lambda: ops.attention_packed(*[torch.ones(2, 1, 8, dtype=torch.float16)] * 3)):
        with pytest.raises(SesaError, match="no CPU fallback"):
            call()


def test_memory_overlap_rules():
    from sesa.token_ops import _apart, _writable
    buf = torch.zeros(7, 48)
    q, k = buf.as_strided((6, 2, 8), (48, 8, 1)), buf.as_strided((6, 2, 8), (48, 8, 1), 16)
    assert _apart(q, k) and _apart(k, q)
    assert not _apart(q, q) and not _apart(q, buf.as_strided((6, 2, 8), (48, 8, 1), 8))
    assert not _apart(q, buf.as_strided((6, 2, 8), (40, 8, 1), 16))
    assert _apart(buf[:2], buf[2:]) and _apart(q, torch.zeros(6, 2, 8))
    assert not _apart(q, buf.as_strided((6, 2, 8), (48, 8, 1), 40))   # wraps into the next row's q
    assert _writable(q) and _writable(buf.t().t()) and not _writable(buf.t())
    assert not _writable(buf.as_strided((6, 2, 8), (8, 8, 1))) and not _writable(torch.zeros(1, 8).expand(4, 8))


def test_memory_overlap_rules_against_sets():
    """Never apart where two views share an element; apart for the layouts that projections write."""
    from sesa.token_ops import _apart, _writable
    import random
    rng = random.Random(0)
    buf = torch.zeros(4000)
    found = 0
    for _ in range(3000):
        views = []
        for _ in range(2):
            shape = [rng.randint(1, 4) for _ in range(rng.randint(1, 4))]
            base = rng.choice([1, 2, 3])
            stride = sorted((base * rng.choice([1, 4, 8, 16, 24, 48, 96]) for _ in shape), reverse=rng.random() < 0.8)
            views.append(buf.as_strided(shape, stride, rng.randint(0, 60)))
        sets = [set((v.storage_offset() + sum(i * s for i, s in zip(ix, v.stride())) for ix in np.ndindex(*v.shape))) for v in views]
        if _apart(*views):
            found += 1
            assert not sets[0] & sets[1], (views[0].shape, views[0].stride(), views[1].shape, views[1].stride())
        for v, st in zip(views, sets):
            assert not _writable(v) or len(st) == v.numel()
    assert found > 100
    rows = torch.zeros(5, 3, 18, 8)
    q, k, v, o = rows.split([6, 3, 3, 6], 2)
    assert all(_apart(a, o) and _apart(o, a) for a in (q, k, v)) and not _apart(rows[:, :, 5:7], q)
    assert _apart(rows[..., :4], rows[..., 4:]) and not _apart(rows[..., :5], rows[..., 4:])


# ---- GPU: linear_i8 -------------------------------------------------------------------------------------
def linear_case(seed, m, k, n, bias=True, full=False):
    g = gen(seed)
    i8 = lambda *s: torch.randint(-128 if full else -127, 128, s, generator=g, device="cuda", dtype=torch.int8)  # noqa: E731
    x, w = i8(m, k), i8(n, k)
    xs = torch.rand(m, generator=g, device="cuda") * 0.02 / math.sqrt(k)
    ws = torch.rand(n, generator=g, device="cuda") * 0.02
    b = torch.randn(n, generator=g, device="cuda") if bias else None
    return x, xs, w, ws, b


def linear_check(got, x, xs, w, ws, b, act="none"):
    prod = (x.double() @ w.double().t()) * xs.double()[..., None] * ws.double()
    v = prod if b is None else prod + b.double()
    # the integer's own rounding, the scales' product, the fused multiply-add: three half-steps of the product, one of v
    tol = 4 * E * (prod.abs() + v.abs())
    if act == "gelu":
        v, tol = 0.5 * v * torch.erfc(-v / math.sqrt(2.0)), 1.13 * tol + 5e-7 * (1 + v.abs())   # |gelu'| <= 1.13
    elif act == "tanh":
        v = torch.tanh(v)
        tol = tol + 20 * E * v.abs()   # exp2 and rcp to one step each, amplified 5x by 1 - e at the series' border
    elif act == "relu":
        v = torch.where(torch.isnan(v), v, v.clamp_min(0))
    close(got, v, tol + HALF[got.dtype] * (v.abs() + tol) + TINY[got.dtype])


SHAPES = [(1, 1, 1), (1, 64, 16), (1, 4096, 300), (2, 15, 17), (3, 17, 5), (16, 640, 64), (17, 100, 33), (33, 129, 70),
          (64, 2048, 96), (65, 128, 64), (100, 130, 129), (128, 15, 300), (257, 512, 513), (300, 1000, 257), (300, 1008, 260),
          (2100, 136, 2100), (2100, 144, 2100), (4090, 250, 4100), (4100, 256, 4100)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_i8_shapes(m, k, n):
    from sesa import ops
    for i, dt in enumerate(DT.values()):
        x, xs, w, ws, b = linear_case(m + k + n + i, m, k, n, bias=i != 1)
        linear_check(ops.linear_i8(x, xs, w, ws, b, out_dtype=dt), x, xs, w, ws, b)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(17, 512, 12304), (33, 100, 8200), (64, 64, 6160), (64, 64, 6144), (16, 48, 30000), (70, 384, 256),
                                   (8200, 320, 2064), (8200, 500, 2064)])
def test_linear_i8_kernel_choice(m, k, n):
    """Either side of the rules that choose between the kernels and tiles."""
    from sesa import ops
    x, xs, w, ws, b = linear_case(m + k + n, m, k, n)
    linear_check(ops.linear_i8(x, xs, w, ws, b, out_dtype=torch.bfloat16), x, xs, w, ws, b)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu", "tanh", "relu"])
@pytest.mark.parametrize("m", [5, 200])
def test_linear_i8_activations(act, m):
    from sesa import ops
    for dt in DT.values():
        x, xs, w, ws, b = linear_case(m, m, 192, 130)
        linear_check(ops.linear_i8(x, xs, w, ws, b, act=act, out_dtype=dt), x, xs, w, ws, b, act)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [7, 150])
def test_linear_i8_strides_and_extremes(m):
    from sesa import ops
    x, xs, w, ws, b = linear_case(3, m, 300, 90, full=True)
    for lo, hi in ((0, 256), (1, 258), (16, 272), (3, 300)):   # aligned and unaligned column ranges, rows 300 apart
        linear_check(ops.linear_i8(x[:, lo:hi], xs, w[:, lo:hi], ws, b, out_dtype=torch.float32), x[:, lo:hi], xs,
                     w[:, lo:hi], ws, b)
    y = ops.linear_i8(x[:, :128].t().contiguous().t(), xs, w[:, :128], ws, b, out_dtype=torch.float32)   # column-major x
    linear_check(y, x[:, :128], xs, w[:, :128], ws, b)
    y = ops.linear_i8(x.view(m, 1, 300).expand(m, 2, 300), xs[:, None].expand(m, 2), w, ws, out_dtype=torch.float16)
    assert y.shape == (m, 2, 90) and torch.equal(y[:, 0], y[:, 1])
    big = torch.full((m, 131071), -128, dtype=torch.int8, device="cuda")   # the largest sum: 2^31 - 2^14
    y = ops.linear_i8(big, torch.ones(m, device="cuda"), big[:3], torch.ones(3, device="cuda"), out_dtype=torch.float32)
    assert bool((y.double() - 131071 * 16384).abs().max() <= 131071 * 16384 * E)
    xs2 = xs.clone()
    xs2[2] = math.nan
    y = ops.linear_i8(x, xs2, w, ws, b, act="relu")
    assert bool(torch.isnan(y[2]).all()) and not bool(torch.isnan(y[:2]).any())
    assert ops.linear_i8(x[:0], xs[:0], w, ws).shape == (0, 90)


@pytest.mark.gpu
def test_linear_i8_refuses_tensors():
    from sesa import ops
    from sesa._native import SesaError
    x, xs, w, ws, b = linear_case(4, 4, 32, 8)
    for bad in (lambda: ops.linear_i8(x.float(), xs, w, ws), lambda: ops.linear_i8(x, xs, w[:, :31], ws),
                lambda: ops.linear_i8(x, xs[:3], w, ws), lambda: ops.linear_i8(x, xs.half(), w, ws),
                lambda: ops.linear_i8(x, xs, w, ws[:7]), lambda: ops.linear_i8(x, xs, w, ws, b.half()),
                lambda: ops.linear_i8(x, xs, w, ws, act="swish"), lambda: ops.linear_i8(x, xs, w, ws, out_dtype=torch.float64),
                lambda: ops.linear_i8(x, xs, w.cpu(), ws), lambda: ops.linear_i8(x, xs, w, ws.clone().requires_grad_())):
        with pytest.raises(SesaError, match="linear_i8"):
            bad()


# ---- GPU: norm_residual ---------------------------------------------------------------------------------
def gate_ref(g, act):
    return {"none": lambda: g, "sigmoid": lambda: torch.sigmoid(g), "silu": lambda: g * torch.sigmoid(g),
            "tanh": lambda: torch.tanh(g)}[act]()


def norm_ref(v, kind, w, b, eps):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    v = v if w is None else v * w.double()
    return v if b is None else v + b.double()


def norm_all(x, res, gate, gate_act, post, pw, pb, scale, pre, nw, nb, eps=1e-6):
    """y, n and, for each, the largest value of the row that entered its chain (the unit of the tolerances)."""
    p = norm_ref(x.double(), post, pw, pb, eps)
    g = 1.0 if gate is None else gate_ref(gate.double(), gate_act)
    sp = p * g * (1.0 if scale is None else scale.double())
    y = sp if res is None else res.double() + sp
    gain = (torch.as_tensor(g).abs() * (torch.ones(1, dtype=torch.double, device=x.device) if scale is None else scale.double().abs()))
    top = gain.amax(-1, keepdim=True) * (p.abs().amax(-1, keepdim=True) + (0 if pb is None else pb.abs().max().double()))
    top = top + (0 if res is None else res.double().abs().amax(-1, keepdim=True))
    n = norm_ref(y, pre, nw, nb, eps)
    if pre == "none":
        return y, n, top, top
    dev = y - y.mean(-1, keepdim=True) if pre == "layer" else y
    r = 1 / torch.sqrt((dev * dev).mean(-1, keepdim=True) + eps)
    wmax = 1.0 if nw is None else nw.abs().max().double()
    # an error of y's unit passes through the norm with its gain, once directly and once through the statistics
    return y, n, top, 2 * top * r * wmax + (0 if nb is None else nb.abs().max().double())


NORM_TOL = 64 * E   # 64 half-steps of fp32: at most 16 roundings in a chain, 2 reductions of at most 24 levels each


def norm_check(op_out, ref, i8=False):
    y, n, top_y, top_n = ref
    close(op_out[0], y, NORM_TOL * top_y + HALF[op_out[0].dtype] * y.abs() * (1 + 1e-6) + TINY[op_out[0].dtype])
    if not i8:
        close(op_out[1], n, NORM_TOL * top_n + HALF[op_out[1].dtype] * n.abs() * (1 + 1e-6) + TINY[op_out[1].dtype])
        return
    q, s = op_out[1].double(), op_out[2].double()
    step = n.abs().amax(-1) / 127
    assert bool(((s - step).abs() <= NORM_TOL * top_n[..., 0] / 127 + 2 * E * step).all())
    # in steps: half a step of rounding, and the chain's error counted in steps
    lim = 0.5 + (NORM_TOL * top_n / step[..., None].clamp_min(1e-300)) * 2 + 127 * 4 * E
    assert bool(((q - n / step[..., None].clamp_min(1e-300)).abs() <= lim).all()) and int(q.abs().max()) <= 127


@pytest.mark.gpu
@pytest.mark.parametrize("d", [1, 7, 8, 64, 511, 512, 513, 1000, 1024, 1031, 2048, 2050, 4096, 4104, 8192, 8200, 16384, 20001,
                               32768])
def test_norm_residual_dims(d):
    from sesa import ops
    kinds = [("f16", "f32", "none", "rms"), ("bf16", "bf16", "rms", "layer"), ("f32", "f32", "layer", "rms"),
             ("f16", "f16", "rms", "rms"), ("bf16", "f32", "layer", "layer")]
    for i, (xt, rt, post, pre) in enumerate(kinds):
        g = gen(d * 8 + i)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        m = [1, 5, 4, 9, 3][i]
        x, res = r(m, d).to(DT[xt]) + 0.5, (2 * r(m, d)).to(DT[rt])
        pw, pb, sc, nw, nb = 1 + 0.1 * r(d), 0.1 * r(d), 0.2 + 0.1 * r(d), 1 + 0.1 * r(d), 0.1 * r(d)
        pb = pb if post == "layer" else None
        nb = nb if pre == "layer" else None
        pw = pw if post != "none" else None
        out = ops.norm_residual(x, res, post=post, post_weight=pw, post_bias=pb, scale=sc, pre=pre, pre_weight=nw, pre_bias=nb)
        assert out[0].dtype == res.dtype and out[1].dtype == x.dtype
        ref = norm_all(x, res, None, "none", post, pw, pb, sc, pre, nw, nb)
        norm_check(out, ref)
        norm_check(ops.norm_residual_i8(x, res, post=post, post_weight=pw, post_bias=pb, scale=sc, pre=pre, pre_weight=nw,
                                        pre_bias=nb), ref, True)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "sigmoid", "silu", "tanh"])
def test_norm_residual_gates(act):
    from sesa import ops
    g = gen(5)
    x, res = torch.randn(2, 3, 40, generator=g, device="cuda").half(), torch.randn(2, 3, 40, generator=g, device="cuda")
    for shape in ((2, 3, 40), (2, 1, 40), (1, 1, 40)):
        gate = 3 * torch.randn(*shape, generator=g, device="cuda").half()
        if shape == (1, 1, 40):
            x, res = x[:1], res[:1]
        norm_check(ops.norm_residual(x, res, gate=gate, gate_act=act, post="rms"),
                   norm_all(x, res, gate, act, "rms", None, None, None, "rms", None, None))
    flat, gate = torch.randn(12, 40, generator=g, device="cuda").half(), torch.randn(3, 40, generator=g, device="cuda").half()
    norm_check(ops.norm_residual(flat, None, gate=gate, gate_act=act),
               norm_all(flat, None, gate.repeat_interleave(4, 0), act, "none", None, None, None, "rms", None, None))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [100, 1500])
def test_norm_residual_strides_and_odd_rows(d):
    from sesa import ops
    g = gen(6)
    wide = torch.randn(9, 2 * d + 3, generator=g, device="cuda").half()
    x, res = wide[:, 1:d + 1], wide[:, d + 2:2 * d + 2]        # rows at odd addresses
    norm_check(ops.norm_residual(x, res), norm_all(x, res, None, "none", "none", None, None, None, "rms", None, None))
    x = torch.randn(4, d, generator=g, device="cuda")
    x[0] = 0
    x[1, 3], x[2, 5] = math.inf, math.nan
    q, s = ops.quantize_i8(x)
    assert float(s[0]) == 0 and bool((q[:3] == 0).all()) and bool(torch.isnan(s[1:3]).all())
    norm_check((x[3:], q[3:], s[3:]), (x[3:].double(), x[3:].double(), x[3:].abs().amax(-1, keepdim=True).double(),
                                       x[3:].abs().amax(-1, keepdim=True).double()), True)
    y, n = ops.norm_residual(x, pre="layer")
    assert torch.equal(y.nan_to_num(7, 7, 7), x.nan_to_num(7, 7, 7)) and bool(torch.isnan(n[1:3]).all())
    assert bool((n[0] == 0).all()) and bool(torch.isfinite(n[3]).all())
    q, s = ops.quantize_i8(x[:1] + 1e-38)   # below the smallest scale: counts as zero, never NaN
    assert float(s[0]) == 0 and bool((q == 0).all())
    assert ops.norm_residual(x[:0])[1].shape == (0, d)
    same = torch.full((3, d), 1000.0, device="cuda")   # LayerNorm of a constant row: no deviation, no cancellation
    assert float(ops.norm_residual(same, pre="layer")[1].abs().max()) <= 1000 * 64 * E / math.sqrt(1e-6)


@pytest.mark.gpu
def test_norm_residual_in_place_c_entry():
    N, L = _lib()
    g = gen(7)
    x, res = torch.randn(33, 700, generator=g, device="cuda").half(), torch.randn(33, 700, generator=g, device="cuda")
    ref = norm_all(x, res, None, "none", "rms", None, None, None, "rms", None, None)
    n = torch.empty_like(x)
    a = N.SesaNormArgs(rows=33, dim=700, x_dtype=1, r_dtype=0, x=x.data_ptr(), x_ld=700, residual=res.data_ptr(), r_ld=700, post=1,
                       pre=1, eps=1e-6, y=res.data_ptr(), y_ld=700, n=n.data_ptr(), n_ld=700)
    N.check(L.sesa_norm_residual(ctypes.byref(a), torch.cuda.current_stream().cuda_stream))
    norm_check((res, n), ref)


@pytest.mark.gpu
def test_norm_residual_refuses_tensors():
    from sesa import ops
    from sesa._native import SesaError
    x = torch.randn(4, 32, device="cuda").half()
    one = torch.ones(32, device="cuda")
    for bad in (lambda: ops.norm_residual(x.double()), lambda: ops.norm_residual(x, x.bfloat16()), lambda: ops.norm_residual(x, x[:3]),
                lambda: ops.norm_residual(x, gate=x.float()), lambda: ops.norm_residual(x, gate=x[:3]),
                lambda: ops.norm_residual(x, gate=x[:, :31]), lambda: ops.norm_residual(x, post="batch"),
                lambda: ops.norm_residual(x, gate_act="gelu"), lambda: ops.norm_residual(x, scale=one.half()),
                lambda: ops.norm_residual(x, pre_weight=one[:31]), lambda: ops.norm_residual(x, eps=-1.0),
                lambda: ops.norm_residual(torch.randn(2, 32769, device="cuda")), lambda: ops.norm_residual(x, x.cpu()),
                lambda: ops.norm_residual(x.float().requires_grad_())):
        with pytest.raises(SesaError, match="norm_residual"):
            bad()


# ---- GPU: rope_axes -------------------------------------------------------------------------------------
def rope_ref(x, pos, freqs, sections, layout):
    P = sum(sections)
    axis = [a for a, s in enumerate(sections) for _ in range(s)]
    ang = (pos.double()[:, axis] * freqs.double())[:, None]
    if float(pos.abs().max()) > 2 ** 26:   # beyond exact products in 64 bits: reduce with whole integers on the host
        turn = [int(round(float(f) / (2 * math.pi) * 2 ** 80)) for f in freqs]
        ang = torch.tensor([[((int(pos[t, a]) * turn[i]) % 2 ** 80) / 2 ** 80 * 2 * math.pi for i, a in enumerate(axis)]
                            for t in range(pos.shape[0])], dtype=torch.double, device=x.device)[:, None]
    c, s, xd = torch.cos(ang), torch.sin(ang), x.double()
    u, v = (xd[..., :2 * P:2], xd[..., 1:2 * P:2]) if layout == "pairs" else (xd[..., :P], xd[..., P:2 * P])
    a, b = u * c - v * s, u * s + v * c
    rot = torch.stack([a, b], -1).flatten(-2) if layout == "pairs" else torch.cat([a, b], -1)
    mag = torch.stack([u.abs() + v.abs()] * 2, -1).flatten(-2) if layout == "pairs" else torch.cat([u.abs() + v.abs()] * 2, -1)
    return torch.cat([rot, xd[..., 2 * P:]], -1), torch.cat([mag, torch.zeros_like(xd[..., 2 * P:])], -1)


def rope_check(got, x, pos, freqs, sections, layout):
    ref, mag = rope_ref(x, pos, freqs, sections, layout)
    # angle 2^-25 half-turns off (pi 2^-25), sine and cosine two steps (2^-23 each), two products and a sum
    close(got, ref, 16 * E * mag + HALF[got.dtype] * ref.abs() * (1 + 1e-6) + TINY[got.dtype])
    P2 = 2 * sum(sections)
    assert torch.equal(got[..., P2:], x[..., P2:])


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("d,sections", [(2, [1]), (8, [4]), (64, [16, 16]), (64, [32, 0]), (64, [0, 32]), (48, [5, 7, 3]), (100, [11, 9, 13, 4]),
                                        (128, [16, 24, 24]), (80, [40]), (6, [1, 1])])
def test_rope_axes(layout, d, sections):
    from sesa import ops
    for i, (dt, hq, hk, t) in enumerate([("f16", 4, 2, 5), ("bf16", 1, 1, 1), ("f32", 3, 8, 70)]):
        g = gen(d + i)
        q, k = (torch.randn(t, h, d, generator=g, device="cuda").to(DT[dt]) for h in (hq, hk))
        pos = torch.randint(-3, 5000, (t, len(sections)), generator=g, device="cuda", dtype=[torch.int32, torch.int64][i % 2])
        freqs = 10000.0 ** -torch.rand(sum(sections), generator=g, device="cuda")
        a, b = ops.rope_axes(q, k, pos, freqs, sections, layout=layout)
        rope_check(a, q, pos, freqs, sections, layout)
        rope_check(b, k, pos, freqs, sections, layout)
        assert torch.equal(ops.rope_axes(q, None, pos, freqs, sections, layout=layout), a)
        # in place, q and k as column ranges of the same rows, the rest of the row left alone
        rows = torch.randn(t, (hq + hk) * d + 3, generator=g, device="cuda").to(DT[dt])
        rows[:, :hq * d], rows[:, hq * d:(hq + hk) * d] = q.reshape(t, -1), k.reshape(t, -1)
        kept = rows[:, -3:].clone()
        ops.rope_axes_(rows[:, :hq * d].unflatten(1, (hq, d)), rows[:, hq * d:-3].unflatten(1, (hk, d)), pos, freqs, sections,
                       layout=layout)
        assert torch.equal(rows[:, :hq * d].reshape(a.shape), a) and torch.equal(rows[:, hq * d:-3].reshape(b.shape), b)
        assert torch.equal(rows[:, -3:], kept)


@pytest.mark.gpu
def test_rope_axes_far_positions():
    """Angles stay exact where an fp32 (and an fp64) product of position and frequency no longer is."""
    from sesa import ops
    g = gen(3)
    q = torch.randn(6, 1, 16, generator=g, device="cuda")
    freqs = 10000.0 ** -torch.rand(8, generator=g, device="cuda")
    for pos in ([0, 1, 10 ** 6, -10 ** 6, 2 ** 31 - 1, -2 ** 31], [0, 1, 2 ** 40, -2 ** 40, 2 ** 45 + 1, 3]):
        p = torch.tensor(pos, device="cuda", dtype=torch.int64)[:, None]
        # freqs / (2 pi) is held to 2^-54 of a turn: at 2^45 the angle is off by up to 2 pi 2^-9
        ref, mag = rope_ref(q, p, freqs, [8], "halves")
        tol = (16 * E + 2 * math.pi * p.double().abs()[:, None] * 2.0 ** -54) * mag + HALF[q.dtype] * ref.abs()
        close(ops.rope_axes(q, None, p, freqs, [8]), ref, tol)


@pytest.mark.gpu
def test_rope_axes_refuses_tensors():
    from sesa import ops
    from sesa._native import SesaError
    q, f = torch.randn(4, 2, 16, device="cuda"), torch.ones(8, device="cuda")
    p = torch.zeros(4, 1, dtype=torch.int32, device="cuda")
    for bad in (lambda: ops.rope_axes(q[0], None, p, f, [8]), lambda: ops.rope_axes(q, q.half(), p, f, [8]),
                lambda: ops.rope_axes(q, q[:3], p, f, [8]), lambda: ops.rope_axes(q, None, p[:3], f, [8]),
                lambda: ops.rope_axes(q, None, p.float(), f, [8]), lambda: ops.rope_axes(q, None, p, f[:7], [8]),
                lambda: ops.rope_axes(q, None, p, torch.ones(9, device="cuda"), [9]), lambda: ops.rope_axes(q, None, p, f, [4, 4]),
                lambda: ops.rope_axes(q, None, p, f, [8], layout="thirds"), lambda: ops.rope_axes(q, None, p.cpu(), f, [8]),
                lambda: ops.rope_axes_(q, q, p, f, [8]), lambda: ops.rope_axes_(q.expand(4, 2, 16)[:1].expand(4, 2, 16), None, p, f, [8]),
                lambda: ops.rope_axes(q.clone().requires_grad_(), None, p, f, [8])):
        with pytest.raises(SesaError, match="rope_axes"):
            bad()


# ---- GPU: attention_packed ------------------------------------------------------------------------------
def attn_ref(q, k, v, cu, causal, scale, gate):
    """[tokens, lanes, heads, d] -> (out, sum_j p_j |v_j|, sum |q_i k_i| scale at its largest) in 64 bits."""
    t, lanes, h, d = q.shape
    grp = h // k.shape[2]
    out, mag = torch.zeros(q.shape, dtype=torch.double, device=q.device), torch.zeros(q.shape, dtype=torch.double, device=q.device)
    big = torch.zeros(q.shape[:-1], dtype=torch.double, device=q.device)
    for a, b in zip(cu[:-1], cu[1:]):
        if b <= a:
            continue
        Q = q[a:b].double().permute(1, 2, 0, 3)
        K, V = (x[a:b].double().permute(1, 2, 0, 3).repeat_interleave(grp, 1) for x in (k, v))
        s = (Q @ K.transpose(-1, -2).contiguous()) * scale
        big[a:b] = ((Q.abs() @ K.abs().transpose(-1, -2).contiguous()) * scale).amax(-1).permute(2, 0, 1)
        if causal:
            hide = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).triu(1)
            s = s.masked_fill(hide, -math.inf)
        p = torch.softmax(s, -1)
        out[a:b], mag[a:b] = ((p @ x).permute(2, 0, 1, 3) for x in (V, V.abs()))
    if gate is not None:
        gt = torch.sigmoid(gate.double())[..., None]
        out, mag = out * gt, mag * gt
    return out, mag, big


def attn_check(got, q, k, v, cu, causal=True, scale=None, gate=None):
    four = q.dim() == 4
    q4, k4, v4, g4 = (x if four or x is None else x.unsqueeze(1) for x in (q, k, v, gate))
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    ref, mag, big = attn_ref(q4, k4, v4, cu, causal, scale, g4)
    u, d = HALF[q.dtype], q.shape[-1]
    # P rounded once (u), the scores' sums of d products (d + 8 half-steps of their largest sum, twice: in P and in the
    # normaliser), exp2 and the row sum (2^-19), then the result's own rounding
    tol = (u + 2 * (d + 8) * E * big[..., None] + 2.0 ** -19) * mag
    if got.dtype == torch.float16:
        # P below 2^-14 of the row's running maximum (itself within 2^8 of the true one) is subnormal: 2^-25 a key at most
        n = max(b - a for a, b in zip(cu[:-1], cu[1:]))
        tol = tol + 2.0 ** -25 * n * float(v.abs().max())
    close((got if four else got.unsqueeze(1)), ref, tol + u * (ref.abs() + tol) + TINY[q.dtype])


def qkv(seed, t, hq, hk, d, dt, lanes=None):
    g = gen(seed)
    lead = (t,) if lanes is None else (t, lanes)
    rows = torch.randn(*lead, hq + 2 * hk, d, generator=g, device="cuda").to(DT[dt])
    return rows.split([hq, hk, hk], -2)


def cu_of(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu, torch.tensor(cu, dtype=torch.int32, device="cuda")


LENS = [[1], [2], [31], [64], [65], [128, 1, 0, 63], [0, 0, 5], [129, 300], [1] * 70, [700], [513, 0, 257, 1], list(range(40))]


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", LENS, ids=lambda v: f"{len(v)}seq{sum(v)}")
def test_attention_packed_lengths(lens, causal):
    from sesa import ops
    cu, cut = cu_of(lens)
    for i, (d, hq, hk, dt) in enumerate([(64, 4, 2, "f16"), (128, 4, 1, "bf16"), (64, 2, 2, "bf16"), (128, 2, 2, "f16")]):
        q, k, v = qkv(sum(lens) * 4 + i, cu[-1], hq, hk, d, dt)
        attn_check(ops.attention_packed(q, k, v, cut, causal=causal), q, k, v, cu, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [8, 24, 40, 48, 56, 72, 80, 96, 120])
def test_attention_packed_head_dims(d):
    from sesa import ops
    cu, cut = cu_of([100, 29])
    for dt in ("f16", "bf16"):
        q, k, v = qkv(d, 129, 6, 2, d, dt)
        gate = torch.randn(129, 6, generator=gen(d), device="cuda").to(q.dtype)
        attn_check(ops.attention_packed(q, k, v, cut, gate=gate), q, k, v, cu, True, None, gate)
        attn_check(ops.attention_packed(q, k, v, cut, causal=False, scale=0.7), q, k, v, cu, False, 0.7)


@pytest.mark.gpu
def test_attention_packed_lanes_gates_and_strides():
    from sesa import ops
    cu, cut = cu_of([70, 0, 131])
    q, k, v = qkv(11, 201, 8, 8, 64, "f16", lanes=5)
    gate = 4 * torch.randn(201, 5, 8, generator=gen(1), device="cuda").half()
    out = ops.attention_packed(q, k, v, cut, causal=False, gate=gate)
    attn_check(out, q, k, v, cu, False, None, gate)
    for ln in (0, 4):   # a lane is what it would be alone
        assert torch.equal(out[:, ln], ops.attention_packed(q[:, ln], k[:, ln], v[:, ln], cut, causal=False, gate=gate[:, ln]))
    flat = [x[:, 0].permute(1, 0, 2).contiguous().permute(1, 0, 2) for x in (q, k, v)]   # head-major storage
    assert torch.equal(ops.attention_packed(*flat, cut, causal=False, gate=gate[:, 0]), out[:, 0])
    odd = [torch.nn.functional.pad(x[:, 0], (1, 2))[..., 1:65] for x in (q, k, v)]       # rows at odd addresses
    assert torch.equal(ops.attention_packed(*odd, cut, causal=False, gate=gate[:, 0]), out[:, 0])
    one = ops.attention_packed(q[:, 0], k[:, 0], v[:, 0])
    attn_check(one, q[:, 0], k[:, 0], v[:, 0], [0, 201], True)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_attention_packed_rest_and_bad_lengths(d):
    """Rows of no sequence: 0, or with out= left as they were; boundaries outside the run are held to it."""
    from sesa import ops
    q, k, v = qkv(12, 300, 2, 1, d, "bf16")
    for lo, mid, hi in ((0, 100, 260), (40, 41, 299), (200, 200, 200), (0, 300, 300)):
        cut = torch.tensor([lo, mid, hi], dtype=torch.int32, device="cuda")
        got = ops.attention_packed(q, k, v, cut)
        attn_check(got, q, k, v, [lo, mid, hi])
        assert bool((got[:lo] == 0).all()) and bool((got[hi:] == 0).all())
        out = torch.full_like(got, 7.0)
        assert ops.attention_packed(q, k, v, cut, out=out) is out
        assert torch.equal(out[lo:hi], got[lo:hi]) and bool((out[:lo] == 7).all()) and bool((out[hi:] == 7).all())
    cut = torch.tensor([0, 120, 10 ** 6], dtype=torch.int32, device="cuda")
    attn_check(ops.attention_packed(q, k, v, cut), q, k, v, [0, 120, 300])
    cut = torch.tensor([-50, 120, 300], dtype=torch.int32, device="cuda")
    attn_check(ops.attention_packed(q, k, v, cut), q, k, v, [0, 120, 300])


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_attention_packed_non_finite(d, dt):
    """A masked key contributes nothing, whatever it holds; a visible one does what the formula says."""
    from sesa import ops
    cu, cut = cu_of([90, 60])
    q, k, v = (x.clone() for x in qkv(13, 150, 2, 2, d, dt))
    clean = ops.attention_packed(q, k, v, cut)
    for bad in (math.inf, -math.inf, math.nan):
        k2, v2 = k.clone(), v.clone()
        k2[70], v2[70] = math.nan, bad          # inside the first sequence: rows 0 .. 69 and the second do not see it
        v2[90:] = v[90:]
        got = ops.attention_packed(q, k2, v2, cut)
        attn_check(got[:70], q[:70], k[:70], v[:70], [0, 70])
        assert torch.equal(got[90:], clean[90:]) and bool(torch.isnan(got[70:90]).all())
        got = ops.attention_packed(q, k, v2, cut)   # v alone: the rows that see it get it
        attn_check(got[:70], q[:70], k[:70], v[:70], [0, 70])
        assert torch.equal(got[90:], clean[90:])
        tail = got[70:90].float()
        assert bool((torch.isnan(tail) if math.isnan(bad) else tail == bad).all())
    v2 = v.clone()
    v2[90:] = math.nan                           # the next sequence's keys, in the same key block as the first's end
    got = ops.attention_packed(q, k, v2, cut, causal=False)
    attn_check(got[:90], q[:90], k[:90], v[:90], [0, 90], False)
    k2 = k.clone()
    k2[5] = torch.where(q[0, :, :] > 0, -math.inf, math.inf).to(k.dtype)   # score -inf for row 0's signs
    got = ops.attention_packed(q[:6], k2[:6], v[:6])
    attn_check(got[:5], q[:5], k[:5], v[:5], [0, 5])


@pytest.mark.gpu
@pytest.mark.parametrize("d", [8, 40, 56, 72, 96, 120])
def test_attention_packed_part_rows(d):
    """Rows narrower than the tile: copied at 16-byte addresses and through registers alike, and nothing of the element
    behind a row (another head's NaN and infinity) reaches it."""
    from sesa import ops
    cu, cut = cu_of([300, 0, 65, 129])
    for causal in (True, False):
        q, k, v = qkv(d + 7, cu[-1], 6, 3, d, "bf16")
        got = ops.attention_packed(q, k, v, cut, causal=causal)
        attn_check(got, q, k, v, cu, causal)
        odd = [torch.nn.functional.pad(x, (1, 2))[..., 1:d + 1] for x in (q, k, v)]
        assert torch.equal(ops.attention_packed(*odd, cut, causal=causal), got)
        k2, v2 = k.clone(), v.clone()
        k2[:, 2], v2[:, 2], k2[:, 0], v2[:, 0] = math.nan, math.inf, math.inf, math.nan
        assert torch.equal(ops.attention_packed(q, k2, v2, cut, causal=causal)[:, 2:4], got[:, 2:4])


@pytest.mark.gpu
def test_attention_packed_large_scores():
    """Scores far apart (the running maximum moves by more than the lazy step, P under- and overflows without it)."""
    from sesa import ops
    for dt in ("f16", "bf16"):
        q, k, v = (x.clone() for x in qkv(14, 400, 2, 2, 64, dt))
        q, k = (q * 6).to(q.dtype), (k * torch.linspace(0.1, 6, 400, device="cuda")[:, None, None]).to(k.dtype)
        attn_check(ops.attention_packed(q, k, v), q, k, v, [0, 400])
        attn_check(ops.attention_packed(q, k.flip(0), v, causal=False), q, k.flip(0), v, [0, 400], False)


@pytest.mark.gpu
def test_attention_packed_refuses_tensors():
    from sesa import ops
    from sesa._native import SesaError
    q, k, v = qkv(15, 8, 4, 2, 64, "f16")
    cu = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    rows = torch.zeros(8, 4, 64, device="cuda", dtype=torch.float16)
    for bad in (lambda: ops.attention_packed(q.float(), k.float(), v.float()), lambda: ops.attention_packed(q, k.bfloat16(), v),
                lambda: ops.attention_packed(q[:, :3], k, v), lambda: ops.attention_packed(q, k[:7], v[:7]),
                lambda: ops.attention_packed(q[..., :60], k[..., :60], v[..., :60]), lambda: ops.attention_packed(q, k, v, cu.long()),
                lambda: ops.attention_packed(q, k, v, cu[:1]), lambda: ops.attention_packed(q, k, v, cu, gate=q[..., 0].float()),
                lambda: ops.attention_packed(q, k, v, cu, gate=k[..., 0]), lambda: ops.attention_packed(q, k, v, cu, scale=0.0),
                lambda: ops.attention_packed(q, k, v, cu.cpu()), lambda: ops.attention_packed(q[0], k[0], v[0]),
                lambda: ops.attention_packed(rows, rows, rows, cu, out=rows), lambda: ops.attention_packed(q, k, v, cu, out=rows[:7]),
                lambda: ops.attention_packed(q, k, v, cu, out=rows[:1].expand(8, 4, 64)),
                lambda: ops.attention_packed(q.detach().clone().requires_grad_(), k, v)):
        with pytest.raises(SesaError, match="attention_packed"):
            bad()


# ---- GPU: together --------------------------------------------------------------------------------------
class Block:
    """One pre-norm transformer block in 8 bits: attention and feed-forward, as a user strings the operators together."""

    def __init__(self, dim, heads, kv, d, seed):
        from sesa import ops
        g = gen(seed)
        r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.heads, self.kv, self.d = heads, kv, d
        self.full = {n: r(o, i) * i ** -0.5 for n, o, i in (("qkv", (heads + 2 * kv) * d, dim), ("out", dim, heads * d),
                                                           ("up", 3 * dim, dim), ("down", dim, 3 * dim))}
        self.w = {n: ops.quantize_i8(w) for n, w in self.full.items()}
        self.norms = [1 + 0.1 * r(dim) for _ in range(3)]
        self.bias = 0.1 * r(3 * dim)
        self.freqs = 10000.0 ** -torch.linspace(0, 1, d // 2, device="cuda")
        self.sections = [d // 4, d // 2 - d // 4]

    def __call__(self, x, pos, cu):
        from sesa import ops
        h, k, d = self.heads, self.kv, self.d
        _, q8, s = ops.norm_residual_i8(x, pre_weight=self.norms[0])
        qkv = ops.linear_i8(q8, s, *self.w["qkv"]).view(-1, h + 2 * k, d)
        qq, kk, vv = qkv.split([h, k, k], 1)
        ops.rope_axes_(qq, kk, pos, self.freqs, self.sections)
        o = ops.attention_packed(qq, kk, vv, cu).view(-1, h * d)
        o = ops.linear_i8(*ops.quantize_i8(o), *self.w["out"])
        x, q8, s = ops.norm_residual_i8(o, x, pre_weight=self.norms[1])
        u = ops.linear_i8(q8, s, *self.w["up"], self.bias, act="gelu")
        u = ops.linear_i8(*ops.quantize_i8(u), *self.w["down"])
        return ops.norm_residual(u, x, pre_weight=self.norms[2])

    def ref(self, x, pos, cu):
        """The same block in 64 bits, the weights as their 8 bits stand for, activations unrounded."""
        w = {n: q.double() * s.double()[:, None] for n, (q, s) in self.w.items()}
        h, k, d = self.heads, self.kv, self.d
        x = x.double()
        qkv = (norm_ref(x, "rms", self.norms[0], None, 1e-6) @ w["qkv"].t()).view(-1, h + 2 * k, d)
        qq, kk, vv = qkv.split([h, k, k], 1)
        qq, kk = (rope_ref(t, pos, self.freqs, self.sections, "halves")[0] for t in (qq, kk))
        o = attn_ref(qq[:, None], kk[:, None], vv[:, None], cu, True, d ** -0.5, None)[0].reshape(-1, h * d)
        x = x + o @ w["out"].t()
        u = norm_ref(x, "rms", self.norms[1], None, 1e-6) @ w["up"].t() + self.bias.double()
        x = x + (0.5 * u * torch.erfc(-u / math.sqrt(2.0))) @ w["down"].t()
        return x, norm_ref(x, "rms", self.norms[2], None, 1e-6)


def block_inputs(seed, t, dim, lens):
    g = gen(seed)
    cu, cut = cu_of(lens)
    return torch.randn(t, dim, generator=g, device="cuda"), torch.randint(0, 900, (t, 2), generator=g, device="cuda"), cu, cut


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1], [3, 60, 0, 17], [200, 150]])
def test_block_of_all_operators(lens):
    blk = Block(256, 4, 2, 64, 1)
    x, pos, cu, cut = block_inputs(2, sum(lens), 256, lens)
    got, ref = blk(x, pos, cut), blk.ref(x, pos, cu)
    # five roundings to 8 bits on the way (a row's step is its largest value / 127, so about 1 % of a value each for
    # normal rows, uniform over a step: 1 / sqrt(12) of it), added as independent errors
    for a, b in zip(got, ref):
        rel = float((a.double() - b).norm() / b.norm())
        assert rel <= math.sqrt(5) * (4.5 / 127 / math.sqrt(12)), rel


@pytest.mark.gpu
def test_block_streams_and_graphs():
    """The same values from another stream, from two streams at once, and from a graph replayed among eager work; two graphs
    of the same block keep apart."""
    blk = Block(256, 4, 2, 64, 1)
    sets = [block_inputs(s, 77, 256, [40, 0, 37]) for s in (3, 4)]
    want = [[t.clone() for t in blk(x, pos, cut)] for x, pos, _, cut in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for st, (x, pos, _, cut) in zip(streams, sets):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(blk(x, pos, cut))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    graphs = []
    for x, pos, _, cut in sets:
        hold = [x.clone(), pos.clone(), cut.clone()]
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = blk(*hold)
        graphs.append((gr, hold, out))
    for i in range(4):
        for (gr, hold, out), j in zip(graphs, ((i % 2), (i + 1) % 2)):
            for h, s in zip(hold, (sets[j][0], sets[j][1], sets[j][3])):
                h.copy_(s)
            gr.replay()
            eager = blk(sets[j][0], sets[j][1], sets[j][3])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want[j]))
            assert all(torch.equal(a, b) for a, b in zip(eager, want[j]))


@pytest.mark.gpu
def test_opcheck_token_ops():
    from sesa import ops  # noqa: F401
    utils = ("test_schema", "test_faketensor")
    x, xs, w, ws, b = linear_case(1, 5, 32, 8)
    torch.library.opcheck(torch.ops.sesa.linear_i8.default, (x, xs, w, ws, b, "gelu", torch.float16), test_utils=utils)
    h = torch.randn(6, 16, device="cuda").half()
    rest = (None, "none", "rms", None, None, None, "layer", None, None, 1e-6)
    torch.library.opcheck(torch.ops.sesa.norm_residual.default, (h, h.float(), *rest), test_utils=utils)
    torch.library.opcheck(torch.ops.sesa.norm_residual_i8.default, (h, None, *rest), test_utils=utils)
    torch.library.opcheck(torch.ops.sesa.quantize_i8.default, (h,), test_utils=utils)
    q, k, v = qkv(2, 6, 2, 1, 16, "f16")
    pos = torch.zeros(6, 1, dtype=torch.int32, device="cuda")
    torch.library.opcheck(torch.ops.sesa.rope_axes.default, ([q, k], pos, torch.ones(8, device="cuda"), [8], "pairs"), test_utils=utils)
    torch.library.opcheck(torch.ops.sesa.attention_packed.default, (q, k, v, None, True, None, None), test_utils=utils)
    torch.library.opcheck(torch.ops.sesa.attention_packed_into.default, (q, k, v, None, True, None, None, torch.zeros_like(q)),
                          test_utils=utils)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows so far apart that an element's offset passes 2^31 (and bytes 2^32): the last rows come out right."""
    from sesa import ops
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GiB of device memory")
    buf = torch.empty(6 << 30, dtype=torch.uint8, device="cuda")
    g = gen(21)
    m, ld = 70000, 65536                                     # 4.3 G elements of int8, rows 64 KiB apart
    x = buf.view(torch.int8).as_strided((m, 64), (ld, 1))
    x.copy_(torch.randint(-127, 128, (m, 64), generator=g, device="cuda", dtype=torch.int8))
    w, ws = ops.quantize_i8(torch.randn(32, 64, generator=g, device="cuda"))
    xs = torch.rand(m, generator=g, device="cuda")
    linear_check(ops.linear_i8(x, xs, w, ws, out_dtype=torch.float32), x, xs, w, ws, None)
    t, ld = 40000, 65536                                     # 2.6 G elements of fp16
    rows = buf.view(torch.float16).as_strided((t, 3, 2, 64), (ld, 128, 64, 1))
    rows.copy_(torch.randn(t, 3, 2, 64, generator=g, device="cuda"))
    q, k, v = rows.unbind(1)
    cu, cut = cu_of([39000, 900, 100])
    out = ops.attention_packed(q, k, v, cut)
    lo = 39000
    attn_check(out[lo:], q[lo:], k[lo:], v[lo:], [0, 900, 1000])
    flat = rows.as_strided((t, 384), (ld, 1))
    norm_check([a[lo:] for a in ops.norm_residual(flat)], norm_all(flat[lo:], None, None, "none", "none", None, None, None, "rms", None, None))
    pos, f = torch.arange(t, device="cuda")[:, None], torch.ones(32, device="cuda")
    want = ops.rope_axes(q[lo:].contiguous(), None, pos[lo:], f, [32])
    ops.rope_axes_(q, None, pos, f, [32])
    assert torch.equal(q[lo:], want)


@pytest.mark.gpu
def test_grids_past_one_row():
    """More workgroups than one row of the launch grid holds (2^18)."""
    from sesa import ops
    g = gen(22)
    x = torch.randn(1_060_000, 16, generator=g, device="cuda").half()
    q, s = ops.quantize_i8(x)
    norm_check((x, q, s), (x.double(), x.double(), x.abs().amax(-1, keepdim=True).double(), x.abs().amax(-1, keepdim=True).double()), True)
    x = torch.randn(262_200, 1032, generator=g, device="cuda", dtype=torch.float16)
    y, n = ops.norm_residual(x)
    at = torch.tensor([0, 262_143, 262_144, 262_199], device="cuda")
    norm_check((y[at], n[at]), norm_all(x[at], None, None, "none", "none", None, None, None, "rms", None, None))
    assert torch.equal(y, x)
    del x, y, n
    t = 300_000                                               # sequences of one token: each attends to itself alone
    rows = torch.randn(t, 3, 1, 8, generator=g, device="cuda").half()
    cut = torch.arange(t + 1, dtype=torch.int32, device="cuda")
    assert torch.equal(ops.attention_packed(*rows.unbind(1), cut), rows[:, 2])
    t = 67_200_000                                            # one pair a token: a thread each
    x = torch.randn(t, 1, 2, generator=g, device="cuda", dtype=torch.float16)
    pos = torch.arange(t, dtype=torch.int32, device="cuda")[:, None]
    got = ops.rope_axes(x, None, pos, torch.full((1,), 0.001, device="cuda"), [1])
    at = torch.tensor([0, 5, 67_108_863, 67_108_864, t - 1], device="cuda")
    rope_check(got[at], x[at], pos[at], torch.full((1,), 0.001, device="cuda"), [1], "halves")


@pytest.mark.gpu
def test_attention_packed_out_ranges_and_lane_groups():
    """Lanes with grouped heads under a causal mask, and out as a column range of wider rows (the rest left alone)."""
    from sesa import ops
    cu, cut = cu_of([0, 130, 1, 60])
    for d, dt in ((64, "bf16"), (128, "f16"), (40, "f16")):
        q, k, v = qkv(31 + d, 191, 6, 3, d, dt, lanes=3)
        gate = torch.randn(191, 3, 6, generator=gen(d), device="cuda").to(q.dtype)
        want = ops.attention_packed(q, k, v, cut, gate=gate)
        attn_check(want, q, k, v, cu, True, None, gate)
        wide = torch.full((191, 3, 8, d + 5), 3.0, device="cuda", dtype=q.dtype)
        ops.attention_packed(q, k, v, cut, gate=gate, out=wide[:, :, 1:7, 2:2 + d])
        assert torch.equal(wide[:, :, 1:7, 2:2 + d], want)
        wide[:, :, 1:7, 2:2 + d] = 3.0
        assert bool((wide == 3).all())
        rows = torch.cat([q, k, v, torch.zeros_like(q)], 2)   # out beside q, k, v in the same rows
        qq, kk, vv, oo = rows.split([6, 3, 3, 6], 2)
        ops.attention_packed(qq, kk, vv, cut, gate=gate, out=oo)
        assert torch.equal(oo, want) and torch.equal(qq, q)


@pytest.mark.gpu
def test_token_ops_under_compile_and_modes():
    """A traced call goes through the registered ops (fullgraph), an intercepting mode sees them."""
    from torch.utils._python_dispatch import TorchDispatchMode
    from sesa import ops
    blk = Block(128, 2, 1, 64, 5)
    x, pos, cu, cut = block_inputs(6, 50, 128, [20, 30])
    want = blk(x, pos, cut)

    def f(x):
        y, q, s = ops.norm_residual_i8(x, pre_weight=blk.norms[0])
        z = ops.linear_i8(q, s, *blk.w["qkv"]).view(-1, 4, 64)
        qq, kk = ops.rope_axes(z[:, :2], z[:, 2:3], pos, blk.freqs, blk.sections)
        return y, ops.attention_packed(qq, kk, z[:, 3:], cut)
    for a, b in zip(torch.compile(f, backend="aot_eager", fullgraph=True)(x), f(x)):
        assert torch.equal(a, b)
    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))
    with Watch():
        got = blk(x, pos, cut)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for name in ("linear_i8", "norm_residual_i8", "norm_residual", "quantize_i8", "rope_axes_", "attention_packed"):
        assert f"sesa.{name}.default" in seen, name


@pytest.mark.gpu
@pytest.mark.parametrize("d", [40, 64, 96, 128])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_attention_packed_non_finite_values_of_long_sequences(d, dt):
    """One infinite value row early in a sequence of several tiles: the rows before it stay finite, the others get it, in
    its own tile (a masked block) and in later ones (whole blocks)."""
    from sesa import ops
    cu, cut = cu_of([300, 80])
    q, k, v = (x.clone() for x in qkv(40 + d, 380, 4, 2, d, dt))
    clean = ops.attention_packed(q, k, v, cut)
    v[5, :, 3] = math.inf
    got = ops.attention_packed(q, k, v, cut)
    attn_check(got[:5], q[:5], k[:5], v[:5], [0, 5])
    assert torch.equal(got[300:], clean[300:])
    tail = got[5:300].float()
    assert bool((tail[..., 3] == math.inf).all()) and bool(torch.isfinite(torch.cat([tail[..., :3], tail[..., 4:]], -1)).all())
    v[5, :, 3] = 0.5   # (finite again: the other columns of those rows were what they are now)
    ref = ops.attention_packed(q, k, v, cut)
    keep = [c for c in range(d) if c != 3]
    u = HALF[q.dtype]
    assert bool(((got[:300][..., keep] - ref[:300][..., keep]).double().abs() <=
                 3 * u * (ref[:300][..., keep].double().abs() + float(v.abs().max()))).all())
