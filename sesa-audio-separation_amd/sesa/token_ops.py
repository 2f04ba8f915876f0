"""Transformer operators over the libsesa C ABI (namespace ``sesa::``), in fp16 / bf16 and 8-bit integers.

``linear_i8`` (Linear layer on 8-bit integers), ``norm_residual`` / ``norm_residual_i8`` / ``quantize_i8`` (norms, gate
and residual between two blocks; rows in 8 bits), ``rope_axes`` / ``rope_axes_`` (rotary positions with several axes),
``attention_packed`` / ``attention_packed_into`` (attention within each sequence of a packed run).  The Roformers'
``int8`` precision runs the same kernels inside libsesa.

Device tensors only, on the current stream of the tensors' device; every result is a new tensor unless the name says
otherwise; nothing waits for the device, so the calls can be captured into a graph.  Inference only: a call whose
inputs would need a gradient, backward or forward mode, raises, also while it is compiled.  The ops are plain
``torch.library`` definitions (schema, device kernel, fake kernel, an autograd kernel that refuses), and a plain eager call
of the functions below goes straight to the device kernel: for a single token the host's share of a call is most of it.
"""
import ctypes
import math

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _native as N

_DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ACT = {"none": 0, "gelu": 1, "tanh": 2, "relu": 3}
_NORM = {"none": 0, "rms": 1, "layer": 2}
_GATE = {"none": 0, "sigmoid": 1, "silu": 2, "tanh": 3}
_LAYOUT = {"halves": 0, "pairs": 1}
_INT4 = ctypes.c_int * 4

_LIB = torch.library.Library("sesa", "FRAGMENT")


def _define(schema):
    """Registers ``schema`` with the decorated function as its device kernel, and the refusal of gradients above it."""
    name = schema.split("(", 1)[0]

    def wrap(fn):
        _LIB.define(schema)
        _LIB.impl(name, fn, "CUDA")
        op = getattr(torch.ops.sesa, name).default
        args = [a.name for a in op._schema.arguments]

        def forward_only(*values):
            _refuse_gradients(name, args, values)
            with torch._C._AutoDispatchBelowAutograd():
                return op(*values)
        _LIB.impl(name, forward_only, "Autograd")
        return fn
    return wrap


def _fail(op, msg):
    raise N.SesaError(f"sesa::{op}: {msg}")


def _refuse_gradients(op, names, values):
    """No argument waits for a gradient or carries a forward-mode tangent.  The dispatcher asks this where autograd would
    record the op, so a compiled graph is refused while it is traced (its own run has gradients off)."""
    grad, forward = torch.is_grad_enabled(), _forward_ad._current_level >= 0
    if not grad and not forward:
        return
    for name, value in zip(names, values):
        for t in value if isinstance(value, (list, tuple)) else (value,):
            if isinstance(t, torch.Tensor) and (grad and t.requires_grad or
                                                forward and _forward_ad.unpack_dual(t).tangent is not None):
                _fail(op, f"{name} requires a gradient and this operator has none (use torch.no_grad())")


def _check(op, idx, names, *tensors):
    """Every tensor (None: absent) on device ``idx``, none of them waiting for a gradient."""
    grad = torch.is_grad_enabled()
    try:
        for t in tensors:
            if t is not None and (t.get_device() != idx or grad and t.requires_grad):
                break
        else:
            return
    except AttributeError:   # not a tensor
        pass
    for name, t in zip(names.split(), tensors):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or t.get_device() != idx:
            _fail(op, f"{name}: expected a HIP device tensor on cuda:{idx} (got {type(t).__name__} on "
                      f"{getattr(t, 'device', None)}); the sesa path has no CPU fallback")
        if grad and t.requires_grad:
            _fail(op, f"{name} requires a gradient and this operator has none (use torch.no_grad())")


def _device(op, t):
    """The index of the device the call runs on."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _fail(op, f"expected a HIP device tensor (got {type(t).__name__} on {getattr(t, 'device', None)}); "
                  "the sesa path has no CPU fallback")
    return t.get_device()


def _launch(op, idx, entry, *args):
    """``entry(*args, stream)`` with device ``idx`` current, on its current stream."""
    if _current_device() == idx:
        rc = entry(*args, _current_stream(idx))
    else:
        with torch.cuda.device(idx):
            rc = entry(*args, _current_stream(idx))
    if rc:
        N.check(rc, f"sesa_{op}")


_Tensor = torch.Tensor
_PLAIN = {torch.Tensor, torch.nn.Parameter, type(None)}
_compiling = torch.compiler.is_compiling
_tracing = torch._C._is_tracing
_dispatch_modes = torch._C._len_torch_dispatch_stack
_function_modes = torch._C._len_torch_function_stack
_transforms = torch._C._are_functorch_transforms_active
_written = torch.autograd.graph.increment_version   # (an op saved such a tensor for its backward: that has to notice)
_current_device = torch.cuda.current_device
_current_stream = torch._C._cuda_getCurrentRawStream


def _plain(*tensors):
    """Whether nothing but the values counts: plain tensors (or None), and no torch.compile or torch.jit trace, no torch.func
    transform, no mode and no forward-mode level that would have to see the op."""
    return set(map(type, tensors)) <= _PLAIN and not (_compiling() or _dispatch_modes() or _function_modes() or _transforms() or
                                                      _tracing() or _forward_ad._current_level >= 0)


def _eager(op, t, *more):
    """Whether a call can go straight to its device kernel: a device tensor, and ``_plain``.  Saves the dispatcher's share of
    the host's time (3 to 4 us a call: a one-token call takes 6 to 9)."""
    if not isinstance(t, _Tensor):
        if hasattr(type(t), "__torch_function__"):   # a stand-in (torch.fx): the op itself goes into its graph
            return False
        _device(op, t)
    elif not t.is_cuda:
        _device(op, t)
    return _plain(t, *more)


def _param(op, name, t, n):
    """An optional fp32 [n] parameter vector, contiguous."""
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.shape != (n,):
        _fail(op, f"{name}: expected float32 [{n}], got {t.dtype} {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _rows(t):
    """[..., n] as [rows, n] with the last dimension contiguous (a copy only where the strides need one)."""
    if t.dim() != 2:
        t = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])   # (-1 has no answer where n is 0)
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _span(t):
    """Elements from a tensor's first to behind its last."""
    return sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1 if t.numel() else 0


def _writable(t):
    """Whether every element has a place of its own and the last dimension is contiguous."""
    reach = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s < reach:
            return False
        reach = s * (n - 1) + reach
    return t.numel() == 0 or t.shape[-1] == 1 or t.stride(-1) == 1


def _disjoint(ts, us, off):
    """Whether two strided sets of elements share none; ts / us: (size, stride) from the widest stride down, u's first
    element ``off`` behind t's.  False also where it is not plain to see."""
    reach = [sum((n - 1) * s for n, s in d) + 1 for d in (ts, us)]
    if off >= reach[0] or -off >= reach[1]:
        return True
    if not ts or not us or ts[0][1] != us[0][1]:
        return False
    row = ts[0][1]
    if any(sum((n - 1) * s for n, s in d[1:]) + 1 > row for d in (ts, us)):
        return False
    at = off % row   # u's rows begin at..row behind, or row - at before, some row of t
    return _disjoint(ts[1:], us[1:], at) and _disjoint(ts[1:], us[1:], at - row)


def _apart(t, u):
    """Whether two tensors share no memory: by storage, by span, or as column ranges of the same rows."""
    if t.untyped_storage().data_ptr() != u.untyped_storage().data_ptr() or not t.numel() or not u.numel():
        return True
    a, b = t.data_ptr(), u.data_ptr()
    if a + _span(t) * t.element_size() <= b or b + _span(u) * u.element_size() <= a:
        return True
    if t.element_size() != u.element_size() or (b - a) % t.element_size():
        return False
    dims = [sorted(((n, s) for n, s in zip(x.shape, x.stride()) if n > 1), key=lambda d: -d[1]) for x in (t, u)]
    return _disjoint(*dims, (b - a) // t.element_size())


def _ptr(t):
    return None if t is None else t.data_ptr()


# ---- linear_i8 ------------------------------------------------------------------------------------------
def _linear_shape(x, x_scale, weight):
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        _fail("linear_i8", f"x {list(x.shape)} and weight {list(weight.shape)} do not share their last dimension")
    if x_scale.shape != x.shape[:-1]:
        _fail("linear_i8", f"x_scale {list(x_scale.shape)}: expected one scale per row of x {list(x.shape)}")
    return [*x.shape[:-1], weight.shape[0]]


@_define("linear_i8(Tensor x, Tensor x_scale, Tensor weight, Tensor w_scale, Tensor? bias, str act, "
         "ScalarType out_dtype) -> Tensor")
def _linear_i8(x, x_scale, weight, w_scale, bias, act, out_dtype):
    op = "linear_i8"
    idx = _device(op, x)
    _check(op, idx, "x x_scale weight w_scale bias", x, x_scale, weight, w_scale, bias)
    shape = _linear_shape(x, x_scale, weight)
    if x.dtype != torch.int8 or weight.dtype != torch.int8:
        _fail(op, f"x and weight: expected int8, got {x.dtype} and {weight.dtype}")
    if x_scale.dtype != torch.float32:
        _fail(op, f"x_scale: expected float32, got {x_scale.dtype}")
    if act not in _ACT or out_dtype not in _DTYPE:
        _fail(op, f"act {act!r} (one of {', '.join(_ACT)}), out_dtype {out_dtype} (float32, float16 or bfloat16)")
    n, k = weight.shape
    ws, b = _param(op, "w_scale", w_scale, n), _param(op, "bias", bias, n)
    xr, wr = _rows(x), _rows(weight)
    xs = x_scale if x_scale.is_contiguous() else x_scale.contiguous()
    out = x.new_empty(shape, dtype=out_dtype)
    _launch(op, idx, N.lib().sesa_linear_i8, xr.data_ptr(), xr.stride(0), xs.data_ptr(), wr.data_ptr(), wr.stride(0),
            ws.data_ptr(), _ptr(b), _ACT[act], xr.shape[0], n, k, out.data_ptr(), _DTYPE[out_dtype], n)
    return out


@torch.library.register_fake("sesa::linear_i8", lib=_LIB)
def _(x, x_scale, weight, w_scale, bias, act, out_dtype):
    return x.new_empty(_linear_shape(x, x_scale, weight), dtype=out_dtype)


# ---- norm_residual --------------------------------------------------------------------------------------
def _gate_groups(x, gate):
    """Rows of x per gate row: the gate has x's shape, or 1 in place of trailing leading dimensions of x."""
    if not x.numel() and gate.shape == x.shape:
        return 1
    lead, g = list(x.shape[:-1]), list(gate.shape[:-1])
    if gate.dim() == 2 and x.dim() == 2:   # [groups, dim] for flat rows
        if gate.shape[0] and x.shape[0] % gate.shape[0] == 0 and gate.shape[1] == x.shape[1]:
            return max(1, x.shape[0] // gate.shape[0])
    elif gate.dim() == x.dim() and gate.shape[-1] == x.shape[-1]:
        cut = len(lead)
        while cut and g[cut - 1] == 1:
            cut -= 1
        if g[:cut] == lead[:cut]:
            per = 1
            for s in lead[cut:]:
                per *= s
            return max(1, per)
    _fail("norm_residual", f"gate {list(gate.shape)} does not cover x {list(x.shape)} (x's shape, 1 in trailing "
                           "dimensions before the last, or [groups, dim] for x [rows, dim])")


def _norm_call(op, x, residual, gate, gate_act, post, post_weight, post_bias, scale, pre, pre_weight, pre_bias, eps, i8):
    idx = _device(op, x)
    _check(op, idx, "x residual gate post_weight post_bias scale pre_weight pre_bias", x, residual, gate, post_weight,
           post_bias, scale, pre_weight, pre_bias)
    if x.dtype not in _DTYPE or x.dim() < 1:
        _fail(op, f"x: expected float32, float16 or bfloat16 [..., dim], got {x.dtype} {list(x.shape)}")
    if post not in _NORM or pre not in _NORM or gate_act not in _GATE:
        _fail(op, f"post {post!r}, pre {pre!r} (one of {', '.join(_NORM)}), gate_act {gate_act!r} (one of "
                  f"{', '.join(_GATE)})")
    d = x.shape[-1]
    if residual is not None and (residual.shape != x.shape or residual.dtype not in (x.dtype, torch.float32)):
        _fail(op, f"residual: expected {list(x.shape)} in {x.dtype} or float32, got {residual.dtype} "
                  f"{list(residual.shape)}")
    if gate is not None and gate.dtype != x.dtype:
        _fail(op, f"gate: expected {x.dtype}, got {gate.dtype}")
    per = 1 if gate is None else _gate_groups(x, gate)
    rt = x.dtype if residual is None else residual.dtype
    xr = _rows(x)
    rr, gr = None if residual is None else _rows(residual), None if gate is None else _rows(gate)
    y = torch.empty_like(x if residual is None else residual, memory_format=torch.contiguous_format)
    n = torch.empty_like(x, dtype=torch.int8 if i8 else None, memory_format=torch.contiguous_format)
    qs = x.new_empty(x.shape[:-1], dtype=torch.float32) if i8 else None
    a = N.SesaNormArgs(xr.shape[0], d, _DTYPE[x.dtype], _DTYPE[rt], xr.data_ptr(), xr.stride(0))
    if rr is not None:
        a.residual, a.r_ld = rr.data_ptr(), rr.stride(0)
    if gr is not None:
        a.gate, a.gate_ld, a.rows_per_gate, a.gate_act = gr.data_ptr(), gr.stride(0), per, _GATE[gate_act]
    a.post, a.pre, a.eps = _NORM[post], _NORM[pre], eps
    kept = []   # copies live until the launch
    for name, t in (("post_weight", post_weight), ("post_bias", post_bias), ("scale", scale), ("pre_weight", pre_weight),
                    ("pre_bias", pre_bias)):
        if t is not None:
            kept.append(_param(op, name, t, d))
            setattr(a, name, kept[-1].data_ptr())
    a.y, a.y_ld = y.data_ptr(), d
    if i8:
        a.q, a.q_ld, a.q_scale = n.data_ptr(), d, qs.data_ptr()
    else:
        a.n, a.n_ld = n.data_ptr(), d
    _launch("norm_residual", idx, N.lib().sesa_norm_residual, ctypes.byref(a))
    return (y, n, qs) if i8 else (y, n)


_NORM_SCHEMA = ("(Tensor x, Tensor? residual, Tensor? gate, str gate_act, str post, Tensor? post_weight, Tensor? post_bias, "
                "Tensor? scale, str pre, Tensor? pre_weight, Tensor? pre_bias, float eps) -> ")


@_define("norm_residual" + _NORM_SCHEMA + "(Tensor, Tensor)")
def _norm_residual(*args):
    return _norm_call("norm_residual", *args, False)


@_define("norm_residual_i8" + _NORM_SCHEMA + "(Tensor, Tensor, Tensor)")
def _norm_residual_i8(*args):
    return _norm_call("norm_residual_i8", *args, True)


@torch.library.register_fake("sesa::norm_residual", lib=_LIB)
def _(x, residual, *rest):
    return torch.empty_like(x if residual is None else residual, memory_format=torch.contiguous_format), \
        torch.empty_like(x, memory_format=torch.contiguous_format)


@torch.library.register_fake("sesa::norm_residual_i8", lib=_LIB)
def _(x, residual, *rest):
    return torch.empty_like(x if residual is None else residual, memory_format=torch.contiguous_format), \
        torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format), \
        x.new_empty(x.shape[:-1], dtype=torch.float32)


@_define("quantize_i8(Tensor x) -> (Tensor, Tensor)")
def _quantize_i8(x):
    op = "quantize_i8"
    idx = _device(op, x)
    _check(op, idx, "x", x)
    if x.dtype not in _DTYPE or x.dim() < 1:
        _fail(op, f"x: expected float32, float16 or bfloat16 [..., dim], got {x.dtype} {list(x.shape)}")
    xr = _rows(x)
    q = torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format)
    s = x.new_empty(x.shape[:-1], dtype=torch.float32)
    a = N.SesaNormArgs(rows=xr.shape[0], dim=x.shape[-1], x_dtype=_DTYPE[x.dtype], r_dtype=_DTYPE[x.dtype],
                       x=xr.data_ptr(), x_ld=xr.stride(0), q=q.data_ptr(), q_ld=x.shape[-1], q_scale=s.data_ptr())
    _launch("norm_residual", idx, N.lib().sesa_norm_residual, ctypes.byref(a))
    return q, s


@torch.library.register_fake("sesa::quantize_i8", lib=_LIB)
def _(x):
    return torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format), \
        x.new_empty(x.shape[:-1], dtype=torch.float32)


# ---- rope_axes ------------------------------------------------------------------------------------------
def _rope_call(op, xs, outs, positions, freqs, sections, layout):
    idx = _device(op, xs[0])
    _check(op, idx, "positions freqs q k", positions, freqs, *xs)
    x0 = xs[0]
    shape, dtype = x0.shape, x0.dtype
    for x in xs:
        if x.dim() != 3 or dtype not in _DTYPE or x.dtype is not dtype or \
                (x is not x0 and (x.shape[0] != shape[0] or x.shape[2] != shape[2])):
            _fail(op, f"expected [tokens, heads, head_dim] tensors of one type, token count and head_dim, got "
                      f"{[(str(t.dtype), list(t.shape)) for t in xs]}")
    if not 1 <= len(sections) <= 4 or positions.dim() != 2 or \
            positions.shape != (shape[0], len(sections)) or \
            positions.dtype not in (torch.int32, torch.int64):
        _fail(op, f"positions: expected int32 or int64 [{x0.shape[0]}, {len(sections)}] (1 to 4 axes), got "
                  f"{positions.dtype} {list(positions.shape)}")
    if layout not in _LAYOUT:
        _fail(op, f"layout {layout!r} (one of {', '.join(_LAYOUT)})")
    f = _param(op, "freqs", freqs, sum(sections))
    p = positions if len(sections) == 1 or positions.stride(1) == 1 else positions.contiguous()
    a = N.SesaRopeArgs(x0.shape[0], x0.shape[2], _DTYPE[x0.dtype], _LAYOUT[layout], len(sections), _INT4(*sections),
                       p.data_ptr(), p.stride(0), p.dtype is torch.int64, f.data_ptr(), len(xs))
    for i, x in enumerate(xs):
        o, r = outs[i], a.t[i]
        r.x, r.out, r.heads = x.data_ptr(), o.data_ptr(), x.shape[1]
        r.x_t, r.x_h, _ = x.stride()
        r.o_t, r.o_h, _ = o.stride()
    _launch("rope_axes", idx, N.lib().sesa_rope_axes, ctypes.byref(a))


@_define("rope_axes(Tensor[] xs, Tensor positions, Tensor freqs, int[] sections, str layout) -> Tensor[]")
def _rope_axes(xs, positions, freqs, sections, layout):
    if not 1 <= len(xs) <= 2:
        _fail("rope_axes", f"one or two tensors, got {len(xs)}")
    _device("rope_axes", xs[0])
    xs = [x if x.dim() < 1 or x.stride(-1) == 1 else x.contiguous() for x in xs]
    outs = [torch.empty_like(x, memory_format=torch.contiguous_format) for x in xs]
    _rope_call("rope_axes", xs, outs, positions, freqs, sections, layout)
    return outs


@torch.library.register_fake("sesa::rope_axes", lib=_LIB)
def _(xs, positions, freqs, sections, layout):
    return [torch.empty_like(x, memory_format=torch.contiguous_format) for x in xs]


@_define("rope_axes_(Tensor(a!)[] xs, Tensor positions, Tensor freqs, int[] sections, str layout) -> ()")
def _rope_axes_(xs, positions, freqs, sections, layout):
    _rope_places(xs)
    _rope_call("rope_axes_", xs, xs, positions, freqs, sections, layout)
    _written(xs)


def _rope_places(xs):
    if not 1 <= len(xs) <= 2:
        _fail("rope_axes_", f"one or two tensors, got {len(xs)}")
    for x in xs:
        _device("rope_axes_", x)
        if x.dim() != 3 or not _writable(x):
            _fail("rope_axes_", f"in place needs [tokens, heads, head_dim] rows that lie apart, contiguous in the last "
                                f"dimension; got {list(x.shape)} with strides {list(x.stride())}")
    if len(xs) == 2 and not _apart(*xs):
        _fail("rope_axes_", "the two tensors overlap")


@torch.library.register_fake("sesa::rope_axes_", lib=_LIB)
def _(xs, positions, freqs, sections, layout):
    return None


# ---- attention_packed -----------------------------------------------------------------------------------
def _attn_call(op, q, k, v, cu, causal, scale, gate, out, zero_rest):
    idx = _device(op, q)
    _check(op, idx, "q k v cu_seqlens gate out", q, k, v, cu, gate, out)
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        _fail(op, f"q, k, v: expected one of float16 and bfloat16, got {q.dtype}, {k.dtype}, {v.dtype}")
    nd = q.dim()
    if nd not in (3, 4) or k.dim() != nd or k.shape != v.shape or k.shape[:nd - 2] != q.shape[:nd - 2] or \
            k.shape[-1] != q.shape[-1]:
        _fail(op, f"expected q [tokens, (lanes,) heads, head_dim] and k, v [tokens, (lanes,) kv_heads, head_dim], got "
                  f"{list(q.shape)}, {list(k.shape)}, {list(v.shape)}")
    if cu is not None and (cu.dtype != torch.int32 or cu.dim() != 1 or cu.shape[0] < 2):
        _fail(op, f"cu_seqlens: expected int32 [sequences + 1], got {cu.dtype} {list(cu.shape)}")
    if gate is not None and (gate.dtype != q.dtype or gate.shape != q.shape[:-1]):
        _fail(op, f"gate: expected {q.dtype} {list(q.shape[:-1])}, got {gate.dtype} {list(gate.shape)}")
    if out.dtype != q.dtype or out.shape != q.shape or (out.numel() and out.stride(-1) != 1):
        _fail(op, f"out: expected {q.dtype} {list(q.shape)}, contiguous in the last dimension")
    if 0 in q.shape:
        return
    q, k, v = (t if t.stride(-1) == 1 else t.contiguous() for t in (q, k, v))
    cu = cu if cu is None or cu.is_contiguous() else cu.contiguous()
    lanes = q.shape[1] if nd == 4 else 1

    def st3(t, last):   # strides of token, lane, head
        s = t.stride()
        return (s[0], s[1], s[2]) if nd == 4 else (s[0], 0, s[1])
    a = N.SesaAttnArgs(q.shape[0], lanes, q.shape[-2], k.shape[-2], q.shape[-1], _DTYPE[q.dtype], q.data_ptr(),
                       k.data_ptr(), v.data_ptr(), *st3(q, 1), *st3(k, 1), *st3(v, 1), _ptr(cu),
                       1 if cu is None else cu.shape[0] - 1, causal,
                       q.shape[-1] ** -0.5 if scale is None else scale, _ptr(gate),
                       *((0, 0, 0) if gate is None else st3(gate, 0)), out.data_ptr(), *st3(out, 1), zero_rest)
    _launch("attention_packed", idx, N.lib().sesa_attention_packed, ctypes.byref(a))


@_define("attention_packed(Tensor q, Tensor k, Tensor v, Tensor? cu_seqlens, bool causal, float? scale, Tensor? gate) "
         "-> Tensor")
def _attention_packed(q, k, v, cu_seqlens, causal, scale, gate):
    _device("attention_packed", q)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    _attn_call("attention_packed", q, k, v, cu_seqlens, causal, scale, gate, out, True)
    return out


@torch.library.register_fake("sesa::attention_packed", lib=_LIB)
def _(q, k, v, cu_seqlens, causal, scale, gate):
    return torch.empty_like(q, memory_format=torch.contiguous_format)


@_define("attention_packed_into(Tensor q, Tensor k, Tensor v, Tensor? cu_seqlens, bool causal, float? scale, Tensor? gate, "
         "Tensor(a!) out) -> ()")
def _attention_packed_into(q, k, v, cu_seqlens, causal, scale, gate, out):
    op = "attention_packed_into"
    for name, t in (("q", q), ("k", k), ("v", v), ("gate", gate), ("cu_seqlens", cu_seqlens), ("out", out)):
        if t is not None:
            _device(op, t)
        if t is not None and name != "out" and not _apart(t, out):
            _fail(op, f"out overlaps {name}")
    if out.dim() < 2 or not _writable(out):
        _fail(op, f"out: rows have to lie apart, contiguous in the last dimension; got {list(out.shape)} with strides "
                  f"{list(out.stride())}")
    _attn_call(op, q, k, v, cu_seqlens, causal, scale, gate, out, False)
    _written(out)


@torch.library.register_fake("sesa::attention_packed_into", lib=_LIB)
def _(q, k, v, cu_seqlens, causal, scale, gate, out):
    return None


# ---- Python entry points --------------------------------------------------------------------------------
def linear_i8(x, x_scale, weight, w_scale, bias=None, *, act="none", out_dtype=torch.float16):
    """``act(x_scale * w_scale * (x @ weight.T) + bias)`` on 8-bit integers -> [..., n] in ``out_dtype``.

    x int8 [..., k] with x_scale fp32 [...] (one scale a token), weight int8 [n, k] with w_scale fp32 [n] (one a channel;
    ``quantize_i8`` makes both pairs), bias fp32 [n] or None; act 'none', 'gelu' (erf), 'tanh' or 'relu'.  The sum is an
    exact 32-bit integer (k <= 131071), everything after it fp32, rounded once."""
    call = _linear_i8 if _eager("linear_i8", x, x_scale, weight, w_scale, bias) else torch.ops.sesa.linear_i8
    return call(x, x_scale, weight, w_scale, bias, act, out_dtype)


def norm_residual(x, residual=None, *, gate=None, gate_act="none", post="none", post_weight=None, post_bias=None,
                  scale=None, pre="rms", pre_weight=None, pre_bias=None, eps=1e-6):
    """``y = residual + scale * gate_act(gate) * post_norm(x)``, ``n = pre_norm(y)`` -> (y, n).

    x [..., dim] fp32 / fp16 / bf16 is a block's output, residual (same shape; x's type or fp32) the stream it joins: y
    comes in residual's type, n in x's.  gate: x's type and shape, with 1 in trailing dimensions before the last for a
    gate that many rows share ([groups, dim] for x [rows, dim]); gate_act 'none', 'sigmoid', 'silu' or 'tanh'.
    post / pre: 'none', 'rms' or 'layer' with fp32 [dim] weights (None: 1) and biases (None: 0), which 'none' does not use;
    scale fp32 [dim].
    Statistics are fp32; y and n are rounded once, n from the unrounded y."""
    eager = _eager("norm_residual", x, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias)
    call = _norm_residual if eager else torch.ops.sesa.norm_residual
    return call(x, residual, gate, gate_act, post, post_weight, post_bias, scale, pre, pre_weight, pre_bias, eps)


def norm_residual_i8(x, residual=None, *, gate=None, gate_act="none", post="none", post_weight=None, post_bias=None,
                     scale=None, pre="rms", pre_weight=None, pre_bias=None, eps=1e-6):
    """``norm_residual`` with n in 8 bits, one scale a row, for ``linear_i8`` -> (y, q int8, q_scale fp32 [...]).

    q_scale = max |n| / 127, q = round(n / q_scale) to even.  A row with nothing above 1.6e-36 has scale 0; a row that holds
    a NaN or an infinity has scale NaN and q 0, so a product with it is NaN in every channel."""
    eager = _eager("norm_residual_i8", x, residual, gate, post_weight, post_bias, scale, pre_weight, pre_bias)
    call = _norm_residual_i8 if eager else torch.ops.sesa.norm_residual_i8
    return call(x, residual, gate, gate_act, post, post_weight, post_bias, scale, pre, pre_weight, pre_bias, eps)


def quantize_i8(x):
    """Rows in 8 bits, one scale a row (``norm_residual_i8``'s rule, no norm): weights [n, k], activations [..., k]."""
    return (_quantize_i8 if _eager("quantize_i8", x) else torch.ops.sesa.quantize_i8)(x)


def rope_axes(q, k, positions, freqs, sections, *, layout="halves"):
    """Rotary positions with several axes on q [tokens, heads, head_dim] and k (same tokens; or None) -> (q', k') or q'.

    positions int32 / int64 [tokens, axes] (angles are off by at most |position| 2^-63 turns), sections the number of pairs
    each axis turns, freqs fp32 [sum(sections)] in radians per position, up to 2^40.  layout 'halves': pair i = elements
    (i, i + P), P = sum(sections); 'pairs': (2 i, 2 i + 1).  Elements behind the pairs pass through."""
    call = _rope_axes if _eager("rope_axes", q, k, positions, freqs) else torch.ops.sesa.rope_axes
    out = call([q] if k is None else [q, k], positions, freqs, sections, layout)
    return out[0] if k is None else (out[0], out[1])


def rope_axes_(q, k, positions, freqs, sections, *, layout="halves"):
    """``rope_axes`` in place on q and k (k may be None)."""
    eager = _eager("rope_axes_", q, k, positions, freqs)
    xs = [q] if k is None else [q, k]
    if not eager and not _compiling() and _tracing():   # (torch.jit drops an op that only writes a list of tensors)
        _rope_places(xs)
        for x, y in zip(xs, torch.ops.sesa.rope_axes(xs, positions, freqs, sections, layout)):
            x.copy_(y)
        return
    call = _rope_axes_ if eager else torch.ops.sesa.rope_axes_
    call(xs, positions, freqs, sections, layout)


def attention_packed(q, k, v, cu_seqlens=None, *, causal=True, scale=None, gate=None, out=None):
    """Softmax attention within each sequence of a packed run of tokens -> q's shape.

    q [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim] (heads a multiple of kv_heads; head_dim a multiple of
    8 up to 128), fp16 or bf16, any strides with a contiguous last dimension.  A fourth dimension [tokens, lanes, ...]
    runs that many columns of the same lengths side by side (a Roformer's bands in its time attention).
    cu_seqlens int32 [sequences + 1] on the device, non-decreasing: sequence s is tokens cu_seqlens[s] ..
    cu_seqlens[s + 1] - 1 (None: one sequence).  It is read by the kernel and held to the run there: a boundary outside
    is taken as the run's end, and boundaries out of order give unspecified rows, never an access outside.  gate: logits
    [tokens, (lanes,) heads], a sigmoid on each head's output.  scale: head_dim ** -0.5.  Rows of no sequence (behind the
    last) come back 0; with ``out`` they are left as they were.  Infinite or NaN values and scores beyond 2.9e6 give what
    the formula says (a key whose score is -inf: nothing), in about three times the time."""
    eager = _eager("attention_packed", q, k, v, cu_seqlens, gate, out)
    if out is None:
        call = _attention_packed if eager else torch.ops.sesa.attention_packed
        return call(q, k, v, cu_seqlens, causal, scale, gate)
    (_attention_packed_into if eager else torch.ops.sesa.attention_packed_into)(q, k, v, cu_seqlens, causal, scale, gate, out)
    return out
