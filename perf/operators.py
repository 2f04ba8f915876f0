"""The transformer operators of ``sesa.ops`` as measured cases: what a pass reads, its plain form and its value in 64 bits.

Four operators, each reached through ``sesa.ops``:

* ``linear_i8``         out = act(x_scale[m] w_scale[n] sum_k x[m, k] w[n, k] + bias[n]), 8-bit integers, 32-bit sums;
* ``norm_residual``     y = residual + scale * gate_act(gate) * post_norm(x), n = pre_norm(y) (``norm_residual_i8``: n in
                        8 bits with one scale a row, the operand of ``linear_i8``);
* ``rope_axes``         rotary positions of several axes on q and k;
* ``attention_packed``  softmax(scale q k^T) v within each of a packed run of sequences, grouped heads.

``run`` computes them in elementary torch operations where ``own`` is false and calls ``sesa.ops`` where it is true.
"""
import math
import os
import sys

import torch

sys.path.insert(1, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sesa-audio-separation_amd"))

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one new token through a wide feed-forward Linear: the weights are read once, nothing else counts
        {"name": "linear one token", "op": "linear", "m": 1, "k": 4096, "n": 16384, "act": "none", "bias": False, "out": "bf16"},
        # a few packed clips through a layer of odd width (K not a multiple of 16, N odd), fp32 out for the next norm
        {"name": "linear odd sizes", "op": "linear", "m": 777, "k": 1000, "n": 1537, "act": "gelu", "bias": True, "out": "f32"},
        # a long batch through the widest Linear: one large product
        {"name": "linear large", "op": "linear", "m": 8192, "k": 4096, "n": 16384, "act": "none", "bias": False, "out": "bf16"},
        # the feed-forward entry of a Roformer layer on one chunk (801 frames x 62 bands, dim 512 -> 2048): the fp32
        # residual takes the attention's output, its RMSNorm leaves in 8 bits and meets the first Linear with its GELU
        {"name": "chunk feed-forward entry", "op": "entry", "m": 49662, "k": 512, "n": 2048, "act": "gelu", "out": "f16"},
        # one new token between two blocks
        {"name": "norm one token", "op": "norm", "m": 1, "d": 4096, "x": "bf16", "res": "bf16", "post": "rms", "pre": "rms", "gate": "none", "groups": 1},
        # LayerNorm before a block after a gated, layer-scaled residual, of odd width
        {"name": "norm odd width", "op": "norm", "m": 3001, "d": 1537, "x": "f16", "res": "f32", "post": "none", "pre": "layer", "gate": "sigmoid", "groups": 3001},
        # norms on both sides of a wide block, one gate row for each of eight clips
        {"name": "norm large", "op": "norm", "m": 16384, "d": 8192, "x": "bf16", "res": "bf16", "post": "rms", "pre": "rms", "gate": "tanh", "groups": 8},
        # sixteen short clips, causal: latency
        {"name": "attention short clips", "op": "attention", "t": 497, "seqs": 16, "lanes": 1, "hq": 8, "hk": 8, "d": 64, "causal": True, "gate": False, "x": "f16"},
        # a Roformer's time attention on two chunks: 801 frames each, the 62 bands side by side, a gate a head
        {"name": "attention over time", "op": "attention", "t": 1602, "seqs": 2, "lanes": 62, "hq": 8, "hk": 8, "d": 64, "causal": False, "gate": True, "x": "f16"},
        # a long causal batch of five sequences of different lengths, four query heads to a key head
        {"name": "attention long causal", "op": "attention", "t": 12289, "seqs": 5, "lanes": 1, "hq": 32, "hk": 8, "d": 128, "causal": True, "gate": False, "x": "bf16"},
        # a few new tokens on the (frame, band) grid
        {"name": "rope few tokens", "op": "rope", "t": 3, "hq": 8, "hk": 8, "d": 64, "axes": 2, "layout": "pairs", "far": 801, "x": "f16"},
        # a long run of tokens on a (time, height, width) grid, far positions
        {"name": "rope long grid", "op": "rope", "t": 24001, "hq": 32, "hk": 8, "d": 128, "axes": 3, "layout": "halves", "far": 1000000, "x": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "entry", "norm", "norm", "attention", "attention", "rope"])
    kind = rng.choice(["f16", "bf16"])
    if op == "linear":
        while True:
            m, k, n = _log(rng, 1, 8192), _log(rng, 64, 4096), _log(rng, 64, 16384)
            if rng.random() < 0.7:
                k = max(64, k // 16 * 16)
            if rng.random() < 0.5:
                n = max(64, n // 64 * 64)
            if 2.0 * m * k * n <= 2.0 * 8192 * 4096 * 16384:
                return {"op": op, "m": m, "k": k, "n": n, "act": rng.choice(["none", "gelu"]), "bias": rng.random() < 0.5, "out": rng.choice(["f16", "bf16", "f32"])}
    if op == "entry":
        return {"op": op, "m": _log(rng, 1, 49662), "k": rng.choice([192, 384, 512, 640, 1000, 1024]), "n": _log(rng, 64, 4096), "act": rng.choice(["none", "gelu"]), "out": kind}
    if op == "norm":
        d = _log(rng, 64, 8192)
        if rng.random() < 0.6:
            d = max(64, d // 8 * 8)
        groups = _log(rng, 1, 64)
        m = max(1, _log(rng, 1, 16384) // groups) * groups
        m = min(m, 16384 // groups * groups)
        gate = rng.choice(["none", "sigmoid", "silu", "tanh", "plain"])
        return {"op": op, "m": m, "d": d, "x": kind, "res": rng.choice([kind, "f32"]), "post": rng.choice(["none", "rms", "layer"]), "pre": rng.choice(["rms", "layer"]),
                "gate": gate, "groups": rng.choice([groups, m])}
    if op == "attention":
        hk, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 8])
        lanes = rng.choice([1, 1, 1, _log(rng, 1, 62)])
        t = _log(rng, 1, 12289)
        while lanes * hk * group * t * t > 32 * 12289 * 12289:
            t //= 2
        return {"op": op, "t": max(t, 1), "seqs": _log(rng, 1, 64), "lanes": lanes, "hq": hk * group, "hk": hk, "d": rng.choice([32, 48, 64, 80, 96, 128]),
                "causal": rng.random() < 0.6, "gate": rng.random() < 0.4, "x": kind}
    hk = rng.choice([1, 2, 8])
    return {"op": op, "t": _log(rng, 1, 24001), "hq": hk * rng.choice([1, 2, 4]), "hk": hk, "d": rng.choice([32, 48, 64, 96, 128]), "axes": rng.choice([1, 2, 3]),
            "layout": rng.choice(["pairs", "halves"]), "far": _log(rng, 64, 1000000), "x": kind}


def _sections(c):
    """The frequency pairs of each axis: all of them together cover the head."""
    p, a = c["d"] // 2, c["axes"]
    return [p - (a - 1) * (p // a)] + [p // a] * (a - 1)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")

    def normal(*shape, kind="f32", std=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(DT[kind])

    def rows_i8(v):
        s = v.abs().amax(-1) / 127.0
        return torch.round(v / s[..., None]).clamp(-127, 127).to(torch.int8), s

    c, s = case, {"case": case}
    if c["op"] in ("linear", "entry"):
        # activations with a few strong channels, as transformers have them, and weights of fan-in variance
        strong = 1.0 + 7.0 * (torch.rand(c["k"], generator=g, device=dev) < 0.02).float()
        s["w"], s["ws"] = rows_i8(normal(c["n"], c["k"], std=c["k"] ** -0.5))
    if c["op"] == "linear":
        s["x"], s["xs"] = rows_i8(normal(c["m"], c["k"]) * strong)
        s["bias"] = normal(c["n"], std=0.1) if c["bias"] else None
    elif c["op"] == "entry":
        s["x"] = normal(c["m"], c["k"], kind=c["out"], std=0.3)
        s["res"] = normal(c["m"], c["k"]) * strong
        s["pre_w"] = 1.0 + normal(c["k"], std=0.1)
        s["bias"] = normal(c["n"], std=0.1)
    elif c["op"] == "norm":
        s["x"] = normal(c["m"], c["d"], kind=c["x"], std=0.5)
        s["res"] = normal(c["m"], c["d"], kind=c["res"], std=2.0)
        s["scale"] = 0.1 + normal(c["d"], std=0.02)
        s["gate"] = normal(c["groups"], c["d"], kind=c["x"]) if c["gate"] != "none" else None
        s["post_w"] = 1.0 + normal(c["d"], std=0.1) if c["post"] != "none" else None
        s["post_b"] = normal(c["d"], std=0.1) if c["post"] == "layer" else None
        s["pre_w"] = 1.0 + normal(c["d"], std=0.1)
        s["pre_b"] = normal(c["d"], std=0.1) if c["pre"] == "layer" else None
    elif c["op"] == "attention":
        shape = (c["t"],) if c["lanes"] == 1 else (c["t"], c["lanes"])
        # q, k and v as one projection writes them: three column ranges of the same rows
        qkv = normal(*shape, (c["hq"] + 2 * c["hk"]), c["d"], kind=c["x"])
        s["q"], s["k"], s["v"] = qkv.split([c["hq"], c["hk"], c["hk"]], dim=-2)
        s["gate"] = normal(*shape, c["hq"], kind=c["x"]) if c["gate"] else None
        if c["seqs"] == 2 and not c["causal"]:
            cut = torch.tensor([c["t"] // 2], device=dev)
        else:  # anywhere, so that lengths differ (some may be empty)
            cut = torch.randint(0, c["t"] + 1, (c["seqs"] - 1,), generator=g, device=dev).sort().values
        s["cu"] = torch.cat([torch.zeros(1, device=dev), cut, torch.full((1,), c["t"], device=dev)]).to(torch.int32)
    else:
        s["q"] = normal(c["t"], c["hq"], c["d"], kind=c["x"])
        s["k"] = normal(c["t"], c["hk"], c["d"], kind=c["x"])
        s["pos"] = torch.randint(0, c["far"], (c["t"], c["axes"]), generator=g, device=dev, dtype=torch.int32)
        s["freqs"] = torch.cat([10000.0 ** (-torch.arange(p, device=dev, dtype=torch.float32) / max(p, 1)) for p in _sections(c)])
    return s


def _act(v, act):
    return 0.5 * v * (1.0 + torch.erf(v * 0.5 ** 0.5)) if act == "gelu" else v


def _gate(g, act):
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-g))
    if act == "silu":
        return g / (1.0 + torch.exp(-g))
    if act == "tanh":
        return torch.tanh(g)
    return g


def _norm(v, kind, w, b, eps=1e-6):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * w
    return v + b if b is not None else v


def _plain(s):
    c = s["case"]
    if c["op"] == "linear":
        acc = s["x"].float() @ s["w"].float().t()
        v = acc * s["xs"][:, None] * s["ws"]
        if s["bias"] is not None:
            v = v + s["bias"]
        return _act(v, c["act"]).to(DT[c["out"]])
    if c["op"] == "entry":
        y = s["res"] + s["x"].float()
        n = _norm(y, "rms", s["pre_w"], None)
        ns = n.abs().amax(-1, keepdim=True) / 127.0
        q = torch.round(n / ns)
        v = (q @ s["w"].float().t()) * ns * s["ws"] + s["bias"]
        return y, _act(v, c["act"]).to(DT[c["out"]])
    if c["op"] == "norm":
        p = s["x"].float()
        if c["post"] != "none":
            p = _norm(p, c["post"], s["post_w"], s["post_b"])
        p = p * s["scale"]
        if s["gate"] is not None:
            gate = _gate(s["gate"].float(), c["gate"])
            p = (p.view(c["groups"], -1, c["d"]) * gate[:, None]).view(c["m"], c["d"])
        y = s["res"].float() + p
        n = _norm(y, c["pre"], s["pre_w"], s["pre_b"])
        return y.to(s["res"].dtype), n.to(s["x"].dtype)
    if c["op"] == "attention":
        t, lanes, hk = c["t"], c["lanes"], c["hk"]
        group, d = c["hq"] // hk, c["d"]
        at = torch.arange(t, device=s["q"].device)
        seq = torch.searchsorted(s["cu"][1:].long(), at, right=True)
        keep = seq[:, None] == seq[None, :]
        if c["causal"]:
            keep = keep & (at[:, None] >= at[None, :])
        q = s["q"].float().view(t, lanes, hk, group, d).permute(1, 2, 3, 0, 4).reshape(lanes * hk, group * t, d)
        k = s["k"].float().view(t, lanes, hk, d).permute(1, 2, 3, 0).reshape(lanes * hk, d, t).contiguous()
        v = s["v"].float().view(t, lanes, hk, d).permute(1, 2, 0, 3).reshape(lanes * hk, t, d).contiguous()
        sc = (torch.matmul(q, k) * d ** -0.5).view(lanes * hk, group, t, t).masked_fill_(~keep, -math.inf)
        p = torch.exp_(sc.sub_(sc.amax(-1, keepdim=True)))
        o = torch.matmul(p.view(lanes * hk, group * t, t), v).view(lanes * hk, group, t, d) / p.sum(-1, keepdim=True)
        o = o.view(lanes, hk, group, t, d).permute(3, 0, 1, 2, 4).reshape(s["q"].shape)
        if s["gate"] is not None:
            o = o * _gate(s["gate"].float(), "sigmoid")[..., None]
        return o.to(s["q"].dtype)
    ang = torch.cat([s["pos"][:, a:a + 1].double() * f for a, f in enumerate(s["freqs"].double().split(_sections(c)))], -1)
    cos, sin = torch.cos(ang).float()[:, None], torch.sin(ang).float()[:, None]

    def turned(x):
        x = x.float()
        a, b = (x[..., 0::2], x[..., 1::2]) if c["layout"] == "pairs" else x.chunk(2, -1)
        u, v = a * cos - b * sin, a * sin + b * cos
        return torch.stack([u, v], -1).flatten(-2) if c["layout"] == "pairs" else torch.cat([u, v], -1)

    return turned(s["q"]).to(s["q"].dtype), turned(s["k"]).to(s["k"].dtype)


def _own(s):
    from sesa import ops

    c = s["case"]
    if c["op"] == "linear":
        return ops.linear_i8(s["x"], s["xs"], s["w"], s["ws"], s["bias"], act=c["act"], out_dtype=DT[c["out"]])
    if c["op"] == "entry":
        y, q, qs = ops.norm_residual_i8(s["x"], s["res"], pre_weight=s["pre_w"])
        return y, ops.linear_i8(q, qs, s["w"], s["ws"], s["bias"], act=c["act"], out_dtype=DT[c["out"]])
    if c["op"] == "norm":
        return ops.norm_residual(s["x"], s["res"], post=c["post"], post_weight=s["post_w"], post_bias=s["post_b"], scale=s["scale"], gate=s["gate"],
                                 gate_act="none" if c["gate"] == "plain" else c["gate"], pre=c["pre"], pre_weight=s["pre_w"], pre_bias=s["pre_b"])
    if c["op"] == "attention":
        return ops.attention_packed(s["q"], s["k"], s["v"], s["cu"], causal=c["causal"], gate=s["gate"])
    return ops.rope_axes(s["q"], s["k"], s["pos"], s["freqs"], _sections(c), layout=c["layout"])


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if c["op"] == "linear":
        return {"bytes": c["m"] * c["k"] + c["n"] * c["k"] + 4 * (c["m"] + c["n"] * (2 if c["bias"] else 1)) + c["m"] * c["n"] * size[c["out"]], "flops": 2.0 * c["m"] * c["n"] * c["k"]}
    if c["op"] == "entry":
        return {"bytes": c["m"] * c["k"] * (size[c["out"]] + 8) + c["n"] * c["k"] + 8 * c["n"] + 4 * c["k"] + c["m"] * c["n"] * size[c["out"]], "flops": 2.0 * c["m"] * c["n"] * c["k"] + 10.0 * c["m"] * c["k"]}
    if c["op"] == "norm":
        gate = c["groups"] * c["d"] * size[c["x"]] if c["gate"] != "none" else 0
        params = 2 + (c["post"] != "none") + (c["post"] == "layer") + (c["pre"] == "layer")
        return {"bytes": c["m"] * c["d"] * 2 * (size[c["x"]] + size[c["res"]]) + gate + 4 * params * c["d"], "flops": 15.0 * c["m"] * c["d"]}
    if c["op"] == "attention":
        # scores of the sequences' own pairs; where the cuts fall is the seed's: the mean over uniform cuts
        n, t = c["seqs"], c["t"]
        pairs = t * t / 2.0 if n == 2 and not c["causal"] else 2.0 * t * t / (n + 1.0)
        pairs = max(float(t), pairs / 2.0 if c["causal"] else pairs)
        rows = t * c["lanes"]
        return {"bytes": rows * 2 * (c["d"] * (2 * c["hq"] + 2 * c["hk"]) + (c["hq"] if c["gate"] else 0)) + 4 * (n + 1), "flops": 4.0 * pairs * c["lanes"] * c["hq"] * c["d"]}
    return {"bytes": c["t"] * (4 * c["d"] * (c["hq"] + c["hk"]) + 4 * c["axes"]) + 2 * c["d"], "flops": 3.0 * c["t"] * (c["hq"] + c["hk"]) * c["d"]}


def exact(case, seed):
    c, s = case, prepare(case, seed)
    s = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}

    def normed(v, kind, w, b):
        mean = v.sum(-1, keepdim=True) / v.shape[-1] if kind == "layer" else 0.0
        var = ((v - mean) ** 2).sum(-1, keepdim=True) / v.shape[-1]
        return (v - mean) / torch.sqrt(var + 1e-6) * w + (0.0 if b is None else b)

    def activated(v):
        return v * 0.5 * torch.erfc(-v / math.sqrt(2.0)) if c["act"] == "gelu" else v

    if c["op"] == "linear":
        out = torch.mm(s["x"] * s["xs"][:, None], (s["w"] * s["ws"][:, None]).t().contiguous())
        return activated(out if s["bias"] is None else out + s["bias"])
    if c["op"] == "entry":
        y = s["x"] + s["res"]
        n = normed(y, "rms", s["pre_w"], None)
        step = n.abs().max(-1, keepdim=True).values / 127.0
        n = torch.round(n / step) * step
        return y, activated(torch.mm(n, (s["w"] * s["ws"][:, None]).t().contiguous()) + s["bias"])
    if c["op"] == "norm":
        p = s["x"] if c["post"] == "none" else normed(s["x"], c["post"], s["post_w"], s["post_b"])
        if s["gate"] is not None:
            g = s["gate"].repeat_interleave(c["m"] // c["groups"], 0)
            p = p * {"sigmoid": torch.sigmoid(g), "silu": g * torch.sigmoid(g), "tanh": torch.tanh(g), "plain": g}[c["gate"]]
        y = s["res"] + s["scale"] * p
        return y, normed(y, c["pre"], s["pre_w"], s["pre_b"])
    if c["op"] == "attention":
        t, group = c["t"], c["hq"] // c["hk"]
        q, k, v = (x.reshape(t, c["lanes"], -1, c["d"]).transpose(0, 2) for x in (s["q"], s["k"], s["v"]))  # [heads, lanes, tokens, d]
        out = torch.zeros_like(q)
        cu = [int(x) for x in s["cu"]]
        for a, b in zip(cu[:-1], cu[1:]):
            for h in range(c["hq"] if b > a else 0):
                logits = torch.matmul(q[h, :, a:b], k[h // group, :, a:b].transpose(-1, -2).contiguous()) / math.sqrt(c["d"])
                if c["causal"]:
                    logits = logits + torch.full((b - a, b - a), -math.inf, dtype=torch.float64, device=q.device).triu(1)
                w = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
                out[h, :, a:b] = torch.matmul(w, v[h // group, :, a:b].contiguous())
        out = out.transpose(0, 2).reshape(s["q"].shape)
        return out if s["gate"] is None else out * torch.sigmoid(s["gate"])[..., None]
    first = [sum(_sections(c)[:a]) for a in range(c["axes"] + 1)]
    turn = torch.cat([torch.polar(torch.ones_like(s["pos"][:, a:a + 1] * s["freqs"][first[a]:first[a + 1]]), s["pos"][:, a:a + 1] * s["freqs"][first[a]:first[a + 1]])
                      for a in range(c["axes"])], -1)[:, None]

    def spun(x):
        if c["layout"] == "pairs":
            z = torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous()) * turn
            return torch.view_as_real(z).reshape(x.shape)
        h = c["d"] // 2
        z = torch.complex(x[..., :h].contiguous(), x[..., h:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    return spun(s["q"]), spun(s["k"])
