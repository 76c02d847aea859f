"""The workloads of the DiT block's operators around its INT8 projections.

Three operators, each in its plain form (elementary torch operations in 32 bits) and as a
program calls it in this library:

  residual_norm   x' = rs x + gate * norm_post(branch), h = norm_pre(x') (1 + scale) + shift,
                  h stored or rotated and quantised to INT8 (the join between two projections)
  qk_norm_rope    per-head RMS norm and rotary positions over several axes, on q and k
  int4_linear     few rows times a 4-bit weight with group scales (modulation tables, the text
                  encoder's projections at few tokens)
"""
import math
import sys

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-6


def listed():
    return [
        # --- residual_norm -----------------------------------------------------------
        # one token of a text encoder (hidden 5120): latency only
        {"name": "norm_one_row", "op": "norm", "rows": 1, "width": 5120, "x": "bf16", "branch": "bf16",
         "post": "rms", "pre": "rms", "tables": 1, "quant": False, "rs": 1.0},
        # the join between attention output and FC1 of a DiT block at the bench's geometry
        {"name": "norm_dit_join", "op": "norm", "rows": 32768, "width": 3072, "x": "f16", "branch": "f16",
         "post": "rms", "pre": "rms", "tables": 9, "quant": True, "rs": 1.0},
        # the geometry of the published TP2 run (M = 6814, hidden 5376), LayerNorm model in bf16
        {"name": "norm_layer_6814", "op": "norm", "rows": 6814, "width": 5376, "x": "bf16", "branch": "bf16",
         "post": "none", "pre": "layer", "tables": 9, "quant": False, "rs": 1.0},
        # odd sizes: an fp32 residual stream of a width that is no multiple of anything
        {"name": "norm_odd_f32", "op": "norm", "rows": 1021, "width": 1001, "x": "f32", "branch": "f32",
         "post": "layer", "pre": "rms", "tables": 3, "quant": False, "rs": 0.5},
        # --- qk_norm_rope -----------------------------------------------------------
        # one token of a text encoder: grouped heads, halves paired, shared frequencies
        {"name": "rope_one_token", "op": "rope", "tokens": 1, "hq": 64, "hk": 8, "dim": 128, "x": "bf16",
         "pairing": "half", "axes": "48,40,40", "order": "interleaved", "freq": "shared", "norm": True,
         "pos": "i64"},
        # a DiT block's q and k at the bench's geometry: 24 heads of 128, time / height / width
        {"name": "rope_dit_video", "op": "rope", "tokens": 32768, "hq": 24, "hk": 24, "dim": 128, "x": "f16",
         "pairing": "interleaved", "axes": "32,48,48", "order": "chunked", "freq": "per_axis", "norm": True,
         "pos": "i32"},
        # one rank of the published TP2 run: 28 local heads, 6814 tokens
        {"name": "rope_tp2_6814", "op": "rope", "tokens": 6814, "hq": 28, "hk": 28, "dim": 128, "x": "bf16",
         "pairing": "interleaved", "axes": "16,56,56", "order": "chunked", "freq": "per_axis", "norm": True,
         "pos": "f32"},
        # a vision tower's heads: 72 wide, two axes, no norm, fp32, odd token count
        {"name": "rope_odd_f32", "op": "rope", "tokens": 1333, "hq": 7, "hk": 7, "dim": 72, "x": "f32",
         "pairing": "half", "axes": "36,36", "order": "chunked", "freq": "per_axis", "norm": False,
         "pos": "i32"},
        # --- int4_linear ------------------------------------------------------------
        # the timestep embedding's first projection: launch latency
        {"name": "int4_time_embed", "op": "int4", "rows": 1, "k": 256, "n": 5376, "x": "f16", "group": 32,
         "zeros": False, "scales": "f16", "bias": True, "out": "f16"},
        # the modulation tables of a block: 9 embedding rows, six vectors of the hidden width each
        {"name": "int4_modulation", "op": "int4", "rows": 9, "k": 5376, "n": 32256, "x": "f16", "group": 128,
         "zeros": False, "scales": "f32", "bias": True, "out": "f32"},
        # a text encoder's gate and up projections at one token
        {"name": "int4_decode_up", "op": "int4", "rows": 1, "k": 5120, "n": 25600, "x": "bf16", "group": 64,
         "zeros": True, "scales": "bf16", "bias": False, "out": "bf16"},
        # a text encoder's down projection for a short batch of tokens
        {"name": "int4_down_32", "op": "int4", "rows": 32, "k": 12800, "n": 5120, "x": "bf16", "group": 128,
         "zeros": True, "scales": "f16", "bias": False, "out": "bf16"},
    ]


def _span(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rope", "int4"])
    if op == "norm":
        quant = rng.random() < 0.4
        width = 256 * rng.randint(1, 28) if quant else _span(rng, 64, 8192)
        x = rng.choice(["f16", "bf16", "f32"])
        rows = _span(rng, 1, 32768)
        rows = max(1, min(rows, 32768 * 3072 // (width * (2 if x == "f32" else 1))))
        return {"op": "norm", "rows": rows, "width": width, "x": x,
                "branch": rng.choice([x, "f32"]) if rows * width < 2 ** 25 else x,
                "post": rng.choice(["none", "rms", "layer"]), "pre": rng.choice(["rms", "layer"]),
                "tables": rng.choice([1, 2, 9]), "quant": quant, "rs": rng.choice([1.0, 0.5])}
    if op == "rope":
        dim, axes = rng.choice([(64, "16,24,24"), (128, "32,48,48"), (128, "48,40,40"), (80, "40,40"),
                                (128, "128"), (256, "64,64,64"), (96, "16,32,32"), (72, "36,36")])
        hk = rng.choice([1, 2, 3, 4, 8, 24, 28])
        hq = hk * rng.choice([1, 1, 2, 4]) if hk <= 8 else hk
        x = rng.choice(["f16", "bf16", "f32"])
        tokens = _span(rng, 1, 65536)
        tokens = max(1, min(tokens, 32768 * 48 * 128 // ((hq + hk) * dim * (2 if x == "f32" else 1))))
        return {"op": "rope", "tokens": tokens, "hq": hq, "hk": hk, "dim": dim, "x": x,
                "pairing": rng.choice(["interleaved", "half"]), "axes": axes,
                "order": rng.choice(["chunked", "interleaved"]), "freq": rng.choice(["per_axis", "shared"]),
                "norm": rng.random() < 0.7, "pos": rng.choice(["i32", "i64", "f32"])}
    group = rng.choice([32, 64, 128])
    k = _span(rng, 128, 16384)
    n = _span(rng, 64, 32768)
    n = max(64, min(n, 32256 * 5376 // k))
    x = rng.choice(["f16", "bf16"])
    return {"op": "int4", "rows": _span(rng, 1, 32), "k": k, "n": n, "x": x, "group": group,
            "zeros": rng.random() < 0.5, "scales": rng.choice(["f16", "bf16", "f32"]),
            "bias": rng.random() < 0.5, "out": rng.choice([x, "f32"])}


# --------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------
def _labels(rows, tables, g, dev):
    """Segments of a packed sequence: `tables` runs of unequal length, in order."""
    if tables == 1:
        return torch.zeros(rows, dtype=torch.int32, device=dev)
    cuts = torch.sort(torch.randint(0, rows + 1, (tables - 1,), generator=g, device=dev)).values
    at = torch.arange(rows, device=dev)
    return torch.searchsorted(cuts, at, right=True).to(torch.int32)


def _axis_of_pairs(sections, order):
    """The axis of every rotated pair: runs in order, or dealt in turn while an axis has pairs left
    (then to the first that has)."""
    left = [d // 2 for d in sections]
    if order == "chunked":
        return [a for a, n in enumerate(left) for _ in range(n)]
    out = []
    for i in range(sum(left)):
        a = i % len(left)
        if left[a] == 0:
            a = next(j for j, n in enumerate(left) if n)
        left[a] -= 1
        out.append(a)
    return out


def _frequencies(sections, order, kind, theta=10000.0):
    axis = _axis_of_pairs(sections, order)
    if kind == "shared":
        total = sum(sections)
        return [theta ** (-2.0 * i / total) for i in range(len(axis))], axis
    seen, freq = [0] * len(sections), []
    for a in axis:
        freq.append(theta ** (-2.0 * seen[a] / sections[a]))
        seen[a] += 1
    return freq, axis


def _positions(tokens, n_axes, kind, g, dev):
    """A few text tokens (the same position on every axis) and then frames of a grid."""
    text = min(tokens, 77)
    at = torch.arange(tokens, device=dev)
    side = 52
    v = torch.clamp(at - text, min=0)
    grid = [v // (side * side), (v // side) % side, v % side, v % 7]
    start = torch.randint(0, 2048, (1,), generator=g, device=dev)
    pos = torch.stack([torch.where(at < text, at, text + grid[a]) for a in range(n_axes)], 1) + start
    if kind == "f32":
        pos = pos.float()
        pos[:, 0] *= 0.96  # frames at another rate than the model's
        return pos.contiguous()
    return pos.to(torch.int32 if kind == "i32" else torch.int64).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(dev)
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale + shift).to(dtype)

    s = dict(case)
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        # a residual stream and a projection's output: near normal, one column in a hundred large
        big = torch.where(torch.rand(width, generator=g, device=dev) < 0.01, 20.0, 1.0)
        s["xt"] = (normal(rows, width) * big).to(_DT[case["x"]])
        s["bt"] = normal(rows, width, scale=3.0).to(_DT[case["branch"]])
        s["labels"] = _labels(rows, case["tables"], g, dev)
        # the modulation: one table of six vectors a row, three of them read here
        mod = normal(case["tables"], 3 * width, scale=0.3)
        s["gate"], s["shift"], s["scale"] = mod[:, :width], mod[:, width:2 * width], mod[:, 2 * width:]
        s["w_post"], s["b_post"] = normal(width, scale=0.2, shift=1.0), normal(width, scale=0.1)
        s["w_pre"] = normal(width, scale=0.2, shift=1.0)
    elif case["op"] == "rope":
        tokens, hq, hk, dim = case["tokens"], case["hq"], case["hk"], case["dim"]
        # q and k are views of a packed projection output [q | k | v]
        qkv = normal(tokens, (hq + 2 * hk) * dim).to(_DT[case["x"]])
        s["q"] = qkv[:, :hq * dim].unflatten(1, (hq, dim))
        s["k"] = qkv[:, hq * dim:(hq + hk) * dim].unflatten(1, (hk, dim))
        sections = [int(v) for v in case["axes"].split(",")]
        s["sections"] = sections
        s["positions"] = _positions(tokens, len(sections), case["pos"], g, dev)
        s["w_q"], s["w_k"] = normal(dim, scale=0.2, shift=1.0), normal(dim, scale=0.2, shift=1.0)
        freq, axis = _frequencies(sections, case["order"], case["freq"])
        s["freq"] = torch.tensor(freq, dtype=torch.float64, device=dev)
        s["axis"] = torch.tensor(axis, device=dev)
        if own:
            _package()
            from h3tp.rms_rope import RotaryAxes
            s["plan"] = RotaryAxes(dim, sections, 10000.0, pairing=case["pairing"], order=case["order"],
                                   frequencies=case["freq"])
    else:
        rows, k, n, group = case["rows"], case["k"], case["n"], case["group"]
        groups = -(-k // group)
        s["xt"] = normal(rows, k).to(_DT[case["x"]])
        s["weight"] = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device=dev, dtype=torch.uint8)
        s["scales_t"] = (torch.rand(n, groups, generator=g, device=dev) * 0.01 + 0.002).to(_DT[case["scales"]])
        s["zeros_t"] = torch.randint(4, 12, (n, groups), generator=g, device=dev, dtype=torch.uint8) \
            if case["zeros"] else None
        s["bias_t"] = normal(n, scale=0.1) if case["bias"] else None
    return s


# --------------------------------------------------------------------------------------
# the operators
# --------------------------------------------------------------------------------------
def _package():
    if "minimax-h3-2xt4_b200" not in sys.path:
        sys.path.insert(0, "minimax-h3-2xt4_b200")


def _rotation(dev):
    """The regular 256-point rotation: the fourfold Kronecker power of the 4x4 matrix with -1 on its
    antidiagonal and 1 elsewhere, over 16."""
    h4 = torch.ones(4, 4, device=dev) - 2 * torch.eye(4, device=dev).flip(1)
    h16 = torch.kron(h4, h4)
    return torch.kron(h16, h16) / 16


def _norm(v, kind, weight, bias):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS)
    v = v * weight
    return v if bias is None else v + bias


def _plain_norm(s):
    x, b = s["xt"].float(), s["bt"].float()
    label = s["labels"].long()
    b = _norm(b, s["post"], s["w_post"], s["b_post"] if s["post"] == "layer" else None)
    x = x * s["rs"] + s["gate"][label] * b
    h = _norm(x, s["pre"], s["w_pre"], None)
    h = h * (1 + s["scale"][label]) + s["shift"][label]
    dtype = s["xt"].dtype
    if not s["quant"]:
        return x.to(dtype), h.to(dtype)
    h = (h.unflatten(1, (-1, 256)) @ _rotation(h.device)).flatten(1)
    step = torch.clamp(h.abs().amax(1, keepdim=True) * (1.0 / 127.0), min=1e-30)
    code = torch.clamp(torch.round(h / step), -128, 127)
    return x.to(dtype), (code * step).to(torch.float16), step


def _plain_rope_one(v, weight, s, cos, sin):
    v = v.float()
    if s["norm"]:
        v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS) * weight
    rot = 2 * cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    out = v.clone()
    if s["pairing"] == "half":
        a, b = v[..., :rot // 2], v[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = v[..., 0:rot:2], v[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    return out


def _plain_rope(s):
    # angles of far positions need 64 bits before the cosine, 32 after it
    angle = s["positions"].double()[:, s["axis"]] * s["freq"]
    cos, sin = angle.cos().float(), angle.sin().float()
    dtype = s["q"].dtype
    return (_plain_rope_one(s["q"], s["w_q"], s, cos, sin).to(dtype),
            _plain_rope_one(s["k"], s["w_k"], s, cos, sin).to(dtype))


def _plain_int4(s):
    k, group = s["k"], s["group"]
    w = s["weight"]
    code = torch.stack((w & 15, w >> 4), 2).flatten(1)[:, :k].float()
    zero = 8.0 if s["zeros_t"] is None else s["zeros_t"].float().repeat_interleave(group, 1)[:, :k]
    w = (code - zero) * s["scales_t"].float().repeat_interleave(group, 1)[:, :k]
    y = s["xt"].float() @ w.T
    if s["bias_t"] is not None:
        y = y + s["bias_t"]
    return y.to(_DT[s["out"]])


def _own_norm(s):
    from h3tp import ops
    post = None
    if s["post"] != "none":
        post = ops.NormSpec(s["post"], s["w_post"], s["b_post"] if s["post"] == "layer" else None, _EPS)
    pre = ops.NormSpec(s["pre"], s["w_pre"], None, _EPS)
    x, h, step = ops.residual_norm(s["xt"], s["bt"], s["gate"], s["labels"], post=post, pre=pre,
                                   shift=s["shift"], scale=s["scale"], residual_scale=s["rs"],
                                   out=torch.empty_like(s["xt"]), quantize=s["quant"])
    if not s["quant"]:
        return x, h
    value = torch.empty(h.shape, dtype=torch.float16, device=h.device)
    return x, torch.mul(h, step, out=value), step


def run(s):
    if not own:
        return {"norm": _plain_norm, "rope": _plain_rope, "int4": _plain_int4}[s["op"]](s)
    _package()
    from h3tp import ops
    if s["op"] == "norm":
        return _own_norm(s)
    if s["op"] == "rope":
        from h3tp.rms_rope import qk_norm_rope
        return qk_norm_rope(s["q"], s["k"], s["positions"], s["plan"], q_weight=s["w_q"], k_weight=s["w_k"],
                            eps=_EPS, norm=s["norm"])
    return ops.int4_linear(s["xt"], s["weight"], s["scales_t"], s["zeros_t"], group=s["group"],
                           bias=s["bias_t"], out_dtype=_DT[s["out"]])


# --------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------
def work(case):
    size = {"f16": 2, "bf16": 2, "f32": 4}
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        sx = size[case["x"]]
        # x and the branch in, x' and h out (the codes and, as values, their fp16 form once)
        moved = n * (2 * sx + size[case["branch"]] + (1 + 1 + 2 if case["quant"] else sx))
        flops = n * (12 + (6 if case["post"] != "none" else 0) + (20 if case["quant"] else 0))
        return {"bytes": moved + 4 * case["width"] * (3 * case["tables"] + 2) + 4 * case["rows"], "flops": flops}
    if case["op"] == "rope":
        n = case["tokens"] * (case["hq"] + case["hk"]) * case["dim"]
        axes = len(case["axes"].split(","))
        pos = {"i32": 4, "i64": 8, "f32": 4}[case["pos"]]
        return {"bytes": 2 * n * size[case["x"]] + case["tokens"] * axes * pos,
                "flops": n * (3 + (4 if case["norm"] else 0))}
    m, k, n = case["rows"], case["k"], case["n"]
    groups = -(-k // case["group"])
    moved = n * ((k + 1) // 2) + n * groups * (size[case["scales"]] + (1 if case["zeros"] else 0))
    moved += m * k * size[case["x"]] + m * n * size[case["out"]] + (4 * n if case["bias"] else 0)
    return {"bytes": moved, "flops": 2 * m * n * k}


# --------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "int4":
        k, group, n = case["k"], case["group"], case["n"]
        total = torch.zeros(case["rows"], n, dtype=f64, device="cuda")
        nibble = torch.empty(n, 2 * s["weight"].shape[1], dtype=f64, device="cuda")
        nibble[:, 0::2] = (s["weight"] % 16).to(f64)
        nibble[:, 1::2] = (s["weight"] // 16).to(f64)
        for at in range(0, k, group):  # the definition, group by group
            end = min(k, at + group)
            z = s["zeros_t"][:, at // group].to(f64)[:, None] if s["zeros_t"] is not None else 8.0
            part = torch.einsum("mk,nk->mn", s["xt"][:, at:end].to(f64), nibble[:, at:end] - z)
            total += part * s["scales_t"][:, at // group].to(f64)
        return total if s["bias_t"] is None else total + s["bias_t"].to(f64)
    if case["op"] == "rope":
        where = s["positions"].to(f64)
        outs = []
        half = sum(s["sections"]) // 2
        turn = torch.polar(torch.ones(case["tokens"], half, dtype=f64, device="cuda"),
                           torch.stack([where[:, a] * f for a, f in zip(s["axis"].tolist(), s["freq"].tolist())], 1))
        for t, w in ((s["q"], s["w_q"]), (s["k"], s["w_k"])):
            v = t.to(f64)
            if case["norm"]:
                v = v / torch.sqrt(v.square().sum(-1, keepdim=True) / case["dim"] + _EPS) * w.to(f64)
            if case["pairing"] == "half":
                first = torch.arange(half, device="cuda")
                second = first + half
            else:
                first = torch.arange(half, device="cuda") * 2
                second = first + 1
            z = torch.complex(v[..., first], v[..., second]) * turn[:, None, :]
            v = v.clone()
            v[..., first], v[..., second] = z.real, z.imag
            outs.append(v)
        return tuple(outs)

    def stat(v, kind, weight, bias):
        if kind == "none":
            return v
        width = v.shape[1]
        mean = v.sum(1) / width if kind == "layer" else torch.zeros(v.shape[0], dtype=f64, device="cuda")
        v = v - mean[:, None]
        dev = torch.sqrt(v.square().sum(1) / width + _EPS)
        v = v / dev[:, None] * weight.to(f64)[None]
        return v if bias is None else v + bias.to(f64)[None]

    xs, hs, steps = [], [], []
    h4 = [[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]]
    for at in range(0, case["rows"], 4096):
        rows = slice(at, at + 4096)
        lab = s["labels"][rows].long()
        b = stat(s["bt"][rows].to(f64), case["post"], s["w_post"], s["b_post"] if case["post"] == "layer" else None)
        x = case["rs"] * s["xt"][rows].to(f64) + torch.index_select(s["gate"], 0, lab).to(f64) * b
        h = stat(x, case["pre"], s["w_pre"], None)
        h = h + h * torch.index_select(s["scale"], 0, lab).to(f64) + torch.index_select(s["shift"], 0, lab).to(f64)
        if case["quant"]:
            m = torch.tensor(h4, dtype=f64, device="cuda") / 2
            h = h.reshape(h.shape[0], -1, 4, 4, 4, 4)
            h = torch.einsum("rgabcd,ai,bj,ck,dl->rgijkl", h, m, m, m, m).reshape(h.shape[0], -1)
            top = h.abs().max(1).values / 127
            step = torch.where(top > 1e-30, top, torch.full_like(top, 1e-30))[:, None]
            h = torch.round(h / step).clamp(-128, 127) * step
            steps.append(step)
        xs.append(x)
        hs.append(h)
    out = (torch.cat(xs), torch.cat(hs))
    return out + (torch.cat(steps),) if case["quant"] else out
