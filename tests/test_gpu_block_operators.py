"""GPU parity of the operators around a block's projections (residual_norm, qk_norm_rope,
int4_linear) against their definitions in 64 bits.

Tolerances.  Every output is rounded once to its type, which moves it by at most half a
step: eps / 2 of the type, relative.  Before that all values are fp32; an fp32 result that
went through d dependent roundings is off by at most about d * 2^-24 times the sum of the
magnitudes that were added to form it (not of the result, which may have cancelled).  Each
check states that sum (`mag`) and a depth d for the longest chain of the kernel: a thread's
own additions, the tree over lanes and warps, and the operations after it.  Below the
smallest normal number of the type the step is fixed: eps * smallest normal is allowed too."""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
U = 2.0 ** -24


def _gen(seed):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _close(got, ref, mag, depth):
    """got (of a float type) is ref rounded once, plus depth roundings of fp32 against mag."""
    info = torch.finfo(got.dtype)
    tol = ref.abs() * (info.eps / 2) + depth * U * mag + info.eps * info.tiny
    err = (got.double() - ref).abs()
    assert got.shape == ref.shape
    assert torch.isfinite(got).all()
    bad = err > tol
    assert not bad.any(), (int(bad.sum()), float((err / tol.clamp(min=1e-300)).max()))


# --------------------------------------------------------------------------------------
# residual_norm
# --------------------------------------------------------------------------------------
def _stat(v, mag, spec):
    """norm of v (64 bits) and the magnitudes behind each of its values."""
    if spec is None:
        return v, mag
    mean = v.mean(1, keepdim=True) if spec.kind == "layer" else torch.zeros_like(v[:, :1])
    d = v - mean
    dev = (d.square().mean(1, keepdim=True) + spec.eps).sqrt()
    y = d / dev
    # an error in the values moves the mean and the deviation as their mean magnitude does
    rel = (mag + mag.mean(1, keepdim=True)) / dev + y.abs() * (mag.square().mean(1, keepdim=True).sqrt() / dev)
    for name, op in (("weight", torch.mul), ("bias", torch.add)):
        t = getattr(spec, name)
        if t is not None:
            y = op(y, t.double())
            rel = rel * t.double().abs() if name == "weight" else rel + t.double().abs()
    return y, rel


H4 = [[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]]


def _rotate(v, absolute=False):
    m = torch.tensor(H4, dtype=torch.float64, device=v.device) / 2
    if absolute:
        m = m.abs()
    v4 = v.reshape(v.shape[0], -1, 4, 4, 4, 4)
    return torch.einsum("rgabcd,ai,bj,ck,dl->rgijkl", v4, m, m, m, m).reshape(v.shape)


def _norm_ref(x, branch, gate, labels, post, pre, shift, scale, rs):
    x = x.double()
    lab = torch.zeros(x.shape[0], dtype=torch.long, device="cuda") if labels is None else labels.long()
    mag = x.abs()
    if branch is not None:
        b, bmag = _stat(branch.double(), branch.double().abs(), post)
        g = torch.ones_like(b) if gate is None else gate.double()[lab]
        x, mag = rs * x + g * b, abs(rs) * mag + g.abs() * bmag
    if pre is None:
        return x, mag, None, None
    h, hmag = _stat(x, mag, pre)
    if scale is not None:
        f = 1 + scale.double()[lab]
        h, hmag = h * f, hmag * (1 + scale.double()[lab].abs())
    if shift is not None:
        h, hmag = h + shift.double()[lab], hmag + shift.double()[lab].abs()
    return x, mag, h, hmag


def _depth(width):
    # a thread adds at most width / 128 + 8 values of its own, then lanes (5), warps (32)
    # and about 20 operations of the formula
    return width / 128 + 8 + 5 + 32 + 20


def _norm_case(g, rows, width, xt, bt, tables):
    x = (_randn(g, rows, width) * 2).to(DT[xt])
    b = (_randn(g, rows, width) * 3).to(DT[bt])
    mod = _randn(g, tables, 3 * width + 1) * 0.4
    lab = torch.randint(0, tables, (rows,), generator=g, device="cuda", dtype=torch.int32)
    gate, shift, scale = mod[:, 1:width + 1], mod[:, width + 1:2 * width + 1], mod[:, 2 * width + 1:]
    return x, b, gate, shift, scale, lab


WIDTHS = [1, 2, 7, 8, 31, 32, 33, 96, 255, 256, 264, 1000, 1001, 1024, 2048, 2056, 4104, 5376, 8192, 8200,
          20000, 32767, 32768]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("xt,bt", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
def test_residual_norm_widths(cuda_device, width, xt, bt):
    from h3tp import ops
    g = _gen(width)
    rows = 5
    x, b, gate, shift, scale, lab = _norm_case(g, rows, width, xt, bt, 3)
    w1, b1, w2, b2 = (_randn(g, width) for _ in range(4))
    kinds = ("rms", "layer") if width > 2 else ("rms", "rms")  # a layer norm of one value divides noise
    post = ops.NormSpec(kinds[width % 2], w1, b1, 1e-5)
    pre = ops.NormSpec(kinds[1 - width % 2], w2, b2, 1e-6)
    want = _norm_ref(x, b, gate, lab, post, pre, shift, scale, 0.75)
    keep = x.clone()
    y, h, s = ops.residual_norm(x, b, gate, lab, post=post, pre=pre, shift=shift, scale=scale,
                                residual_scale=0.75, out=torch.empty_like(x))
    assert s is None and torch.equal(x, keep)
    _close(y, want[0], want[1], _depth(width))
    _close(h, want[2], want[3], 2 * _depth(width))
    z, h2, _ = ops.residual_norm(x, b, gate, lab, post=post, pre=pre, shift=shift, scale=scale,
                                 residual_scale=0.75)
    assert z is x and torch.equal(x, y) and torch.equal(h2, h)  # in place: the same bits


FORMS = [(post, pre, gate, mod) for post, pre, gate, mod in itertools.product(
    [None, "rms", "layer"], [None, "rms", "layer"], [False, True], ["none", "shift", "scale", "both"])
    if pre is not None or mod == "none"]  # the tables belong to the pre-norm


@pytest.mark.parametrize("post,pre,gate,mod", FORMS)
def test_residual_norm_forms(cuda_device, post, pre, gate, mod):
    from h3tp import ops
    g = _gen(7)
    width = 520
    x, b, gt, shift, scale, lab = _norm_case(g, 37, width, "bf16", "bf16", 4)
    gt = gt if gate else None
    shift = shift if mod in ("shift", "both") else None
    scale = scale if mod in ("scale", "both") else None
    lab = lab if any(t is not None for t in (gt, shift, scale)) else None
    ps = None if post is None else ops.NormSpec(post, _randn(g, width), None, 1e-6)
    ns = None if pre is None else ops.NormSpec(pre, None, _randn(g, width), 1e-6)
    want = _norm_ref(x, b, gt, lab, ps, ns, shift, scale, 1.0)
    y, h, _ = ops.residual_norm(x.clone(), b, gt, lab, post=ps, pre=ns, shift=shift, scale=scale)
    _close(y, want[0], want[1], _depth(width))
    if pre is None:
        assert h is None
    else:
        _close(h, want[2], want[3], 2 * _depth(width))


@pytest.mark.parametrize("width,convrot", [(w, False) for w in (16, 17, 256, 272, 1001, 4096, 32768)]
                         + [(w, True) for w in (256, 768, 1280, 4096, 5376, 8192, 8448, 16384, 32768)])
@pytest.mark.parametrize("xt", ["f16", "bf16", "f32"])
def test_residual_norm_quantized(cuda_device, width, convrot, xt):
    """Each code times its scale is within half a step of the exact value (plus the fp32
    error of that value), and the scale is the exact row maximum over 127."""
    from h3tp import ops
    g = _gen(width + 1)
    x, b, gate, shift, scale, lab = _norm_case(g, 9, width, xt, xt, 2)
    x[:, ::97] *= 20
    post, pre = ops.NormSpec("rms", _randn(g, width)), ops.NormSpec("layer")
    _, _, h, mag = _norm_ref(x, b, gate, lab, post, pre, shift, scale, 1.0)
    if convrot:
        h, mag = _rotate(h), _rotate(mag, absolute=True)
    y, q, s = ops.residual_norm(x, b, gate, lab, post=post, pre=pre, shift=shift, scale=scale,
                                quantize=True, convrot=convrot)
    err = (2 * _depth(width) + 16) * U * mag
    assert q.dtype == torch.int8 and s.shape == (9, 1)
    top = h.abs().amax(1, keepdim=True) / 127
    assert ((s.double() - top).abs() <= err.amax(1, keepdim=True) / 127 + 4 * U * top).all()
    step = s.double()
    off = (q.double() * step - h).abs()
    assert (off <= step * (0.5 + 128 * 4 * U) + err).all(), float((off / step).max())
    assert (q.double().abs().amax(1) == 127).all()


def test_residual_norm_without_branch_is_the_pre_norm(cuda_device):
    from h3tp import ops
    g = _gen(3)
    x, _, _, shift, scale, lab = _norm_case(g, 19, 768, "f16", "f16", 3)
    pre = ops.NormSpec("rms", _randn(g, 768), None, 1e-6)
    keep = x.clone()
    y, h, _ = ops.residual_norm(x, labels=lab, pre=pre, shift=shift, scale=scale)
    assert y is x and torch.equal(x, keep)
    want = _norm_ref(x, None, None, lab, None, pre, shift, scale, 1.0)
    _close(h, want[2], want[3], _depth(768))
    # the existing fp16 producer computes the same norm: one rounding apart at most
    _, _, old = ops.modulated_norm_quantize(x, pre.weight, pre.eps, shift.contiguous(), scale.contiguous(),
                                            lab, quantize=False)
    _close(old, want[2], want[3], 2 * _depth(768))


@pytest.mark.parametrize("rows", [0, 1, 2, 147, 149, 1025, 4099])
def test_residual_norm_rows_are_independent(cuda_device, rows):
    """A row's bits do not depend on the rows around it; rows of one label or of many."""
    from h3tp import ops
    g = _gen(11)
    x, b, gate, shift, scale, lab = _norm_case(g, 4099, 768, "f16", "f16", 5)
    post, pre = ops.NormSpec("rms"), ops.NormSpec("rms")
    kw = dict(post=post, pre=pre, shift=shift, scale=scale)
    full = ops.residual_norm(x.clone(), b, gate, lab, **kw)
    part = ops.residual_norm(x[:rows].clone(), b[:rows], gate, lab[:rows], **kw)
    assert torch.equal(part[0], full[0][:rows]) and torch.equal(part[1], full[1][:rows])
    qfull = ops.residual_norm(x.clone(), b, gate, lab, quantize=True, **kw)
    qpart = ops.residual_norm(x[:rows].clone(), b[:rows], gate, lab[:rows], quantize=True, **kw)
    assert torch.equal(qpart[1], qfull[1][:rows]) and torch.equal(qpart[2], qfull[2][:rows])


def test_residual_norm_unaligned_rows(cuda_device):
    """Tensors that start off a 16-byte boundary give the bits of aligned ones."""
    from h3tp import ops
    g = _gen(12)
    rows, width = 7, 512
    x, b, gate, shift, scale, lab = _norm_case(g, rows, width, "f16", "f16", 2)

    def moved(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    w = _randn(g, width)
    kw = dict(labels=lab, shift=shift, scale=scale)
    want = ops.residual_norm(x.clone(), b, gate, pre=ops.NormSpec("rms", w), post=ops.NormSpec("layer", w), **kw)
    got = ops.residual_norm(moved(x), moved(b), gate, pre=ops.NormSpec("rms", moved(w)),
                            post=ops.NormSpec("layer", moved(w)), **kw)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    want = ops.residual_norm(x.clone(), b, gate, pre=ops.NormSpec("rms", w), quantize=True, **kw)
    got = ops.residual_norm(moved(x), moved(b), gate, pre=ops.NormSpec("rms", w), quantize=True, **kw)
    assert torch.equal(want[1], got[1]) and torch.equal(want[2], got[2])


def test_residual_norm_special_values(cuda_device):
    """Rows of zeros, infinities and NaN stay in their rows."""
    from h3tp import ops
    width = 512
    x = torch.ones(6, width, dtype=torch.float16, device="cuda")
    b = torch.ones_like(x)
    x[1], b[1] = 0, 0
    x[2, 5] = float("inf")
    b[3, 7] = float("nan")
    x[4], b[4] = 60000, 60000  # x' overflows fp16, its norm does not
    _, h, _ = ops.residual_norm(x.clone(), b, pre=ops.NormSpec("rms", eps=1e-6))
    y, q, s = ops.residual_norm(x.clone(), b, pre=ops.NormSpec("rms", eps=1e-6), quantize=True)
    assert torch.equal(h[0], torch.ones_like(h[0])) and torch.equal(h[5], h[0])
    assert (h[1] == 0).all() and (q[1] == 0).all() and s[1, 0] == torch.tensor(1e-30)
    assert torch.isnan(h[2, 5]) and torch.isnan(h[3]).all()
    assert torch.isinf(y[4]).all() and torch.equal(h[4], h[0])
    assert torch.isfinite(s).all()


def test_residual_norm_label_out_of_range(cuda_device):
    from h3tp import _native, ops
    x = torch.ones(4, 256, dtype=torch.float16, device="cuda")
    table = torch.tensor([[0.0], [1.0]], device="cuda").expand(2, 256).contiguous()
    assert _native.device_error(0) == 0
    lab = torch.tensor([0, 1, 7, -1], dtype=torch.int32, device="cuda")
    _, h, _ = ops.residual_norm(x, labels=lab, pre=ops.NormSpec("rms", eps=0.0), shift=table)
    assert h[:, 0].tolist() == [1.0, 2.0, 1.0, 1.0]
    assert _native.device_error(0) == _native.H3_ERR_INVALID
    assert _native.device_error(0) == 0


# --------------------------------------------------------------------------------------
# qk_norm_rope
# --------------------------------------------------------------------------------------
def _rope_ref(x, w, pos, plan, norm, eps):
    """The turned heads in 64 bits and the magnitudes behind each value."""
    v = x.double()
    if norm:
        v = v / (v.square().mean(-1, keepdim=True) + eps).sqrt()
        if w is not None:
            v = v * w.double()
    f = torch.tensor(plan.inv_freq, dtype=torch.float64, device="cuda")
    ax = torch.tensor(plan.axis_of_pair, device="cuda")
    ang = pos.double().reshape(x.shape[0], plan.n_axes)[:, ax] * f
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    n = plan.pairs
    i = torch.arange(n, device="cuda") if plan.half else torch.arange(n, device="cuda") * 2
    j = i + n if plan.half else i + 1
    out, mag = v.clone(), v.abs()
    a, b = v[..., i], v[..., j]
    out[..., i], out[..., j] = a * c - b * s, b * c + a * s
    mag[..., i] = mag[..., j] = a.abs() + b.abs()
    return out, mag


ROPE_DEPTH = 8 + 8 + 5 + 20  # a lane's squares, the tree, the formula with its sine and cosine

PLANS = [
    (128, (32, 48, 48), dict()),
    (128, (48, 40, 40), dict(pairing="half", order="interleaved", frequencies="shared")),
    (64, (16, 24, 24), dict(pairing="half")),
    (80, (40, 40), dict(pairing="half")),
    (72, (36, 36), dict(pairing="half")),
    (96, (16, 32, 32), dict()),
    (256, (64, 64, 64), dict(pairing="half")),
    (256, (256,), dict()),
    (248, (2, 4, 240), dict()),
    (10, (4, 2), dict(pairing="half")),
    (33, (8, 6, 10), dict(pairing="half", order="interleaved")),
    (33, (8, 6, 10), dict()),
    (2, (2,), dict()),
    (127, (0, 64), dict(order="interleaved")),
    (120, (20, 20, 20, 20, 20), dict(theta=(100.0, 1e4, 1e4, 1e6, 5e5))),
]


def _positions(g, tokens, axes, kind, far=4096):
    p = torch.randint(-5, far, (tokens, axes), generator=g, device="cuda")
    if kind == "f32":
        return p.float() + 0.37
    return p.to(torch.int32 if kind == "i32" else torch.int64)


@pytest.mark.parametrize("plan", PLANS, ids=[str(p[:2]) for p in PLANS])
@pytest.mark.parametrize("xt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("norm", [True, False])
def test_qk_norm_rope_plans(cuda_device, plan, xt, norm):
    from h3tp.rms_rope import RotaryAxes, qk_norm_rope
    dim, sections, kw = plan
    axes = RotaryAxes(dim, sections, **kw)
    g = _gen(dim)
    q = _randn(g, 13, 5, dim).to(DT[xt])
    k = _randn(g, 13, 2, dim).to(DT[xt])
    wq, wk = _randn(g, dim), _randn(g, dim)
    for kind in ("i32", "i64", "f32"):
        pos = _positions(g, 13, len(sections), kind)
        oq, ok = qk_norm_rope(q, k, pos, axes, q_weight=wq, k_weight=wk, eps=1e-5, norm=norm)
        for got, src, w in ((oq, q, wq), (ok, k, wk)):
            ref, mag = _rope_ref(src, w, pos, axes, norm, 1e-5)
            _close(got, ref, mag, ROPE_DEPTH)


@pytest.mark.parametrize("tokens,hq,hk", [(0, 2, 1), (1, 1, 0), (1, 64, 8), (2, 3, 3), (5, 40, 1), (147, 7, 7),
                                          (149, 24, 24), (1000, 1, 1), (4099, 2, 2)])
@pytest.mark.parametrize("half", [False, True])
def test_qk_norm_rope_sizes(cuda_device, tokens, hq, hk, half):
    from h3tp.rms_rope import RotaryAxes, qk_norm_rope
    axes = RotaryAxes(128, (16, 56, 56), pairing="half" if half else "interleaved")
    g = _gen(tokens)
    q = _randn(g, tokens, hq, 128).half()
    k = _randn(g, tokens, hk, 128).half() if hk else None
    pos = _positions(g, tokens, 3, "i32")
    w = _randn(g, 128)
    oq, ok = qk_norm_rope(q, k, pos, axes, q_weight=w)
    _close(oq, *_rope_ref(q, w, pos, axes, True, 1e-6), ROPE_DEPTH)
    if hk:
        _close(ok, *_rope_ref(k, None, pos, axes, True, 1e-6), ROPE_DEPTH)
    else:
        assert ok is None


@pytest.mark.parametrize("xt", ["f16", "f32"])
def test_qk_norm_rope_strides(cuda_device, xt):
    """Packed rows in place, head-major outputs, rows off a 16-byte boundary and rows of a
    wider tensor: the bits of contiguous tensors."""
    from h3tp.rms_rope import RotaryAxes, packed_qk_norm_rope, qk_norm_rope
    axes = RotaryAxes(64, (16, 24, 24), pairing="half")
    g = _gen(5)
    S, H, K, D = 70, 6, 2, 64
    qkv = _randn(g, S, (H + 2 * K) * D).to(DT[xt])
    q, k = qkv[:, :H * D].reshape(S, H, D), qkv[:, H * D:(H + K) * D].reshape(S, K, D)
    pos = _positions(g, S, 3, "i64")
    w = _randn(g, D)
    wq, wk = qk_norm_rope(q.contiguous(), k.contiguous(), pos, axes, q_weight=w, k_weight=w)
    _close(wq, *_rope_ref(q, w, pos, axes, True, 1e-6), ROPE_DEPTH)

    packed = qkv.clone()
    pq, pk, pv = packed_qk_norm_rope(packed, H, K, pos, axes, q_weight=w, k_weight=w)
    assert pq.data_ptr() == packed.data_ptr()
    assert torch.equal(pq, wq) and torch.equal(pk, wk)
    assert torch.equal(packed[:, (H + K) * D:], qkv[:, (H + K) * D:])  # v is left as it was

    hq = torch.empty(H, S, D, dtype=DT[xt], device="cuda")
    hk = torch.empty(K, S, D, dtype=DT[xt], device="cuda")
    qk_norm_rope(q, k, pos, axes, q_weight=w, k_weight=w, out_q=hq.transpose(0, 1), out_k=hk.transpose(0, 1))
    assert torch.equal(hq.transpose(0, 1), wq) and torch.equal(hk.transpose(0, 1), wk)

    wide = torch.zeros(S, (H + 2 * K) * D + 3, dtype=DT[xt], device="cuda")
    wide[:, 1:-2] = qkv
    off = wide[:, 1:-2]
    oq, ok = qk_norm_rope(off[:, :H * D].unflatten(1, (H, D)), off[:, H * D:(H + K) * D].unflatten(1, (K, D)),
                          pos.flip(1).flip(1), axes, q_weight=w, k_weight=w)
    assert torch.equal(oq, wq) and torch.equal(ok, wk)
    one = q[:, :1].expand(S, H, D)  # a broadcast head as input
    oq, _ = qk_norm_rope(one, None, pos, axes, q_weight=w)
    assert torch.equal(oq, wq[:, :1].expand(S, H, D))


def test_qk_norm_rope_far_positions(cuda_device):
    """Positions up to 2^31: the angle keeps its fraction of a turn."""
    from h3tp.rms_rope import RotaryAxes, qk_norm_rope
    axes = RotaryAxes(64, (32, 32))
    pos = torch.tensor([[2 ** 31 - 1, 0], [-2 ** 31, 1], [123456789, 987654321], [2 ** 30 + 1, 7]],
                       dtype=torch.int32, device="cuda")
    q = _randn(_gen(1), 4, 2, 64)
    got, _ = qk_norm_rope(q, None, pos, axes, norm=False)
    ref, mag = _rope_ref(q, None, pos, axes, False, 0.0)
    # the 64-bit product of a position of 2^31 radians is off by 2^31 * 2^-52 on each side
    tol = ref.abs() * U + ROPE_DEPTH * U * mag + 4 * 2.0 ** 31 * 2.0 ** -52 * mag
    assert ((got.double() - ref).abs() <= tol).all()


def test_qk_norm_rope_special_values(cuda_device):
    from h3tp.rms_rope import RotaryAxes, qk_norm_rope
    axes = RotaryAxes(32, (16,))
    q = torch.zeros(1, 4, 32, device="cuda")
    q[0, 1, 20] = float("inf")  # an element that is not turned
    q[0, 2, 3] = float("nan")
    q[0, 3] = 1.0
    pos = torch.zeros(1, dtype=torch.int32, device="cuda")
    got, _ = qk_norm_rope(q, None, pos, axes, norm=False)
    assert (got[0, 0] == 0).all()
    assert got[0, 1, 20] == float("inf") and (got[0, 1, :20] == 0).all() and (got[0, 1, 21:] == 0).all()
    assert torch.isnan(got[0, 2]).sum() == 2
    assert (got[0, 3] == 1).all()
    got, _ = qk_norm_rope(q, None, pos, axes, norm=True)
    assert (got[0, 0] == 0).all() and torch.isnan(got[0, 2]).all()


# --------------------------------------------------------------------------------------
# int4_linear
# --------------------------------------------------------------------------------------
def _int4_inputs(g, m, k, n, xt, group, zeros, st):
    x = _randn(g, m, k).to(DT[xt])
    w = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device="cuda", dtype=torch.uint8)
    groups = -(-k // group)
    s = (_randn(g, n, groups) * 0.01).to(DT[st])
    z = torch.randint(0, 16, (n, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return x, w, s, z


def _int4_ref(x, w, s, z, group, bias):
    k = x.shape[1]
    code = torch.stack((w & 15, w >> 4), 2).flatten(1)[:, :k].double()
    zero = 8.0 if z is None else z.double().repeat_interleave(group, 1)[:, :k]
    wd = (code - zero) * s.double().repeat_interleave(group, 1)[:, :k]
    y, mag = x.double() @ wd.T, x.double().abs() @ wd.abs().T
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    return y, mag


def _int4_depth(k, group):
    # inside a group at most 8 products of 16 terms follow one another, then the groups do;
    # the tensor cores may truncate where fp32 additions round, hence the factor 2
    return 2 * (16 + -(-k // group) + 16)


@pytest.mark.parametrize("m", [1, 2, 3, 7, 8, 9, 16, 17, 31, 32, 33, 70])
@pytest.mark.parametrize("xt", ["f16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_int4_linear_rows(cuda_device, m, xt, group):
    from h3tp import ops
    g = _gen(m)
    x, w, s, z = _int4_inputs(g, m, 1280, 200, xt, group, m % 2 == 0, "f32")
    bias = _randn(g, 200)
    y = ops.int4_linear(x, w, s, z, group=group, bias=bias, out_dtype=torch.float32)
    _close(y, *_int4_ref(x, w, s, z, group, bias), _int4_depth(1280, group))
    y = ops.int4_linear(x, w, s, z, group=group)
    assert y.dtype == x.dtype
    _close(y, *_int4_ref(x, w, s, z, group, None), _int4_depth(1280, group))


@pytest.mark.parametrize("k", [1, 2, 15, 16, 31, 32, 33, 63, 64, 100, 127, 128, 129, 255, 256, 257, 384, 1000, 1001,
                               2080, 4096, 6144])
@pytest.mark.parametrize("n", [1, 15, 16, 17, 65, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_int4_linear_odd_sizes(cuda_device, k, n, zeros):
    from h3tp import ops
    g = _gen(k * 131 + n)
    group = (32, 64, 128)[(k + n) % 3]
    for m, xt, st in ((1, "f16", "f16"), (5, "bf16", "bf16"), (12, "f16", "f32")):
        x, w, s, z = _int4_inputs(g, m, k, n, xt, group, zeros, st)
        y = ops.int4_linear(x, w, s, z, group=group, out_dtype=torch.float32)
        _close(y, *_int4_ref(x, w, s, z, group, None), _int4_depth(k, group))


@pytest.mark.parametrize("m,k,n", [(1, 17000, 96), (32, 20000, 64), (40, 12800, 300), (9, 5376, 4096)])
def test_int4_linear_long(cuda_device, m, k, n):
    from h3tp import ops
    g = _gen(k)
    x, w, s, z = _int4_inputs(g, m, k, n, "bf16", 128, True, "f16")
    y = ops.int4_linear(x, w, s, z, group=128, out_dtype=torch.float32)
    _close(y, *_int4_ref(x, w, s, z, 128, None), _int4_depth(k, 128))


def test_int4_linear_strides_and_alignment(cuda_device):
    from h3tp import ops
    g = _gen(4)
    x, w, s, z = _int4_inputs(g, 6, 512, 80, "f16", 64, True, "f16")
    want = ops.int4_linear(x, w, s, z, group=64)
    wide = torch.zeros(6, 515, dtype=torch.float16, device="cuda")
    wide[:, 2:-1] = x
    assert torch.equal(ops.int4_linear(wide[:, 2:-1], w, s, z, group=64), want)
    assert torch.equal(ops.int4_linear(x.t().contiguous().t(), w, s, z, group=64), want)
    flat = torch.empty(w.numel() + 3, dtype=torch.uint8, device="cuda")
    flat[3:] = w.reshape(-1)
    assert torch.equal(ops.int4_linear(x, flat[3:].view(w.shape), s, z, group=64), want)
    same = ops.int4_linear(x[:1].expand(6, 512), w, s, z, group=64)  # a broadcast row
    assert torch.equal(same, want[:1].expand(6, 80))
    assert ops.int4_linear(x[:0], w, s, z, group=64).shape == (0, 80)


def test_int4_linear_special_values(cuda_device):
    """Infinities and NaN of x reach the outputs of their row only, also when the row is
    shorter than the tile it is computed in."""
    from h3tp import ops
    x = torch.ones(3, 40, dtype=torch.float16, device="cuda")
    x[1, 39] = float("inf")
    x[2, 0] = float("nan")
    w = torch.full((20, 20), 0x99, dtype=torch.uint8, device="cuda")  # every code 9: weight 1
    s = torch.ones(20, 1, device="cuda")
    s2 = torch.ones(20, 2, device="cuda")
    for group, sc in ((64, s), (32, s2)):
        y = ops.int4_linear(x, w, sc, group=group)
        assert (y[0] == 40).all() and (y[1] == float("inf")).all() and torch.isnan(y[2]).all()


def test_quantize_int4_round_trip(cuda_device):
    """The quantised weight is within half a step of the weight everywhere, and the module
    multiplies by exactly that weight."""
    from h3tp.int4_linear import ColumnParallelLinearINT4, quantize_int4
    g = _gen(8)
    w = _randn(g, 48, 333)
    for zp in (False, True):
        packed, s, z = quantize_int4(w, 64, zp)
        code = torch.stack((packed & 15, packed >> 4), 2).flatten(1)[:, :333].double()
        zero = 8.0 if z is None else z.double().repeat_interleave(64, 1)[:, :333]
        wd = (code - zero) * s.double().repeat_interleave(64, 1)[:, :333]
        step = s.double().repeat_interleave(64, 1)[:, :333]
        # half a step, and with zero points the rounded zero moves the range by another half
        assert ((wd - w.double()).abs() <= step * (1.0 if zp else 0.5) * (1 + 8 * U)).all()
        bias = _randn(g, 48)
        mods = [ColumnParallelLinearINT4(333, 48, r, 2, 64, zp, True, out_dtype=torch.float32,
                                         device="cuda", components=3) for r in range(2)]
        x = _randn(g, 2, 2, 333).half()
        ref = x.double() @ wd.T + bias.double()
        mag = x.double().abs() @ wd.abs().T + bias.double().abs()
        outs = []
        for m in mods:
            m.load_quantized(packed, s, z, bias)
            other = ColumnParallelLinearINT4(333, 48, m.rank, 2, 64, zp, True, out_dtype=torch.float32,
                                             device="cuda", components=3)
            other.load_from_full(w, bias)
            outs.append(m(x))
            assert torch.equal(outs[-1], other(x))
        both = torch.cat([o.unflatten(-1, (3, 8)) for o in outs], -1).flatten(-2)
        _close(both, ref, mag, _int4_depth(333, 64))


# --------------------------------------------------------------------------------------
# streams, graphs, refusals
# --------------------------------------------------------------------------------------
def _three_calls(seed=0):
    """One call of each operator on fresh inputs: (inputs, call) pairs."""
    from h3tp import ops
    from h3tp.rms_rope import RotaryAxes, qk_norm_rope
    g = _gen(seed)
    x, b, gate, shift, scale, lab = _norm_case(g, 33, 768, "f16", "f16", 3)
    axes = RotaryAxes(64, (16, 24, 24))
    q, k = _randn(g, 50, 4, 64).half(), _randn(g, 50, 2, 64).half()
    pos = _positions(g, 50, 3, "i32")
    xi, w, s, z = _int4_inputs(g, 4, 512, 96, "f16", 64, True, "f16")
    pre = ops.NormSpec("rms")
    return [
        ([x, b], lambda: ops.residual_norm(x, b, gate, lab, post=pre, pre=pre, shift=shift, scale=scale,
                                           out=torch.empty_like(x), quantize=True)),
        ([x, b], lambda: ops.residual_norm(x, b, gate, lab, post=pre, pre=pre, shift=shift, scale=scale,
                                           out=torch.empty_like(x))),
        ([q, k], lambda: qk_norm_rope(q, k, pos, axes)),
        ([xi], lambda: ops.int4_linear(xi, w, s, z, group=64)),
    ]


def _flat(r):
    return [t for t in (r if isinstance(r, tuple) else (r,)) if t is not None]


def test_block_operators_on_other_streams(cuda_device):
    calls = _three_calls()
    want = [[t.clone() for t in _flat(c())] for _, c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = []
    for (_, c), st in zip(calls, streams):
        with torch.cuda.stream(st):
            got.append(_flat(c()))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_block_operators_captured(cuda_device):
    """Two graphs of all operators, replayed in turn on changed inputs."""
    sets = [_three_calls(1), _three_calls(2)]
    graphs, outs = [], []
    for calls in sets:
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            for _, c in calls:
                c()
        torch.cuda.current_stream().wait_stream(st)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append([_flat(c()) for _, c in calls])
        graphs.append(gr)
    for _ in range(2):
        for calls in sets:
            for inputs, _ in calls:
                for t in inputs:
                    t.mul_(0.75)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for calls, held in zip(sets, outs):
            for (_, c), h in zip(calls, held):
                assert all(torch.equal(u, v) for u, v in zip(_flat(c()), h))


def test_block_operators_repeat_bit_for_bit(cuda_device):
    calls = _three_calls(3)
    first = [[t.clone() for t in _flat(c())] for _, c in calls]
    for _ in range(3):
        for (_, c), f in zip(calls, first):
            assert all(torch.equal(u, v) for u, v in zip(_flat(c()), f))


def _refused(call, *args, **kw):
    with pytest.raises(ValueError):
        call(*args, **kw)


def test_residual_norm_refusals(cuda_device):
    from h3tp import ops
    x = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    b = torch.zeros_like(x)
    t = torch.zeros(2, 64, device="cuda")
    lab = torch.zeros(4, dtype=torch.int32, device="cuda")
    rms = ops.NormSpec("rms")
    r = lambda *a, **k: _refused(ops.residual_norm, *a, **k)
    r(x.cpu(), b.cpu())
    r(x.double(), b)
    r(x[0], b[0])
    r(x.t(), b.t())
    r(x, b[:3])
    r(x, b.to(torch.bfloat16))
    r(x, b, out=torch.empty(4, 64, device="cuda"))
    r(x, x)                                              # the branch would be read while x is written
    r(x, b, out=b)
    big = torch.zeros(8, 64, dtype=torch.float16, device="cuda")
    r(big[:4], b, out=big[2:6])                          # a partial overlap
    r(x)                                                 # neither a branch nor a norm
    r(x, pre=rms, post=rms)
    r(x, pre=rms, gate=t, labels=lab)
    r(x, pre=rms, residual_scale=0.5)
    r(x, b, quantize=True)
    r(x, b, shift=t, labels=lab)
    r(x, b, pre=rms, quantize=True)                      # 64 is no multiple of 256
    r(x, b, t)                                           # two rows and no labels
    r(x, b, t, lab[:3])
    r(x, b, t, lab.long())
    r(x, b, t.half(), lab)
    r(x, b, t[:, :32], lab)
    r(x, b, t, lab, pre=rms, shift=t[:1])
    r(x, b, t[:0], lab)
    r(x, b, t.cpu(), lab)
    r(x, b, pre=ops.NormSpec("batch"))
    r(x, b, pre=ops.NormSpec("rms", torch.zeros(63, device="cuda")))
    r(x, b, pre=ops.NormSpec("rms", torch.zeros(64)))
    r(x, b, pre=ops.NormSpec("rms", eps=-1.0))
    r(x, b, pre=ops.NormSpec("rms", eps=float("nan")))
    r(torch.zeros(2, 32776, dtype=torch.float16, device="cuda"), pre=rms)
    r(torch.zeros(2, 0, dtype=torch.float16, device="cuda"), pre=rms)
    w = torch.ones(64, device="cuda", requires_grad=True)
    with torch.enable_grad():
        r(x, b, pre=ops.NormSpec("rms", w))
    with torch.no_grad():
        ops.residual_norm(x, b, pre=ops.NormSpec("rms", w))


def test_qk_norm_rope_refusals(cuda_device):
    from h3tp.rms_rope import RotaryAxes, packed_qk_norm_rope, qk_norm_rope
    axes = RotaryAxes(64, (32, 32))
    q = torch.zeros(4, 6, 64, dtype=torch.float16, device="cuda")
    k = torch.zeros(4, 2, 64, dtype=torch.float16, device="cuda")
    pos = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    r = lambda *a, **kw: _refused(qk_norm_rope, *a, **kw)
    r(q.cpu(), k.cpu(), pos.cpu(), axes)
    r(q.double(), None, pos, axes)
    r(q[..., ::2], None, pos, RotaryAxes(32, (32,)))
    r(q[:, :0], None, pos, axes)
    r(q, k[:, :0], pos, axes)
    r(q, k.float(), pos, axes)
    r(q, k[:3], pos, axes)
    r(q, k[..., :32], pos, axes)
    r(q, k, pos, RotaryAxes(128, (32, 32)))
    r(q, k, pos[:, :1], axes)
    r(q, k, pos[:, 0], axes)
    r(q, k, pos[:3], axes)
    r(q, k, pos.half(), axes)
    r(q, k, pos.cpu(), axes)
    r(q, k, pos, axes, eps=-1.0)
    r(q, k, pos, axes, q_weight=torch.zeros(32, device="cuda"))
    r(q, k, pos, axes, q_weight=torch.zeros(64, dtype=torch.float16, device="cuda"))
    r(q, k, pos, axes, out_q=torch.empty(4, 5, 64, dtype=torch.float16, device="cuda"))
    r(q, None, pos, axes, out_k=torch.empty_like(k))
    r(q, k, pos, axes, out_q=q[:, :1].expand(4, 6, 64))
    r(q, q, pos, axes, out_q=q)                          # q turned in place while k reads it
    r(q[:, :2], k, pos, axes, out_q=k)
    buf = torch.zeros(5, 6, 64, dtype=torch.float16, device="cuda")
    r(buf[:4], None, pos, axes, out_q=buf[1:])
    same = torch.empty_like(k)
    r(k, k.clone(), pos, axes, out_q=same, out_k=same)
    r(q.requires_grad_(), k, pos, axes)
    _refused(packed_qk_norm_rope, torch.zeros(4, 640, dtype=torch.float16, device="cuda"), 6, 3, pos, axes)


def test_int4_linear_refusals(cuda_device):
    from h3tp import ops
    g = _gen(1)
    x, w, s, z = _int4_inputs(g, 3, 128, 16, "f16", 64, True, "f16")
    r = lambda *a, **kw: _refused(ops.int4_linear, *a, **{"group": 64, **kw})
    r(x.cpu(), w, s, z)
    r(x.float(), w, s, z)
    r(x[0], w, s, z)
    r(x, w.cpu(), s, z)
    r(x, w.to(torch.int8), s, z)
    r(x, w[:, :63], s, z)
    r(x, w.t().contiguous().t(), s, z)
    r(x, w, s[:, :1], z)
    r(x, w, s.double(), z)
    r(x, w, s, z[:15])
    r(x, w, s, z.to(torch.int8))
    r(x, w, s, z, group=48)
    r(x, w, s, z, group=128)
    r(x, w, s, z, out_dtype=torch.bfloat16)
    r(x, w, s, z, bias=torch.zeros(15, device="cuda"))
    r(x, w, s, z, bias=torch.zeros(16, dtype=torch.float16, device="cuda"))
    r(x, w[:0], s[:0], z[:0])
    r(x[:, :0], w[:, :0], s[:, :0], z[:, :0])
    r(x.clone().requires_grad_(), w, s, z)


# --------------------------------------------------------------------------------------
# a block of them
# --------------------------------------------------------------------------------------
def _block(hidden, ffn, heads, axes, cond, seed):
    from h3tp.tp_dit import TPDiTModulatedBlockINT8
    g = _gen(seed)
    block = TPDiTModulatedBlockINT8(hidden, ffn, heads, axes, cond, device="cuda", group=64)
    for m in (block.qkv_proj, block.out_proj, block.fc1, block.fc2):
        m.weight.data.copy_(torch.randint(-127, 128, m.weight.shape, generator=g, device="cuda", dtype=torch.int8))
        m.weight_scale.data.copy_(torch.rand(m.weight_scale.shape, generator=g, device="cuda") * 2e-4 + 1e-4)
    block.modulation.load_from_full(_randn(g, 6 * hidden, cond) * 0.05, _randn(g, 6 * hidden) * 0.2)
    for w in (block.attn_norm, block.attn_post_norm, block.mlp_norm, block.mlp_post_norm, block.q_norm, block.k_norm):
        w.data.copy_(1 + 0.1 * _randn(g, w.numel()))
    return block, g


def _dequantised(module, x):
    """x through an INT8 projection's weights in 64 bits (the rotation is orthonormal and the
    weights are stored rotated, so x is rotated and not the weights)."""
    w = module.weight.double() * module.weight_scale.double()
    return _rotate(x) @ w.T


def _softmax_attention(q, k, v):
    s = torch.einsum("shd,thd->hst", q.double(), k.double()) / q.shape[-1] ** 0.5
    return torch.einsum("hst,thd->shd", s.softmax(-1), v.double())


@pytest.mark.parametrize("rows,cond_rows", [(1, 1), (300, 3)])
def test_modulated_block(cuda_device, rows, cond_rows):
    """The whole block against its definition in 64 bits.  INT8 activations dominate: a code is
    off by half a step, a step is 1/127 of the rotated row's maximum, about 4 of its standard
    deviations, so each quantised activation carries an error of about (4 / 127) / sqrt(12) =
    0.9% of its norm; four of them in a row, through norms that keep ratios, stay within 4 *
    0.9% of the branches' norm, and twice that is allowed."""
    from h3tp.rms_rope import RotaryAxes
    axes = RotaryAxes(64, (16, 24, 24))
    block, g = _block(512, 1024, 8, axes, 192, rows)
    x = _randn(g, rows, 512).half()
    cond = _randn(g, cond_rows, 192).half()
    pos = _positions(g, rows, 3, "i32", far=64)
    cuts = [0, rows // 3, rows // 2, rows]
    segments = [(cuts[i], cuts[i + 1], i) for i in range(3)] if cond_rows > 1 else None
    labels = torch.zeros(rows, dtype=torch.int32, device="cuda")
    for a, b, r in segments or []:
        labels[a:b] = r
    m = block.modulation
    mods, _ = _int4_ref(cond, m.weight, m.weight_scale, None, 64, m.bias)
    sa, ca, ga, sm, cm, gm = [t.contiguous() for t in mods.chunk(6, 1)]

    def norm(v, w):
        return v / (v.square().mean(-1, keepdim=True) + block.eps).sqrt() * w.double()

    lab = labels.long()
    h = norm(x.double(), block.attn_norm) * (1 + ca[lab]) + sa[lab]
    q, k, v = _dequantised(block.qkv_proj, h).reshape(rows, 3, 8, 64).unbind(1)
    q, _ = _rope_ref(q, block.q_norm, pos, axes, True, block.eps)
    k, _ = _rope_ref(k, block.k_norm, pos, axes, True, block.eps)
    y = _dequantised(block.out_proj, _softmax_attention(q, k, v).reshape(rows, 512))
    want = x.double() + ga[lab] * norm(y, block.attn_post_norm)
    h = norm(want, block.mlp_norm) * (1 + cm[lab]) + sm[lab]
    gate, up = _dequantised(block.fc1, h).chunk(2, 1)
    y = _dequantised(block.fc2, torch.nn.functional.silu(gate) * up)
    delta = want - x.double() + gm[lab] * norm(y, block.mlp_post_norm)

    before = x.clone()
    out = block(x, cond, pos, lambda q, k, v: _softmax_attention(q, k, v).half(), segments)
    assert out is x
    got = out.double() - before.double()
    assert torch.isfinite(out).all()
    err = ((got - delta).norm() / delta.norm()).item()
    assert err <= 0.072, err


def test_modulated_block_captured(cuda_device):
    """A captured block replayed on new inputs gives the bits of an eager one."""
    from h3tp.rms_rope import RotaryAxes
    axes = RotaryAxes(64, (16, 24, 24), pairing="half")
    block, g = _block(512, 1024, 8, axes, 192, 5)
    x0, cond = _randn(g, 640, 512).half(), _randn(g, 2, 192).half()
    pos = _positions(g, 640, 3, "i32")
    segments = [(0, 77, 0), (77, 640, 1)]
    x = x0.clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        block(x, cond, pos, segments=segments)
    torch.cuda.current_stream().wait_stream(st)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        block(x, cond, pos, segments=segments)
    for i in range(2):
        cond.mul_(0.5)
        x.copy_(x0 * (i + 1))
        gr.replay()
        y = x0 * (i + 1)
        block(y, cond, pos, segments=segments)
        assert torch.equal(x, y)


def test_modulated_block_refusals(cuda_device):
    from h3tp.rms_rope import RotaryAxes
    from h3tp.tp_dit import TPDiTModulatedBlockINT8
    axes = RotaryAxes(64, (64,))
    _refused(TPDiTModulatedBlockINT8, 500, 1024, 8, axes, 192, device="cuda")
    _refused(TPDiTModulatedBlockINT8, 512, 1024, 6, axes, 192, device="cuda")
    _refused(TPDiTModulatedBlockINT8, 512, 1024, 9, axes, 192, world_size=2, device="cuda")
    block, g = _block(512, 1024, 8, axes, 192, 6)
    x, cond = torch.zeros(4, 512, dtype=torch.float16, device="cuda"), _randn(g, 2, 192).half()
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    _refused(block, x, cond, pos)
    _refused(block, x, cond, pos, segments=[(0, 3, 0)])
    _refused(block, x, cond[:1], pos[:3])


def test_first_labelled_call_in_a_capture(cuda_device):
    """A process whose first call with labels is captured: the error word is made without
    breaking the capture."""
    import subprocess
    import sys
    from pathlib import Path
    code = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from h3tp import ops
x = torch.ones(5, 256, dtype=torch.float16, device="cuda")
shift = torch.tensor([[0.0], [1.0]], device="cuda").expand(2, 256).contiguous()
labels = torch.tensor([0, 1, 0, 1, 1], dtype=torch.int32, device="cuda")
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    _, h, _ = ops.residual_norm(x, labels=labels, pre=ops.NormSpec("rms", eps=0.0), shift=shift)
graph.replay()
torch.cuda.synchronize()
assert h[:, 0].tolist() == [1.0, 2.0, 1.0, 2.0, 2.0], h[:, 0]
"""
    pkg = Path(__file__).resolve().parents[1] / "minimax-h3-2xt4_b200"
    r = subprocess.run([sys.executable, "-c", code, str(pkg)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


@pytest.mark.parametrize("width", [32, 64, 1280, 2056, 5376, 6144, 6400])
@pytest.mark.parametrize("xt,bt", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm_many_rows_equal_few(cuda_device, width, xt, bt, kind):
    """Enough rows for the kernel that takes two at a time, an odd number of them, labels that
    change inside a pair, and a row with an infinity beside a finite one: the bits of the same
    rows in small calls."""
    from h3tp import ops
    g = _gen(width)
    rows = 741
    x, b, gate, shift, scale, lab = _norm_case(g, rows, width, xt, bt, 3)
    b[600] = float("inf")
    spec = ops.NormSpec(kind, _randn(g, width), _randn(g, width))
    quants = (False, True) if width % 256 == 0 else (False,)
    for quant in quants:
        kw = dict(post=spec, pre=spec, shift=shift, scale=scale, quantize=quant, residual_scale=0.5)
        whole = ops.residual_norm(x.clone(), b, gate, lab, **kw)
        first = ops.residual_norm(x, pre=spec, labels=lab, shift=shift, scale=scale, quantize=quant)
        for at in range(0, rows, 137):
            part = slice(at, at + 137)
            few = ops.residual_norm(x[part].clone(), b[part], gate, lab[part], **kw)
            alone = ops.residual_norm(x[part], pre=spec, labels=lab[part], shift=shift, scale=scale, quantize=quant)
            for a, w in ((few, whole), (alone, first)):
                for u, v in zip(a, w):
                    assert u is None or torch.equal(torch.nan_to_num(u.float(), 7.0), torch.nan_to_num(v[part].float(), 7.0))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("xt", ["f16", "f32"])
def test_qk_norm_rope_many_tokens_equal_few(cuda_device, half, xt):
    """More tokens than the GPU holds lane groups for: the bits of the same tokens in small
    calls, whose heads are split, and in place on packed rows."""
    from h3tp.rms_rope import RotaryAxes, packed_qk_norm_rope, qk_norm_rope
    for dim, axes in ((64, (16, 24, 24)), (80, (40, 40)), (33, (8, 6, 10))):
        plan = RotaryAxes(dim, axes, pairing="half" if half else "interleaved")
        g = _gen(dim)
        S, H, K = 25013, 3, 2
        qkv = _randn(g, S, (H + 2 * K) * dim).to(DT[xt])
        pos = _positions(g, S, len(axes), "i32")
        wq, wk = _randn(g, dim), _randn(g, dim)
        q = qkv[:, :H * dim].unflatten(1, (H, dim))
        k = qkv[:, H * dim:(H + K) * dim].unflatten(1, (K, dim))
        oq, ok = qk_norm_rope(q, k, pos, plan, q_weight=wq, k_weight=wk)
        _close(oq, *_rope_ref(q, wq, pos, plan, True, 1e-6), ROPE_DEPTH)
        _close(ok, *_rope_ref(k, wk, pos, plan, True, 1e-6), ROPE_DEPTH)
        for at in range(0, S, 6007):
            part = slice(at, at + 6007)
            fq, fk = qk_norm_rope(q[part], k[part], pos[part], plan, q_weight=wq, k_weight=wk)
            assert torch.equal(fq, oq[part]) and torch.equal(fk, ok[part])
        pq, pk, _ = packed_qk_norm_rope(qkv, H, K, pos, plan, q_weight=wq, k_weight=wk)
        assert torch.equal(pq, oq) and torch.equal(pk, ok)


@pytest.mark.parametrize("m,k,n,group", [(3, 512, 40000, 32), (20, 300, 50001, 64), (32, 4096, 20000, 128),
                                         (32, 4099, 20000, 64)])
def test_int4_linear_many_columns(cuda_device, m, k, n, group):
    """Several rounds of column tiles a CTA, with x held whole and in chunks."""
    from h3tp import ops
    g = _gen(n)
    x, w, s, z = _int4_inputs(g, m, k, n, "f16", group, True, "f16")
    bias = _randn(g, n)
    y = ops.int4_linear(x, w, s, z, group=group, bias=bias, out_dtype=torch.float32)
    _close(y, *_int4_ref(x, w, s, z, group, bias), _int4_depth(k, group))
