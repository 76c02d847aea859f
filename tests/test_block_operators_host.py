"""The operators around a block's projections, as far as they can be checked without a
GPU: plans, packing, module loaders, and the refusals of the C entry points (returned
before anything is launched, and before a pointer is looked at)."""
import ctypes
import math

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from h3tp import _native
    return _native.load()


# --------------------------------------------------------------------------------------
# rotary plans
# --------------------------------------------------------------------------------------
def test_chunked_plan():
    from h3tp.rms_rope import RotaryAxes
    p = RotaryAxes(16, (4, 6, 6), theta=100.0)
    assert p.axis_of_pair == (0, 0, 1, 1, 1, 2, 2, 2) and p.pairs == 8 and p.n_axes == 3 and not p.half
    want = [1, 100 ** (-2 / 4), 1, 100 ** (-2 / 6), 100 ** (-4 / 6), 1, 100 ** (-2 / 6), 100 ** (-4 / 6)]
    assert p.inv_freq == pytest.approx(want, rel=1e-15)
    assert list(p.axis) == list(p.axis_of_pair)
    assert [t * 2 * math.pi for t in p.turns] == pytest.approx(want, rel=1e-15)


def test_interleaved_plan_deals_in_turn():
    from h3tp.rms_rope import RotaryAxes
    p = RotaryAxes(128, (48, 40, 40), order="interleaved", frequencies="shared", pairing="half")
    assert p.axis_of_pair == (0, 1, 2) * 20 + (0,) * 4 and p.half
    assert p.inv_freq[1] == pytest.approx(1e4 ** (-2 / 128)) and p.inv_freq[63] == pytest.approx(1e4 ** (-126 / 128))
    p = RotaryAxes(32, (4, 0, 8), order="interleaved")
    assert p.axis_of_pair == (0, 0, 2, 2, 2, 2)
    assert sorted(p.axis_of_pair) == sorted((0,) * 2 + (2,) * 4)


def test_plan_with_given_frequencies():
    from h3tp.rms_rope import RotaryAxes
    p = RotaryAxes(8, (4,), inv_freq=[0.5, 0.25])
    assert p.inv_freq == (0.5, 0.25)
    p = RotaryAxes(8, (4, 4), theta=(10.0, 1000.0))
    assert p.inv_freq == pytest.approx([1, 10 ** -0.5, 1, 1000 ** -0.5])


@pytest.mark.parametrize("args,kw", [
    ((1, (1,)), {}), ((258, (258,)), {}), ((8, ()), {}), ((8, (0,)), {}), ((8, (3, 5)), {}), ((8, (6, 4)), {}),
    ((8, (-2, 4)), {}), ((8, (4,)), {"pairing": "thirds"}), ((8, (4,)), {"order": "random"}),
    ((8, (4,)), {"frequencies": "none"}), ((8, (4,)), {"inv_freq": [1.0]}),
    ((8, (4,)), {"inv_freq": [1.0, float("nan")]}), ((8, (4, 4)), {"theta": (1.0,)}), ((8, (4,)), {"theta": 0.0}),
])
def test_plan_refusals(args, kw):
    from h3tp.rms_rope import RotaryAxes
    with pytest.raises(ValueError):
        RotaryAxes(*args, **kw)


# --------------------------------------------------------------------------------------
# 4-bit packing
# --------------------------------------------------------------------------------------
def test_quantize_int4_layout():
    from h3tp.int4_linear import quantize_int4
    w = torch.tensor([[-7.0, 7.0, 3.0, 0.0, 1.0]])
    packed, s, z = quantize_int4(w, 32)
    assert packed.tolist() == [[1 | (15 << 4), 11 | (8 << 4), 9]] and z is None
    assert s.tolist() == [[1.0]]
    packed, s, z = quantize_int4(torch.tensor([[-5.0, 10.0, 0.0]]), 32, zero_points=True)
    assert s.tolist() == [[1.0]] and z.tolist() == [[5]] and packed.tolist() == [[0 | (15 << 4), 5]]


def test_quantize_int4_of_zeros_and_half_scales():
    from h3tp.int4_linear import quantize_int4
    for zp in (False, True):
        for st in (torch.float32, torch.float16, torch.bfloat16):
            packed, s, z = quantize_int4(torch.zeros(3, 70), 64, zp, st)
            assert s.dtype == st and s.shape == (3, 2) and (s > 0).all()
            offset = 8 if z is None else z.long()[:, :1]
            assert ((packed[:, :32] & 15).long() == offset).all()


@pytest.mark.parametrize("bad", [torch.zeros(4), torch.zeros(2, 4, dtype=torch.int8), torch.zeros(0, 4)])
def test_quantize_int4_refusals(bad):
    from h3tp.int4_linear import quantize_int4
    with pytest.raises(ValueError):
        quantize_int4(bad, 32)
    with pytest.raises(ValueError):
        quantize_int4(torch.zeros(2, 4), 48)


def test_int4_module_shards_by_component():
    from h3tp.int4_linear import ColumnParallelLinearINT4
    full = torch.arange(12, dtype=torch.float32).reshape(12, 1).repeat(1, 32)
    mods = [ColumnParallelLinearINT4(32, 12, r, 2, 32, device="cpu", components=3) for r in range(2)]
    assert [m._rows(full)[:, 0].tolist() for m in mods] == [[0, 1, 4, 5, 8, 9], [2, 3, 6, 7, 10, 11]]
    with pytest.raises(ValueError):
        ColumnParallelLinearINT4(32, 10, 0, 2, 32, device="cpu", components=3)
    with pytest.raises(ValueError):
        mods[0].load_quantized(torch.zeros(12, 16, dtype=torch.uint8), torch.zeros(12, 1), None, torch.zeros(12))
    with pytest.raises(ValueError):
        mods[0].load_quantized(torch.zeros(12, 15, dtype=torch.uint8), torch.zeros(12, 1))
    with pytest.raises(ValueError):
        mods[0](torch.zeros(1, 32, dtype=torch.float16))  # no CPU path


# --------------------------------------------------------------------------------------
# overlaps of views
# --------------------------------------------------------------------------------------
def test_head_windows():
    from h3tp import ops
    t = torch.zeros(10, 64)
    q, k = t[:, :32].unflatten(1, (4, 8)), t[:, 32:48].unflatten(1, (2, 8))
    assert ops._head_windows_apart(q, k) and ops._head_windows_apart(k, q)
    assert not ops._head_windows_apart(q, q)
    assert not ops._head_windows_apart(q, t[:, 24:40].unflatten(1, (2, 8)))
    assert not ops._head_windows_apart(t[:9, :32].unflatten(1, (4, 8)), t[1:, 24:56].unflatten(1, (4, 8)))
    assert ops._head_windows_apart(t[:4, :32].unflatten(1, (4, 8)), t[4:8, :32].unflatten(1, (4, 8)))
    assert ops._head_windows_apart(t[:8, :32].unflatten(1, (4, 8)), t[1:9, 32:].unflatten(1, (4, 8)))
    one = t[:1]
    assert not ops._head_windows_apart(one[:, :32].unflatten(1, (4, 8)), one[:, 16:48].unflatten(1, (4, 8)))
    assert ops._head_windows_apart(one[:, :32].unflatten(1, (4, 8)), one[:, 32:].unflatten(1, (4, 8)))


# --------------------------------------------------------------------------------------
# the C entry points' refusals
# --------------------------------------------------------------------------------------
P = 4096  # a pointer that is never read: every call below is refused by its geometry


def _norm(lib, **kw):
    a = dict(x=P, xt=1, b=P, bt=1, rows=4, width=256, rs=1.0, gate=None, gld=256, shift=None, sld=256,
             scale=None, cld=256, mod=1, lab=None, post=0, pw=None, pb=None, pe=0.0, pre=1, nw=None, nb=None,
             ne=0.0, out=P, h=P, rot=0, q=None, s=None, stream=None)
    a.update(kw)
    return lib.h3_residual_norm(*a.values())


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(rows=-1), dict(width=0), dict(width=32769), dict(mod=0), dict(mod=2), dict(post=3),
    dict(pre=-1), dict(b=None), dict(out=None), dict(b=None, out=None, gate=P), dict(b=None, out=None, post=1),
    dict(b=None, out=None, rs=0.5), dict(b=None, out=None, pre=0, h=None), dict(h=None), dict(q=P, h=None),
    dict(q=P, s=P), dict(pre=0), dict(pre=0, h=None, q=P, s=P), dict(h=None, q=P, s=P, rot=1, width=264),
    dict(xt=3), dict(bt=3), dict(xt=1, bt=2), dict(xt=0, bt=1),
])
def test_residual_norm_entry_refuses(lib, kw):
    assert _norm(lib, **kw) == 1


def _rope(lib, **kw):
    turns, axis = (ctypes.c_double * 128)(), (ctypes.c_uint8 * 128)()
    if kw.pop("bad_axis", False):
        axis[3] = 2
    a = dict(q=P, qt=512, qh=64, hq=8, qo=P, qot=512, qoh=64, k=P, kt=512, kh=64, hk=2, ko=P, kot=512, koh=64,
             tokens=4, dim=64, type=1, pos=P, kind=0, axes=2, turns=turns, axis=axis, pairs=32, half=0, norm=1,
             wq=None, wk=None, eps=0.0, stream=None)
    a.update(kw)
    return lib.h3_qk_norm_rope(*a.values())


@pytest.mark.parametrize("kw", [
    dict(q=None), dict(qo=None), dict(ko=None), dict(tokens=-1), dict(hq=0), dict(hq=70000), dict(hk=-1),
    dict(dim=1), dict(dim=257), dict(pos=None), dict(axes=0), dict(axes=256), dict(turns=None), dict(axis=None),
    dict(pairs=0), dict(pairs=33), dict(kind=3), dict(kind=-1), dict(bad_axis=True), dict(type=3), dict(type=-1),
])
def test_qk_norm_rope_entry_refuses(lib, kw):
    assert _rope(lib, **kw) == 1


def _int4(lib, **kw):
    a = dict(x=P, xt=1, ld=256, m=2, k=256, w=P, n=32, s=P, st=1, z=None, group=64, bias=None, out=P, ot=0,
             stream=None)
    a.update(kw)
    return lib.h3_int4_linear(*a.values())


@pytest.mark.parametrize("kw", [
    dict(x=None), dict(w=None), dict(s=None), dict(out=None), dict(m=-1), dict(k=0), dict(n=0), dict(ld=255),
    dict(group=16), dict(group=256), dict(st=3), dict(xt=0), dict(xt=3), dict(ot=2), dict(k=1 << 25),
    dict(n=1 << 25),
])
def test_int4_linear_entry_refuses(lib, kw):
    assert _int4(lib, **kw) == 1


def test_empty_calls_are_no_calls(lib):
    assert _norm(lib, rows=0) == 0 and _rope(lib, tokens=0) == 0 and _int4(lib, m=0) == 0


@pytest.mark.parametrize("call", [_norm, _rope, _int4])
def test_host_pointers_are_refused(lib, call):
    """A pointer that no GPU owns (host memory, or a machine without one) is an error."""
    buf = ctypes.create_string_buffer(1 << 16)
    name = {"_norm": "x", "_rope": "q", "_int4": "x"}[call.__name__]
    assert call(lib, **{name: ctypes.addressof(buf)}) != 0
