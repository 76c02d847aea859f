"""Calls of the operators around a block's projections that the layout and refusal tests do not
make, as far as they need no GPU."""
import pytest
import torch


# --------------------------------------------------------------------------------------
# 4-bit quantisation
# --------------------------------------------------------------------------------------
def _dequantised(packed, scales, zeros, k, group):
    code = torch.stack((packed & 15, packed >> 4), 2).flatten(1)[:, :k].double()
    zero = 8.0 if zeros is None else zeros.double().repeat_interleave(group, 1)[:, :k]
    return (code - zero) * scales.double().repeat_interleave(group, 1)[:, :k]


@pytest.mark.parametrize("magnitude", [1.0, 3e-4, 8e-6, 4e-7, 1e-8])
@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("zero_points", [False, True])
def test_quantize_int4_of_small_weights(magnitude, scale_dtype, zero_points):
    """Whatever the weights' magnitude, the scale follows them as far as its type reaches (fp16: in
    steps of 2^-24 at the lowest) and a weight is off by half a scale: its code's rounding, and
    with zero points the border codes' by what the scale's rounding moves 15 of it."""
    from h3tp.int4_linear import quantize_int4
    g = torch.Generator().manual_seed(1)
    w = torch.randn(40, 200, generator=g) * magnitude
    packed, s, z = quantize_int4(w, 64, zero_points, scale_dtype)
    padded = torch.nn.functional.pad(w, (0, 56)).unflatten(1, (4, 64)).double()
    span = padded.amax(2).clamp(min=0) - padded.amin(2).clamp(max=0) if zero_points else padded.abs().amax(2)
    want = span / (15 if zero_points else 7)
    eps = torch.finfo(scale_dtype).eps
    step = 2.0 ** -24 if scale_dtype == torch.float16 else 0.0
    assert ((s.double() - want).abs() <= want * (eps / 2 + 2.0 ** -22) + step).all()
    off = (_dequantised(packed, s, z, 200, 64) - w.double()).abs()
    assert (off <= s.double().repeat_interleave(64, 1)[:, :200] * (0.5 + 16 * (eps / 2 + 2.0 ** -22))).all()


@pytest.mark.parametrize("w,scale_dtype,zero_points", [
    (float("nan"), torch.float32, False), (float("inf"), torch.float32, False), (float("-inf"), torch.bfloat16, True),
    (5e5, torch.float16, False), (1.1e6, torch.float16, True), (1.0, torch.float64, False), (1.0, torch.int32, False)])
def test_quantize_int4_refuses_what_scales_cannot_hold(w, scale_dtype, zero_points):
    """A group that no finite scale of the type spans would come back as NaN."""
    from h3tp.int4_linear import quantize_int4
    full = torch.ones(2, 64)
    full[1, 40] = w
    with pytest.raises(ValueError):
        quantize_int4(full, 32, zero_points, scale_dtype)


def test_quantize_int4_at_the_ends_of_the_range():
    from h3tp.int4_linear import quantize_int4
    for w, dtype in ((4.5e5, torch.float16), (3.4e38, torch.float32), (3.3e38, torch.bfloat16)):
        for zero_points in (False, True):
            packed, s, z = quantize_int4(torch.tensor([[w, -w, 0.0, w / 3]]), 32, zero_points, dtype)
            got = _dequantised(packed, s, z, 4, 32)
            assert torch.isfinite(s.float()).all()
            assert (got - torch.tensor([[w, -w, 0.0, w / 3]]).double()).abs().max() <= 0.6 * s.double().max()


# --------------------------------------------------------------------------------------
# the 4-bit module's loaders
# --------------------------------------------------------------------------------------
def _module(rank=0, world=1, components=1, zero_points=False, bias=True):
    from h3tp.int4_linear import ColumnParallelLinearINT4
    return ColumnParallelLinearINT4(64, 12, rank, world, 32, zero_points=zero_points, bias=bias, device="cpu",
                                    components=components)


def _quantised(n, zero_points=False):
    from h3tp.int4_linear import quantize_int4
    return quantize_int4(torch.linspace(-1, 1, n * 64).reshape(n, 64), 32, zero_points)


def test_int4_loaders_take_whole_tensors_only():
    """A bias of one value is not spread over the rows, and tensors of another number of rows than
    the module's are refused even where a rank's share of them would fit."""
    full, bias = torch.ones(12, 64), torch.arange(12.0)
    m = _module()
    m.load_from_full(full, bias)
    assert torch.equal(m.bias.data, bias)
    packed, scales, _ = _quantised(12)
    for bad in (torch.ones(1), torch.ones(12, 1), torch.ones(13), torch.tensor(1.0)):
        with pytest.raises(ValueError):
            m.load_from_full(full, bad)
        with pytest.raises(ValueError):
            m.load_quantized(packed, scales, None, bad)
    assert torch.equal(m.bias.data, bias)  # nothing was loaded by a refused call
    for rank, rows in ((1, 13), (0, 11), (1, 14)):  # chunks of 7 + 6, 6 + 5 and 7 + 7 rows
        m = _module(rank, 2, bias=False)
        with pytest.raises(ValueError):
            m.load_from_full(torch.ones(rows, 64))
        with pytest.raises(ValueError):
            m.load_quantized(*_quantised(rows)[:2])


def test_int4_loader_refuses_zero_points_above_15():
    m = _module(zero_points=True, bias=False)
    packed, scales, zeros = _quantised(12, True)
    m.load_quantized(packed, scales, zeros)
    assert torch.equal(m.weight_zero.data, zeros)
    bad = zeros.clone()
    bad[7, 1] = 16
    with pytest.raises(ValueError):
        m.load_quantized(packed, scales, bad)
    assert torch.equal(m.weight_zero.data, zeros)


# --------------------------------------------------------------------------------------
# arguments that are no tensors, inputs of another width
# --------------------------------------------------------------------------------------
def test_int4_module_refuses_other_widths():
    """Rows are not cut anew to the module's width."""
    m = _module()
    for shape in ((3, 32), (2, 128), (64, 3), (128,), ()):
        with pytest.raises(ValueError, match="in_features|64"):
            m(torch.zeros(shape, dtype=torch.float16))
