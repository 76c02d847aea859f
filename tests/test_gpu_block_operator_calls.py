"""GPU tests of the operators around a block's projections beyond one call's agreement with its
definition: codes against the library's other quantisers' rule, calls that meet other calls."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _randn(seed, *shape):
    g = torch.Generator("cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda")


# --------------------------------------------------------------------------------------
# residual_norm: codes
# --------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,width", [(4096, 2048), (4096, 520), (512, 1001), (64, 16384)])
def test_codes_are_the_rounded_quotient(cuda_device, rows, width):
    """A code is round(h / scale) with the correctly rounded quotient, as the library's other
    quantisers give it: h in fp32 is stored as it is before the quantiser, so the codes follow
    from it bit for bit (torch divides fp32 correctly rounded and rounds ties to even)."""
    from h3tp import ops
    x, b = _randn(width, rows, width), _randn(width + 1, rows, width)
    pre = ops.NormSpec("rms", _randn(2, width))
    shift, scale = _randn(3, 1, width) * 0.3, _randn(4, 1, width) * 0.3
    kw = dict(pre=pre, shift=shift, scale=scale)
    y, h, _ = ops.residual_norm(x, b, out=torch.empty_like(x), **kw)
    z, q, s = ops.residual_norm(x, b, out=torch.empty_like(x), quantize=True, convrot=False, **kw)
    assert torch.equal(y, z)
    want_s = h.abs().amax(1, keepdim=True) * torch.tensor(1 / 127, device="cuda")
    assert torch.equal(s, want_s)
    want = torch.round(h / s).clamp(-128, 127).to(torch.int8)
    wrong = int((q != want).sum())
    assert wrong == 0, (wrong, q.numel())
