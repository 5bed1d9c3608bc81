"""What the 8-bit operators promise beside their results: gradients that are not lost, bounds of sums, bits of scales."""
import pytest
import torch
from torch.autograd import forward_ad

import protenix_amd as P
from protenix_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_quantizing_loses_no_gradient(native, monkeypatch):
    """What passes a gradient on is refused, in every direction; leaves, and what is detached or not recorded, are taken."""
    monkeypatch.setattr(ops, "native_enabled", native)
    w = torch.randn((130, 200), device="cuda", requires_grad=True)
    want = P.quantize_fp8(w.detach(), square=True)
    ways = [dict(), dict(along=-2), dict(along=(-1, -2)), dict(square=True)]
    for way in ways:
        for x in (w * 1.0, w[:64], w.t()):
            with pytest.raises(RuntimeError, match="no gradients"):
                P.quantize_fp8(x, **way)
            P.quantize_fp8(x.detach(), **way)
            with torch.no_grad():
                P.quantize_fp8(x, **way)
        with forward_ad.dual_level():
            x = forward_ad.make_dual(w.detach(), torch.ones_like(w))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    P.quantize_fp8(x, **way)
            P.quantize_fp8(w.detach(), **way)
    got = P.quantize_fp8(w, square=True)
    assert torch.equal(got.scales, want.scales) and torch.equal(got.values.view(torch.uint8), want.values.view(torch.uint8))


@pytest.mark.parametrize("native", [True, False])
def test_operands_of_parameters(native, monkeypatch):
    """A checkpoint's blocks as leaves are copied without a graph; what passes a gradient on is refused."""
    monkeypatch.setattr(ops, "native_enabled", native)
    q = P.quantize_fp8(torch.randn((130, 200), device="cuda"), square=True)
    scales = q.scales.clone().requires_grad_()
    t = P.Fp8Tensor(q.values.clone(), scales, square=True)
    assert not t.scales.requires_grad and torch.equal(t.scales, q.scales) and t.scales.data_ptr() != scales.data_ptr()
    with pytest.raises(RuntimeError, match="no gradients"):
        P.Fp8Tensor(q.values, scales * 1.0, square=True)
    with torch.no_grad():
        P.Fp8Tensor(q.values, scales * 1.0, square=True)
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        P.Fp8Tensor(q.values, forward_ad.make_dual(q.scales, q.scales.clone()), square=True)
