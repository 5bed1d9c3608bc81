"""What the 8-bit operators promise beside their results: gradients that are not lost, bounds of sums, bits of scales."""
import pytest
import torch
from torch.autograd import forward_ad

import protenix_amd as P
from protenix_amd import ops
from tests import fp8_oracle as Q
from tests.residual_oracle import half_step, smallest

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


def test_scales_and_their_inverses_at_every_mantissa():
    """s = a / 448 and i = 1 / s are each rounded once: for all 2^23 mantissas of a, s itself, and i by values that lie where one unit of i
    decides between two numbers of 8 bits."""
    ties = torch.arange(17, 32, 2, dtype=torch.float64, device="cuda")      # in the middle of two e4m3 numbers
    steps = torch.arange(-7, 8, dtype=torch.int32, device="cuda")
    told = 0
    for first in range(0, 1 << 23, 1 << 18):
        a = (torch.arange(first, first + (1 << 18), dtype=torch.int32, device="cuda") + (140 << 23)).view(torch.float32)
        s = (a.double() / 448).float()
        i = (1 / s.double()).float()
        near = (ties[None, :] / i.double()[:, None]).float()
        x = torch.zeros((1 << 18, 128), device="cuda")
        x[:, 0] = a
        x[:, 1:121] = (near.view(torch.int32)[:, :, None] + steps).view(torch.float32).reshape(1 << 18, 120)
        t = P.quantize_fp8(x)
        assert torch.equal(t.scales[:, 0], s), first
        rounded = lambda inverse: Q.round_e4m3((x.double() * inverse.double()[:, None]).float().double()).float()
        want = rounded(i)
        assert torch.equal(t.values.float(), want), first
        for unit in (-1, 1):
            told += (rounded((i.view(torch.int32) + unit).view(torch.float32)) != want).any(1).sum().item()
    assert told > 1.9 * 2**23, told / 2**23      # (an inverse off by a unit either way shows)


@pytest.mark.parametrize("shape", [(5, 1024, 96), (70, 1000, 130), (300, 1024, 290), (1300, 500, 1290), (2500, 256, 2600), (3000, 256, 4100)])
@pytest.mark.parametrize("square", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_large_products_that_cancel(shape, square, dtype):
    """Channels that stand out, two of each 8, whose products cancel: results in 16 bits are off by no more than is said of them (each of
    the other products of a group by 2^-13 of its largest), those in fp32 by no more than fp32 sums are."""
    m, k, n = shape
    g = torch.Generator().manual_seed(sum(shape))
    x, w = torch.randn((m, k), generator=g), torch.randn((n, k), generator=g)
    x[:, ::8] *= 100
    x[:, 3::8] = -x[:, ::8][:, :x[:, 3::8].shape[1]]
    w[:, 3::8] = w[:, ::8][:, :w[:, 3::8].shape[1]]
    a, b = P.quantize_fp8(x.cuda()), P.quantize_fp8(w.cuda(), square=square)
    ad, bd = Q.held_by(a), Q.held_by(b)
    got = P.matmul_fp8(a, b, dtype=dtype).cpu().double()
    want = torch.mm(ad, bd.t().contiguous())
    off, said = (got - want).abs(), half_step(dtype) * want.abs() + smallest(dtype)
    size = torch.mm(ad.abs(), bd.abs().t().contiguous())
    blocks = -(-k // 128)
    said = said + (2.0**-16 + (blocks + 3) * 2.0**-24) * size
    if dtype != torch.float32:
        # the largest of a group of 8 is one of the two that stand out, or no more than the sum of the others
        rest = torch.ones(k, dtype=torch.bool)
        rest[::8] = rest[3::8] = False
        one = torch.mm(ad[:, ::8].abs(), bd[:, ::8].abs().t().contiguous())
        said = said + 7 * 2.0**-13 * (one + torch.mm(ad[:, rest].abs(), bd[:, rest].abs().t().contiguous()))
    assert (off <= said).all(), ((off / said).max().item(), (off > said).sum().item())


@pytest.mark.parametrize("leaf", ["x", "w", "b"])
def test_each_gradient_against_differences(leaf):
    """Along a leaf's own direction (it times 1 + t, which moves its scales alone): dy close to y makes the slopes as large as their
    share of the sum of magnitudes, that of b is exact but for fp32, and neither allows a gradient that is 0 or has the wrong sign."""
    g = torch.Generator().manual_seed(7)
    x, w, b = (torch.randn(s, generator=g).mul(v).cuda().requires_grad_() for s, v in (((130, 256), 1.0), ((140, 256), 0.1), ((140,), 1.0)))
    y = P.linear_fp8(x, w, b)
    dy = y.detach() + 0.1 * torch.randn(y.shape, generator=g).cuda()
    grads = dict(zip("xwb", torch.autograd.grad(y, (x, w, b), dy)))
    leaves, t = dict(x=x.detach(), w=w.detach(), b=b.detach()), 2.0**-3
    value = lambda s: (P.linear_fp8(*(v * s if n == leaf else v for n, v in leaves.items())).double() * dy.double()).sum().item()
    slope = (value(1 + t) - value(1 - t)) / (2 * t)
    got = (grads[leaf].double() * leaves[leaf].double()).sum().item()
    xd, wd, dd = leaves["x"].double(), leaves["w"].double(), dy.double()
    size = (y.double() * dd).abs().sum().item()
    # two values of y in fp32 on either side, off by half a step and the 2^-16 of their sums' magnitudes (product_bound()); db's own additions
    magnitudes = torch.mm(xd.abs(), wd.abs().t().contiguous())
    if leaf == "b":
        # (what the products are off by is the same on both sides)
        tol = 2.0**-23 * ((magnitudes + y.double().abs()) * dd.abs()).sum().item() / t + 140 * 2.0**-24 * (dd.abs().sum(0) * leaves["b"].double().abs()).sum().item()
    else:
        # dx and dW take dy in 8 bits, x and W as blocks along other axes or in full: a rounding is off by at most half a step, evenly on both
        # sides of 0, so by a third of its square in the mean; 8 times the deviation of all of them, and 2^-10 for slopes of their density
        step = lambda v: 2.0**-4 * v.abs() + 2.0**-18 * v.abs().max()
        spread = [(step(dd) * torch.mm(xd, wd.t().contiguous())), (step(xd) * torch.mm(dd, wd)), (step(wd) * torch.mm(dd.t().contiguous(), xd))]
        tol = 8 * sum(v.square().sum().item() / 3 for v in spread)**0.5 * 2**0.5 + 2.0**-10 * size
    assert abs(slope - got) <= tol, (slope, got, tol)
    # (of y's variance 256 0.1^2 = 2.56 is the products', 1 the bias': 0.72 and 0.28 of it)
    assert abs(slope) > 8 * tol and abs(slope) > (0.2 if leaf == "b" else 0.6) * size, (slope, tol, size)


@pytest.mark.parametrize("native", [True, False])
def test_gradients_over_more_rows_than_a_product_sums_are_refused_in_front(native, monkeypatch):
    """Before anything is launched, not in the backward pass."""
    monkeypatch.setattr(ops, "native_enabled", native)
    long = torch.zeros((1, 8), dtype=torch.bfloat16, device="cuda").expand((1 << 24) + 1, 8)
    short = torch.zeros((3, 8), dtype=torch.bfloat16, device="cuda")
    for x, w in ((long, short.clone().requires_grad_()), (short.clone().requires_grad_(), long)):
        before = torch.cuda.memory_allocated()
        with pytest.raises(RuntimeError, match="at most 16777216"):
            P.linear_fp8(x, w)
        assert torch.cuda.memory_allocated() == before
