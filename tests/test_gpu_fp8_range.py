"""Products in 8 bits of operands at the ends of fp32's range: the product of a block's two scales lies beyond it where the result does not."""
import pytest
import torch

import protenix_amd as P
from tests import fp8_oracle as Q
from tests.residual_oracle import half_step, smallest

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
# one of every kernel, with 16-bit and with fp32 results: few rows, 64 x 64 with and without parts of k and with two workgroups to a compute unit,
# 128 x 128 with k shared by waves and without, 256 x 128, 192 x 256, 256 x 256; odd sizes, more tiles than workgroups, a last block of a few columns
SHAPES = [(1, 300, 70), (13, 4300, 33), (70, 300, 130), (130, 9001, 100), (1300, 300, 1290), (1600, 200, 1500), (2500, 260, 2600), (2900, 130, 2950),
          (3000, 300, 4100), (4500, 300, 4600), (100, 130, 40000), (100000, 130, 100), (4100, 260, 4100), (8300, 130, 8300)]


def _operand(rows, cols, square, seed, odd):
    """Values of all sizes with scales from one end of the range to the other; every fourth row has values at even (odd) columns alone."""
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn((rows, cols), generator=g) * torch.randn((rows, 1), generator=g).exp() * 40).clamp(-448, 448)
    q[odd::4, 1 - odd::2] = 0
    lead, blocks = -(-rows // 128) if square else rows, -(-cols // 128)
    ends = torch.tensor([-126, -110, -80, -64, -40, 0, 40, 64, 100])
    s = torch.rand((lead, blocks), generator=g).add(1) * 2.0 ** ends[torch.randint(len(ends), (lead, blocks), generator=g)]
    return P.Fp8Tensor(q.to(torch.float8_e4m3fn).cuda(), s.float().cuda(), square=square)


def _held(t):
    q, s = t.values.double(), t.scales.double()
    return q * Q.spread(s, q.shape, t.square)


def _check(got, a, b):
    """Against 64 bits, where no block's products reach fp32's end."""
    ad, bd = _held(a), _held(b)
    dtype, blocks = got.dtype, -(-ad.shape[1] // 128)
    want, size = torch.mm(ad, bd.t().contiguous()), torch.mm(ad.abs(), bd.abs().t().contiguous())
    # as product_bound(), the largest of 8 neighbouring products taken as no more than their sum; two roundings of a block's result at
    # the lower end, each by half of the smallest number
    lost = 2.0**-16 + (blocks + 4) * 2.0**-24 + (0 if dtype == F32 else 7 * 2.0**-13)
    tol = lost * size + half_step(dtype) * want.abs() + smallest(dtype) + (blocks + 1) * 2.0**-148
    # a block whose scale is 2^-126 or less (values below 448 2^-126): the product of the scales may be off by 2^-150, its sum is below 2^25
    least = lambda t: (t.scales <= 2.0**-126).sum(-1).repeat_interleave(128 if t.square else 1)[:t.shape[0]]
    tol = tol + torch.maximum(least(a)[:, None], least(b)[None, :]) * 2.0**-125
    inside = size < 2.0**126
    off = (got.double() - want).abs()
    bad = inside & ~(off <= tol)
    assert inside.float().mean() > 0.02 and not bad.any(), (bad.sum().item(), got[bad][:4], want[bad][:4])
    return inside


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("square", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scales_of_all_sizes(shape, square, dtype):
    m, k, n = shape
    a, b = _operand(m, k, False, sum(shape), 0), _operand(n, k, square, sum(shape) + 1, 1)
    got = P.matmul_fp8(a, b, dtype=dtype)
    _check(got, a, b)
    # values at columns that the other operand has none at: 0, whatever the scales
    assert (got[::4, 1::4] == 0).all()


@pytest.mark.parametrize("m", [5, 70])
def test_scales_whose_product_is_infinite(m):
    """Blocks of a with 1e24 and 1e19 against a block of b with 1e20 and 1e15, where the large values do not meet."""
    x, w = torch.zeros((m, 128), device="cuda"), torch.zeros((130, 128), device="cuda")
    x[:, 0], x[:, 1] = 1e24, 1e19
    w[3, 2], w[4, 1] = 1e20, 1e15
    a = P.quantize_fp8(x)
    for square in (True, False):
        b = P.quantize_fp8(w, square=square)
        got = P.matmul_fp8(a, b, dtype=F32)
        assert _check(got, a, b).all()
        # (1e19 beside 1e24, and 1e15 beside 1e20 in a square block, are 2.29 steps of 2^-9 of the largest / 448: 2 of them, 0.872 of the value)
        assert (got[:, 4] > (7.5e33 if square else 8.6e33)).all()
        assert (got[:, [i for i in range(130) if i != 4]] == 0).all()


@pytest.mark.parametrize("m", [3, 300])
@pytest.mark.parametrize("size", [(1e-18, 1e-19), (1e-19, 1e-19), (1e-30, 1e-8), (1e-36, 1e-1), (1e30, 1e-36), (1e18, 1e17)])
def test_sizes_of_operands(m, size):
    g = torch.Generator().manual_seed(m)
    x, w = (torch.randn(s, generator=g).mul(v).cuda() for s, v in zip(((m, 1024), (200, 1024)), size))
    for square in (True, False):
        a, b = P.quantize_fp8(x), P.quantize_fp8(w, square=square)
        assert _check(P.matmul_fp8(a, b, dtype=F32), a, b).all()


@pytest.mark.parametrize("square", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_row_has_the_same_bits_beside_any_scales(square, dtype):
    """Rows and columns of ordinary scales beside others', and beside what lies behind the last row."""
    for m, k, n in ((14, 300, 130), (62, 4300, 50), (302, 300, 290), (1602, 300, 1502), (2502, 260, 2602), (2902, 130, 2950)):
        g = torch.Generator().manual_seed(m)
        a = P.quantize_fp8(torch.randn((m, k), generator=g).cuda())
        b = P.quantize_fp8(torch.randn((n, k), generator=g).cuda(), square=square)
        want = P.matmul_fp8(a, b, dtype=dtype)
        for extreme in (2.0**-70, 2.0**-120, 2.0**-126, 2.0**100, 2.0**125, 0.0, float("nan"), float("inf")):
            other = P.Fp8Tensor(a.values, torch.where((torch.arange(m, device="cuda") % 3 == 1)[:, None], extreme, a.scales))
            if extreme < 1:
                other._operand[1][:, m:] = 2.0**-126      # (read along with the others)
            rest = torch.arange(m, device="cuda") % 3 != 1
            assert torch.equal(P.matmul_fp8(other, b, dtype=dtype)[rest], want[rest])
            if not square:
                columns = P.Fp8Tensor(b.values, torch.where((torch.arange(n, device="cuda") % 3 == 1)[:, None], extreme, b.scales))
                keep = torch.arange(n, device="cuda") % 3 != 1
                assert torch.equal(P.matmul_fp8(a, columns, dtype=dtype)[:, keep], want[:, keep])


def test_scales_of_zero_and_below():
    g = torch.Generator().manual_seed(0)
    q = torch.randn((40, 256), generator=g).mul(50).to(torch.float8_e4m3fn).cuda()
    s = torch.randn((40, 2), generator=g).cuda()
    s[3], s[5, 0], s[7] = 0, -(2.0**-126), 2.0**-140
    a = P.Fp8Tensor(q, s)
    for scale in (1.0, -(2.0**127), 2.0**-149):
        b = P.Fp8Tensor(q, torch.full((1, 2), scale, device="cuda"), square=True)
        for operand in (a, P.Fp8Tensor(q[:9], s[:9])):
            got = P.matmul_fp8(operand, b, dtype=F32)
            assert (got[3] == 0).all()
            _check(got, operand, b) if scale != -(2.0**127) else None
