"""Every kernel that a product in 8 bits may take, with every type of result and both kinds of b's scales, against 64 bits: which kernel a shape takes is
asked of the profiler, so that a change of the rule that leaves one without a test is noticed."""
import re

import pytest
import torch

import protenix_amd as P
from tests import fp8_oracle as Q
from tests.residual_oracle import half_step, smallest

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAMES = {F32: ("float", "f"), BF16: ("__bf16", "DF16b"), F16: ("_Float16", "DF16_")}
# tiles of 64 x 64 with k in parts and without, two workgroups of them to a compute unit, 128 x 128 with k shared by waves and without, 256 x 128,
# 192 x 256, 256 x 256; of those whose workgroups walk over tiles one shape with fewer tiles than workgroups and one with more; odd sizes
SHAPES = [(70, 300, 130), (130, 9001, 100), (1300, 300, 1290), (1600, 200, 1500), (100, 130, 40000), (2500, 260, 2600), (100000, 130, 100), (4100, 260, 4100),
          (2900, 130, 2950), (4500, 300, 4600), (3000, 300, 4100), (8300, 130, 8300)]
# up to 16 rows: one, two and four blocks at a time
FEW = [(1, 128, 70), (5, 1100, 130), (16, 2100, 70), (1, 3100, 130), (5, 4096, 130), (16, 8200, 130), (1, 12300, 70)]
# (rows and columns of a tile, waves along both, groups that share k, buffers)
TILES = {(64, 64, 4, 1, 2, 4), (64, 64, 4, 1, 2, 2), (128, 128, 2, 2, 2, 2), (128, 128, 2, 2, 1, 2)}
TILES16 = TILES | {(256, 128, 4, 2, 1, 2), (192, 256, 2, 4, 1, 2), (256, 256, 2, 4, 1, 2)}


def _operand(m, k, seed, square=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=g) * torch.randn((m, 1), generator=g).mul(0.7).exp() * torch.randn((1, k), generator=g).mul(0.7).exp()
    return P.quantize_fp8(x.cuda(), square=square)


def _check(a, b, dtype):
    got = P.matmul_fp8(a, b, dtype=dtype)
    ad, bd = (t.values.double() * Q.spread(t.scales.double(), t.values.shape, t.square) for t in (a, b))
    want = torch.mm(ad, bd.t().contiguous())
    if dtype == F16 and want.abs().max() > 60000:      # (half has no such numbers)
        ad, want = ad / 2**8, want / 2**8
        got = P.matmul_fp8(P.Fp8Tensor(a.values, a.scales / 2**8), b, dtype=dtype)
    size = torch.mm(ad.abs(), bd.abs().t().contiguous())
    blocks = -(-ad.shape[1] // 128)
    # as product_bound(), the largest of 8 neighbouring products taken as no more than their sum
    lost = 2.0**-16 + (blocks + 3) * 2.0**-24 + (0 if dtype == F32 else 7 * 2.0**-13)
    off = (got.double() - want).abs()
    tol = lost * size + half_step(dtype) * want.abs() + smallest(dtype)
    assert (off <= tol).all(), (ad.shape, bd.shape, (off / tol).max().item(), (off > tol).sum().item())


def _launched(profile):
    """(what, template arguments) of the products' kernels."""
    found = set()
    for name in {e.name for e in profile.events()}:
        what = re.search(r"fp8_(tile_product|few_rows_product|join_kernel)", name)
        if what:
            numbers = re.findall(r"Li(\d+)E", name) or re.findall(r"(\d+),", name.split(what.group(0))[1])
            by_row = bool(re.search(r"Lb1E|true", name))
            kind = next(t for t, (plain, short) in NAMES.items() if re.search(rf"[<, ]{plain}>|[EI]{short}E", name))
            found.add((what.group(1), tuple(int(n) for n in numbers), by_row, kind))
    return found


@pytest.mark.parametrize("square", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_every_kernel_is_right(dtype, square):
    operands = [(_operand(m, k, 1), _operand(n, k, 2, square)) for m, k, n in SHAPES + FEW]
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU, torch.profiler.ProfilerActivity.CUDA]) as profile:
        for a, b in operands:
            P.matmul_fp8(a, b, dtype=dtype)
        torch.cuda.synchronize()
    tiles = TILES16 if dtype != F32 else TILES if square else TILES - {(64, 64, 4, 1, 2, 2)}
    want = {("tile_product", tile, not square, dtype) for tile in tiles} | {("join_kernel", (), False, dtype)}
    if square:
        want.add(("few_rows_product", (), False, dtype))
    got = _launched(profile)
    assert got == want, (want - got, got - want)
    for a, b in operands:
        _check(a, b, dtype)
