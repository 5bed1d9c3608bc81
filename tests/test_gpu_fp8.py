"""8-bit blocks and their products against 64-bit forms: layouts, roundings, gradients, sizes on all sides of the tiles."""
import threading

import pytest
import torch
from torch.autograd import forward_ad

import protenix_amd as P
from protenix_amd import ops
from tests import fp8_oracle as Q
from tests.residual_oracle import half_step, smallest

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def _matrix(m, k, dtype, seed=0, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=g)
    if spread:      # rows and columns of different sizes
        x = x * torch.randn((m, 1), generator=g).exp() * torch.randn((1, k), generator=g).exp()
    return x.to(dtype).cuda()


def _same(t: P.Fp8Tensor, x: torch.Tensor, square=False):
    q, s = Q.quantize(x, square)
    assert t.values.dtype == torch.float8_e4m3fn and t.values.shape == x.shape and t.square == square
    assert torch.equal(t.scales.cpu().double(), s)
    assert torch.equal(t.values.cpu().float().double(), q)


SHAPES = [(1, 1), (1, 128), (1, 2048), (2, 7), (3, 8), (5, 9), (127, 127), (128, 128), (129, 129), (130, 255), (257, 136), (64, 1411),
          (999, 64), (300, 640), (17, 130)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize_every_way(shape, dtype):
    x = _matrix(*shape, dtype, sum(shape))
    for square in (False, True):
        rows, cols = P.quantize_fp8(x, square=square, along=(-1, -2))
        _same(rows, x, square)
        _same(cols, x.t(), square)
        _same(P.quantize_fp8(x, square=square), x, square)
        _same(P.quantize_fp8(x, square=square, along=-2), x.t(), square)
        # (what stands behind the last column is read by products)
        for t in (rows, cols):
            assert (t._operand[0].view(torch.uint8)[:, t.shape[1]:-(-t.shape[1] // 128) * 128] & 0x7f == 0).all()


def test_quantize_more_dimensions_and_strides():
    x = _matrix(30, 300, BF16).view(5, 6, 300)
    t = P.quantize_fp8(x)
    assert t.shape == x.shape and t.values.shape == x.shape and t.scales.shape == (5, 6, 3)
    q, s = Q.quantize(x.view(30, 300))
    assert torch.equal(t.values.cpu().float().double().view(30, 300), q) and torch.equal(t.scales.cpu().double().view(30, 3), s)
    assert P.quantize_fp8(x, along=-2).shape == (300, 30)
    wide = _matrix(64, 400, F32)
    for view in (wide.t(), wide[::2], wide[:, 3:200], wide[:, ::3]):
        _same(P.quantize_fp8(view), view)
        _same(P.quantize_fp8(view, along=-2), view.t())
    row = _matrix(1, 200, F16)[0]
    assert P.quantize_fp8(row).values.shape == (200,) and P.quantize_fp8(row).scales.shape == (2,)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_extremes(dtype):
    """Zeros, the smallest and largest values, values between two e4m3 ones, blocks far apart in size."""
    top = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    x = torch.zeros((9, 256), dtype=dtype)
    x[1, :] = tiny
    x[2, 5] = top
    x[3, :128] = torch.linspace(-448, 448, 128).to(dtype)
    x[4, 130] = -tiny
    x[5, :] = top
    x[6, :128] = torch.arange(128).to(dtype) / 512 * 3.5      # many lie in the middle of two
    x[6, 0] = 448
    x[7, :] = -0.0
    x[8, ::2] = 2.0**-14
    x = x.cuda()
    _same(P.quantize_fp8(x), x)
    _same(P.quantize_fp8(x, along=-2), x.t())
    for square in (True,):
        a, b = P.quantize_fp8(x, square=square, along=(-1, -2))
        _same(a, x, True)
        _same(b, x.t(), True)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_blocks_that_are_not_finite_stay_that(bad):
    """Their products are not finite, and no other block's are touched."""
    x, w = _matrix(70, 300, F32, spread=False), _matrix(130, 300, F32, 1, spread=False)
    clean = P.linear_fp8(x, w)
    x2 = x.clone()
    x2[33, 200] = bad
    out = P.linear_fp8(x2, w)
    rest = [i for i in range(70) if i != 33]
    assert not out[33].isfinite().any() and torch.equal(out[rest], clean[rest])
    few = P.linear_fp8(x2[30:40], w)
    assert not few[3].isfinite().any() and torch.equal(few[[0, 1, 2, 4]], P.linear_fp8(x[30:40], w)[[0, 1, 2, 4]])
    # in a weight: the outputs of its 128 rows
    w2 = w.clone()
    w2[129, 0] = bad
    out = P.linear_fp8(x, w2)
    assert not out[:, 128:].isfinite().any() and torch.equal(out[:, :128], clean[:, :128])
    for axis in (-1, -2):
        t = P.quantize_fp8(x2, along=axis)
        assert (~t.scales.isfinite()).sum() == 1


# rows of a on both sides of the kernels' borders (16 rows at a time up to 64, tiles of 64, 128, 256), odd columns and blocks
PRODUCTS = [(1, 128, 16), (1, 2048, 1000), (2, 100, 17), (15, 384, 130), (16, 1000, 128), (17, 130, 64), (33, 1, 1), (48, 129, 200),
            (64, 640, 257), (65, 640, 257), (65, 64, 3), (100, 4096, 72), (128, 128, 128), (200, 8200, 136), (257, 513, 300),
            (1035, 1000, 777), (1536, 256, 1792), (4100, 128, 520), (3000, 130, 4100), (40, 150001, 70),
            (130, 20000, 17), (1300, 300, 1290), (1600, 200, 1500), (2500, 129, 2600),
            (2900, 130, 2950), (4500, 64, 4600), (70, 20000, 3), (20, 20000, 1)]


def _check_product(got, a, b, bias=None):
    want = a @ b.t() + (0 if bias is None else bias.detach().cpu().double())
    tol = Q.product_bound(a, b, got.dtype) + half_step(got.dtype) * want.abs() + smallest(got.dtype)
    if bias is not None:
        tol = tol + 2.0**-23 * want.abs()
    off = (got.detach().cpu().double() - want).abs()
    assert (off <= tol).all(), ((off / tol).max().item(), (off > tol).sum().item())


@pytest.mark.parametrize("shape", PRODUCTS)
@pytest.mark.parametrize("square", [True, False])
def test_products(shape, square):
    m, k, n = shape
    a, b = P.quantize_fp8(_matrix(m, k, BF16, 1)), P.quantize_fp8(_matrix(n, k, BF16, 2), square=square)
    ad, bd = Q.held_by(a), Q.held_by(b)
    bias = torch.randn(n).cuda()
    for dtype in TYPES if m * n < 1 << 20 else (BF16,):
        if dtype == F16 and (ad @ bd.t()).abs().max() > 60000:
            continue
        got = P.matmul_fp8(a, b, dtype=dtype)
        assert got.dtype == dtype and got.shape == (m, n)
        _check_product(got, ad, bd)
        _check_product(P.matmul_fp8(a, b, bias.to(dtype), dtype=dtype), ad, bd, bias.to(dtype))


def test_products_behind_each_other_and_twice_are_the_same():
    for m in (3, 70, 700, 2600):
        a, b = P.quantize_fp8(_matrix(m, 1000, BF16, 1)), P.quantize_fp8(_matrix(2700, 1000, BF16, 2), square=True)
        first = P.matmul_fp8(a, b)
        for _ in range(5):
            assert torch.equal(P.matmul_fp8(a, b), first)


def test_operands_of_a_checkpoint():
    x, w = _matrix(40, 500, BF16, 1), _matrix(300, 500, BF16, 2)
    a, b = P.quantize_fp8(x), P.quantize_fp8(w, square=True)
    given = P.Fp8Tensor(b.values.clone(), b.scales.clone(), square=True)
    mine = P.Fp8Tensor(a.values.clone(), a.scales.clone())
    assert torch.equal(P.matmul_fp8(mine, given), P.matmul_fp8(a, b))
    assert torch.equal(mine.values.view(torch.uint8), a.values.view(torch.uint8)) and torch.equal(mine.scales, a.scales)
    # any scales, of either sign
    s = torch.randn((40, 4)).cuda()
    t = P.Fp8Tensor(a.values, s)
    _check_product(P.matmul_fp8(t, b, dtype=F32), Q.held_by(t), Q.held_by(b))
    batch = P.Fp8Tensor(a.values.reshape(5, 8, 500), a.scales.reshape(5, 8, 4))
    assert torch.equal(P.matmul_fp8(batch, b), P.matmul_fp8(a, b).view(5, 8, 300))


def _train(m, k, n, tx=BF16, tw=None, tb=None, seed=0, lead=None):
    x = _matrix(m, k, tx, seed, spread=False)
    x = (x if lead is None else x.view(*lead, k)).requires_grad_()
    w = _matrix(n, k, tw or tx, seed + 1, spread=False).requires_grad_()
    b = None if tb is None else _matrix(1, n, tb, seed + 2, spread=False)[0].requires_grad_()
    dy = _matrix(m, n, tx, seed + 3)
    return x, w, b, dy if lead is None else dy.view(*lead, n)


def _check_training(x, w, b, dy):
    y = P.linear_fp8(x, w, b)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    assert [g.dtype for g in grads] == [t.dtype for t in leaves] and [g.shape for g in grads] == [t.shape for t in leaves]
    xm, dm = x.detach().reshape(-1, x.shape[-1]), dy.reshape(-1, dy.shape[-1])
    wd = Q.held(w, True)
    _check_product(y.reshape(-1, y.shape[-1]), Q.held(xm), wd, b)
    _check_product(grads[0].reshape(xm.shape), Q.held(dm), wd.t())
    _check_product(grads[1], Q.held(dm.t()), Q.held(xm.t()))
    if b is not None:
        d = dm.cpu().double()
        # at most 128 additions in a tile and one per tile after it, each off by half a step of at most the sum of magnitudes
        tol = (128 + d.shape[0] / 128 + 8) * 2.0**-24 * d.abs().sum(0) + half_step(b.dtype) * d.sum(0).abs() + smallest(b.dtype)
        assert ((grads[2].cpu().double() - d.sum(0)).abs() <= tol).all()


@pytest.mark.parametrize("shape", [(1, 128, 128), (1, 5, 3), (3, 200, 17), (64, 384, 300), (129, 1000, 77), (300, 130, 520), (1035, 257, 384)])
@pytest.mark.parametrize("types", [(F32, F32, F32), (BF16, BF16, None), (F16, F16, F16), (BF16, F32, F32)])
def test_linear_and_its_gradients(shape, types):
    _check_training(*_train(*shape, *types, seed=sum(shape)))


def test_linear_of_batches_and_strides():
    _check_training(*_train(90, 200, 60, lead=(3, 5, 6)))
    x, w, _, dy = _train(90, 200, 60)
    turned = x.detach().t().contiguous().t().requires_grad_()
    y = P.linear_fp8(turned, w.detach().t().contiguous().t())
    assert torch.equal(y, P.linear_fp8(x.detach(), w.detach()))
    # a gradient that is a view: of a sum, every element the same
    s = P.linear_fp8(turned, w).sum()
    g = torch.autograd.grad(s, turned)[0]
    assert torch.equal(g, torch.autograd.grad(P.linear_fp8(x, w), x, torch.ones_like(dy))[0])


def test_linear_under_autocast():
    x, w, b, dy = _train(30, 200, 60, F32, F32, F32)
    for dtype in (BF16, F16):
        with torch.autocast("cuda", dtype=dtype):
            y = P.linear_fp8(x, w, b)
            assert y.dtype == dtype and P.linear_fp8(x.to(BF16), w).dtype == BF16
            assert P.linear_fp8(x, w, b, dtype=F32).dtype == F32
        assert torch.equal(y, P.linear_fp8(x, w, b, dtype=dtype))
        assert [g.dtype for g in torch.autograd.grad(y, (x, w, b), dy.to(dtype))] == [F32] * 3


def test_linear_frozen_inputs():
    x, w, b, dy = _train(150, 200, 130, tb=F32)
    full = torch.autograd.grad(P.linear_fp8(x, w, b), (x, w, b), dy)
    for mask in range(1, 7):
        some = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((x, w, b))]
        grads = torch.autograd.grad(P.linear_fp8(*some), [t for t in some if t.requires_grad], dy)
        assert all(torch.equal(g, full[i]) for g, i in zip(grads, [i for i in range(3) if mask >> i & 1]))


def test_gradients_against_differences():
    """The directional derivative of the product of what the operands stand for: along steps that move only the scales (a matrix
    times 1 + t), the rounding stands still and the product is exactly linear."""
    x, w, b, dy = _train(130, 256, 140, F32, F32, F32, seed=5)
    y = P.linear_fp8(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), dy)
    t = 2.0**-3
    value = lambda xs, ws, bs: (P.linear_fp8(x.detach() * xs, w.detach() * ws, b.detach() * bs).double() * dy.double()).sum().item()
    size = (y.double() * dy.double()).abs().sum().item()
    # (dx and dW come from dy in 8 bits and x along another axis: each value off by at most half a step, 2^-4, at random, so that the
    # sum over 130 x 140 x 256 products with two roundings is off by far less than 2^-4 of the sum of its magnitudes / 2^5)
    for (got, leaf), args in zip(((gx, x), (gw, w), (gb, b)), ((1, 0, 0), (0, 1, 0), (0, 0, 1))):
        slope = (value(*(1 + t * a for a in args)) - value(*(1 - t * a for a in args))) / (2 * t)
        want = (got.double() * leaf.detach().double()).sum().item()
        assert abs(slope - want) < 2.0**-9 * size, (slope, want, size)


def test_empty_sizes():
    w = _matrix(30, 200, BF16).requires_grad_()
    x = torch.empty((0, 200), dtype=BF16, device="cuda", requires_grad=True)
    b = torch.ones(30, device="cuda", requires_grad=True)
    y = P.linear_fp8(x, w, b)
    assert y.shape == (0, 30)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert gx.shape == (0, 200) and gw.shape == w.shape and (gw == 0).all() and (gb == 0).all()
    none = torch.empty((0, 200), dtype=BF16, device="cuda", requires_grad=True)
    y = P.linear_fp8(w, none)
    assert y.shape == (30, 0)
    gx, gw = torch.autograd.grad(y, (w, none), torch.empty_like(y))
    assert (gx == 0).all() and gw.shape == (0, 200)
    t = P.quantize_fp8(x.detach())
    assert t.values.shape == (0, 200) and t.scales.shape == (0, 2)
    assert P.matmul_fp8(t, P.quantize_fp8(w.detach(), square=True)).shape == (0, 30)
    again = P.Fp8Tensor(t.values, t.scales)
    assert again.values.shape == (0, 200) and P.matmul_fp8(again, P.quantize_fp8(w.detach(), square=True)).shape == (0, 30)


def test_workspaces_hold_nothing(monkeypatch):
    """Results do not depend on what the workspaces held."""
    x, w, b, dy = _train(300, 4096, 136, tb=F32)
    first = torch.autograd.grad(P.linear_fp8(x, w, b), (x, w, b), dy)
    y = P.linear_fp8(x.detach(), w.detach(), b.detach())
    monkeypatch.setattr(ops, "poison_workspaces", True)
    assert torch.equal(P.linear_fp8(x.detach(), w.detach(), b.detach()), y)
    assert all(torch.equal(a, c) for a, c in zip(first, torch.autograd.grad(P.linear_fp8(x, w, b), (x, w, b), dy)))


def test_python_and_native_paths_give_the_same_bits(monkeypatch):
    for types in ((BF16, F32, F32), (F32, F32, None), (F16, F16, F16)):
        x, w, b, dy = _train(90, 200, 60, *types, lead=(3, 5, 6))

        def every():
            y = P.linear_fp8(x, w, b)
            wq = P.quantize_fp8(w, square=True)
            pair = P.quantize_fp8(x, along=(-1, -2))
            with torch.no_grad():
                served = P.linear_fp8(x, wq, b, dtype=F16), P.matmul_fp8(pair[0], wq, b), P.linear_fp8(x, w)
            return (y, *torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], dy), *served,
                    *(u for t in (wq, *pair) for u in (t.values.view(torch.uint8), t.scales)))

        first = every()
        with monkeypatch.context() as m:
            m.setattr(ops, "native_enabled", False)
            second = every()
        assert len(first) == len(second) and all(a.shape == c.shape and a.dtype == c.dtype and torch.equal(a, c) for a, c in zip(first, second))


def test_rows_behind_the_last_are_left_alone():
    """Nothing outside the results is written."""
    lib, dev = ops._lib.load(), "cuda"
    for m, n, k in ((5, 21, 130), (70, 130, 300), (300, 300, 300)):
        a, b = P.quantize_fp8(_matrix(m, k, BF16)), P.quantize_fp8(_matrix(n, k, BF16, 1), square=True)
        room = torch.full((m * n + 512,), 7.0, device=dev)
        ws = torch.empty((max(lib.ptx_fp8_matmul_workspace_elems(m, n, k, 1, 0), 1),), device=dev)
        ops._lib.check(lib.ptx_fp8_matmul(a._operand[0].data_ptr(), a._operand[1].data_ptr(), b._operand[0].data_ptr(), b._operand[1].data_ptr(),
                                          1, None, room.data_ptr() + 4 * 256, ws.data_ptr(), m, n, k, 0, 0, ops._stream()), "matmul")
        assert (room[:256] == 7).all() and (room[256 + m * n:] == 7).all()
        assert torch.equal(room[256:256 + m * n].view(m, n), P.matmul_fp8(a, b, dtype=F32))
        x = _matrix(m, k, F32)
        rows, cols = P.quantize_fp8(x, along=(-1, -2))
        for t, at in ((rows, 0), (cols, 2)):
            data, scales = t._operand[:2]
            blocks = -(-t.shape[1] // 128) * 128
            q = torch.full((data.numel() + 512,), 9, dtype=torch.uint8, device=dev)
            s = torch.full((scales.numel() + 512,), 9.0, device=dev)
            ptrs = [None] * 4
            ptrs[at], ptrs[at + 1] = q.data_ptr() + 256, s.data_ptr() + 4 * 256
            ops._lib.check(lib.ptx_fp8_quantize(x.data_ptr(), *ptrs, None, None, m, k, 0, 0, 0, ops._stream()), "quantize")
            assert (q[:256] == 9).all() and (q[256 + data.numel():] == 9).all() and (q[256:256 + data.numel()].view(data.shape)[:, blocks:] == 9).all() and (s[:256] == 9).all() and (s[256 + scales.numel():] == 9).all()
            assert torch.equal(q[256:256 + data.numel()].view(data.shape)[:, :blocks], data.view(torch.uint8)[:, :blocks])


def test_streams_and_graphs():
    x, w, b, dy = _train(130, 384, 520, tb=F32)
    wq = P.quantize_fp8(w.detach(), square=True)
    eager = P.linear_fp8(x.detach(), wq)
    grads = torch.autograd.grad(P.linear_fp8(x, w, b), (x, w, b), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(P.linear_fp8(x.detach(), wq), eager)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    static = x.detach().clone().requires_grad_()
    leaf_w, leaf_b = w.detach().clone().requires_grad_(), b.detach().clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = P.linear_fp8(static, leaf_w, leaf_b)
        got = torch.autograd.grad(out, (static, leaf_w, leaf_b), dy)
        served = P.linear_fp8(static.detach(), wq)
    for turn in range(3):
        with torch.no_grad():
            static.copy_(x * (turn + 1))
        graph.replay()
        torch.cuda.synchronize()
        now = x.detach().mul(turn + 1).requires_grad_()
        want = torch.autograd.grad(P.linear_fp8(now, w, b), (now, w, b), dy)
        assert torch.equal(served, P.linear_fp8(now.detach(), wq)) and all(torch.equal(g, v) for g, v in zip(got, want))
    assert all(torch.equal(g, v) for g, v in zip(grads, torch.autograd.grad(P.linear_fp8(x, w, b), (x, w, b), dy)))


def test_large_offsets():
    """More than 2^32 bytes in and out: the last rows are as those of a short matrix (whose products are summed in another order)."""
    m, k = (1 << 32) // 1152 + 77, 1152
    x = torch.empty((m, k), dtype=BF16, device="cuda")
    x[:-200] = 1.0
    tail = _matrix(200, k, BF16)
    x[-200:] = tail
    t = P.quantize_fp8(x)
    short = P.quantize_fp8(tail)
    assert torch.equal(t.values[-200:].view(torch.uint8), short.values.view(torch.uint8)) and torch.equal(t.scales[-200:], short.scales)
    w = P.quantize_fp8(_matrix(1300, k, BF16, 1), square=True)
    y = P.matmul_fp8(t, w)
    _check_product(y[-200:], Q.held_by(short), Q.held_by(w))
    assert torch.equal(y[5], y[m // 2])
    del y, t
    # (x's rows in whole tiles of 128, so that the last tile holds the tail alone)
    m = (1 << 31) // 1152 // 128 * 128 + 128
    u = P.quantize_fp8(x[:m], along=-2)
    last = P.quantize_fp8(x[m - 128:m].contiguous(), along=-2)
    assert torch.equal(u.values[:, -128:].view(torch.uint8), last.values.view(torch.uint8)) and torch.equal(u.scales[:, -1:], last.scales)


def test_more_columns_than_a_launch_has_threads_for():
    """One row by 2^27 of a weight: 512 threads for 16 columns each would be more than 2^32."""
    n = (1 << 27) + 70
    last = P.quantize_fp8(_matrix(256, 128, BF16), square=True)      # (n ends 70 rows behind a block of rows: the last block and the one before)
    values = torch.zeros((n, 128), dtype=torch.uint8, device="cuda")
    values[-70 - 128:] = last.values.view(torch.uint8)[:70 + 128]
    scales = torch.zeros((n // 128 + 1, 1), device="cuda")
    scales[-2:] = last.scales
    w = P.Fp8Tensor(values.view(torch.float8_e4m3fn), scales, square=True)
    del values
    x = P.quantize_fp8(_matrix(1, 128, BF16, 1))
    y = P.matmul_fp8(x, w, dtype=F32)
    short = P.Fp8Tensor(last.values[:70 + 128], last.scales, square=True)
    _check_product(y[:, -70 - 128:], Q.held_by(x), Q.held_by(short))
    assert (y[:, :-70 - 128] == 0).all()


@pytest.mark.parametrize("native", [True, False])
def test_forward_mode_derivatives_are_refused(native, monkeypatch):
    monkeypatch.setattr(ops, "native_enabled", native)
    x, w, b = (torch.randn(s, device="cuda") for s in ((8, 16), (16, 16), (16,)))
    xq, wq = P.quantize_fp8(x), P.quantize_fp8(w, square=True)
    calls = [lambda t: P.linear_fp8(t(x), w), lambda t: P.linear_fp8(x, t(w)), lambda t: P.linear_fp8(x, w, t(b)), lambda t: P.linear_fp8(t(x), wq),
             lambda t: P.linear_fp8(xq, wq, t(b)), lambda t: P.matmul_fp8(xq, wq, t(b)), lambda t: P.add_rms_norm(t(x)),
             lambda t: P.add_rms_norm(x, t(x)), lambda t: P.add_rms_norm(x, None, t(b)), lambda t: P.add_rms_norm(x, x, t(b), quantize=True)]
    with forward_ad.dual_level():
        for f in calls:
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    f(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
            f(lambda t: t)


@pytest.mark.parametrize("native", [True, False])
def test_recorded_gradients_of_a_leaf_that_an_eager_graph_holds_are_refused(native, monkeypatch):
    monkeypatch.setattr(ops, "native_enabled", native)
    x, w, g = (torch.randn(s, device="cuda", requires_grad=True) for s in ((8, 16), (16, 16), (16,)))
    calls = [lambda: P.linear_fp8(x, w.detach()), lambda: P.linear_fp8(x.detach(), w), lambda: P.linear_fp8(x.detach(), w.detach(), g),
             lambda: P.add_rms_norm(x)[0], lambda: P.add_rms_norm(x.detach(), x)[0], lambda: P.add_rms_norm(x.detach(), None, g)[0]]
    alive = [f() for f in calls]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for f in calls:
            with pytest.raises(RuntimeError, match="eager graph that is still alive"):
                f()
        with torch.no_grad():      # (nothing to accumulate: taken)
            out = [f() for f in calls]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, alive))


def test_threads():
    x, w, b, dy = _train(130, 384, 520, tb=F32)
    gain = torch.ones(384, device="cuda", requires_grad=True)

    def call():
        y, h = P.add_rms_norm(x, None, gain)
        out = P.linear_fp8(y, w, b)
        with torch.no_grad():
            used = P.linear_fp8(P.add_rms_norm(x, None, gain, quantize=True)[0], P.quantize_fp8(w, square=True), b)
        return (out, used, *torch.autograd.grad(out, (x, gain, w, b), dy))

    want = call()
    torch.cuda.synchronize()
    got = {}

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                mine = call()
        s.synchronize()
        got[i] = mine

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert len(got) == 3 and all(torch.equal(a, c) for g in got.values() for a, c in zip(g, want))


def test_one_tensor_in_both_places():
    w = _matrix(200, 200, F32).requires_grad_()
    copies = [w.detach().clone().requires_grad_() for _ in range(2)]
    dy = _matrix(200, 200, F32, 1)
    got, = torch.autograd.grad(P.linear_fp8(w, w), w, dy)
    a, c = torch.autograd.grad(P.linear_fp8(*copies), copies, dy)
    assert torch.equal(got, a + c)


def test_a_layer_in_training_and_in_use():
    """Norm, product, gate and product, as a transition has them: differentiable as a whole, and in 8 bits from end to end."""
    g = torch.Generator().manual_seed(0)
    draw = lambda *s, scale=1.0: torch.randn(s, generator=g).mul(scale).cuda().requires_grad_()
    x, res, gain = draw(2, 75, 256), draw(2, 75, 256), draw(256)
    w_a, w_b, w_o = draw(1024, 256, scale=0.06), draw(1024, 256, scale=0.06), draw(256, 1024, scale=0.03)

    def layer(x, res, gain, w_a, w_b, w_o, linear):
        y, h = P.add_rms_norm(x, res, gain)
        return h + linear(torch.nn.functional.silu(linear(y, w_a)) * linear(y, w_b), w_o)

    leaves = (x, res, gain, w_a, w_b, w_o)
    out = layer(*leaves, P.linear_fp8)
    dy = torch.randn(out.shape, generator=g).cuda()
    grads = torch.autograd.grad(out, leaves, dy)
    # with the products in fp32: each of up to five 8-bit roundings on the way is off by 2^-4 of a value at most, some 2^-5.3 at a root mean
    # square, and they are independent: 5^(1/2) 2^-5.3 2^(1/2) (two operands) is 0.08
    exact = layer(*leaves, torch.nn.functional.linear)
    for got, want in zip((out, *grads), (exact, *torch.autograd.grad(exact, leaves, dy))):
        assert (got - want).norm() < 0.08 * want.norm()
    with torch.no_grad():
        y, h = P.add_rms_norm(x, res, gain, quantize=True)
        q = [P.quantize_fp8(w, square=True) for w in (w_a, w_b, w_o)]
        u = torch.nn.functional.silu(P.matmul_fp8(y, q[0], dtype=F32)) * P.matmul_fp8(y, q[1], dtype=F32)
        used = h + P.linear_fp8(u, q[2])
    # the same operands but for roundings that fall the other way (y here straight from the norm's sums)
    assert torch.equal(h, P.add_rms_norm(x, res, gain)[1]) and (used - out).norm() < 2.0**-10 * out.norm()


def test_refusals():
    x, w = _matrix(4, 200, BF16), _matrix(30, 200, BF16)
    xq, wq = P.quantize_fp8(x), P.quantize_fp8(w, square=True)
    grad = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        P.linear_fp8(grad, wq)
    with pytest.raises(RuntimeError, match="no gradients"):
        P.linear_fp8(xq, w.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no gradients"):
        P.matmul_fp8(xq, wq, torch.zeros(30, device="cuda", requires_grad=True))
    with torch.no_grad():
        assert torch.equal(P.linear_fp8(grad, wq), P.linear_fp8(x, wq))
    with pytest.raises(RuntimeError, match="scale per 128 values of a row"):
        P.matmul_fp8(P.quantize_fp8(x, square=True), wq)
    for bad in (lambda: P.matmul_fp8(xq, P.quantize_fp8(_matrix(30, 201, BF16))), lambda: P.linear_fp8(x, w[:, :100]),
                lambda: P.linear_fp8(x, w, torch.zeros(29, device="cuda")), lambda: P.linear_fp8(x, w, dtype=torch.float64),
                lambda: P.linear_fp8(x.double(), w), lambda: P.linear_fp8(x, w[0]), lambda: P.matmul_fp8(x, wq),
                lambda: P.quantize_fp8(x, along=0), lambda: P.quantize_fp8(x[None], square=True), lambda: P.quantize_fp8(x[:, :0]),
                lambda: P.Fp8Tensor(xq.values, xq.scales[:, :1]), lambda: P.Fp8Tensor(x, xq.scales),
                lambda: P.Fp8Tensor(xq.values, xq.scales.double()), lambda: P.linear_fp8(x, w, torch.zeros(30)),
                lambda: P.linear_fp8(x, w.cpu())):
        with pytest.raises(RuntimeError):
            bad()
    y = P.linear_fp8(grad, w)
    with pytest.raises(RuntimeError, match="differentiable"):
        torch.autograd.grad(y, grad, torch.ones_like(y), create_graph=True)[0].sum().backward()
