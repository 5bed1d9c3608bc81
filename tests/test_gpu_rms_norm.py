"""The residual sum and its RMS norm, forward, backward and into 8-bit blocks, against the 64-bit form."""
import pytest
import torch

import protenix_amd as P
from protenix_amd import ops
from tests import fp8_oracle as Q
from tests.residual_oracle import half_step, smallest

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)]
EPS = 1e-6


def _inputs(shape, tx, tr=None, tw=F32, seed=0):
    g = torch.Generator().manual_seed(seed)
    draw = lambda size, t, scale=1.0, add=0.0: torch.randn(size, generator=g).mul(scale).add(add).to(t).cuda()
    x = draw(shape, tx, 0.7).requires_grad_()
    r = None if tr is None else draw(shape, tr, 2.0, 0.4).requires_grad_()
    w = None if tw is None else draw(shape[-1:], tw, 0.2, 1.0).requires_grad_()
    return x, r, w, draw(shape, tx), draw(shape, tr or tx)


def _parts(x, r, w, eps=EPS):
    h = x.detach().cpu().double() + (0 if r is None else r.detach().cpu().double())
    rstd = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    wd = torch.ones(x.shape[-1], dtype=torch.double) if w is None else w.detach().cpu().double()
    return h, rstd, wd


def _near(got, want, extra, what):
    got = got.detach().cpu()
    tol = half_step(got.dtype) * want.abs() + extra + smallest(got.dtype)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, bad.sum().item(), got[bad][:4], want[bad][:4])


def _compare(x, r, w, dy, dh, y, h, grads, eps=EPS):
    """fp32 sums of a row: at most 64 terms in turn per lane and exchange (8 columns, 2 blocks, 6 exchanges, 16 waves), so their error is
    below 64 2^-24 = 2^-18 of the sum of magnitudes; all squares have one sign, so rstd is off by 2^-18 of itself, and U = 2^-16
    counts it with the roundings of each factor."""
    hd, rstd, wd = _parts(x, r, w, eps)
    U = 2.0**-16
    if r is not None:
        _near(h, hd, 2.0**-23 * (x.detach().cpu().double().abs() + r.detach().cpu().double().abs()), "h")
    _near(y, hd * rstd * wd, U * (hd * rstd * wd).abs() + 2.0**-22 * rstd * wd.abs() * (0 if r is None else 1) *
          (x.detach().cpu().double().abs() + hd.abs()), "y")
    if grads is None:
        return
    dyd, dhd = (torch.zeros_like(hd) if t is None else t.cpu().double() for t in (dy, dh))
    g, xh = dyd * wd, hd * rstd
    c = (g * xh).mean(-1, keepdim=True)
    dres = rstd * (g - xh * c) + dhd
    size = (g * xh).abs().mean(-1, keepdim=True)
    lost = U * rstd * (g.abs() + xh.abs() * size) * 2 + 2.0**-22 * dhd.abs()
    for name in ("x", "r"):
        if name in grads:
            _near(grads[name], dres, lost, "d" + name)
    if "w" in grads:
        dims = tuple(range(hd.dim() - 1))
        rows = max(hd[..., 0].numel(), 1)
        # (a walk over rows / 1024 of them, then at most 1024 / 64 partial sums and 16 exchanges in turn)
        turn = U + 2.0**-24 * (rows / 1024 + 64)
        _near(grads["w"], (dyd * xh).sum(dims), (turn * (dyd * xh).abs()).sum(dims), "dw")


def _run(x, r, w, dy, dh, eps=EPS):
    y, h = P.add_rms_norm(x, r, w, eps)
    leaves = {n: t for n, t in zip("xrw", (x, r, w)) if t is not None}
    pairs = [(o, g) for o, g in ((y, dy), (h, dh)) if g is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [g for _, g in pairs], allow_unused=True)
    return y, h, {n: g for n, g in zip(leaves, grads) if g is not None}


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("cols", [1, 7, 8, 24, 64, 67, 128, 200, 256, 384, 512, 513, 768, 1000, 1025, 2048, 2051, 4096, 4100, 8192, 16384])
def test_row_lengths(types, cols):
    args = _inputs((3, 37, cols) if cols <= 1024 else (5, cols), *types, seed=cols)
    y, h, grads = _run(*args)
    assert y.dtype == types[0] and h.dtype == types[1]
    assert grads["x"].dtype == types[0] and grads["r"].dtype == types[1] and grads["w"].dtype == F32
    _compare(*args, y, h, grads)


@pytest.mark.parametrize("rows", [1, 2, 5, 64, 1023, 5000])
@pytest.mark.parametrize("cols", [16, 128, 600])
def test_row_counts(rows, cols):
    args = _inputs((rows, cols), BF16, F32, seed=rows)
    _compare(*args, *_run(*args))


@pytest.mark.parametrize("tx", [F32, BF16, F16])
@pytest.mark.parametrize("tw", [F32, BF16, F16, None])
def test_no_residual_and_parameters(tx, tw):
    args = _inputs((41, 72), tx, None, tw)
    y, h, grads = _run(*args)
    assert torch.equal(h, args[0]) and h.data_ptr() == args[0].data_ptr() and (tw is None or grads["w"].dtype == tw)
    _compare(*args, y, h, grads)
    args = _inputs((41, 72), tx, tx, tw)
    _compare(*args, *_run(*args))


@pytest.mark.parametrize("types", [(BF16, BF16), (BF16, F32), (F32, None)])
@pytest.mark.parametrize("which", ["y", "h"])
def test_one_of_the_two_results_unused(types, which):
    x, r, w, dy, dh = _inputs((12, 320), *types)
    args = (x, r, w, dy if which == "y" else None, dh if which == "h" else None)
    _compare(*args, *_run(*args))


@pytest.mark.parametrize("types", [(BF16, BF16), (F16, F32)])
def test_frozen_inputs(types):
    args = _inputs((19, 200), *types)
    full = _run(*args)[2]
    for mask in range(1, 7):
        some = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(args[:3])]
        y, h = P.add_rms_norm(*some, EPS)
        outs = [(o, g) for o, g in ((y, args[3]), (h, args[4])) if o.requires_grad]
        grads = torch.autograd.grad([o for o, _ in outs], [t for t in some if t.requires_grad], [g for _, g in outs])
        assert all(torch.equal(g, full[n]) for n, g in zip([n for i, n in enumerate("xrw") if mask >> i & 1], grads))


@pytest.mark.parametrize("types", TYPES + [(BF16, None)])
@pytest.mark.parametrize("cols", [1, 7, 64, 65, 127, 128, 129, 200, 256, 384, 513, 1000, 2048, 4100, 8192, 9000, 16384])
def test_into_eight_bits(types, cols):
    """The values are those of the block's rounding of y in 64 bits, but where y lies within fp32's error of the middle of two."""
    x, r, w, _, _ = _inputs((3, 11, cols), *types, seed=cols)
    with torch.no_grad():
        t, h = P.add_rms_norm(x, r, w, EPS, quantize=True)
        y = P.add_rms_norm(x, r, w, EPS)
    assert t.shape == x.shape and t.values.shape == x.shape and t.scales.shape == (3, 11, -(-cols // 128))
    assert torch.equal(h, y[1]) and (r is not None or h is x)
    hd, rstd, wd = _parts(x, r, w)
    yd = (hd * rstd * wd).view(33, cols)
    s = Q.scales_of(yd)
    # y is off by U of itself and by fp32's rounding of the sum
    err = 2.0**-16 * yd.abs() + 2.0**-22 * (rstd * wd.abs() * (x.detach().cpu().double().abs() + hd.abs())).view(33, cols)
    off = Q.spread(torch.nn.functional.pad(err, (0, -cols % 128)).view(33, -1, 128).amax(-1), yd.shape, False)
    sd = t.scales.cpu().double().view(33, -1)
    assert ((sd - s).abs() * 448 <= Q.spread(s, yd.shape, False).new_tensor(0) + off.view(33, -1)[:, ::128][:, :s.shape[1]] + 2.0**-22 * s * 448).all()
    q = t.values.cpu().float().double().view(33, cols)
    at = yd / Q.spread(sd, yd.shape, False)
    slack = (err + off * at.abs() / 448) / Q.spread(sd, yd.shape, False) + 2.0**-22 * at.abs()
    low, high = Q.round_e4m3((at - slack).clamp(-448, 448)), Q.round_e4m3((at + slack).clamp(-448, 448))
    assert ((q >= low) & (q <= high)).all()
    assert (t._operand[0].view(torch.uint8)[:, cols:-(-cols // 128) * 128] & 0x7f == 0).all()


@pytest.mark.parametrize("rows", [1, 3, 100, 5000])
def test_into_eight_bits_row_counts(rows):
    x, r, w, _, _ = _inputs((rows, 2048), BF16, BF16, BF16, seed=rows)
    with torch.no_grad():
        t, _ = P.add_rms_norm(x, r, w, EPS, quantize=True)
        y = P.add_rms_norm(x.float(), r.float(), w.float(), EPS)[0]
        want = P.quantize_fp8(y)
    assert torch.equal(t.scales, want.scales) and torch.equal(t.values.view(torch.uint8), want.values.view(torch.uint8))


def test_rows_of_zeros_and_rows_with_nan():
    x, r, w, dy, dh = _inputs((40, 136), BF16, F32)
    zero = torch.zeros((3, 136), device="cuda", requires_grad=True)
    y, h = P.add_rms_norm(zero, None, w, EPS)
    assert (y == 0).all()
    g = torch.autograd.grad(y, zero, torch.ones_like(y))[0]
    assert torch.allclose(g, (w / EPS**0.5).expand_as(g), rtol=1e-5)
    with torch.no_grad():
        t = P.add_rms_norm(zero, None, w, EPS, quantize=True)[0]
        assert (t.values.float() == 0).all() and (t.scales == 2.0**-126).all()
        clean = P.add_rms_norm(x, r, w)
        x2 = x.clone()
        x2[7, 3], x2[9, 135] = float("nan"), float("inf")
        y, h = P.add_rms_norm(x2, r, w)
        t = P.add_rms_norm(x2, r, w, quantize=True)[0]
    rest = [i for i in range(40) if i not in (7, 9)]
    assert torch.equal(y[rest], clean[0][rest]) and torch.equal(h[rest], clean[1][rest])
    assert y[7].isnan().all() and y[9, 135].isnan() and not t.scales[7].isfinite().any() and t.scales[rest].isfinite().all()


def test_against_differences():
    x, r, w, dy, dh = _inputs((6, 96), F32, F32, seed=4)
    y, h, grads = _run(x, r, w, dy, dh)
    g = torch.Generator().manual_seed(5)
    step, leaves = 2.0**-7, [x, r, w]
    way = [torch.randn(t.shape, generator=g).cuda() for t in leaves]

    def value(sign):
        with torch.no_grad():
            yy, hh = P.add_rms_norm(*(t + sign * step * v for t, v in zip(leaves, way)), EPS)
        return (yy.double() * dy.double()).sum() + (hh.double() * dh.double()).sum()

    slope = ((value(1) - value(-1)) / (2 * step)).item()
    want = sum((grads[n].double() * v.double()).sum().item() for n, v in zip("xrw", way))
    # values of y and h are off by 2^-20 or less of their size here; the third derivative of a row's norm, whose size is 2, is below the
    # number of elements
    bound = 2.0**-20 * ((y.double() * dy.double()).abs().sum() + (h.double() * dh.double()).abs().sum()).item() / step + x.numel() * step**2
    assert abs(slope - want) < bound, (slope, want, bound)


def test_strides_and_empty_tensors():
    x, r, w, dy, dh = _inputs((24, 200), BF16, F32)
    first = _run(x, r, w, dy, dh)
    turned = [t.detach().t().contiguous().t().requires_grad_() for t in (x, r)]
    again = _run(*turned, w, dy.t().contiguous().t(), dh.t().contiguous().t())
    assert torch.equal(first[0], again[0]) and all(torch.equal(first[2][n], again[2][n]) for n in "xrw")
    odd = torch.empty((24 * 200 + 1,), dtype=BF16, device="cuda")[1:].view(24, 200).copy_(x.detach())
    with torch.no_grad():
        assert torch.equal(P.add_rms_norm(odd, r, w)[0], first[0])
        assert torch.equal(P.add_rms_norm(odd, r, w, quantize=True)[0].scales, P.add_rms_norm(x, r, w, quantize=True)[0].scales)
    none = torch.empty((0, 200), dtype=BF16, device="cuda", requires_grad=True)
    y, h = P.add_rms_norm(none, none.float(), w)
    gx, gw = torch.autograd.grad(y, (none, w), torch.empty_like(y))
    assert y.shape == (0, 200) and gx.shape == (0, 200) and (gw == 0).all()
    with torch.no_grad():
        t, _ = P.add_rms_norm(none, None, w, quantize=True)
    assert t.values.shape == (0, 200) and t.scales.shape == (0, 2)


def test_workspaces_graphs_and_streams(monkeypatch):
    x, r, w, dy, dh = _inputs((700, 384), BF16, F32)
    first = _run(x, r, w, dy, dh)
    with monkeypatch.context() as m:
        m.setattr(ops, "poison_workspaces", True)
        again = _run(x, r, w, dy, dh)
    assert torch.equal(first[0], again[0]) and all(torch.equal(first[2][n], again[2][n]) for n in "xrw")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        y = P.add_rms_norm(x, r, w)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, first[0])
    leaves = [t.detach().clone().requires_grad_() for t in (x, r, w)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, h = P.add_rms_norm(*leaves)
        got = torch.autograd.grad((y, h), leaves, (dy, dh))
        with torch.no_grad():
            t = P.add_rms_norm(*leaves, quantize=True)[0]
    for turn in range(3):
        with torch.no_grad():
            leaves[0].copy_(x * (turn + 1))
        graph.replay()
        torch.cuda.synchronize()
        now = (x.detach() * (turn + 1)).requires_grad_()
        want = _run(now, r, w, dy, dh)
        with torch.no_grad():
            eager = P.add_rms_norm(now, r, w, quantize=True)[0]
        assert torch.equal(y, want[0]) and all(torch.equal(a, want[2][n]) for a, n in zip(got, "xrw"))
        assert torch.equal(t.scales, eager.scales) and torch.equal(t.values.view(torch.uint8), eager.values.view(torch.uint8))


def test_python_and_native_paths_give_the_same_bits(monkeypatch):
    for types in ((BF16, F32), (BF16, BF16), (F32, None), (F16, None)):
        x, r, w, dy, dh = _inputs((5, 31, 200), *types)

        def every():
            y, h, grads = _run(x, r, w, dy, dh)
            with torch.no_grad():
                t, h2 = P.add_rms_norm(x, r, w, quantize=True)
                plain = P.add_rms_norm(x, r, w)
            return (y, h, *(grads[n] for n in "xrw" if n in grads), t.values.view(torch.uint8), t.scales, h2, *plain)

        first = every()
        with monkeypatch.context() as m:
            m.setattr(ops, "native_enabled", False)
            second = every()
        assert len(first) == len(second) and all(a.shape == c.shape and a.dtype == c.dtype and torch.equal(a, c) for a, c in zip(first, second))


def test_one_tensor_as_update_and_residual():
    x, _, w, dy, dh = _inputs((7, 200), F32)
    copies = [x.detach().clone().requires_grad_() for _ in range(2)]
    got, = torch.autograd.grad(P.add_rms_norm(x, x, w), x, (dy, dh))
    a, c = torch.autograd.grad(P.add_rms_norm(*copies, w), copies, (dy, dh))
    assert torch.equal(got, a + c)


@pytest.mark.parametrize("cols", [7, 64, 67, 600, 1025, 4100, 9001])
def test_written_in_place(cols):
    """The C entry point's y over x and h over the residual."""
    lib = ops._lib.load()
    for tx, tr in TYPES:
        x, r, w, _, _ = _inputs((333, cols), tx, tr, seed=cols)
        with torch.no_grad():
            y, h = P.add_rms_norm(x, r, w)
            a, b = x.detach().clone(), r.detach().clone()
            ops._lib.check(lib.ptx_add_rms_norm_fwd(a.data_ptr(), b.data_ptr(), w.data_ptr(), a.data_ptr(), None, b.data_ptr(), None, 333, cols, EPS,
                                                    ops._LN_DTYPES[tx], ops._LN_DTYPES[tr], ops._LN_DTYPES[w.dtype], ops._stream()), "add_rms_norm")
        assert torch.equal(a, y) and torch.equal(b, h)


def test_columns_beyond_32_bits_are_refused():
    x = torch.ones((), device="cuda").expand(1, (1 << 32) + 128)
    for call in (lambda: P.add_rms_norm(x), lambda: P.add_rms_norm(x, quantize=True)):
        with pytest.raises(RuntimeError, match="16384"):
            call()


def test_large_offsets():
    """More than 2^32 elements: the last rows are those of a short call, with their gradients."""
    rows, cols = (1 << 32) // 4096 + 77, 4096
    x = torch.empty((rows, cols), dtype=BF16, device="cuda")
    x[:-50] = 1.0
    tail = _inputs((50, cols), BF16)[0].detach()
    x[-50:] = tail
    t = tail.clone().requires_grad_()
    y, h = P.add_rms_norm(t)
    dt, = torch.autograd.grad((y, h), t, (tail, tail))
    x.requires_grad_()
    far, same = P.add_rms_norm(x)
    assert torch.equal(far[-50:], y) and torch.equal(far[3], far[rows // 2])
    dx, = torch.autograd.grad((far, same), x, (x.detach(), x.detach()))
    assert torch.equal(dx[-50:], dt) and torch.equal(dx[3], dx[rows // 2])
    del far, same, dx
    with torch.no_grad():
        q, short = P.add_rms_norm(x, quantize=True)[0], P.add_rms_norm(t, quantize=True)[0]
    assert torch.equal(q.values[-50:].view(torch.uint8), short.values.view(torch.uint8)) and torch.equal(q.scales[-50:], short.scales)


def test_refusals():
    x, r, w, _, _ = _inputs((4, 200), BF16, F32)
    with pytest.raises(RuntimeError, match="no gradients"):
        P.add_rms_norm(x, r, w, quantize=True)
    for bad in (lambda: P.add_rms_norm(x, r[:3], w), lambda: P.add_rms_norm(x, r.half(), w), lambda: P.add_rms_norm(x, r, w[:10]),
                lambda: P.add_rms_norm(x.double(), None, w), lambda: P.add_rms_norm(x, r, w.cpu()), lambda: P.add_rms_norm(x[:, :0]),
                lambda: P.add_rms_norm(torch.zeros((2, 16385), device="cuda")), lambda: P.add_rms_norm(x, r.cpu(), w)):
        with pytest.raises(RuntimeError):
            bad()
