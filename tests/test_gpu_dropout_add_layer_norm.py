"""The residual sum with dropout and its LayerNorm, forward and backward, against the 64-bit form."""
import pytest
import torch

import protenix_amd as P
from protenix_amd import ops
from tests import residual_oracle as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)]


def _inputs(shape, tx, tr, tw=F32, seed=0, residual=True, shift=0.4):
    g = torch.Generator().manual_seed(seed)
    draw = lambda size, t, scale=1.0, add=0.0: torch.randn(size, generator=g).mul(scale).add(add).to(t).cuda()
    x = draw(shape, tx, 0.7).requires_grad_()
    r = draw(shape, tr, 2.0, shift).requires_grad_() if residual else None
    w, b = draw(shape[-1:], tw, 0.2, 1.0).requires_grad_(), draw(shape[-1:], tw, 0.2).requires_grad_()
    return x, r, w, b, draw(shape, tx), draw(shape, tr if residual else tx)


def _near(got, want, extra, what):
    """One rounding to got's type beside `extra`, the bound of what the fp32 arithmetic loses."""
    got, want = got.detach().cpu(), want.detach()
    tol = R.half_step(got.dtype) * want.abs() + extra + R.smallest(got.dtype)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, bad.sum().item(), got[bad][:4], want[bad][:4], extra.expand_as(want)[bad][:4])


def _compare(x, r, w, b, dy, dh, p, seed, shared_dim, eps, y, h, grads):
    """fp32 sums of a row: at most 64 terms in turn per lane (8 columns, up to 4 blocks, 6 exchanges, 16 waves), so their
    error is below 64 2^-24 = 2^-18 of the mean absolute value; the variance twice that.  The bounds below count those of every
    row in units of 2^-16, with C = rstd max|h|, how much of a row's scale is its mean."""
    hd, m = R.update(x, r, p, seed, shared_dim)
    yd, xh, rstd = R.norm_parts(hd, w, b, eps)
    top = lambda t: t.abs().amax(-1, keepdim=True)
    C = rstd * top(hd) + 1
    wd = torch.ones(x.shape[-1], dtype=torch.double) if w is None else w.detach().cpu().double()
    scale = top(xh) + 1
    u = 2.0**-16
    kept = torch.where(m != 0, x.detach().cpu().double() * m, torch.zeros_like(hd))
    _near(h, hd, 2.0**-23 * (kept.abs() + (hd - kept).abs()), "h")
    _near(y, yd, u * C * scale * wd.abs() + 2.0**-23 * yd.abs(), "y")
    if grads is None:
        return
    dyd, dhd = (torch.zeros_like(hd) if t is None else t.cpu().double() for t in (dy, dh))
    g = dyd * wd
    a, c = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dres = rstd * (g - a - xh * c) + dhd
    lost = u * rstd * top(g) * scale**2 * C + 2.0**-22 * dhd.abs()
    want = {"x": (torch.where(m != 0, dres * m, torch.zeros_like(dres)), lost * m + 2.0**-22 * (dres * m).abs()),
            "r": (dres, lost)}
    dims = tuple(range(hd.dim() - 1))
    rows = max(hd[..., 0].numel(), 1)
    # (a walk over rows / 4096 of them, then at most 1024 / 64 partial sums and 16 exchanges in turn)
    turn = 2.0**-24 * (rows / 4096 + 64)
    want["w"] = ((dyd * xh).sum(dims), (dyd.abs() * (u * C * scale + turn * xh.abs())).sum(dims))
    want["b"] = (dyd.sum(dims), turn * dyd.abs().sum(dims))
    for name, got in grads.items():
        _near(got, *want[name], "d" + name)


def _run(x, r, w, b, dy, dh, p, seed, shared_dim=None, eps=1e-5):
    y, h = P.dropout_add_layer_norm(x, r, w, b, p, eps, shared_dim=shared_dim, seed=seed)
    leaves = {n: t for n, t in zip("xrwb", (x, r, w, b)) if t is not None}
    pairs = [(o, g) for o, g in ((y, dy), (h, dh)) if g is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], list(leaves.values()), [g for _, g in pairs], allow_unused=True)
    return y, h, {n: g for n, g in zip(leaves, grads) if g is not None}


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("cols", [1, 7, 8, 24, 64, 67, 128, 200, 256, 384, 512, 513, 768, 1000, 1025, 2048, 2051, 4096, 4100, 8192])
def test_row_lengths(types, cols):
    rows = (3, 37) if cols <= 1024 else (1, 5)
    args = _inputs((*rows, cols), *types, seed=cols)
    y, h, grads = _run(*args, 0.15, 21)
    assert y.dtype == types[0] and h.dtype == types[1]
    assert grads["x"].dtype == types[0] and grads["r"].dtype == types[1] and grads["w"].dtype == F32
    _compare(*args, 0.15, 21, None, 1e-5, y, h, grads)


@pytest.mark.parametrize("cols", [8193, 12288, 16383, 16384])
@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F16, F32)])
def test_very_long_rows(types, cols):
    args = _inputs((3, cols), *types, seed=cols)
    _compare(*args, 0.1, 5, None, 1e-5, *_run(*args, 0.1, 5))


@pytest.mark.parametrize("rows", [1, 2, 5, 64, 1023, 5000])
@pytest.mark.parametrize("cols", [16, 128, 600])
def test_row_counts(rows, cols):
    args = _inputs((rows, cols), BF16, F32, seed=rows)
    _compare(*args, 0.25, 9, None, 1e-5, *_run(*args, 0.25, 9))


@pytest.mark.parametrize("shared_dim", [None, -2, -3, 0])
@pytest.mark.parametrize("types", [(BF16, F32), (F16, F16)])
def test_shared_masks(types, shared_dim):
    args = _inputs((2, 13, 11, 128), *types, seed=1)
    _compare(*args, 0.25, 77, shared_dim, 1e-5, *_run(*args, 0.25, 77, shared_dim))


@pytest.mark.parametrize("p", [0.0, 1e-5, 0.5, 1.0])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F16, F32)])
def test_probabilities_and_no_residual(types, residual, p):
    if not residual:
        types = (types[0], types[0])
    args = _inputs((9, 30, 136), *types, seed=2, residual=residual)
    y, h, grads = _run(*args, p, 3)
    _compare(*args, p, 3, None, 1e-5, y, h, grads)
    if p == 1.0 and not residual:      # rows of zeros: their norm is the bias
        assert torch.equal(y, args[3].detach().to(y.dtype).expand_as(y)) and (h == 0).all()


@pytest.mark.parametrize("tw", [F32, BF16, F16])
@pytest.mark.parametrize("have", ["wb", "w", "b", ""])
def test_parameters(tw, have):
    x, r, w, b, dy, dh = _inputs((41, 72), BF16, BF16, tw)
    args = (x, r, w if "w" in have else None, b if "b" in have else None, dy, dh)
    y, h, grads = _run(*args, 0.1, 3)
    _compare(*args, 0.1, 3, None, 1e-5, y, h, grads)
    assert all(grads[n].dtype == tw for n in have)


@pytest.mark.parametrize("types", [(BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("which", ["y", "h"])
def test_one_of_the_two_results_unused(types, which):
    x, r, w, b, dy, dh = _inputs((12, 320), *types)
    args = (x, r, w, b, dy if which == "y" else None, dh if which == "h" else None)
    _compare(*args, 0.2, 3, None, 1e-5, *_run(*args, 0.2, 3))


@pytest.mark.parametrize("types", [(BF16, BF16), (F16, F32)])
def test_frozen_inputs(types):
    """Any subset of the four may want no gradient."""
    args = _inputs((19, 200), *types)
    full = _run(*args, 0.2, 3)[2]
    for mask in range(1, 15):
        some = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(args[:4])]
        y, h = P.dropout_add_layer_norm(*some, 0.2, seed=3)
        wanted = [n for i, n in enumerate("xrwb") if mask >> i & 1]
        outs = [(o, g) for o, g in ((y, args[4]), (h, args[5])) if o.requires_grad]
        grads = torch.autograd.grad([o for o, _ in outs], [t for t in some if t.requires_grad], [g for _, g in outs])
        assert all(torch.equal(g, full[n]) for n, g in zip(wanted, grads)), wanted


def test_rows_far_from_zero_and_of_one_value():
    """A mean a thousand times the deviation; rows of one value, whose variance is 0."""
    x, r, w, b, dy, dh = _inputs((20, 256), F32, F32, shift=2000.0)
    _compare(x, r, w, b, dy, dh, 0.1, 3, None, 1e-5, *_run(x, r, w, b, dy, dh, 0.1, 3))
    c = torch.full((4, 256), 3.0, device="cuda")
    y, h = P.dropout_add_layer_norm(c, c, w, b)
    assert torch.equal(h, c + c) and torch.equal(y, b.detach().expand_as(y))


def test_rows_with_nan_stay_among_themselves():
    x, r, w, b, dy, dh = _inputs((40, 128), BF16, F32)
    clean = P.dropout_add_layer_norm(x, r, w, b, 0.25, seed=1)
    x2 = x.detach().clone()
    x2[7] = float("nan")
    x2[9, 5] = float("inf")
    y, h = P.dropout_add_layer_norm(x2, r, w, b, 0.25, seed=1)
    rest = [i for i in range(40) if i not in (7, 9)]
    assert torch.equal(y[rest], clean[0][rest]) and torch.equal(h[rest], clean[1][rest])
    keep = R.keep_mask((40, 128), 0.25, 1)[9, 5]
    assert bool(h[9, 5].isinf()) == bool(keep) and bool(y[7].isnan().all())


def test_against_differences():
    """The directional derivative along a random direction, from the forward pass alone."""
    x, r, w, b, dy, dh = _inputs((6, 96), F32, F32, seed=4)
    y, h, grads = _run(x, r, w, b, dy, dh, 0.25, 8)
    g = torch.Generator().manual_seed(5)
    step, leaves = 2.0**-7, [x, r, w, b]
    way = [torch.randn(t.shape, generator=g).cuda() for t in leaves]

    def value(sign):
        with torch.no_grad():
            yy, hh = P.dropout_add_layer_norm(*(t + sign * step * v for t, v in zip(leaves, way)), 0.25, seed=8)
        return (yy.double() * dy.double()).sum() + (hh.double() * dh.double()).sum()

    slope = ((value(1) - value(-1)) / (2 * step)).item()
    want = sum((grads[n].double() * v.double()).sum().item() for n, v in zip("xrwb", way))
    # values of y and h are off by 2^-20 or less of their size here; the third derivative of a row's norm, whose deviation is 2, is
    # below the number of elements
    bound = 2.0**-20 * ((y.double() * dy.double()).abs().sum() + (h.double() * dh.double()).abs().sum()).item() / step + x.numel() * step**2
    assert abs(slope - want) < bound, (slope, want, bound)


def test_python_and_native_paths_give_the_same_bits(monkeypatch):
    seed = torch.tensor([77], device="cuda")
    for types in [(BF16, F32), (BF16, BF16), (F32, F32)]:
        for p in (0.2, 0.0):
            args = _inputs((5, 31, 200), *types)
            first = _run(*args, p, seed, -2)
            with monkeypatch.context() as m:
                m.setattr(ops, "poison_workspaces", True)
                second = _run(*args, p, seed, -2)
                with torch.no_grad():
                    y, h = P.dropout_add_layer_norm(*args[:4], p, seed=seed, shared_dim=-2)
            with torch.no_grad():
                y2, h2 = P.dropout_add_layer_norm(*args[:4], p, seed=seed, shared_dim=-2)
            for a in (second[0], y, y2):
                assert torch.equal(first[0], a)
            for a in (second[1], h, h2):
                assert torch.equal(first[1], a)
            assert all(torch.equal(first[2][n], second[2][n]) for n in "xrwb")


def test_repeated_calls_give_the_same_bits():
    args = _inputs((4000, 384), BF16, BF16)
    a, b = _run(*args, 0.1, 1), _run(*args, 0.1, 1)
    assert torch.equal(a[0], b[0]) and all(torch.equal(a[2][n], b[2][n]) for n in "xrwb")


def test_same_mask_as_dropout_add():
    x, r, *_ = _inputs((3, 40, 128), BF16, F32)
    _, h = P.dropout_add_layer_norm(x, r, p=0.25, shared_dim=0, seed=5)
    assert torch.equal(h, P.dropout_add(x, r, 0.25, shared_dim=0, seed=5))


def test_strides_and_offsets():
    x, r, w, b, *_ = _inputs((17, 130), BF16, F32)
    want = P.dropout_add_layer_norm(x[:, 1:129].contiguous(), r[:, 2:].contiguous(), w[1:129].clone(), b[2:].clone(), 0.2, seed=3)
    got = P.dropout_add_layer_norm(x[:, 1:129], r[:, 2:], w[1:129], b[2:], 0.2, seed=3)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("shape", [(0, 16), (3, 0, 16)])
def test_no_rows(shape):
    x, r, w, b, dy, dh = _inputs(shape, BF16, F32)
    y, h, grads = _run(x, r, w, b, dy, dh, 0.2, 3)
    assert y.shape == h.shape == shape and (grads["w"] == 0).all() and (grads["b"] == 0).all() and grads["x"].shape == shape


def test_refusals():
    x = torch.zeros(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    for args, kw, match in [((x, x, w[:4]), {}, "weight and bias"), ((x, x, w, w.to(BF16)), {}, "weight and bias"),
                            ((x, x, w.cpu()), {}, "weight and bias"), ((x, x, w.double()), {}, "float32"), ((x.to(BF16), x.to(F16)), {}, "type"),
                            ((x[:, :0],), {}, "empty"), ((torch.zeros(2, 16385, device="cuda"),), {}, "unsupported shape"),
                            ((x, x), {"p": 2.0}, "probability"), ((x, x), {"shared_dim": -1, "p": 0.1}, "last"), ((x, x[:1]), {}, "differ")]:
        with pytest.raises(RuntimeError, match=match):
            P.dropout_add_layer_norm(*args, **kw)
    x.requires_grad_()
    y, h = P.dropout_add_layer_norm(x, None, w)
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(y.sum(), x, create_graph=True)
        g.sum().backward()


def test_recorded_and_replayed():
    x, r, w, b, dy, dh = _inputs((3, 50, 128), BF16, F32)
    seed = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step():
        y, h, g = _run(x, r, w, b, dy, dh, 0.25, seed, 0)
        return y.detach(), h.detach(), *g.values()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    with torch.cuda.graph(other):
        outs2 = step()
    for rep in range(4):
        seed.fill_(1000 + rep)
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(a, c) for a, c in zip(outs, want)), rep
        assert all(torch.equal(a, c) for a, c in zip(outs2, want)), rep


@pytest.mark.parametrize("types", TYPES)
def test_few_columns(types):
    # one, two and four lanes to a row, every length of its last block
    for cols in (*range(2, 7), *range(9, 20), 23, 25, 31, 32, 33):
        args = _inputs((3, 101, cols), *types, seed=cols)
        _compare(*args, 0.15, cols, None, 1e-5, *_run(*args, 0.15, cols))


@pytest.mark.parametrize("types", [(BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("rows,cols", [(300001, 5), (70001, 27), (2600, 1500), (1900, 2800), (1100, 5001), (800, 7000)])
def test_walks_of_several_turns(types, rows, cols):
    args = _inputs((rows, cols), *types, seed=cols)
    _compare(*args, 0.1, 3, None, 1e-5, *_run(*args, 0.1, 3))


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("cols", [7, 24, 67, 128, 136, 384, 768, 1035, 2056, 8200, 9000])
def test_dropped_values_do_not_matter(types, cols):
    """Infinities, NaN and values that the factor would carry beyond the type, in all dropped places: the results and gradients are, bit by
    bit, those of zeros there.  Lanes of a row without columns of their own hold its last 8 columns under another block's mask."""
    for shared_dim in (None, 0):
        x, r, w, b, dy, dh = _inputs((3, 37 if cols < 2000 else 5, cols), *types, seed=cols)
        keep = R.keep_mask(x.shape, 0.25, 31, shared_dim).cuda()
        odd = torch.tensor([float("inf"), float("nan"), float("-inf"), torch.finfo(types[0]).max], device="cuda").to(types[0])
        odd = odd[torch.arange(x.numel(), device="cuda") % 4].view(x.shape)
        runs = [_run(torch.where(keep, x.detach(), there).requires_grad_(), r, w, b, dy, dh, 0.25, 31, shared_dim)
                for there in (torch.zeros_like(odd), odd)]
        for name, want, got in zip(("y", "h", *"xrwb"), *((y, h, *(g[n] for n in "xrwb")) for y, h, g in runs)):
            assert want.isfinite().all() and torch.equal(want, got), (name, shared_dim)


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("cols", [64, 136, 1035])
def test_the_sum_alone_asks_nothing_of_the_norm(types, cols):
    """Where y is not used, h's gradient goes on as it is: through rows without a norm (an infinity in them, or one value and
    eps = 0) and columns whose weight is infinite too."""
    x, r, w, b, _, dh = _inputs((6, cols), *types)
    with torch.no_grad():
        x[1, 3], r[2, cols - 1], r[3, 0] = float("inf"), float("-inf"), float("nan")
        x[4], r[4] = 0.0, 2.0
        w[5] = float("inf")
    _, _, grads = _run(x, r, w, b, None, dh, 0.5, 7, eps=0.0)
    keep = R.keep_mask(x.shape, 0.5, 7).cuda()
    assert torch.equal(grads["r"], dh)
    assert torch.equal(grads["x"], torch.where(keep, dh.float() * 2, 0.0).to(types[0]))
    assert (grads["w"] == 0).all() and (grads["b"] == 0).all()
