"""residual + dropout(x) and its gradients against the 64-bit form, element by element, and the ways it is called."""
import threading

import pytest
import torch

import protenix_amd as P
from protenix_amd import ops
from tests import residual_oracle as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)]


def _inputs(shape, tx, tr, seed=0, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g).to(tx).cuda().requires_grad_()
    r = torch.randn(shape, generator=g).mul(3).to(tr).cuda().requires_grad_() if residual else None
    d = torch.randn(shape, generator=g).to(tr if residual else tx).cuda()
    return x, r, d


def _check(got, want, parts, what):
    """`got` is one rounding to its type of a value formed from `parts` in fp32 (two roundings: the factor's and the product's
    or the sum's)."""
    got, want = got.detach().cpu(), want.cpu()
    tol = R.half_step(got.dtype) * want.abs() + 2.0**-23 * sum(p.abs() for p in parts) + R.smallest(got.dtype)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, bad.sum().item(), got[bad][:4], want[bad][:4])


def _compare(x, r, d, p, seed, shared_dim, out, grads):
    h, m = R.update(x, r, p, seed, shared_dim)
    xd, dd = x.detach().cpu().double(), d.cpu().double()
    kept = torch.where(m != 0, xd * m, torch.zeros_like(xd))
    _check(out, h, [kept] + ([] if r is None else [r.detach().cpu().double()]), "out")
    _check(grads[0], torch.where(m != 0, dd * m, torch.zeros_like(dd)), [dd * m], "dx")
    # what is dropped leaves the residual as it is, and no gradient
    gone = m == 0
    assert torch.equal(out.detach().cpu()[gone], (torch.zeros_like(xd).to(out.dtype) if r is None else r.detach().cpu().to(out.dtype))[gone])
    assert (grads[0].cpu()[gone] == 0).all()
    if r is not None:
        assert torch.equal(grads[1], d)


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape,shared_dim", [((1,), None), ((7,), None), ((3, 1), None), ((5, 8), None), ((1, 93, 384), None),
                                              ((2, 3, 5, 67), -2), ((2, 9, 5, 64), -3), ((2, 17, 33, 13), 0), ((40, 3, 16), 0),
                                              ((4, 131, 1030), 1), ((1, 1, 128), -2), ((70000, 9), 0), ((1000, 3, 1), -2)])
def test_values_and_gradients(types, shape, shared_dim):
    x, r, d = _inputs(shape, *types, seed=len(shape))
    out = P.dropout_add(x, r, 0.1, shared_dim=shared_dim, seed=99)
    assert out.dtype == types[1] and out.shape == x.shape
    grads = torch.autograd.grad(out, [x, r], d)
    assert grads[0].dtype == types[0]
    _compare(x, r, d, 0.1, 99, shared_dim, out, grads)


@pytest.mark.parametrize("p", [0.0, 1e-6, 0.25, 0.5, 0.999, 1.0, 1 / 3])
@pytest.mark.parametrize("residual", [True, False])
def test_probabilities(p, residual):
    x, r, d = _inputs((61, 1003), BF16, F32 if residual else BF16, seed=3, residual=residual)
    leaves = [x] if r is None else [x, r]
    out = P.dropout_add(x, r, p, seed=(1 << 63) + 12345)
    _compare(x, r, d, p, (1 << 63) + 12345, None, out, torch.autograd.grad(out, leaves, d))
    still = P.dropout_add(x, r, p, training=False)
    assert torch.equal(still, P.dropout_add(x, r, 0.0))


def test_numbers_at_the_threshold_are_told_apart():
    """A million elements have some sixteen whose first 16 bits equal the threshold's: below and above it."""
    n, seed, p = 1 << 20, 5, 0.1
    assert round(p * 2**32) & 0xFFFF
    out = P.dropout_add(torch.ones(n // 64, 64, device="cuda"), None, p, seed=seed)
    assert torch.equal(out.cpu() != 0, R.keep_mask((n // 64, 64), p, seed))


def test_dropped_infinities_and_nan_leave_nothing():
    x = torch.full((64, 64), float("nan"), device="cuda")
    x[::2] = float("inf")
    keep = R.keep_mask((64, 64), 0.5, 3).cuda()
    r = torch.randn(64, 64, device="cuda")
    out = P.dropout_add(x, r, 0.5, seed=3)
    assert torch.equal(out[~keep], r[~keep])
    assert out[keep].isfinite().logical_not().all()


def test_strides_offsets_and_expanded_gradients():
    base, resb = torch.randn(37, 29, 66, device="cuda"), torch.randn(29, 37, 64, device="cuda")
    x, r = base[:, :, 1:65].transpose(0, 1), resb
    want = P.dropout_add(x.contiguous(), r, 0.3, seed=8, shared_dim=0)
    assert torch.equal(P.dropout_add(x, r, 0.3, seed=8, shared_dim=0), want)
    assert torch.equal(P.dropout_add(x, r.expand(29, 37, 64), 0.3, seed=8, shared_dim=-3), want)
    flat = torch.randn(1 + 24 * 40, device="cuda").to(BF16)
    off = flat[1:].view(24, 40)             # starts at an odd element
    assert torch.equal(P.dropout_add(off, None, 0.3, seed=1), P.dropout_add(off.clone(), None, 0.3, seed=1))
    y = x.detach().clone().requires_grad_()
    g, = torch.autograd.grad(P.dropout_add(y, r, 0.3, seed=8).sum(), y)     # the gradient of a sum is an expanded one
    assert torch.equal(g != 0, R.keep_mask((29, 37, 64), 0.3, 8).cuda())


def test_python_and_native_paths_give_the_same_bits(monkeypatch):
    x, r, d = _inputs((5, 31, 200), BF16, F32)
    seed = torch.tensor([77], device="cuda")
    for kw in ({"seed": 12}, {"seed": seed, "shared_dim": -2}):
        out = P.dropout_add(x, r, 0.2, **kw)
        grads = torch.autograd.grad(out, [x, r], d)
        with monkeypatch.context() as m:
            m.setattr(ops, "native_enabled", False)
            out2 = P.dropout_add(x, r, 0.2, **kw)
            grads2 = torch.autograd.grad(out2, [x, r], d)
            with torch.no_grad():
                assert torch.equal(P.dropout_add(x, r, 0.2, **kw), out)
        assert torch.equal(out, out2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


def test_seeds():
    x = torch.ones(64, 96, device="cuda")
    a = P.dropout_add(x, None, 0.5, seed=4)
    assert torch.equal(a, P.dropout_add(x, None, 0.5, seed=torch.tensor(4, device="cuda")))
    assert torch.equal(P.dropout_add(x, None, 0.5, seed=-1), P.dropout_add(x, None, 0.5, seed=(1 << 64) - 1))
    assert not torch.equal(a, P.dropout_add(x, None, 0.5, seed=4 + (1 << 32)))
    torch.manual_seed(11)
    b, c = P.dropout_add(x, None, 0.5), P.dropout_add(x, None, 0.5)
    assert not torch.equal(b, c)
    torch.manual_seed(11)
    assert torch.equal(b, P.dropout_add(x, None, 0.5))
    # the mask does not depend on the type, nor does it on the residual
    assert torch.equal(a != 0, P.dropout_add(x.to(BF16), None, 0.5, seed=4) != 0)


@pytest.mark.parametrize("native", [True, False])
def test_a_changed_seed_tensor_is_noticed_in_backward(native, monkeypatch):
    monkeypatch.setattr(ops, "native_enabled", native)
    x, seed = torch.ones(8, 8, device="cuda", requires_grad=True), torch.tensor([4], device="cuda")
    out = P.dropout_add(x, None, 0.5, seed=seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("native", [True, False])
def test_gradients_of_gradients_are_refused(native, monkeypatch):
    monkeypatch.setattr(ops, "native_enabled", native)
    x = torch.ones(8, 8, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(P.dropout_add(x, x, 0.5, seed=1).pow(2).sum(), x, create_graph=True)
        g.sum().backward()


def test_one_tensor_as_update_and_residual():
    x = torch.randn(16, 40, device="cuda", requires_grad=True)
    P.dropout_add(x, x, 0.5, seed=6).sum().backward()
    assert torch.equal(x.grad.cpu(), 1 + 2 * R.keep_mask((16, 40), 0.5, 6).float())


def test_what_needs_no_gradient_gets_none():
    x, r, d = _inputs((6, 24), BF16, F32)
    out = P.dropout_add(x.detach(), r, 0.5, seed=2)
    out.backward(d)
    assert torch.equal(r.grad, d)
    out = P.dropout_add(x, r.detach(), 0.5, seed=2)
    out.backward(d)
    assert x.grad is not None
    with torch.no_grad():
        assert not P.dropout_add(x, r, 0.5, seed=2).requires_grad


@pytest.mark.parametrize("shape", [(0,), (0, 8), (4, 0), (2, 0, 3, 8)])
def test_empty(shape):
    x = torch.zeros(shape, device="cuda", requires_grad=True, dtype=BF16)
    r = torch.zeros(shape, device="cuda", requires_grad=True)
    out = P.dropout_add(x, r, 0.5, shared_dim=0 if len(shape) > 1 else None)
    assert out.shape == x.shape and out.dtype == F32
    out.sum().backward()
    assert x.grad.shape == x.shape and r.grad.shape == r.shape


def test_refusals():
    x = torch.zeros(4, 6, 8, device="cuda")
    for args, kw, match in [((x, x[:2]), {}, "differ"), ((x, x.cpu()), {}, "differ"), ((x.to(BF16), x.to(F16)), {}, "type"),
                            ((x, x.to(BF16)), {}, "type"), ((x.double(),), {}, "float32, bfloat16 or float16"),
                            ((x.long(),), {}, "float32"), ((x[0, 0, 0],), {}, "dimension"), ((x, x, -0.1), {}, "probability"),
                            ((x, x, 1.5), {}, "probability"), ((x, x, float("nan")), {}, "probability"),
                            ((x, x), {"shared_dim": -1}, "last"), ((x, x), {"shared_dim": 2}, "last"), ((x, x), {"shared_dim": 3}, "last"),
                            ((x, x), {"shared_dim": -4}, "last"), ((x, x), {"seed": 1 << 64}, "64 bits"),
                            ((x, x), {"seed": torch.zeros(2, dtype=torch.int64, device="cuda")}, "seed tensor"),
                            ((x, x), {"seed": torch.zeros(1, device="cuda")}, "seed tensor"),
                            ((x, x), {"seed": torch.zeros(1, dtype=torch.int64)}, "seed tensor")]:
        with pytest.raises(RuntimeError, match=match):
            P.dropout_add(*args, **kw)
    with pytest.raises(RuntimeError, match="unsupported"):
        P.dropout_add(x[0, 0, :1].expand(1 << 31))
    with pytest.raises(TypeError):
        P.dropout_add(x, x, seed=1.5)


def _graphed(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_replays_draw_with_the_seed_the_tensor_holds_then():
    x, r, d = _inputs((3, 50, 128), BF16, F32)
    seed = torch.zeros(1, dtype=torch.int64, device="cuda")

    def step():
        out = P.dropout_add(x, r, 0.25, shared_dim=0, seed=seed)
        return (out.detach(), *torch.autograd.grad(out, [x, r], d))

    graph, outs = _graphed(step)
    for rep in range(4):
        seed.fill_(1000 + rep)
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step())), rep


def test_a_recorded_call_needs_its_seed_and_leaves_of_its_own():
    x = torch.randn(8, 16, device="cuda", requires_grad=True)
    alive = P.dropout_add(x, None, 0.5, seed=1)          # an eager graph that holds x's accumulator
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="needs its seed"):
            P.dropout_add(x.detach(), None, 0.5)
        with pytest.raises(RuntimeError, match="eager graph that is still alive"):
            P.dropout_add(x, None, 0.5, seed=1)
        out = P.dropout_add(x.detach(), None, 0.5, seed=1)
    graph.replay()
    assert torch.equal(out, alive)


def test_side_streams_and_threads():
    x, r, d = _inputs((64, 1024), BF16, F32)
    want = P.dropout_add(x, r, 0.2, seed=3)
    want_g = torch.autograd.grad(want, [x, r], d)
    torch.cuda.synchronize()
    got = {}

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                out = P.dropout_add(x, r, 0.2, seed=3)
                grads = torch.autograd.grad(out, [x, r], d)
        s.synchronize()
        got[i] = (out, *grads)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert len(got) == 3
    for g in got.values():
        assert torch.equal(g[0], want) and torch.equal(g[1], want_g[0]) and torch.equal(g[2], want_g[1])


@pytest.mark.parametrize("native", [True, False])
def test_recorded_gradients_of_a_leaf_that_an_eager_graph_holds_are_refused(native, monkeypatch):
    # in each operator and on both host paths (the Python one also takes what the native one hands back: int32 positions, large seeds)
    monkeypatch.setattr(ops, "native_enabled", native)
    x, w = (torch.randn(s, device="cuda", requires_grad=True) for s in ((8, 16), (16,)))
    table, buckets = torch.randn(9, 2, device="cuda", requires_grad=True), P.RelativeBuckets(4)
    pos = torch.arange(5, device="cuda", dtype=torch.int32)
    calls = [lambda: P.dropout_add(x, None, 0.5, seed=1), lambda: P.dropout_add(x, None, 0.5, seed=1 << 63),
             lambda: P.dropout_add_layer_norm(x.detach(), None, w, None, 0.5, seed=1),
             lambda: P.dropout_add_layer_norm(x.detach(), x, None, None, 0.5, seed=1 << 63),
             lambda: P.relative_position_bias(table, buckets, range(5), range(5)),
             lambda: P.relative_position_bias(table, buckets, pos, pos)]
    alive = [f() for f in calls]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for f in calls:
            with pytest.raises(RuntimeError, match="eager graph that is still alive"):
                f()
        with torch.no_grad():      # (nothing to accumulate: taken)
            out = [f() for f in calls]
    graph.replay()
    torch.cuda.synchronize()
    flat = lambda l: [t for o in l for t in (o if isinstance(o, tuple) else (o,))]
    assert all(torch.equal(a, b) for a, b in zip(flat(out), flat(alive)))


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shared_dim", [None, 0])
def test_rows_that_end_anywhere_in_a_block(types, shared_dim):
    for cols in range(1, 24):
        x, r, d = _inputs((6, 3, cols), *types, seed=cols)
        out = P.dropout_add(x, r, 0.2, shared_dim=shared_dim, seed=cols)
        _compare(x, r, d, 0.2, cols, shared_dim, out, torch.autograd.grad(out, [x, r], d))
