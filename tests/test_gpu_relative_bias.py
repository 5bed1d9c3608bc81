"""The learned bias by buckets of relative position and its table's gradient against the 64-bit form."""
import numpy as np
import pytest
import torch

import protenix_amd as P
from protenix_amd import ops
from tests import residual_oracle as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SCHEMES = [(32, None, True), (1, None, True), (5, None, False), (128, 32, True), (128, 32, False), (100, 254, True), (8192, 255, False)]


def _buckets(scheme):
    return P.RelativeBuckets(scheme[0], scheme[1], bidirectional=scheme[2])


def _tensor(p, batch):
    t = torch.arange(p.start, p.stop) if isinstance(p, range) else p.cpu()
    return (t if t.dim() == 2 else t[None]).expand(batch, -1)


def _oracle_buckets(scheme, q, k, groups=None):
    """[B, Q, K] bucket numbers of whole-number tensors."""
    top, count, both = scheme
    lut = np.array([R.bucket(d, top, count, both) for d in range(-top, top + 1)])
    # (Python's whole numbers: differences of 64-bit positions do not fit 64 bits)
    d = np.empty((len(q), q.shape[1], k.shape[1]), np.int64)
    for b in range(len(q)):
        kk = [int(v) for v in k[b]]
        for i, a in enumerate(int(v) for v in q[b]):
            d[b, i] = [max(-top, min(top, c - a)) for c in kk]
    u = lut[d + top]
    if groups is not None:
        gq, gk = (g.numpy() for g in groups)
        u = np.where(gk[:, None, :] == gq[:, :, None], u, lut.max() + 1 if count is None else count)
    return torch.from_numpy(u)


def _check(scheme, table, q, k, groups, dtype, out, dout=None, grad=None):
    batch = out.shape[0] if out.dim() == 4 else 1
    gs = None if groups is None else tuple(_tensor(g, batch) for g in groups)
    u = _oracle_buckets(scheme, _tensor(q, batch), _tensor(k, batch), gs)
    want = table.detach().cpu().to(dtype)[u].movedim(-1, 1)          # (a value of the table, rounded once: equal, not near)
    assert out.dtype == dtype and torch.equal(out.detach().cpu().reshape(want.shape), want)
    if grad is None:
        return
    d = dout.detach().cpu().double().reshape(want.shape).movedim(1, -1).reshape(-1, table.shape[1])
    sums = torch.zeros(table.shape, dtype=torch.double).index_add_(0, u.reshape(-1), d)
    size = torch.zeros(table.shape, dtype=torch.double).index_add_(0, u.reshape(-1), d.abs())
    # fp32 sums: a lane adds at most all its elements in turn, (elements of a head) / (65536 lanes / heads), at least 8, then
    # 4 waves, 6 exchanges and 1024 / 64 slices
    turn = 2.0**-24 * (d.shape[0] * table.shape[1] / 16384 + 64)
    tol = R.half_step(grad.dtype) * sums.abs() + turn * size + R.smallest(grad.dtype)
    got = grad.cpu()
    bad = ~((got.double() - sums).abs() <= tol)
    assert not bad.any(), (bad.nonzero()[:4], got[bad][:4], sums[bad][:4])


def _run(scheme, heads, q, k, groups=None, table_dtype=F32, dtype=F32, seed=0):
    g = torch.Generator().manual_seed(seed)
    b = _buckets(scheme)
    table = torch.randn(b.num_buckets + (groups is not None), heads, generator=g).to(table_dtype).cuda().requires_grad_()
    out = P.relative_position_bias(table, b, q, k, groups=groups, dtype=dtype)
    dout = torch.randn(out.shape, generator=g).to(dtype).cuda()
    grad, = torch.autograd.grad(out, table, dout)
    assert grad.dtype == table_dtype and grad.shape == table.shape
    _check(scheme, table, q, k, groups, dtype, out, dout, grad)
    return table, out


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("q,k", [(range(1), range(1)), (range(9), range(9)), (range(0, 50), range(0, 300)), (range(299, 300), range(0, 300)),
                                 (range(700, 713), range(3, 1030)), (range(-5, 30), range(0, 8)), (range(1 << 40, (1 << 40) + 7), range(0, 20))])
def test_ranges(scheme, q, k):
    _run(scheme, 3, q, k)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("table_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads", [1, 4, 16])
def test_types_and_heads(dtype, table_dtype, heads):
    _run((128, 32, True), heads, range(130), range(211), table_dtype=table_dtype, dtype=dtype)


def _chains(batch, n, seed):
    rng = np.random.default_rng(seed)
    pos, grp = np.zeros((batch, n), np.int64), np.zeros((batch, n), np.int64)
    for b in range(batch):
        at, c = 0, 0
        while at < n:
            m = min(int(rng.integers(1, 60)), n - at)
            pos[b, at:at + m] = int(rng.integers(-9, 50)) + np.arange(m)
            grp[b, at:at + m] = c % 3
            at, c = at + m, c + 1
    return torch.from_numpy(pos).cuda(), torch.from_numpy(grp).cuda()


@pytest.mark.parametrize("scheme", SCHEMES)
@pytest.mark.parametrize("n", [1, 7, 130, 411])
def test_chains(scheme, n):
    pos, grp = _chains(2, n, n)
    _run(scheme, 4, pos, pos, (grp, grp), dtype=BF16)
    _run(scheme, 4, pos[:, n // 2:], pos, (grp[:, n // 2:], grp))
    _run(scheme, 2, pos[0], pos[0], (grp[0].int(), grp[0].int()))


def test_positions_without_order_repeated_and_at_the_ends_of_64_bits():
    top = (1 << 63) - 1
    p = torch.tensor([5, 5, -7, top, -top - 1, 0, 1, top - 3, -top, 5, 12], device="cuda")
    _run((8, None, True), 2, p, p)
    _run((128, 32, False), 2, p.flip(0), p)
    _run((100, 254, True), 2, torch.tensor([3, -100], device="cuda", dtype=torch.int32), p)


def test_groups_of_any_numbers():
    """Group numbers that differ by 2^32 and more, or by everything 64 bits hold."""
    pos, grp = _chains(2, 97, 6)
    for numbers in ([5, 5 + (1 << 32), -5], [(1 << 63) - 1, -(1 << 63), 0], [0, 1 << 30, -(1 << 30)]):
        g = torch.tensor(numbers, device="cuda")[grp]
        _run((8, None, True), 3, pos, pos, (g, g), dtype=BF16)
    # positions and groups that jump from query to query and from key to key
    perm = torch.randperm(97, generator=torch.Generator().manual_seed(1)).cuda()
    _run((128, 32, True), 3, pos[:, perm], pos, (grp[:, perm], grp))
    _run((128, 32, True), 3, pos, pos[:, perm], (grp, grp[:, perm]))


def test_batched_positions_beside_single_ones():
    pos, grp = _chains(3, 40, 1)
    _run((32, None, True), 4, pos, range(25))
    _run((32, None, True), 4, pos[0], pos)
    _run((32, None, True), 4, range(40), range(40), (grp, grp[0]))


@pytest.mark.parametrize("heads", [1, 5, 300])
def test_many_heads_and_buckets(heads):
    _run((127, None, True), heads, range(20), range(60))
    pos, grp = _chains(1, 50, 3)
    _run((127, None, True), heads, pos, pos, (grp, grp), dtype=F16)


def test_long_sums():
    """Two million elements a head in a handful of buckets."""
    _run((1, None, True), 2, range(1500), range(1400), dtype=BF16)


@pytest.mark.parametrize("q,k", [(range(0), range(5)), (range(5), range(0)), (range(0), range(0))])
def test_empty(q, k):
    table = torch.randn(32, 4, device="cuda", requires_grad=True)
    out = P.relative_position_bias(table, P.RelativeBuckets(128, 32), q, k)
    assert out.shape == (4, len(q), len(k))
    g, = torch.autograd.grad(out.sum(), table)
    assert (g == 0).all()
    none = P.relative_position_bias(table, P.RelativeBuckets(128, 32), torch.zeros(0, 3, dtype=torch.int64, device="cuda"), range(3))
    assert none.shape == (0, 4, 3, 3)


def test_infinite_entries_and_nan_stay_in_their_buckets():
    b = P.RelativeBuckets(3)
    table = torch.zeros(7, 2, device="cuda")
    table[0], table[6, 1] = float("-inf"), float("nan")
    out = P.relative_position_bias(table, b, range(20), range(20))
    d = torch.arange(20)[None] - torch.arange(20)[:, None]
    assert torch.equal(out.cpu()[0].isinf(), d <= -3) and torch.equal(out.cpu()[1].isnan(), d >= 3)
    # a gradient's NaN reaches its own bucket and head only
    table.requires_grad_()
    dout = torch.ones(2, 20, 20, device="cuda")
    dout[1, 4, 5] = float("nan")
    g, = torch.autograd.grad(P.relative_position_bias(table, b, range(20), range(20)), table, dout)
    assert g.isnan().nonzero().tolist() == [[4, 1]]


def test_paths_and_repeats_give_the_same_bits(monkeypatch):
    pos, grp = _chains(2, 333, 5)
    b = _buckets((32, None, True))
    table = torch.randn(66, 4, device="cuda", requires_grad=True)
    dout = torch.randn(2, 4, 333, 333, device="cuda").to(BF16)

    def run():
        out = P.relative_position_bias(table, b, pos, pos, groups=(grp, grp), dtype=BF16)
        return out, *torch.autograd.grad(out, table, dout)

    first = run()
    assert all(torch.equal(a, c) for a, c in zip(first, run()))
    monkeypatch.setattr(ops, "poison_workspaces", True)
    assert all(torch.equal(a, c) for a, c in zip(first, run()))
    with torch.no_grad():
        assert torch.equal(first[0], P.relative_position_bias(table, b, pos, pos, groups=(grp, grp), dtype=BF16))


def test_gradient_layouts():
    """Gradients that are expanded or transposed."""
    table = torch.randn(32, 4, device="cuda", requires_grad=True)
    b = P.RelativeBuckets(128, 32)
    out = P.relative_position_bias(table, b, range(60), range(60))
    g, = torch.autograd.grad(out, table, torch.ones(1, device="cuda").expand(4, 60, 60), retain_graph=True)
    assert g.sum().item() == 4 * 3600
    d = torch.randn(4, 60, 60, device="cuda")
    a, = torch.autograd.grad(out, table, d.transpose(1, 2), retain_graph=True)
    c, = torch.autograd.grad(out, table, d.transpose(1, 2).contiguous())
    assert torch.equal(a, c)
    wide = torch.randn(4, 32, device="cuda").t()
    assert torch.equal(P.relative_position_bias(wide, b, range(9), range(9)), P.relative_position_bias(wide.contiguous(), b, range(9), range(9)))


def test_refusals():
    b = P.RelativeBuckets(128, 32)
    t = torch.zeros(32, 4, device="cuda")
    i = torch.zeros(2, 5, dtype=torch.int64, device="cuda")
    for args, kw, match in [((t[:31], b, range(3), range(3)), {}, "table is"), ((t, b, range(3), range(3)), {"groups": (i[0, :3], i[0, :3])}, "table is"),
                            ((t[0], b, range(3), range(3)), {}, "table is"), ((t[:, :0], b, range(3), range(3)), {}, "table is"),
                            ((t.double(), b, range(3), range(3)), {}, "float32"), ((t, b, range(0, 6, 2), range(3)), {}, "step 1"),
                            ((t, b, i.float(), range(3)), {}, "whole numbers"), ((t, b, 3, range(3)), {}, "whole numbers"),
                            ((t, b, i[None], range(3)), {}, "whole numbers"), ((t, b, i.cpu(), range(3)), {}, "table on"),
                            ((t, b, i, i[:1].expand(3, 5)), {}, "batch sizes"), ((t, b, range(3), range(3)), {"dtype": torch.float64}, "float32"),
                            ((t, b, range(1 << 62, (1 << 62) + 3), range(3)), {}, "positions from"),
                            ((torch.zeros(33, 4, device="cuda"), b, range(3), range(3)), {"groups": (i[0], i[0])}, "groups of"),
                            ((t, b, range((1 << 32) + 3), range(1)), {}, "unsupported"), ((t, b, range(1), range((1 << 30) + 1)), {}, "unsupported")]:
        with pytest.raises(RuntimeError, match=match):
            P.relative_position_bias(*args, **kw)
    m = P.RelativePositionBias(4, b, grouped=True).cuda()
    assert m.weight.shape == (33, 4)
    with pytest.raises(RuntimeError, match="grouped"):
        m(range(3), range(3))
    t.requires_grad_()
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(P.relative_position_bias(t, b, range(3), range(3)).pow(2).sum(), t, create_graph=True)
        g.sum().backward()


def test_recorded_and_replayed():
    pos, grp = _chains(1, 100, 5)
    m = P.RelativePositionBias(4, P.RelativeBuckets(32), grouped=True).cuda()
    dout = torch.randn(1, 4, 100, 100, device="cuda")

    def step():
        out = m(pos, pos, (grp, grp))
        return out.detach(), *torch.autograd.grad(out, m.weight, dout)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for rep in range(4):
        with torch.no_grad():
            m.weight.copy_(torch.randn_like(m.weight))
            new, g2 = _chains(1, 100, 50 + rep)
            pos.copy_(new)
            grp.copy_(g2)
            dout.copy_(torch.randn_like(dout))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(outs, step())), rep


def test_batches_beyond_the_units_a_launch_can_number_are_refused():
    b, t = P.RelativeBuckets(4), torch.zeros(9, 1, device="cuda")
    one = torch.zeros(1, 1, dtype=torch.int64, device="cuda")
    for n in ((1 << 30) + 1, (1 << 32) + 1):
        with pytest.raises(RuntimeError, match="unsupported"):
            P.relative_position_bias(t, b, one.expand(n, 1), range(1))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("heads", [1, 5])
def test_rows_that_end_anywhere_in_a_block(dtype, heads):
    for k in range(1, 24):
        _run((5, None, False), heads, range(7, 20), range(k), dtype=dtype, seed=k)


@pytest.mark.parametrize("batch,heads,q", [(700, 16, 1), (300, 40, 3), (1, 300, 2)])
def test_heads_side_by_side(batch, heads, q):
    g = torch.Generator().manual_seed(batch)
    pos = torch.randint(-40, 40, (batch, 65), generator=g).cuda()
    _run((32, None, True), heads, pos[:, :q].contiguous(), pos, dtype=BF16)


def test_ranges_whose_length_passes_63_bits_are_refused():
    b, t = P.RelativeBuckets(4), torch.zeros(9, 2, device="cuda")
    for far in (range(-(1 << 62), 1 << 62), range(-(1 << 62), (1 << 63) - 1), range(-(1 << 62), (1 << 62) + 3), range(0, 1 << 70)):
        for sides in ((far, range(3)), (range(3), far)):
            with pytest.raises(RuntimeError, match="unsupported"):
                P.relative_position_bias(t, b, *sides)
    assert P.relative_position_bias(t, b, range(5, 3), range(3)).shape == (2, 0, 3)
    assert P.relative_position_bias(t, b, range(5, -(1 << 70)), range(3)).shape == (2, 0, 3)
