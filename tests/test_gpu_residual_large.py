"""Residual dropout, its norm and the position bias on tensors of more than 2^31 elements: the last of them are where they should be."""
import numpy as np
import pytest
import torch

import protenix_amd as P
from tests import residual_oracle as R

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _keep_rows(first, rows, cols, p, seed):
    """keep_mask of mask rows first .. first + rows - 1."""
    blocks = -(-cols // 8)
    counter = np.zeros((rows, blocks, 4), np.uint64)
    counter[..., 0] = np.arange(blocks)[None, :]
    counter[..., 1] = (first + np.arange(rows))[:, None]
    u = np.zeros((rows, blocks, 8), np.uint64)
    for draw in (0, 1):
        counter[..., 3] = draw
        w = R.philox(counter, (seed & 0xFFFFFFFF, seed >> 32))
        u = (u << np.uint64(16)) | np.stack((w & np.uint64(0xFFFF), w >> np.uint64(16)), -1).reshape(rows, blocks, 8)
    return torch.from_numpy(u.reshape(rows, blocks * 8)[:, :cols] >= np.uint64(round(p * 2.0**32)))


@pytest.mark.parametrize("rows,cols,shared", [(33001, 65600, False), (2, 33001 * 32800, True), ((1 << 21) + 7, 1025, False)])
def test_dropout_add(rows, cols, shared):
    x = torch.ones(rows, cols, device="cuda", dtype=BF16)
    out = P.dropout_add(x, None, 0.5, seed=(7 << 32) + 1, shared_dim=0 if shared else None)
    tail = slice(cols - 4096, cols) if shared else slice(0, cols)
    if shared:      # one mask row: the columns at the end of both rows
        assert torch.equal(out[0, -(1 << 20):], out[1, -(1 << 20):])
        blocks = np.arange((cols - 4096) // 8, -(-cols // 8), dtype=np.uint64)
        counter = np.zeros((len(blocks), 4), np.uint64)
        counter[:, 0] = blocks
        w = R.philox(counter, (1, 7))
        keep = torch.from_numpy(np.stack((w & np.uint64(0xFFFF), w >> np.uint64(16)), -1).reshape(-1)[:4096] >= np.uint64(1 << 15))
        assert cols % 8 == 0 and torch.equal(out[1, tail].cpu() != 0, keep)
    else:
        assert torch.equal(out[-3:].cpu() != 0, _keep_rows(rows - 3, 3, cols, 0.5, (7 << 32) + 1))
    assert abs(out[-1].float().mean().item() - 1) < 0.1


def test_dropout_add_layer_norm():
    rows, cols, seed = 140001, 16000, 11
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, cols, device="cuda", dtype=BF16, generator=g).requires_grad_()
    w = torch.ones(cols, device="cuda", requires_grad=True)
    y, h = P.dropout_add_layer_norm(x, None, w, None, 0.25, seed=seed)
    dx, dw = torch.autograd.grad(y, [x, w], x.detach())
    keep = _keep_rows(rows - 2, 2, cols, 0.25, seed).double() / 0.75
    xe = x[-2:].detach().cpu().double().requires_grad_()
    he = xe * keep
    ye = R.norm_parts(he, None, None, 1e-5)[0]
    ge, = torch.autograd.grad(ye, xe, xe.detach())
    for got, want in ((y[-2:], ye), (h[-2:], he), (dx[-2:], ge)):
        err = (got.detach().cpu().double() - want.detach()).abs().max().item()
        assert err <= 2.0**-8 * want.abs().max().item(), err      # half a step of bf16 beside what fp32 loses (a thousandth of that)
    assert dw.isfinite().all()


def test_relative_position_bias():
    n, heads = 17001, 8
    b = P.RelativeBuckets(128, 32)
    table = torch.randn(32, heads, device="cuda", requires_grad=True)
    out = P.relative_position_bias(table, b, range(n), range(n), dtype=BF16)
    u = torch.tensor([b.bucket(j - (n - 1)) for j in range(n)])
    assert torch.equal(out[-1, -1].detach().cpu(), table.detach().cpu().to(BF16)[u, heads - 1])
    dout = torch.zeros_like(out)
    dout[:, -1] = 1.0
    grad, = torch.autograd.grad(out, table, dout)
    assert torch.equal(grad.cpu(), torch.bincount(u, minlength=32).float()[:, None].expand(32, heads))
