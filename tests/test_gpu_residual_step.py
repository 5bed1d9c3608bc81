"""The operators as a training step has them: positions make the attention's bias, the attention's result is dropped out
onto the residual stream, and the next layer reads its norm."""
import pytest
import torch

import protenix_amd as P
from tests import residual_oracle as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 2e-2)])
@pytest.mark.parametrize("n,rows", [(37, 5), (64, 64)])
def test_bias_attention_dropout_norm(dtype, tol, n, rows):
    H, D, C = 4, 32, 128
    g = torch.Generator().manual_seed(n)
    draw = lambda *s, t=dtype, scale=1.0: torch.randn(*s, generator=g).mul(scale).to(t)
    q, k, v = draw(1, rows, n, H, D, scale=0.3), draw(1, rows, n, H, D), draw(1, rows, n, H, D)
    z = draw(1, rows, n, C, t=torch.float32, scale=2.0)
    table, w, b = draw(18, H, t=torch.float32), draw(C, t=torch.float32, scale=0.1) + 1, draw(C, t=torch.float32, scale=0.1)
    mask = torch.zeros(1, rows, 1, 1, n)
    mask[..., n - 3:] = -1e9
    dy, dh = draw(1, rows, n, C), draw(1, rows, n, C, t=torch.float32)
    chain = torch.arange(n) // 20
    pos = torch.arange(n) % 20

    leaves = [t.cuda().requires_grad_() for t in (q, k, v, z, table, w, b)]
    qg, kg, vg, zg, tg, wg, bg = leaves
    bias = P.relative_position_bias(tg, P.RelativeBuckets(8), pos.cuda(), pos.cuda(), groups=(chain.cuda(), chain.cuda()), dtype=dtype)
    o = P.TriAttentionFunction.apply(qg, kg, vg, mask.cuda().to(dtype), bias[None, None])
    z1 = P.dropout_add(o.reshape(1, rows, n, C), zg, 0.25, shared_dim=-3, seed=5)
    y, h = P.dropout_add_layer_norm(o.reshape(1, rows, n, C), z1, wg, bg, 0.25, shared_dim=-2, seed=6)
    grads = torch.autograd.grad((y, h), leaves, (dy.cuda(), dh.cuda()))

    exact = [t.double().requires_grad_() for t in (q, k, v, z, table, w, b)]
    qe, ke, ve, ze, te, we, be = exact
    d = (pos[None, :] - pos[:, None]).clamp(-8, 8) + 8
    u = torch.where(chain[None, :] == chain[:, None], d, torch.full_like(d, 17))
    s = torch.einsum("bnihd,bnjhd->bnhij", qe, ke) + mask.double() + te[u].movedim(-1, 0)[None, None]
    oe = torch.einsum("bnhij,bnjhd->bnihd", s.softmax(-1), ve).reshape(1, rows, n, C)
    m1, m2 = (R.keep_mask((1, rows, n, C), 0.25, sd, dim).double() / 0.75 for sd, dim in ((5, -3), (6, -2)))
    he = ze + oe * m1 + oe * m2
    ye = R.norm_parts(he, None, None, 1e-5)[0] * we + be
    want = torch.autograd.grad((ye, he), exact, (dy.double(), dh.double()))
    for name, got, ref in [("y", y, ye), ("h", h, he)] + list(zip("qkvztwb", grads, want)):
        err = ((got.detach().cpu().double() - ref.detach()).abs().max() / ref.abs().max()).item()
        assert err < tol, (name, err)
