"""Residual dropout, its norm and the position bias beside forward-mode differentiation."""
import pytest
import torch
from torch.autograd import forward_ad

import protenix_amd as P
from protenix_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_forward_mode_derivatives_are_refused(native, monkeypatch):
    """The operators have none: a result without a tangent would say that it is zero."""
    monkeypatch.setattr(ops, "native_enabled", native)
    x, w, table = (torch.randn(s, device="cuda") for s in ((8, 16), (16,), (9, 2)))
    buckets, pos = P.RelativeBuckets(4), torch.arange(5, device="cuda", dtype=torch.int32)
    calls = {"update": lambda t: P.dropout_add(t(x), x, 0.5, seed=1), "residual": lambda t: P.dropout_add(x, t(x), 0.5, seed=1 << 63),
             "of the norm": lambda t: P.dropout_add_layer_norm(t(x)), "its residual": lambda t: P.dropout_add_layer_norm(x, t(x), w, w, 0.5, seed=1),
             "weight": lambda t: P.dropout_add_layer_norm(x, None, t(w)), "bias": lambda t: P.dropout_add_layer_norm(x, None, w, t(w)),
             "table": lambda t: P.relative_position_bias(t(table), buckets, range(5), range(5)),
             "table, int32": lambda t: P.relative_position_bias(t(table), buckets, pos, pos)}
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for name, f in calls.items():
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    f(dual)
            with pytest.raises(RuntimeError, match="forward-mode"):
                f(lambda t: dual(t.clone().requires_grad_()))
            f(lambda t: t)
        with forward_ad._set_fwd_grad_enabled(False):      # (as in the forward of a user's own function, which has its own rule)
            [f(dual) for f in calls.values()]
