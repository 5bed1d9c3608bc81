"""8-bit blocks and the RMS norm without a GPU: what is refused, and the oracle against torch's own 8-bit type."""
import pytest
import torch

import protenix_amd as P
from protenix_amd import _lib
from tests import fp8_oracle as Q


def test_the_oracle_rounds_as_the_type_does():
    g = torch.Generator().manual_seed(0)
    v = torch.cat([torch.randn(20000, generator=g) * 100, torch.randn(20000, generator=g) * 0.01, torch.linspace(-448, 448, 7169)]).clamp(-448, 448)
    assert torch.equal(Q.round_e4m3(v.double()), v.to(torch.float8_e4m3fn).double())
    x = torch.randn((130, 300), generator=g)
    for square in (False, True):
        q, s = Q.quantize(x, square)
        assert (q.abs().amax() == 448) and s.shape == ((2, 3) if square else (130, 3))
        assert ((Q.held(x, square) - x.double()).abs() <= 2.0**-4 * x.double().abs() + Q.spread(s, x.shape, square) * 2.0**-10).all()


def test_sizes():
    lib = _lib.load()
    assert [lib.ptx_fp8_pitch(n) for n in (1, 128, 129)] == [128, 128, 256]
    assert [lib.ptx_fp8_scale_pitch(n) for n in (1, 4, 5)] == [4, 4, 8]
    assert lib.ptx_fp8_scale_elems(5, 129, 0) == 16 and lib.ptx_fp8_scale_elems(129, 129, 1) == 4
    assert lib.ptx_fp8_matmul_workspace_elems(1, 4096, 4096, 1, 1) == 0
    assert lib.ptx_add_rms_norm_bwd_workspace_elems(0, 128) == 0 and lib.ptx_add_rms_norm_bwd_workspace_elems(10, 128) >= 128


def test_c_refusals():
    """Bad arguments come back as codes before anything is launched."""
    lib = _lib.load()

    def quantize(x=16, q=16, s=16, qt=None, st=None, sums=None, ws=None, rows=4, cols=8, dtype=0, sums_dtype=0):
        return lib.ptx_fp8_quantize(x, q, s, qt, st, sums, ws, rows, cols, 0, dtype, sums_dtype, None)

    assert quantize(dtype=2) == 1 and quantize(rows=-1) == 1 and quantize(cols=-1) == 1 and quantize(x=None) == 1
    assert quantize(s=None) == 1 and quantize(q=None) == 1 and quantize(qt=16) == 1 and quantize(st=16) == 1
    assert quantize(q=None, s=None) == 1 and quantize(q=24) == 1 and quantize(sums=16) == 1 and quantize(sums=16, ws=16, sums_dtype=9) == 1
    assert quantize(rows=1 << 28) == 2 and quantize(rows=1 << 40) == 2 and quantize(rows=1 << 20, cols=1 << 20) == 2
    assert quantize(rows=0) == 0 and quantize(cols=0) == 0

    def matmul(a=16, sa=16, b=16, sb=16, bias=None, out=16, ws=None, m=4, n=8, k=128, out_dtype=1, bias_dtype=0):
        return lib.ptx_fp8_matmul(a, sa, b, sb, 1, bias, out, ws, m, n, k, out_dtype, bias_dtype, None)

    assert matmul(out_dtype=2) == 1 and matmul(bias=16, bias_dtype=5) == 1 and matmul(m=-1) == 1 and matmul(n=-1) == 1 and matmul(k=0) == 1
    assert all(matmul(**{name: None}) == 1 for name in ("a", "sa", "b", "sb", "out"))
    assert all(matmul(**{name: 8}) == 1 for name in ("a", "sa", "b", "sb"))
    assert matmul(k=(1 << 24) + 1) == 2 and matmul(m=1 << 31) == 2 and matmul(m=1 << 20, n=1 << 20) == 2
    assert matmul(m=0) == 0 and matmul(n=0) == 0
    if lib.ptx_fp8_matmul_workspace_elems(70, 128, 8192, 1, 1):
        assert matmul(m=70, n=128, k=8192) == 1 and b"workspace" in lib.ptx_last_error_string()

    def norm(x=16, r=16, w=None, y=16, s=None, h=16, rows=4, cols=8, tx=1, ts=1, tw=0):
        return lib.ptx_add_rms_norm_fwd(x, r, w, y, s, h, None, rows, cols, 1e-6, tx, ts, tw, None)

    assert norm(tx=2) == 1 and norm(ts=4) == 1 and norm(tw=-1) == 1 and norm(rows=-1) == 1 and norm(cols=0) == 1
    assert norm(x=None) == 1 and norm(y=None) == 1 and norm(h=None) == 1 and norm(r=None, ts=0) == 1 and norm(y=24, s=16) == 1
    assert norm(tx=0, ts=1) == 2 and norm(tx=1, ts=3) == 2 and norm(cols=16385) == 2 and norm(rows=1 << 31) == 2 and norm(rows=0) == 0

    def back(dy=16, x=16, h=None, rstd=16, dw=None, ws=None, rows=4, cols=8, tx=1, ts=1):
        return lib.ptx_add_rms_norm_bwd(dy, None, x, None, h, rstd, None, 16, None, dw, ws, rows, cols, tx, ts, 0, None)

    assert back(x=None) == 1 and back(rstd=None) == 1 and back(ts=0) == 1 and back(dw=16) == 1 and back(cols=16385) == 2
    assert back(tx=3, ts=1) == 2 and back(rows=0) == 0


def test_python_refuses_cpu_tensors():
    x = torch.zeros((4, 128))
    for call in (lambda: P.quantize_fp8(x), lambda: P.linear_fp8(x, x), lambda: P.add_rms_norm(x), lambda: P.add_rms_norm(x, quantize=True),
                 lambda: P.Fp8Tensor(x.to(torch.float8_e4m3fn), torch.ones((4, 1)))):
        with pytest.raises(RuntimeError, match="GPU|on cpu"):
            call()
