"""Residual dropout and the relative position bias on the CPU: the oracle's generator against published numbers, the
buckets, and what the entry points refuse before anything is launched."""
import copy
import ctypes
import math
import pickle

import numpy as np
import pytest
import torch

import protenix_amd as P
from protenix_amd import _lib
from tests import residual_oracle as R


@pytest.mark.parametrize("counter,key,want", [
    # the known answers published with the generator (philox4x32, 10 rounds)
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_oracle_generator_gives_the_published_numbers(counter, key, want):
    assert tuple(int(v) for v in R.philox(np.array(counter), key)) == want


def test_oracle_mask_keeps_the_share_it_should():
    n = 1 << 18
    for p in (0.1, 0.25, 0.9):
        kept = R.keep_mask((n // 64, 64), p, 1234).double().mean().item()
        # five standard deviations of a binomial share
        assert abs(kept - (1 - p)) < 5 * math.sqrt(p * (1 - p) / n)
    m = R.keep_mask((3, 5, 7, 9), 0.5, 7, shared_dim=-3)
    assert torch.equal(m, m[:, :1].expand_as(m)) and not torch.equal(m[:, :, :1].expand_as(m), m)


@pytest.mark.parametrize("distance,count,both", [(1, None, True), (32, None, True), (120, None, True), (254, None, False), (5, None, False),
                                                 (128, 32, True), (128, 32, False), (9, 32, True), (17, 32, False), (8192, 254, True),
                                                 (8192, 255, False), (2, 2, False), (2, 4, True), (3, 4, True), (1000, 3, False)])
def test_buckets_follow_their_formula(distance, count, both):
    b = P.RelativeBuckets(distance, count, bidirectional=both)
    assert b.num_buckets == (count or (2 * distance + 1 if both else distance + 1))
    near = range(-min(distance, 400) - 3, min(distance, 400) + 4)
    far = [s * (distance + o) for s in (-1, 1) for o in (-2, -1, 0, 1, 1000, 1 << 40)]
    edges = [s * (int(n) + o) for n in b._struct.starts[:b._struct.side] for s in (-1, 1) for o in (-1, 0, 1) if n + o >= 0]
    for d in [*near, *far, *edges]:
        got = b.bucket(d)
        assert got == R.bucket(max(-distance, min(distance, d)), distance, count, both), d
        assert 0 <= got < b.num_buckets


def test_common_buckets_by_value():
    # 32 buckets to 128, two sides: 8 single distances, then 8, 12, 16, 23, 32, 46, 64, 91 and on
    b = P.RelativeBuckets(128, 32)
    assert [min(n for n in range(200) if b.bucket(-n) == j) for j in range(16)] == [0, 1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91]
    assert b.bucket(1) == 17 and b.bucket(10**9) == 31 and b.bucket(-(10**9)) == 15


@pytest.mark.parametrize("args,kw", [((0,), {}), ((8193, 32), {}), ((128,), {}), ((255,), {"bidirectional": False}), ((128, 256), {}),
                                     ((128, 33), {}), ((128, 1), {"bidirectional": False}), ((128, 2), {}), ((8, 32), {}),
                                     ((16, 32), {"bidirectional": False})])
def test_buckets_that_no_kernel_takes_are_refused(args, kw):
    with pytest.raises(ValueError):
        P.RelativeBuckets(*args, **kw)


def test_buckets_and_module_are_copied_whole():
    m = P.RelativePositionBias(4, P.RelativeBuckets(128, 32), grouped=True)
    for c in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        assert c.buckets._struct is not m.buckets._struct and bytes(c.buckets._struct) == bytes(m.buckets._struct)
        assert c.buckets.bucket(50) == m.buckets.bucket(50) and c.weight.shape == (33, 4)
    assert list(m.state_dict()) == ["weight"]


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        P.dropout_add(x, x)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        P.dropout_add_layer_norm(x, x)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        P.relative_position_bias(torch.zeros(32, 4), P.RelativeBuckets(128, 32), range(3), range(3))


def _buckets(**changes):
    s = P.RelativeBuckets(128, 32)._struct
    c = _lib.RelativeBucketsStruct.from_buffer_copy(s)
    for n, v in changes.items():
        if n == "starts":
            for i, start in v.items():
                c.starts[i] = start
        else:
            setattr(c, n, v)
    return c


def test_c_entry_points_refuse_before_a_launch():
    lib = _lib.load()
    add = lambda rows=4, cols=8, shared=1, inner=1, p=0.5, xt=0, st=0, res=None: lib.ptx_dropout_add(
        None, res, None, rows, cols, shared, inner, p, 1, None, xt, st, None)
    assert add(rows=0) == 0                                     # nothing to do
    assert add() == 1 and b"null" in lib.ptx_last_error_string()
    assert add(xt=9) == 1 and add(xt=2) == 1 and add(st=2) == 1
    assert add(xt=1, st=3) == 2 and add(xt=0, st=1, res=8) == 2   # two 16-bit types; fp32 onto a 16-bit residual
    assert add(rows=-1) == 1 and add(cols=0) == 1 and add(rows=1 << 31) == 2
    assert add(p=-0.1) == 1 and add(p=1.1) == 1 and add(p=float("nan")) == 1
    assert add(rows=12, shared=5) == 1 and add(shared=0) == 1 and add(inner=0) == 1
    fwd = lambda rows=4, cols=8, p=0.0, xt=0, st=0, wt=0: lib.ptx_dropout_add_layernorm_fwd(
        *([None] * 8), rows, cols, 1, 1, p, 1e-5, 1, None, xt, st, wt, None)
    assert fwd(rows=0) == 0 and fwd() == 1
    assert fwd(cols=16385) == 2 and fwd(xt=0, st=1) == 2 and fwd(xt=1, st=3) == 2 and fwd(wt=2) == 1 and fwd(p=2.0) == 1
    bwd = lambda rows=4, cols=8, dw=None, xt=0, st=0: lib.ptx_dropout_add_layernorm_bwd(
        *([None] * 10), dw, None, None, rows, cols, 1, 1, 0.0, 1, None, xt, st, 0, None)
    assert bwd(rows=0) == 0 and bwd() == 1 and bwd(dw=8) == 1 and bwd(cols=20000) == 2 and bwd(xt=3, st=1) == 2
    assert lib.ptx_dropout_add_layernorm_bwd_workspace_elems(0, 8) == 0
    assert lib.ptx_dropout_add_layernorm_bwd_workspace_elems(5, 8) >= 2 * 8


def test_c_relative_bias_refuses_before_a_launch():
    lib = _lib.load()

    def fwd(buckets, batch=1, heads=4, q=3, k=3, gq=None, gk=None, tt=0, ot=0):
        p = None if buckets is None else ctypes.addressof(buckets)
        return lib.ptx_relative_bias_fwd(p, None, None, batch, heads, q, k, None, None, 0, 0, gq, gk, tt, ot, None)

    ok = _buckets()
    assert fwd(ok, q=0) == 0 and fwd(ok, k=0) == 0 and fwd(ok, batch=0) == 0
    assert fwd(ok) == 1 and b"null" in lib.ptx_last_error_string()
    assert fwd(None) == 1 and fwd(ok, heads=0) == 1 and fwd(ok, q=-1) == 1 and fwd(ok, tt=2) == 1 and fwd(ok, ot=7) == 1
    assert fwd(ok, gq=8) == 1 and fwd(ok, gk=8) == 1
    assert fwd(ok, batch=1 << 20, q=1 << 20, k=1 << 10) == 2
    # buckets that would be read from beyond the table, or distances from beyond the look-up
    for bad, rc in ((_buckets(count=0), 2), (_buckets(count=256), 2), (_buckets(count=31), 1), (_buckets(max_distance=8193), 2),
                    (_buckets(max_distance=-1), 2), (_buckets(side=0), 1), (_buckets(side=257), 1), (_buckets(neg_base=-1), 1),
                    (_buckets(pos_base=17), 1), (_buckets(pos_step=-2), 1), (_buckets(neg_step=1 << 30), 1),
                    (_buckets(starts={0: 1}), 1), (_buckets(starts={5: 3}), 1)):
        assert fwd(bad, q=0) == rc
        assert lib.ptx_relative_bias_bwd(ctypes.addressof(bad), None, None, None, 1, 4, 3, 3, None, None, 0, 0, None, None, 0, 0, None) == rc
    assert lib.ptx_relative_bias_bwd(ctypes.addressof(ok), None, None, None, 1, 4, 3, 3, None, None, 0, 0, None, None, 0, 0, None) == 1
    assert lib.ptx_relative_bias_bwd_workspace_elems(4, 32) >= 4 * 32


def test_c_relative_bias_refuses_batches_whose_units_it_cannot_number():
    lib = _lib.load()
    buckets = P.RelativeBuckets(32)._struct
    for batch in ((1 << 30) + 1, (1 << 31) - 1):
        args = (batch, 1, 1, 1, None, None, 0, 0, None, None, 0, 0, None)
        assert lib.ptx_relative_bias_fwd(ctypes.addressof(buckets), None, None, *args) == 2
        assert lib.ptx_relative_bias_bwd(ctypes.addressof(buckets), None, None, None, *args) == 2


def test_c_relative_bias_refuses_buckets_that_come_back():
    """The kernels take the differences of a bucket for an interval: |d| in buckets of its own has 2 1 0 1 2 around the query."""
    lib = _lib.load()

    def rc(buckets):
        args = (1, 4, 0, 3, None, None, 0, 0, None, None, 0, 0, None)      # (no query: nothing to launch)
        fwd = lib.ptx_relative_bias_fwd(ctypes.addressof(buckets), None, None, *args)
        text = lib.ptx_last_error_string()
        if fwd:
            assert lib.ptx_relative_bias_bwd(ctypes.addressof(buckets), None, None, None, *args) == fwd
        return fwd, text

    both = dict(neg_base=0, neg_step=1, pos_base=0, pos_step=1)
    singles = {i: i for i in range(16)}
    for bad in (_buckets(max_distance=2, side=3, starts=singles, **both), _buckets(**both), _buckets(neg_base=5, neg_step=0, pos_base=2),
                _buckets(max_distance=1, side=2, starts=singles, neg_base=0, neg_step=1, pos_base=1, pos_step=0, count=2),
                _buckets(max_distance=2, side=3, starts=singles, neg_base=2, neg_step=-1, pos_base=2, pos_step=-1)):
        got, text = rc(bad)
        assert got == 2 and b"interval" in text, (got, text)
    # the same numbers where each is met once: beyond max_distance, in empty buckets, in the query's own or on one side only
    for good in (_buckets(max_distance=2, side=16, starts={**singles, 1: 3, 2: 3}, **both),
                 _buckets(neg_base=3, neg_step=0, pos_base=3, pos_step=0), _buckets(neg_base=5, neg_step=0, pos_base=4),
                 _buckets(max_distance=4, side=5, starts=singles, neg_base=4, neg_step=-1, pos_base=4, pos_step=1),
                 _buckets(max_distance=1, side=2, starts=singles, neg_base=0, neg_step=1, pos_base=0, pos_step=0),
                 _buckets(max_distance=8, side=2, starts={1: 0}, **both)):
        assert rc(good)[0] == 0, rc(good)
    for scheme in ((1, None, True), (120, None, True), (254, None, False), (128, 32, True), (128, 32, False), (8192, 254, True), (8192, 255, False),
                   (2, 2, False), (2, 4, True), (3, 4, True)):
        assert rc(P.RelativeBuckets(scheme[0], scheme[1], bidirectional=scheme[2])._struct)[0] == 0, scheme


def test_c_relative_bias_refuses_a_distance_of_zero():
    """Every d > 0 would have n = 0 and the first bucket of its side, which a look-up by min(|d|, max_distance) cannot tell from d = 0's."""
    lib = _lib.load()
    args = (1, 4, 0, 3, None, None, 0, 0, None, None, 0, 0, None)
    for most, rc in ((0, 2), (1, 0)):
        s = _buckets(max_distance=most, count=2, side=1, neg_base=0, neg_step=0, pos_base=1, pos_step=0)
        assert lib.ptx_relative_bias_fwd(ctypes.addressof(s), None, None, *args) == rc
        assert lib.ptx_relative_bias_bwd(ctypes.addressof(s), None, None, None, *args) == (rc or 1)      # (1: null pointers, refused later)


def test_a_drawn_seed_asks_the_updates_device_whether_it_records(monkeypatch):
    """The recording may be on the stream of another device than the current one."""
    current = [0]

    class Device:
        def __init__(self, d):
            self.index = d.index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *_):
            current.pop()

    class Update:      # (what a tensor on the second GPU says of itself)
        is_cuda, device = True, torch.device("cuda", 1)

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[-1] == 1)
    for call in (P.dropout_add, P.dropout_add_layer_norm):
        with pytest.raises(RuntimeError, match="needs its seed"):
            call(Update(), p=0.5)
