"""The operators on packed blocks refuse bad arguments before they touch CUDA."""

import ctypes

import pytest
import torch

from kernels import _native, ops

E, OK = _native.QS_EINVAL, _native.QS_OK
A = 1 << 20  # an aligned address that is never read


def lib():
    return _native.lib()


def norm(x=A, xt=30, xs=64, r=None, rs=0, t=None, ts=0, w=A, eps=1e-6, n=2, k=64, d=A, db=68):
    return lib().qs_rms_norm_q8(x, xt, xs, r, rs, t, ts, w, eps, n, k, d, db, None)


@pytest.mark.parametrize("bad", [dict(xt=5), dict(k=0), dict(k=48), dict(k=-32), dict(n=-1), dict(n=1 << 31), dict(eps=0.0),
                                 dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(r=A, rs=64), dict(t=A, ts=64),
                                 dict(db=67), dict(xs=63), dict(x=None), dict(w=None), dict(d=None), dict(x=A + 2), dict(xs=68),
                                 dict(w=A + 4), dict(r=A + 8, rs=64, t=A, ts=64), dict(r=A, rs=64, t=A, ts=66), dict(r=A, rs=32, t=A, ts=64)])
def test_norm(bad):
    assert norm(**bad) == E


def test_nothing_to_do():
    assert norm(n=0, x=None, w=None, d=None) == OK
    assert route(n=0, z=None, ids=None, w=None) == OK
    assert matmul(rows=0, w=None, x=None, out=None) == OK
    assert experts(tokens=0, w=None) == OK


def route(z=A, zt=0, zs=8, n=2, e=8, k=2, score=0, bias=None, g=1, kept=1, gscore=0, ren=1, scale=1.0, ids=A, w=A):
    return lib().qs_route(z, zt, zs, n, e, k, score, bias, g, kept, gscore, ren, scale, ids, w, None)


@pytest.mark.parametrize("bad", [dict(zt=2), dict(e=0), dict(e=1025, zs=2000), dict(score=2), dict(score=-1), dict(gscore=2), dict(g=0),
                                 dict(g=3), dict(g=65, e=130, zs=130), dict(kept=0), dict(kept=2), dict(k=0), dict(k=9),
                                 dict(g=4, kept=1, k=3), dict(k=33, e=64, zs=64), dict(n=-1), dict(n=1 << 31), dict(zs=7), dict(z=None),
                                 dict(ids=None), dict(w=None), dict(z=A + 2), dict(ids=A + 1), dict(bias=A + 2)])
def test_route(bad):
    assert route(**bad) == E


def test_route_two_best_of_groups_of_one():
    """A group of one expert has no second best; a single group's score decides nothing."""
    assert route(g=8, kept=2, k=2, gscore=1) == E
    assert route(n=0, z=None, ids=None, w=None, g=8, kept=2, k=2, gscore=0) == OK
    assert route(n=0, z=None, ids=None, w=None, g=4, kept=2, k=2, gscore=1) == OK
    assert route(n=0, z=None, ids=None, w=None, g=1, kept=1, e=1, zs=1, k=1, gscore=1) == OK


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=(1 << 20) + 1), dict(e=0), dict(e=1025), dict(ids=None), dict(order=None), dict(off=None), dict(ids=A + 2)])
def test_plan(bad):
    a = dict(ids=A, n=4, e=8, order=A, off=A) | bad
    assert lib().qs_expert_plan(a["ids"], a["n"], a["e"], a["order"], a["off"], None) == E


def matmul(t=12, w=A, wr=144, n=8, k=256, x=A, xr=272, rows=2, out=A, ot=0, os=8, ws=None, wb=0):
    return lib().qs_matmul(t, w, wr, n, k, x, xr, rows, out, ot, os, ws, wb, None)


@pytest.mark.parametrize("bad", [dict(k=0), dict(k=128), dict(k=1 << 31), dict(n=0), dict(n=1 << 31), dict(rows=-1), dict(rows=(1 << 20) + 1),
                                 dict(rows=1 << 20, n=1 << 19, os=1 << 19), dict(w=None), dict(x=None), dict(out=None), dict(ot=2),
                                 dict(wr=128), dict(wr=152), dict(xr=271), dict(os=7), dict(w=A + 8), dict(out=A + 2)])
def test_matmul(bad):
    assert matmul(**bad) == E


def test_matmul_type():
    assert matmul(t=20) == _native.QS_ENOTSUP
    n = ctypes.c_int64()
    assert lib().qs_matmul_workspace(20, 8, 256, 1, 0, ctypes.byref(n)) == _native.QS_ENOTSUP
    assert lib().qs_matmul_workspace(12, 8, 100, 1, 0, ctypes.byref(n)) == E
    assert lib().qs_matmul_workspace(12, 8, 256, 1, 0, ctypes.byref(n)) == OK and n.value == 0
    assert lib().qs_matmul_workspace(12, 8, 256, 1, 2, ctypes.byref(n)) == E
    assert lib().qs_matmul_workspace(12, 8, 256, 0, 0, ctypes.byref(n)) == OK and n.value == 0
    assert lib().qs_matmul_experts_workspace(12, 4, 8, 256, 2, 2, 0, 0, 0, ctypes.byref(n)) == OK and n.value == 0
    assert lib().qs_matmul_experts_workspace(12, 4, 8, 256, 2, 2, 0, 1, 0, ctypes.byref(n)) == OK and n.value == 2 * 2 * 8 * 4


@pytest.mark.parametrize("t,al", [(12, 16), (13, 16), (7, 8), (23, 8), (3, 4), (10, 4), (2, 2), (14, 2), (18, 2)])
def test_matmul_alignment(t, al):
    qk, nb = _native.block_info(t)
    assert matmul(t=t, w=A + al // 2, wr=16 * nb, k=qk) == E
    assert matmul(t=t, wr=16 * nb + al // 2, k=qk) == E


def experts(t=12, w=A, wr=144, we=144 * 8, e=4, n=8, k=256, x=A, xr=272, per=0, ids=A, order=A, off=A, tokens=2, top=2, wt=None, out=A, ot=0,
            os=8, ws=None, wb=0):
    return lib().qs_matmul_experts(t, w, wr, we, e, n, k, x, xr, per, ids, order, off, tokens, top, wt, out, ot, os, ws, wb, None)


@pytest.mark.parametrize("bad", [dict(e=0), dict(e=1025), dict(top=0), dict(top=1025), dict(tokens=-1), dict(tokens=1 << 20), dict(we=144 * 7),
                                 dict(we=144 * 8 + 8), dict(ids=None), dict(order=None), dict(off=None), dict(ids=A + 2), dict(wt=A + 2),
                                 dict(wt=A), dict(wt=A, ws=A, wb=127), dict(wt=A, ws=A + 8, wb=128), dict(wt=A, wb=128), dict(wr=143), dict(xr=200), dict(os=4), dict(k=32), dict(ot=7)])
def test_experts(bad):
    assert experts(**bad) == E


def test_cpu_tensors_and_shapes():
    """No fallback on CPU tensors."""
    x = torch.zeros(2, 64)
    for call in (lambda: ops.rms_norm_q8(x, torch.ones(64)), lambda: ops.route(x, 2), lambda: ops.expert_plan(torch.zeros(2, 2, dtype=torch.int32), 4),
                 lambda: ops.matmul(torch.zeros(4, 144, dtype=torch.uint8), 12, torch.zeros(1, 272, dtype=torch.uint8))):
        with pytest.raises(_native.QsError) as e:
            call()
        assert e.value.code == E
