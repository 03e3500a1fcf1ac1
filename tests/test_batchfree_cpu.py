"""Group norm, linear layer and dropout without a GPU: the generator against known answers, workspaces, and every refused call (nothing
may be launched: the operand addresses are not memory)."""
import ctypes as C

import pytest

from pl_yolo_amd import _lib
from pl_yolo_amd._lib import GnDesc, LinearDesc, PlyoloError, call
import batchfree as bf

P = 0x10000      # a 16-byte aligned address that nobody may touch


def gn_desc(**k):
    d = GnDesc()
    v = dict(dtype=0, N=2, HW=16, C=32, groups=4, act=1, eps=1e-5, x_ld=32, o_ld=32, r_ld=32)
    v.update(k)
    for n, x in v.items():
        setattr(d, n, x)
    return d


def lin_desc(**k):
    d = LinearDesc()
    v = dict(dtype=0, M=10, N=16, K=24, act=1, x_ld=24, w_ld=24, y_ld=16, z_ld=16, r_ld=16)
    v.update(k)
    for n, x in v.items():
        setattr(d, n, x)
    return d


def test_philox_known_answers():
    # the known-answer vectors that the generator's authors publish with it (philox4x32, 7 rounds)
    assert bf.philox7((0, 0, 0, 0), (0, 0)) == [0x5f6fb709, 0x0d893f64, 0x4f121f81, 0x4f730a48]
    f = bf.M32
    assert bf.philox7((f, f, f, f), (f, f)) == [0x5207ddc2, 0x45165e59, 0x4d8ee751, 0x8c52f662]


def test_keep_mask_follows_the_integer_form():
    seed, step, site, p = 0x123456789abcdef0, 7, 3, 0.25
    m = bf.keep_mask(seed, step, site, 5, 7, p)
    for i in range(35):
        w = bf.philox7((i // 4, 0, step, site), (seed & bf.M32, seed >> 32))[i % 4]
        assert bool(m.flat[i]) == ((w >> 8) >= 0.25 * (1 << 24))
    far = bf.keep_mask(seed, step, site, 1, 9, p, first=(1 << 34) + 1)      # counters beyond 32 bits
    for j in range(9):
        i = (1 << 34) + 1 + j
        w = bf.philox7(((i // 4) & bf.M32, (i // 4) >> 32, step, site), (seed & bf.M32, seed >> 32))[i % 4]
        assert bool(far.flat[j]) == ((w >> 8) >= 0.25 * (1 << 24))


def gn_fwd(d, x=P, ga=P, be=P, res=None, out=P, stats=P, ws=P, n=1 << 30):
    call("plyolo_gn_act_fwd", C.byref(d) if d is not None else None, x, ga, be, res, out, stats, ws, n, None)


def gn_bwd(d, dout=P, d_ld=32, x=P, stats=P, dx=P, dx_ld=32, ws=P, n=1 << 30):
    call("plyolo_gn_act_bwd", C.byref(d) if d is not None else None, dout, d_ld, x, stats, P, P, dx, dx_ld, 0, P, P, 0, ws, n, None)


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(N=0), dict(HW=0), dict(HW=-4), dict(C=0), dict(groups=0), dict(groups=5), dict(C=8192, x_ld=8192, o_ld=8192),
                                 dict(act=6), dict(act=-1), dict(eps=-1.0), dict(eps=float("nan")), dict(x_ld=31), dict(N=65536, HW=65536),
                                 dict(N=1 << 22, HW=1)])
def test_gn_refuses_descriptors(bad):
    d = gn_desc(**bad)
    assert _lib.lib().plyolo_gn_workspace(C.byref(d)) == 0
    with pytest.raises(PlyoloError, match="gn_act_fwd"):
        gn_fwd(d)
    with pytest.raises(PlyoloError, match="gn_act_bwd"):
        gn_bwd(d)


def test_gn_refuses_operands():
    need = _lib.lib().plyolo_gn_workspace(C.byref(gn_desc()))
    assert need > 0
    for kw in (dict(x=None), dict(out=None), dict(stats=None), dict(ws=None), dict(ws=P + 4), dict(n=need - 1), dict(x=P + 1), dict(ga=P + 2)):
        with pytest.raises(PlyoloError, match="gn_act_fwd"):
            gn_fwd(gn_desc(), **kw)
    for kw in (dict(o_ld=31),):
        with pytest.raises(PlyoloError, match="o_ld"):
            gn_fwd(gn_desc(**kw))
    with pytest.raises(PlyoloError, match="r_ld"):
        gn_fwd(gn_desc(r_ld=8), res=P)
    for kw in (dict(dout=None), dict(x=None), dict(stats=None), dict(dx=None), dict(d_ld=31), dict(dx_ld=31), dict(ws=None), dict(n=need - 1), dict(dx=P + 1)):
        with pytest.raises(PlyoloError, match="gn_act_bwd"):
            gn_bwd(gn_desc(), **kw)
    with pytest.raises(PlyoloError, match="null descriptor"):
        gn_fwd(None)


def lin_fwd(d, x=P, w=P, b=P, res=None, z=None, y=P):
    call("plyolo_linear_fwd", C.byref(d) if d is not None else None, x, w, b, res, z, y, P, 1 << 40, None)


def lin_bwd(d, dy=P, z=P, x=P, w=P, dx=P, dx_ld=24, dw=P, dwt=0, db=P, ws=P, n=1 << 40):
    call("plyolo_linear_bwd", C.byref(d) if d is not None else None, dy, z, x, w, dx, dx_ld, 0, dw, dwt, db, 0, ws, n, None)


@pytest.mark.parametrize("bad", [dict(dtype=7), dict(M=0), dict(N=0), dict(K=-1), dict(act=9), dict(x_ld=23), dict(w_ld=23), dict(N=1 << 21, y_ld=1 << 21),
                                 dict(N=1 << 15, K=1 << 15, x_ld=1 << 15, w_ld=1 << 15, y_ld=1 << 15)])
def test_linear_refuses_descriptors(bad):
    d = lin_desc(**bad)
    with pytest.raises(PlyoloError, match="linear_fwd"):
        lin_fwd(d)
    with pytest.raises(PlyoloError, match="linear_bwd"):
        lin_bwd(d)
    assert _lib.lib().plyolo_linear_workspace(C.byref(d), 1) == 0


def test_linear_refuses_operands():
    for kw in (dict(x=None), dict(w=None), dict(y=None), dict(y=P + 1), dict(b=P + 2)):
        with pytest.raises(PlyoloError, match="linear_fwd"):
            lin_fwd(lin_desc(), **kw)
    for dk, kw in ((dict(y_ld=15), {}), (dict(z_ld=15), dict(z=P)), (dict(r_ld=15), dict(res=P))):
        with pytest.raises(PlyoloError, match="pitch"):
            lin_fwd(lin_desc(**dk), **kw)
    need = _lib.lib().plyolo_linear_workspace(C.byref(lin_desc()), 1)
    assert need > 0
    for kw in (dict(dy=None), dict(z=None), dict(w=None), dict(x=None), dict(dx=None, dw=None, db=None), dict(dx_ld=23), dict(dwt=3), dict(dwt=-1), dict(ws=None),
               dict(ws=P + 8), dict(n=need - 1), dict(dy=P + 1), dict(dw=P + 2, dwt=1)):
        with pytest.raises(PlyoloError, match="linear_bwd"):
            lin_bwd(lin_desc(), **kw)
    for f in (lin_fwd, lin_bwd):            # more tiles than one launch has room for
        with pytest.raises(PlyoloError, match="workgroups"):
            f(lin_desc(M=2147480000, N=64, K=1, y_ld=64, z_ld=64), z=P)
    with pytest.raises(PlyoloError, match="dw_dtype"):
        lin_bwd(lin_desc(dtype=1), dwt=0)      # bf16 weight gradients of an fp32 layer


def drop(M=4, Cc=8, x=P, x_ld=8, p=0.5, rng=P, res=None, r_ld=0, out=P, o_ld=8, dt=0):
    call("plyolo_dropout_fwd", dt, M, Cc, x, x_ld, p, rng, 1, res, r_ld, out, o_ld, None)


@pytest.mark.parametrize("kw", [dict(M=0), dict(Cc=0), dict(x=None), dict(rng=None), dict(out=None), dict(x_ld=7), dict(o_ld=7), dict(res=P, r_ld=7), dict(p=-0.1),
                                dict(p=1.5), dict(p=float("nan")), dict(dt=4), dict(x=P + 1), dict(rng=P + 4),
                                dict(M=2147483647, Cc=1024, x_ld=1024, o_ld=1024)])
def test_dropout_refuses(kw):
    with pytest.raises(PlyoloError, match="dropout_fwd"):
        drop(**kw)
    if "res" in kw:
        return
    a = dict(M=4, Cc=8, x=P, x_ld=8, p=0.5, rng=P, out=P, o_ld=8, dt=0)
    a.update(kw)
    with pytest.raises(PlyoloError, match="dropout_bwd"):
        call("plyolo_dropout_bwd", a["dt"], a["M"], a["Cc"], a["x"], a["x_ld"], a["p"], a["rng"], 1, a["out"], a["o_ld"], 0, None)


def test_rng_next_refuses():
    for a, b in ((None, P), (P, None), (P + 4, P)):
        with pytest.raises(PlyoloError, match="rng_next"):
            call("plyolo_rng_next", a, b, None)
