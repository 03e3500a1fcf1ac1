"""-m gpu: group norm + activation, linear layer and counter-based dropout through the C ABI against their definitions in 64 bits.

Tolerances, fixed before the first run.  Stored values: UNIT[dtype] relative (half a step).  fp32 arithmetic: a sum of n terms t_i is off by
at most n * E32 * sum |t_i| in any order; elementwise chains (normalise, activation with the hardware exponential, whose relative error grows
with its argument) by CH = 64 half steps of fp32 relative to the magnitudes that enter them."""
import ctypes as C

import pytest
import torch

import hiputil as hu
from batchfree import ACTS, E32, GUARD, TD, UNIT, Mat, act64, act_grad64, assert_close, gn64, gn_bwd64, keep_mask
from pl_yolo_amd import _lib
from pl_yolo_amd._lib import BF16, F32, GnDesc, LinearDesc, call, ptr

pytestmark = pytest.mark.gpu
DEV = hu.DEV
CH = 64 * E32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rnd(m, c, seed, scale=1.0):
    return torch.randn(m, c, generator=gen(seed), device=DEV) * scale


# ------------------------------------------------------------------------------------------------ group norm
class Gn:
    def __init__(self, dt, n, hw, c, groups, act="silu", pad=0, off=0, eps=1e-5, affine=True, data=None, seed=1):
        self.dt, self.n, self.hw, self.c, self.groups, self.act, self.eps = dt, n, hw, c, groups, act, eps
        x = data if data is not None else rnd(n * hw, c, seed, 1.3) + rnd(1, c, seed + 1, 0.7)
        self.x = Mat(n * hw, c, dt, pad, off, x)
        self.gamma = 1.0 + rnd(1, c, seed + 2, 0.2).flatten() if affine else None
        self.beta = rnd(1, c, seed + 3, 0.3).flatten() if affine else None
        d = GnDesc()
        d.dtype, d.N, d.HW, d.C, d.groups, d.act, d.eps, d.x_ld, d.o_ld, d.r_ld = dt, n, hw, c, groups, ACTS[act], eps, self.x.ld, self.x.ld, self.x.ld
        self.d, self.pad, self.off = d, pad, off
        self.nws = _lib.lib().plyolo_gn_workspace(C.byref(d))
        assert self.nws > 0
        self.ws = torch.full((self.nws + 256,), 171, dtype=torch.uint8, device=DEV)

    def mat(self, data=None):
        return Mat(self.n * self.hw, self.c, self.dt, self.pad, self.off, data)

    def fwd(self, res=None, out=None, stats=None, stream=None):
        out = out or self.mat()
        st = stats if stats is not None else torch.full((self.n, self.groups, 2), GUARD, device=DEV)
        call("plyolo_gn_act_fwd", C.byref(self.d), self.x.ptr, ptr(self.gamma), ptr(self.beta), res.ptr if res else None, out.ptr, st.data_ptr(),
             self.ws.data_ptr(), self.nws, stream if stream is not None else hu.stream())
        return out, st

    def bwd(self, dout, st, dx=None, acc=0, dga=None, dbe=None, acc_par=0):
        dx = dx or self.mat()
        call("plyolo_gn_act_bwd", C.byref(self.d), dout.ptr, dout.ld, self.x.ptr, st.data_ptr(), ptr(self.gamma), ptr(self.beta), dx.ptr, dx.ld, acc,
             ptr(dga), ptr(dbe), acc_par, self.ws.data_ptr(), self.nws, hu.stream())
        return dx

    def ws_kept(self):
        return bool((self.ws[self.nws:] == 171).all())

    def check_fwd(self, out, st, res=None, what="gn_fwd"):
        xh, u, mu, rs = gn64(self.x.v, self.n, self.hw, self.groups, self.gamma, self.beta, self.eps)
        want = act64(u, self.act)
        # the mean is stored in fp32: u moves by rstd |mean| half steps, the chain by CH of what enters it
        mag = self.chain(xh, mu, rs)
        tol = mag * CH
        if res is not None:
            want = want + res.v.double()
        tol = tol + UNIT[self.dt] * (want.abs() + tol) + E32 * want.abs()
        assert_close(out.v, want, tol, what)
        n = self.hw * (self.c // self.groups)
        spread = 1.0 / rs
        assert_close(st[:, :, 0], mu, 8 * E32 * (mu.abs() + spread), what + " mean")
        assert_close(st[:, :, 1], rs, 64 * E32 * rs * (1.0 + 0 * n), what + " rstd")
        assert out.untouched() and self.ws_kept()

    def chain(self, xh, mu, rs):
        ga = self.gamma.double().abs() if self.gamma is not None else 1.0
        be = self.beta.double().abs() if self.beta is not None else 0.0
        m = (mu.abs() * rs).view(self.n, 1, self.groups, 1).expand(self.n, self.hw, self.groups, self.c // self.groups).reshape(self.n * self.hw, self.c)
        return ga * (xh.abs() + m + 1.0) + be

    def check_bwd(self, dx, dout, dga=None, dbe=None, base=None, what="gn_bwd"):
        wdx, wga, wbe, size = gn_bwd64(self.x.v, dout.v, self.n, self.hw, self.groups, self.gamma, self.beta, self.eps, self.act)
        xh, u, mu, rs = gn64(self.x.v, self.n, self.hw, self.groups, self.gamma, self.beta, self.eps)
        ga = self.gamma.double().abs() if self.gamma is not None else torch.ones(self.c, dtype=torch.float64, device=DEV)
        mag = self.chain(xh, mu, rs)
        # dx = rstd (v - m1 - xh m2): each term with the chain's error; the means are averages of |v| (1 + |xh|) with 64 half steps each
        v = (dout.v.double().abs() * ga * 1.2).view(self.n, self.hw, self.groups, -1)
        xg = xh.abs().view(self.n, self.hw, self.groups, -1)
        m1, m2 = v.mean(dim=(1, 3), keepdim=True), (v * (xg + mag.view_as(xg) * 0)).mean(dim=(1, 3), keepdim=True)
        t = (v * (1.0 + mag.view_as(v)) + m1 * 4 + (xg + mag.view_as(xg)) * m2 * 4) * rs.view(self.n, 1, self.groups, 1)
        want = wdx if base is None else wdx + base
        tol = t.reshape(self.n * self.hw, self.c) * CH
        tol = tol + UNIT[self.dt] * (want.abs() + tol) + E32 * want.abs()
        assert_close(dx.v, want, tol, what + " dx")
        # parameter gradients: no partial sum is longer than rows-per-thread + joins; 512 covers both at the tested sizes
        x1 = dout.v.double().abs() * 1.2 * (1.0 + mag)
        if dga is not None:
            assert_close(dga, wga, 512 * E32 * size[0] + CH * (x1 * (1.0 + xh.abs())).sum(0) + 1e-30, what + " dgamma")
        if dbe is not None:
            assert_close(dbe, wbe, 512 * E32 * size[1] + CH * x1.sum(0) + 1e-30, what + " dbeta")
        assert dx.untouched() and self.ws_kept()


GN_SHAPES = [  # n, hw, c, groups, pad, off
    (2, 400, 64, 32, 0, 0),         # two channels a group: a vector spans four groups
    (1, 1, 8, 1, 0, 0),             # one pixel
    (3, 945, 60, 12, 7, 0),         # five channels a group, odd pitch
    (2, 77, 40, 5, 8, 0),           # wide rows with a pitch
    (1, 333, 7, 7, 0, 1),           # instance norm, rows at odd addresses
    (2, 50, 1, 1, 2, 0),            # one channel
    (1, 9, 2064, 3, 0, 0),          # more vectors than threads in a row, 688 channels a group
    (5, 6400, 128, 32, 0, 0),       # many chunks
    (1, 20011, 24, 8, 0, 0),        # one long image, ragged last chunk
    (33, 3, 16, 4, 0, 0),           # many short images
    (1, 130, 4096, 4096, 0, 0),     # as many groups as the largest channel count
    (8, 9000, 64, 32, 0, 0),        # held in registers by 1024 threads
    (13, 1500, 200, 5, 0, 0),       # ... by a slice of five vectors
    (6, 6400, 132, 12, 0, 0),       # streamed, four channels behind the last bf16 vector
    (2, 20000, 13, 13, 0, 0),       # ... five (one fp32)
    (1, 30000, 9, 3, 3, 1),         # ... one, rows at odd addresses
    (2, 9000, 15, 1, 0, 0),         # ... seven (three fp32)
]


@pytest.mark.parametrize("dt", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", GN_SHAPES, ids=lambda s: "n%d_hw%d_c%d_g%d_p%d_o%d" % s)
def test_gn_forward_backward(shape, dt):
    n, hw, c, groups, pad, off = shape
    t = Gn(dt, n, hw, c, groups, "silu", pad, off, eps=1e-3 if hw * (c // groups) < 8 else 1e-5)
    res = t.mat(rnd(n * hw, c, 9))
    out, st = t.fwd()
    t.check_fwd(out, st)
    out2, st2 = t.fwd(res)
    t.check_fwd(out2, st2, res, "gn_fwd + res")
    assert torch.equal(st, st2)
    dout = t.mat(rnd(n * hw, c, 11, 0.1))
    dga, dbe = torch.full((c,), GUARD, device=DEV), torch.full((c,), GUARD, device=DEV)
    dx = t.bwd(dout, st, dga=dga, dbe=dbe)
    t.check_bwd(dx, dout, dga, dbe)
    # again: bit for bit
    out3, st3 = t.fwd()
    dga2, dbe2 = torch.empty_like(dga), torch.empty_like(dbe)
    dx2 = t.bwd(dout, st, dga=dga2, dbe=dbe2)
    assert torch.equal(out.v, out3.v) and torch.equal(st, st3) and torch.equal(dx.v, dx2.v) and torch.equal(dga, dga2) and torch.equal(dbe, dbe2)


@pytest.mark.parametrize("dt", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("act", sorted(ACTS))
def test_gn_activations_accumulation_and_in_place(act, dt):
    t = Gn(dt, 2, 130, 48, 6, act)
    out, st = t.fwd()
    t.check_fwd(out, st)
    dout, base = t.mat(rnd(260, 48, 12, 0.1)), rnd(260, 48, 13, 0.1)
    dx = t.mat(base)
    b64 = dx.v.double().clone()
    dga, dbe = torch.full((48,), 2.0, device=DEV), torch.full((48,), -3.0, device=DEV)
    t.bwd(dout, st, dx=dx, acc=1, dga=dga, dbe=dbe, acc_par=1)
    t.check_bwd(dx, dout, base=b64, what="accumulated")
    d1, e1 = torch.zeros(48, device=DEV), torch.zeros(48, device=DEV)
    plain = t.bwd(dout, st, dga=d1, dbe=e1)
    assert_close(dga, d1.double() + 2.0, 2 * E32 * (d1.double().abs() + 2.0), "dgamma +=")
    assert_close(dbe, e1.double() - 3.0, 2 * E32 * (e1.double().abs() + 3.0), "dbeta +=")
    # without parameter gradients the same dx
    assert torch.equal(t.bwd(dout, st).v, plain.v)
    # dx over dout, out over x
    d2 = t.mat(dout.v)
    t.bwd(d2, st, dx=d2)
    assert torch.equal(d2.v, plain.v)
    keep = out.v.clone()
    t.fwd(out=t.x)
    assert torch.equal(t.x.v, keep)


@pytest.mark.parametrize("dt", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("c,groups", [(13, 13), (132, 12), (10, 1)])
def test_gn_streamed_in_place_with_a_ragged_last_vector(c, groups, dt):
    """The last vector of a row overlaps its neighbour: in place, what is read there may be new already and must not count."""
    n, hw = 2, 12000
    t = Gn(dt, n, hw, c, groups, "gelu")
    want, st = t.fwd()
    t.check_fwd(want, st)
    dout = t.mat(rnd(n * hw, c, 11, 0.1))
    wdx = t.bwd(dout, st)
    t.check_bwd(wdx, dout)
    base = t.mat(rnd(n * hw, c, 12, 0.1))
    b64 = base.v.double().clone()
    t.bwd(dout, st, dx=base, acc=1)
    t.check_bwd(base, dout, base=b64)
    t.bwd(dout, st, dx=dout)
    assert torch.equal(dout.v, wdx.v) and dout.untouched()
    _, st2 = t.fwd(out=t.x)
    assert torch.equal(t.x.v, want.v) and torch.equal(st, st2) and t.x.untouched()


def test_gn_without_affine():
    for dt in (BF16, F32):
        t = Gn(dt, 2, 64, 24, 4, "relu", affine=False)
        out, st = t.fwd()
        t.check_fwd(out, st)
        dout = t.mat(rnd(128, 24, 5))
        t.check_bwd(t.bwd(dout, st), dout)


def test_gn_large_mean_and_one_huge_value():
    """A mean 4000 times the spread, and one value 1e5 times the rest: no digits may be lost to E[x^2] - E[x]^2 (fp32)."""
    x = rnd(2 * 3000, 16, 3) + 4096.0
    t = Gn(F32, 2, 3000, 16, 2, "none", data=x)
    out, st = t.fwd()
    t.check_fwd(out, st)
    for row in (0, 1234, 5999):
        x = rnd(2 * 3000, 16, 4)
        x[row, 3] = 1e5
        t = Gn(F32, 2, 3000, 16, 2, "none", data=x)
        out, st = t.fwd()
        t.check_fwd(out, st, what="huge value in row %d" % row)


def test_gn_constant_group():
    x = torch.full((2 * 100, 8), 3.0, device=DEV)
    t = Gn(F32, 2, 100, 8, 2, "none", data=x)
    out, st = t.fwd()
    assert torch.equal(out.v, t.beta.expand(200, 8)) and bool(((st[:, :, 1] - 1e5 ** 0.5).abs() < 1e-3).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dt", [BF16, F32], ids=["bf16", "fp32"])
def test_gn_keeps_nan_and_infinity_in_their_group(dt, bad):
    x = rnd(3 * 200, 32, 6)
    ok = Gn(dt, 3, 200, 32, 4, data=x)
    o0, s0 = ok.fwd()
    x2 = x.clone()
    x2[200 + 57, 9] = bad          # image 1, group 1
    t = Gn(dt, 3, 200, 32, 4, data=x2)
    o1, s1 = t.fwd()
    hit = torch.zeros(600, 32, dtype=torch.bool, device=DEV)
    hit[200:400, 8:16] = True
    assert bool(torch.isnan(o1.v[hit]).all()) and torch.equal(o1.v[~hit], o0.v[~hit])
    assert bool(torch.isnan(s1[1, 1, 1]))
    dout = t.mat(rnd(600, 32, 7))
    a, b = ok.bwd(dout, s0), t.bwd(dout, s1)
    assert bool(torch.isnan(b.v[hit]).all()) and torch.equal(a.v[~hit], b.v[~hit])


def test_gn_gradient_against_differences():
    """d(sum out * r) along random directions by central differences of the fp32 forward."""
    t = Gn(F32, 2, 60, 12, 3, "gelu")
    r = rnd(120, 12, 21)
    x0 = t.x.v.clone()
    out, st = t.fwd()
    dga, dbe = torch.zeros(12, device=DEV), torch.zeros(12, device=DEV)
    dx = t.bwd(t.mat(r), st, dga=dga, dbe=dbe)
    h = 2.0 ** -7

    def f():
        return float((t.fwd()[0].v.double() * r.double()).sum())
    for seed in (31, 32, 33):
        v = rnd(120, 12, seed)
        t.x.v.copy_(x0 + h * v)
        up = f()
        t.x.v.copy_(x0 - h * v)
        dn = f()
        t.x.v.copy_(x0)
        want = float((dx.v.double() * v.double()).sum())
        # third derivatives of order 1 over 1440 values with |v|^3 ~ 1.6: h^2 / 6 * their root sum; rounding 1e-6 / h
        assert abs((up - dn) / (2 * h) - want) < 2e-2 + 1e-3 * abs(want), ((up - dn) / (2 * h), want)
    g0 = t.gamma.clone()
    v = rnd(1, 12, 34).flatten()
    t.gamma.copy_(g0 + h * v)
    up = f()
    t.gamma.copy_(g0 - h * v)
    dn = f()
    t.gamma.copy_(g0)
    want = float((dga.double() * v.double()).sum())
    assert abs((up - dn) / (2 * h) - want) < 2e-2 + 1e-3 * abs(want)


# ------------------------------------------------------------------------------------------------ linear
class Lin:
    def __init__(self, dt, m, n, k, act="silu", bias=True, pad=0, off=0, wpad=0, seed=1):
        self.dt, self.m, self.n, self.k, self.act, self.pad, self.off = dt, m, n, k, act, pad, off
        self.x = Mat(m, k, dt, pad, off, rnd(m, k, seed))
        self.w = Mat(n, k, dt, wpad, off, rnd(n, k, seed + 1, k ** -0.5))
        self.b = rnd(1, n, seed + 2, 0.2).flatten() if bias else None
        d = LinearDesc()
        d.dtype, d.M, d.N, d.K, d.act = dt, m, n, k, ACTS[act]
        d.x_ld, d.w_ld, d.y_ld, d.z_ld, d.r_ld = self.x.ld, self.w.ld, n + pad, n + pad, n + pad
        self.d = d
        lib = _lib.lib()
        self.nf, self.nb = lib.plyolo_linear_workspace(C.byref(d), 0), lib.plyolo_linear_workspace(C.byref(d), 1)
        self.ws = torch.full((max(self.nf, self.nb) + 256,), 171, dtype=torch.uint8, device=DEV)

    def rows(self, data=None):
        return Mat(self.m, self.n, self.dt, self.pad, self.off, data)

    def fwd(self, res=None, z=True, y=None):
        y = y or self.rows()
        zm = self.rows() if z else None
        call("plyolo_linear_fwd", C.byref(self.d), self.x.ptr, self.w.ptr, ptr(self.b), res.ptr if res else None, zm.ptr if z else None, y.ptr,
             self.ws.data_ptr(), self.nf, hu.stream())
        return y, zm

    def check_fwd(self, y, zm, res=None):
        x, w = self.x.v.double(), self.w.v.double()
        z = x @ w.t()
        size = x.abs() @ w.abs().t()
        if self.b is not None:
            z, size = z + self.b.double(), size + self.b.double().abs()
        tz = (self.k + 4) * E32 * size
        if zm is not None:
            assert_close(zm.v, z, tz + UNIT[self.dt] * (z.abs() + tz), "z")
            assert zm.untouched()
        want = act64(z, self.act)
        ty = 1.2 * tz + CH * (want.abs() + E32)          # |act'| <= 1.13; the activation's own error
        if res is not None:
            want = want + res.v.double()
        assert_close(y.v, want, ty + E32 * want.abs() + UNIT[self.dt] * (want.abs() + ty), "y")
        assert y.untouched() and bool((self.ws[self.nf:] == 171).all() if self.nf == 0 else True)

    def bwd(self, dy, z, dx=True, dw=None, dwt=None, db=True, acc_dx=0, acc_par=0, dxm=None, dbt=None):
        dxm = dxm or (Mat(self.m, self.k, self.dt, self.pad, self.off) if dx else None)
        dwt = self.dt if dwt is None else dwt
        dwm = dw if dw is not None else torch.full((self.n, self.k), GUARD, dtype=TD[dwt], device=DEV)
        dbt = dbt if dbt is not None else (torch.full((self.n,), GUARD, device=DEV) if db else None)
        call("plyolo_linear_bwd", C.byref(self.d), dy.ptr, z.ptr if z is not None else None, self.x.ptr, self.w.ptr, dxm.ptr if dxm else None,
             dxm.ld if dxm else 0, acc_dx, dwm.data_ptr() if dw is not False else None, dwt, ptr(dbt), acc_par, self.ws.data_ptr(), self.nb, hu.stream())
        return dxm, dwm, dbt

    def check_bwd(self, dy, z, dxm, dwm, db, base=None, dwt=None):
        dwt = self.dt if dwt is None else dwt
        x, w = self.x.v.double(), self.w.v.double()
        g = act_grad64(z.v.double(), self.act) if z is not None else 1.0
        dz = dy.v.double() * g
        # dz is rounded to the operand type once for the products; its own chain: CH relative to |dy| (1 + |z|)
        edz = (UNIT[self.dt] if self.act != "none" else 0.0) * dz.abs() + (CH * dy.v.double().abs() * (1.0 + z.v.double().abs()) if z is not None else 0.0 * dz)
        if dxm is not None:
            want = dz @ w
            tol = edz @ w.abs() + (self.n + 4) * E32 * (dz.abs() @ w.abs())
            if base is not None:
                want = want + base
            assert_close(dxm.v, want, tol + E32 * want.abs() + UNIT[self.dt] * (want.abs() + tol), "dx")
            assert dxm.untouched()
        if dwm is not None:
            want = dz.t() @ x
            tol = edz.t() @ x.abs() + (min(self.m, 4096) + 64) * E32 * (dz.abs().t() @ x.abs())
            assert_close(dwm, want, tol + UNIT[dwt] * (want.abs() + tol), "dw")
        if db is not None:
            echain = (CH * dy.v.double().abs() * (1.0 + (z.v.double().abs() if z is not None else 0.0))).sum(0)
            assert_close(db, dz.sum(0), echain + 1100 * E32 * dz.abs().sum(0) + 1e-30, "db")
        assert bool((self.ws[self.nb:] == 171).all())


LIN_SHAPES = [  # m, n, k, pad, off, wpad
    (1, 1, 1, 0, 0, 0),
    (1, 64, 128, 0, 0, 0),          # a single row
    (3, 85, 179, 5, 0, 0),          # nothing divides anything
    (4, 1024, 1024, 0, 0, 0),
    (16, 40, 72, 8, 0, 8),
    (17, 130, 257, 0, 1, 0),        # odd addresses
    (64, 256, 512, 0, 0, 0),
    (65, 8, 2048, 0, 0, 0),         # one vector of columns
    (129, 127, 65, 0, 0, 3),        # one beyond and one short of a tile
    (400, 255, 320, 0, 0, 0),
    (1000, 1, 33, 1, 0, 0),         # one output column
    (2037, 85, 200, 3, 0, 0),
    (5000, 192, 96, 0, 0, 0),
    (20000, 16, 8, 0, 0, 0),        # tall and narrow
    (4099, 264, 136, 24, 0, 0),     # wide path with a pitch, ragged tiles
    (3000, 640, 1, 0, 0, 0),        # one input channel
]


@pytest.mark.parametrize("dt", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", LIN_SHAPES, ids=lambda s: "m%d_n%d_k%d_p%d_o%d_w%d" % s)
def test_linear_forward_backward(shape, dt):
    m, n, k, pad, off, wpad = shape
    t = Lin(dt, m, n, k, "silu", True, pad, off, wpad)
    y, z = t.fwd()
    t.check_fwd(y, z)
    res = t.rows(rnd(m, n, 8))
    y2, _ = t.fwd(res, z=False)
    t.check_fwd(y2, None, res)
    dy = t.rows(rnd(m, n, 9, 0.1))
    dx, dw, db = t.bwd(dy, z)
    t.check_bwd(dy, z, dx, dw, db)
    # again: bit for bit
    y3, z3 = t.fwd()
    dx3, dw3, db3 = t.bwd(dy, z)
    assert torch.equal(y.v, y3.v) and torch.equal(z.v, z3.v) and torch.equal(dx.v, dx3.v) and torch.equal(dw, dw3) and torch.equal(db, db3)


LIN_LARGE = [  # m, n, k, pad, off: each the smallest kind of layer that takes the tile
    (8200, 1032, 520, 0, 0),        # 224 x 256 forward, ragged in every direction
    (8200, 520, 1032, 8, 0),        # 224 x 256 dx
    (11600, 1288, 520, 0, 0),       # 256 x 256 forward
    (11600, 520, 1288, 0, 0),       # 256 x 256 dx
    (12900, 264, 248, 0, 0),        # 128 x 128, dx and dw in one launch
    (12900, 259, 251, 1, 0),        # ... through registers
    (400, 512, 512, 0, 0),          # 32 x 32 blocks
    (333, 515, 509, 0, 1),          # ... with cut rows
    (3300, 500, 300, 0, 0),         # 64 x 64 tiles, rows of whole fp32 vectors but not of bf16 ones
]


@pytest.mark.parametrize("dt", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", LIN_LARGE, ids=lambda s: "m%d_n%d_k%d_p%d_o%d" % s)
def test_linear_large(shape, dt):
    m, n, k, pad, off = shape
    t = Lin(dt, m, n, k, "silu", True, pad, off, pad)
    res = t.rows(rnd(m, n, 8))
    y, z = t.fwd(res)
    t.check_fwd(y, z, res)
    dy = t.rows(rnd(m, n, 9, 0.1))
    base = Mat(m, k, dt, pad, off, rnd(m, k, 10, 0.1))
    b64 = base.v.double().clone()
    dx, dw, db = t.bwd(dy, z, dxm=base, acc_dx=1)
    t.check_bwd(dy, z, dx, dw, db, base=b64)
    y2, _ = t.fwd(res, z=False)
    assert torch.equal(y.v, y2.v)
    base.v.copy_(b64.to(base.v.dtype))
    dx2, dw2, db2 = t.bwd(dy, z, dxm=base, acc_dx=1)
    t.check_bwd(dy, z, dx2, None, None, base=b64)
    assert torch.equal(dw, dw2) and torch.equal(db, db2)


def test_linear_first_call_captured():
    """The first launch of a kernel that needs more than 64 KiB of LDS may be a captured one."""
    t = Lin(BF16, 8200, 1032, 520, "gelu")
    y, z = t.rows(), t.rows()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call("plyolo_linear_fwd", C.byref(t.d), t.x.ptr, t.w.ptr, ptr(t.b), None, z.ptr, y.ptr, None, 0, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        y.v.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        t.check_fwd(y, z)


@pytest.mark.parametrize("dt", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("m", [5, 300])
def test_linear_activations_parts_and_accumulation(act, dt, m):
    n, k = 96, 72
    t = Lin(dt, m, n, k, act, bias=act != "relu")
    y, z = t.fwd()
    t.check_fwd(y, z)
    dy = t.rows(rnd(m, n, 9, 0.1))
    zz = z if act != "none" else None
    dx, dw, db = t.bwd(dy, zz)
    t.check_bwd(dy, zz, dx, dw, db)
    # each gradient alone is the same
    a = t.bwd(dy, zz, dw=False, db=False)[0]
    b = t.bwd(dy, zz, dx=False, db=False)[1]
    c = t.bwd(dy, zz, dx=False, dw=False)[2]
    assert torch.equal(a.v, dx.v) and torch.equal(b, dw) and torch.equal(c, db)
    # fp32 weight gradients, all three added to what is there
    base = Mat(m, k, dt, data=rnd(m, k, 10, 0.1))
    b64 = base.v.double().clone()
    w0, b0 = rnd(n, k, 11, 0.1), rnd(1, n, 12).flatten()
    ref = t.bwd(dy, zz, dwt=F32)[1]
    t.check_bwd(dy, zz, None, ref, None, dwt=F32)
    dw2, db2 = w0.clone(), b0.clone()
    t.bwd(dy, zz, dw=dw2, dwt=F32, dxm=base, acc_dx=1, acc_par=1, dbt=db2)
    t.check_bwd(dy, zz, base, None, None, base=b64)
    assert_close(dw2, ref.double() + w0.double(), 2 * E32 * (ref.double().abs() + w0.double().abs()), "dw +=")
    assert_close(db2, db.double() + b0.double(), 2 * E32 * (db.double().abs() + b0.double().abs()), "db +=")


def test_linear_gradient_against_differences():
    t = Lin(F32, 40, 24, 36, "gelu")
    r = rnd(40, 24, 41)
    y, z = t.fwd()
    dx, dw, db = t.bwd(t.rows(r), z)
    h = 2.0 ** -7

    def f():
        return float((t.fwd()[0].v.double() * r.double()).sum())
    x64, w64 = t.x.v.double().clone(), t.w.v.double().clone()
    for buf, grad, shape in ((t.x.v, dx.v, (40, 36)), (t.w.v, dw, (24, 36)), (t.b, db, (24,))):
        v = torch.randn(shape, generator=gen(50), device=DEV)
        # The central difference of r * gelu(z + s d) is off by at most h^2 / 6 * sup |gelu3| * |r| |d|^3, with the third derivative
        # gelu3(z) = phi(z) z (z^2 - 4), |gelu3| < 0.8, and d = the change of z along v; the two forward passes by
        # (K + 64) E32 (|x| |w| + |b|) |r| each, divided by 2 h
        v64 = v.double()
        d = v64 @ w64.t() if shape == (40, 36) else x64 @ v64.t() if shape == (24, 36) else v64.expand(40, 24)
        cut = h * h / 6 * 0.8 * float((r.double().abs() * d.abs() ** 3).sum())
        size = (x64.abs() + h * 5) @ (w64.abs() + h * 5).t() + t.b.double().abs() + h * 5
        rounding = (36 + 64) * E32 * float((size * r.double().abs()).sum()) / h
        keep = buf.clone()
        buf.copy_(keep + h * v)
        up = f()
        buf.copy_(keep - h * v)
        dn = f()
        buf.copy_(keep)
        want = float((grad.double() * v.double()).sum())
        assert abs((up - dn) / (2 * h) - want) < cut + rounding, (cut, rounding)


@pytest.mark.parametrize("m", [3, 200])
def test_linear_keeps_nan_in_its_row(m):
    """A NaN or infinity in one input row reaches that output row only; padding columns full of NaN reach nothing."""
    t = Lin(BF16, m, 72, 40, "none", pad=8)
    y0, _ = t.fwd()
    t.x.buf[:].masked_fill_(t.x.buf == GUARD, float("nan"))
    y1, _ = t.fwd()
    assert torch.equal(y0.v, y1.v)
    t.x.v[1, 3] = float("inf")
    y2, _ = t.fwd()
    assert torch.equal(y0.v[[0, 2]], y2.v[[0, 2]]) and not bool(torch.isfinite(y2.v[1]).any())


# ------------------------------------------------------------------------------------------------ dropout
def drop(dt, m, c, p, rng, site, x, res=None, out=None, bwd=False, acc=0):
    out = out or Mat(m, c, dt, x.ld - c, x.off)
    if bwd:
        call("plyolo_dropout_bwd", dt, m, c, x.ptr, x.ld, p, rng.data_ptr(), site, out.ptr, out.ld, acc, hu.stream())
    else:
        call("plyolo_dropout_fwd", dt, m, c, x.ptr, x.ld, p, rng.data_ptr(), site, res.ptr if res else None, res.ld if res else 0, out.ptr, out.ld, hu.stream())
    return out


DROP_SHAPES = [(1, 1, 0, 0), (1, 13, 0, 0), (5, 8, 0, 0), (7, 12, 4, 0), (33, 24, 8, 0), (400, 256, 0, 0), (129, 85, 3, 0), (129, 85, 0, 0), (50, 16, 0, 1), (1000, 3, 1, 0),
               (3, 4099, 0, 0)]


@pytest.mark.parametrize("dt", [BF16, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
@pytest.mark.parametrize("shape", DROP_SHAPES, ids=lambda s: "m%d_c%d_p%d_o%d" % s)
def test_dropout(shape, p, dt):
    m, c, pad, off = shape
    seed, step, site = 0x7edcba9876543210, (1 << 32) + 41, 5        # the upper half of the step is not used
    rng = torch.tensor([seed, step], dtype=torch.int64, device=DEV)
    x, res = Mat(m, c, dt, pad, off, rnd(m, c, 2)), Mat(m, c, dt, pad + 8, off, rnd(m, c, 3))
    keep = torch.from_numpy(keep_mask(seed, step, site, m, c, p)).to(DEV)
    scale = 1.0 / (1.0 - float(torch.tensor(p, dtype=torch.float32))) if p < 1.0 else 0.0
    want = torch.where(keep, x.v.double() * scale, torch.zeros((), dtype=torch.float64, device=DEV))
    out = drop(dt, m, c, p, rng, site, x)
    assert torch.equal(out.v != 0, keep & (x.v != 0))
    assert_close(out.v, want, 4 * E32 * want.abs() + UNIT[dt] * want.abs(), "out")
    o2 = drop(dt, m, c, p, rng, site, x, res)
    w2 = want + res.v.double()
    assert_close(o2.v, w2, 4 * E32 * (want.abs() + w2.abs()) + UNIT[dt] * w2.abs(), "out + res")
    # the backward is the same mask; accumulation; in place
    assert torch.equal(drop(dt, m, c, p, rng, site, x, bwd=True).v, out.v)
    acc = Mat(m, c, dt, pad, off, res.v)
    drop(dt, m, c, p, rng, site, x, out=acc, bwd=True, acc=1)
    assert torch.equal(acc.v, o2.v) and acc.untouched() and out.untouched() and o2.untouched()
    drop(dt, m, c, p, rng, site, x, out=x)
    assert torch.equal(x.v, out.v)


def test_dropout_element_index_is_pitch_free_and_paths_agree():
    """The mask depends on (row, column) and not on pitch, alignment, type or the kernel that the sizes choose."""
    rng = torch.tensor([99, 7], dtype=torch.int64, device=DEV)
    one = None
    for dt in (BF16, F32):
        for pad, off in ((0, 0), (8, 0), (1, 0), (0, 1), (3, 5)):
            x = Mat(61, 24, dt, pad, off, torch.ones(61, 24, device=DEV))
            k = drop(dt, 61, 24, 0.5, rng, 2, x).v != 0
            one = k if one is None else one
            assert torch.equal(k, one)
    other = drop(BF16, 61, 24, 0.5, rng, 3, Mat(61, 24, BF16, data=torch.ones(61, 24, device=DEV))).v != 0
    assert not torch.equal(other, one)


def test_dropout_drops_infinities_and_nan():
    x = torch.full((64, 64), float("inf"), device=DEV)
    x[::2] = float("nan")
    rng = torch.tensor([1, 1], dtype=torch.int64, device=DEV)
    keep = torch.from_numpy(keep_mask(1, 1, 0, 64, 64, 0.5)).to(DEV)
    for dt in (BF16, F32):
        o = drop(dt, 64, 64, 0.5, rng, 0, Mat(64, 64, dt, data=x)).v.float()
        assert bool((o[~keep] == 0).all()) and not bool(torch.isfinite(o[keep]).any())


def test_dropout_rate():
    rng = torch.tensor([5, 5], dtype=torch.int64, device=DEV)
    x = Mat(4096, 256, F32, data=torch.ones(4096, 256, device=DEV))
    for p in (0.05, 0.3, 0.9):
        n = 4096 * 256
        kept = int((drop(F32, 4096, 256, p, rng, 1, x).v != 0).sum())
        assert abs(kept - n * (1 - p)) < 5 * (n * p * (1 - p)) ** 0.5       # five standard deviations


def test_rng_next_counts_steps():
    state, out = torch.tensor([11, 41], dtype=torch.int64, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    for i in range(3):
        call("plyolo_rng_next", state.data_ptr(), out.data_ptr(), hu.stream())
        assert out.tolist() == [11, 41 + i] and state.tolist() == [11, 42 + i]


# ------------------------------------------------------------------------------------------------ together
class Block:
    """y = x + dropout(W2 silu(W1 silu(gn(x)) + b1) + b2) on pixel rows, and its backward: the three operators as a training step uses them."""

    def __init__(self, dt, n, hw, c, hid):
        self.m, self.c = n * hw, c
        self.gn = Gn(dt, n, hw, c, 8, "silu", seed=61)
        self.l1 = Lin(dt, self.m, hid, c, "silu", seed=71)
        self.l2 = Lin(dt, self.m, c, hid, "none", seed=81)
        self.state = torch.tensor([1234, 0], dtype=torch.int64, device=DEV)
        self.rng = torch.zeros(2, dtype=torch.int64, device=DEV)
        self.dt = dt
        self.out, self.dy = Mat(self.m, c, dt), Mat(self.m, c, dt, data=rnd(self.m, c, 91, 0.1))
        self.h, self.t = self.gn.mat(), Mat(self.m, hid, dt)
        self.zm, self.u = Mat(self.m, hid, dt), Mat(self.m, c, dt)
        self.st = torch.zeros(n, 8, 2, device=DEV)
        self.g3, self.g2, self.g1, self.dx = Mat(self.m, c, dt), Mat(self.m, hid, dt), Mat(self.m, c, dt), Mat(self.m, c, dt)
        self.dw1, self.dw2 = torch.zeros(hid, c, device=DEV), torch.zeros(c, hid, device=DEV)
        self.db1, self.db2 = torch.zeros(hid, device=DEV), torch.zeros(c, device=DEV)
        self.dga, self.dbe = torch.zeros(c, device=DEV), torch.zeros(c, device=DEV)

    def step(self, s):
        g, a, b, p = self.gn, self.l1, self.l2, 0.25
        call("plyolo_rng_next", self.state.data_ptr(), self.rng.data_ptr(), s)
        g.fwd(out=self.h, stats=self.st, stream=s)
        call("plyolo_linear_fwd", C.byref(a.d), self.h.ptr, a.w.ptr, ptr(a.b), None, self.zm.ptr, self.t.ptr, a.ws.data_ptr(), a.nf, s)
        call("plyolo_linear_fwd", C.byref(b.d), self.t.ptr, b.w.ptr, ptr(b.b), None, None, self.u.ptr, b.ws.data_ptr(), b.nf, s)
        call("plyolo_dropout_fwd", self.dt, self.m, self.c, self.u.ptr, self.u.ld, p, self.rng.data_ptr(), 4, g.x.ptr, g.x.ld, self.out.ptr, self.out.ld, s)
        call("plyolo_dropout_bwd", self.dt, self.m, self.c, self.dy.ptr, self.dy.ld, p, self.rng.data_ptr(), 4, self.g3.ptr, self.g3.ld, 0, s)
        call("plyolo_linear_bwd", C.byref(b.d), self.g3.ptr, None, self.t.ptr, b.w.ptr, self.g2.ptr, self.g2.ld, 0, self.dw2.data_ptr(), F32, self.db2.data_ptr(), 0,
             b.ws.data_ptr(), b.nb, s)
        call("plyolo_linear_bwd", C.byref(a.d), self.g2.ptr, self.zm.ptr, self.h.ptr, a.w.ptr, self.g1.ptr, self.g1.ld, 0, self.dw1.data_ptr(), F32, self.db1.data_ptr(),
             0, a.ws.data_ptr(), a.nb, s)
        call("plyolo_copy_add", self.dt, self.m, self.c, self.dy.ptr, self.dy.ld, self.dx.ptr, self.dx.ld, 0, s)        # the shortcut's gradient
        call("plyolo_gn_act_bwd", C.byref(g.d), self.g1.ptr, self.g1.ld, g.x.ptr, self.st.data_ptr(), ptr(g.gamma), ptr(g.beta), self.dx.ptr, self.dx.ld, 1,
             self.dga.data_ptr(), self.dbe.data_ptr(), 0, g.ws.data_ptr(), g.nws, s)

    def results(self):
        return [t.clone() for t in (self.out.v, self.dx.v, self.dw1, self.dw2, self.db1, self.db2, self.dga, self.dbe, self.rng)]


def test_block_gradients_against_automatic_differentiation():
    k = Block(F32, 2, 90, 32, 48)
    k.step(hu.stream())
    x = k.gn.x.v.double().clone().requires_grad_(True)
    par = [t.double().clone().requires_grad_(True) for t in (k.l1.w.v, k.l2.w.v, k.l1.b, k.l2.b, k.gn.gamma, k.gn.beta)]
    w1, w2, b1, b2, ga, be = par
    t = x.view(2, 90, 8, 4)
    xh = ((t - t.mean(dim=(1, 3), keepdim=True)) / torch.sqrt(t.var(dim=(1, 3), keepdim=True, unbiased=False) + 1e-5)).reshape(180, 32)
    h = act64(xh * ga + be, "silu")
    u = act64(h @ w1.t() + b1, "silu") @ w2.t() + b2
    keep = torch.from_numpy(keep_mask(1234, 0, 4, 180, 32, 0.25)).to(DEV)
    y = x + torch.where(keep, u / 0.75, torch.zeros_like(u))
    y.backward(k.dy.v.double())
    got = k.results()
    for a, b, name in zip(got, [y.detach(), x.grad] + [q.grad for q in par], ("out", "dx", "dw1", "dw2", "db1", "db2", "dgamma", "dbeta")):
        # chains of three layers with sums of at most 180 terms of mixed sign: 1e-5 of the largest value covers 180 * E32 many times over
        assert_close(a, b, 1e-5 * float(b.abs().max()), name)


@pytest.mark.parametrize("dt", [BF16, F32], ids=["bf16", "fp32"])
def test_block_captured_and_replayed(dt):
    """A captured step replays with the generator's state moving on: every replay equals the eager step of the same number."""
    eager, cap = Block(dt, 2, 70, 32, 40), Block(dt, 2, 70, 32, 40)
    want = []
    for _ in range(4):
        eager.step(hu.stream())
        want.append(eager.results())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        cap.step(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(cap.results(), want[i]):
            assert torch.equal(a, b), i
        torch.randn(1000, device=DEV).sum().item()       # eager work between replays
    assert not torch.equal(want[0][0], want[1][0])       # another mask each step


def test_block_recorded_in_a_plan():
    eager, rec = Block(BF16, 2, 70, 32, 40), Block(BF16, 2, 70, 32, 40)
    lib = _lib.lib()
    plan = lib.plyolo_plan_create()
    _lib.check(lib.plyolo_plan_begin(plan))
    rec.step(None)
    _lib.check(lib.plyolo_plan_end(plan))
    for i in range(3):
        eager.step(hu.stream())
        _lib.check(lib.plyolo_plan_run(plan, hu.stream()))
        torch.cuda.synchronize()
        for a, b in zip(rec.results(), eager.results()):
            assert torch.equal(a, b), i
    lib.plyolo_plan_destroy(plan)


def test_two_streams_with_their_own_workspaces():
    a, b = Block(BF16, 4, 400, 64, 128), Block(BF16, 4, 400, 64, 128)
    a.step(hu.stream())
    torch.cuda.synchronize()
    want = a.results()
    a.state.copy_(torch.tensor([1234, 0], device=DEV))
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    a.step(s1.cuda_stream)
    b.step(s2.cuda_stream)
    torch.cuda.synchronize()
    for x, y, z in zip(a.results(), b.results(), want):
        assert torch.equal(x, z) and torch.equal(y, z)


def test_rows_beyond_32_bit_offsets():
    """Pitches that put the last rows more than 2^31 elements behind the first: bit for bit what packed rows give."""
    m, c, ld = 70000, 16, 32000
    big = torch.empty(m * ld, dtype=torch.bfloat16, device=DEV)

    def col(i, data=None):
        v = big.as_strided((m, c), (ld, 1), 64 * i)
        if data is not None:
            v.copy_(data)
        return v
    data = {s: rnd(m, c, s).bfloat16() for s in (1, 2, 3)}
    w, b, ga, be = rnd(c, c, 4, 0.3).bfloat16(), rnd(1, c, 5).flatten(), rnd(1, c, 6).flatten(), rnd(1, c, 7).flatten()
    rng = torch.tensor([77, 5], dtype=torch.int64, device=DEV)
    lib, s = _lib.lib(), hu.stream()

    def run(place, ld):
        x, res, dy = place(0, data[1]), place(1, data[2]), place(2, data[3])
        z, y, dx, o, dg, dd = (place(i) for i in range(3, 9))
        d = LinearDesc()
        d.dtype, d.M, d.N, d.K, d.act, d.x_ld, d.w_ld, d.y_ld, d.z_ld, d.r_ld = BF16, m, c, c, ACTS["silu"], ld, c, ld, ld, ld
        nws = lib.plyolo_linear_workspace(C.byref(d), 1)
        ws = torch.empty(nws, dtype=torch.uint8, device=DEV)
        dw, db = torch.empty(c, c, dtype=torch.bfloat16, device=DEV), torch.empty(c, device=DEV)
        call("plyolo_linear_fwd", C.byref(d), x.data_ptr(), w.data_ptr(), ptr(b), res.data_ptr(), z.data_ptr(), y.data_ptr(), None, 0, s)
        call("plyolo_linear_bwd", C.byref(d), dy.data_ptr(), z.data_ptr(), x.data_ptr(), w.data_ptr(), dx.data_ptr(), ld, 0, dw.data_ptr(), BF16, ptr(db), 0,
             ws.data_ptr(), nws, s)
        g = GnDesc()
        g.dtype, g.N, g.HW, g.C, g.groups, g.act, g.eps, g.x_ld, g.o_ld, g.r_ld = BF16, 2, m // 2, c, 4, ACTS["silu"], 1e-5, ld, ld, ld
        nws = lib.plyolo_gn_workspace(C.byref(g))
        ws2 = torch.empty(nws, dtype=torch.uint8, device=DEV)
        st, dga, dbe = torch.empty(2, 4, 2, device=DEV), torch.empty(c, device=DEV), torch.empty(c, device=DEV)
        call("plyolo_gn_act_fwd", C.byref(g), x.data_ptr(), ptr(ga), ptr(be), res.data_ptr(), o.data_ptr(), ptr(st), ws2.data_ptr(), nws, s)
        call("plyolo_gn_act_bwd", C.byref(g), dy.data_ptr(), ld, x.data_ptr(), ptr(st), ptr(ga), ptr(be), dg.data_ptr(), ld, 0, ptr(dga), ptr(dbe), 0,
             ws2.data_ptr(), nws, s)
        call("plyolo_dropout_fwd", BF16, m, c, x.data_ptr(), ld, 0.25, rng.data_ptr(), 3, res.data_ptr(), ld, dd.data_ptr(), ld, s)
        return [t.clone() for t in (z, y, dx, dw, db, o, st, dg, dga, dbe, dd)]
    far = run(col, ld)
    near = run(lambda i, v=None: v.clone() if v is not None else torch.empty(m, c, dtype=torch.bfloat16, device=DEV), c)
    for name, a, e in zip(("z", "y", "dx", "dw", "db", "gn", "stats", "gn dx", "dgamma", "dbeta", "dropout"), far, near):
        assert torch.equal(a, e), name
