"""-m gpu: the batch-free units where their documentation allows more than the shipped models ask for: any channel count, shortcuts on odd
rows, probabilities that change, several streams.

Tolerances: bf16 stored values are off by half a step, 2^-8 relative (UNIT); the linear unit rounds x and W on their way in (the references
here start from the rounded ones), z, dz and its outputs once each."""
import ctypes as C
import math
import os

import pytest
import torch
import torch.nn.functional as F
import yaml

import hiputil as hu
import pl_yolo_amd
from batchfree import ACTS, E32, UNIT, Mat, act64, act_grad64, assert_close, keep_mask
from conftest import ROOT
from oracle import detector as odet
from pl_yolo_amd import _lib
from pl_yolo_amd._lib import BF16, F32, GnDesc, LinearDesc, call
from pl_yolo_amd.layers import BaseConv, Dropout, HipModule, dropout_state, get_normalization

pytestmark = pytest.mark.gpu
DEV = hu.DEV
TYPES = {"bf16": 0, "fp32": 1}


def rnd(shape, seed, dtype="fp32", scale=1.0):
    x = (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV)
    return hu.rnd_bf16(x) if dtype == "bf16" else x


def rows(x):
    """[N, C, H, W] -> pixel rows [N H W, C] in 64 bits."""
    return x.double().permute(0, 2, 3, 1).reshape(-1, x.shape[1])


def linear_bounds(x, w, b, act, dy, u, ez):
    """(z, y, dx, dw, db) of the unit on rows in 64 bits and how far each may be off: sums of n terms by n E32 of their sizes, the
    activation's chain by 64 E32, stored values by u; the stored z is off by ez |z| more, and act' moves by at most |act''| <= 1.2 of that."""
    n, k = w.shape
    z = x @ w.t() + b
    tz = (k + 4) * E32 * (x.abs() @ w.abs().t() + b.abs())
    y = act64(z, act)
    ty = 1.2 * tz + 64 * E32 * (y.abs() + E32)
    dz = dy * act_grad64(z, act)
    tdz = dy.abs() * (1.2 * (tz + ez * (z.abs() + tz)) + 64 * E32 * (1.0 + z.abs()))
    td = tdz + u * (dz.abs() + tdz)          # dz as the operand of the two products
    dx, dw = dz @ w, dz.t() @ x
    tdx = td @ w.abs() + (n + 4) * E32 * (dz.abs() @ w.abs())
    tdw = td.t() @ x.abs() + (len(x) + 64) * E32 * (dz.abs().t() @ x.abs())
    return ((y, ty + u * (y.abs() + ty)), (dx, tdx + u * (dx.abs() + tdx)), (dw, tdw + E32 * dw.abs()),
            (dz.sum(0), tdz.sum(0) + 1100 * E32 * dz.abs().sum(0) + 1e-30))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("cin,cout,hw,n", [(179, 85, (7, 5), 3), (1, 3, (4, 4), 2), (85, 179, (1, 1), 4), (13, 8, (33, 17), 2)])
def test_linear_unit_of_any_channel_count(cin, cout, hw, n, dtype):
    torch.manual_seed(31)
    m = BaseConv(cin, cout, 1, 1, bias=True, norm=None, act="gelu").to(DEV).train()
    m.compute_dtype = dtype
    x, r = rnd((n, cin) + hw, 32, dtype), rnd((n, cout) + hw, 33, dtype, 0.1)
    w = (hu.rnd_bf16(m.conv.weight) if dtype == "bf16" else m.conv.weight).detach().double().view(cout, cin)
    u = UNIT[TYPES[dtype]]
    want = linear_bounds(rows(x), w, m.conv.bias.detach().double(), "gelu", rows(r), u, u)
    for _ in range(2):
        xi = x.clone().requires_grad_(True)
        m.zero_grad()
        y = m(xi)
        y.backward(r)
        for got, (ref, tol), what in zip((rows(y.detach()), rows(xi.grad), m.conv.weight.grad.view(cout, cin), m.conv.bias.grad), want, ("y", "dx", "dw", "db")):
            assert_close(got, ref, tol, what)
    m.eval()
    with torch.no_grad():
        assert torch.equal(m(x), y)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("c", [1, 3, 85])
def test_dropout_of_any_channel_count(c, dtype):
    m = Dropout(0.3).train()
    m.compute_dtype = dtype
    x, r = rnd((2, c, 5, 7), 34, dtype), rnd((2, c, 5, 7), 35, dtype)
    seed = dropout_state(m).tolist()[0]
    u = UNIT[TYPES[dtype]]
    for step in range(2):
        xi = x.clone().requires_grad_(True)
        y = m(xi)
        y.backward(r)
        keep = torch.from_numpy(keep_mask(seed, step, 0, 70, c, 0.3)).to(DEV)
        for got, src, what in ((y.detach(), x, "y"), (xi.grad, r, "dx")):
            want = torch.where(keep, rows(src) / 0.7, torch.zeros((), dtype=torch.float64, device=DEV))
            assert_close(rows(got), want, (8 * E32 + u) * want.abs(), what)


# ------------------------------------------------------------------------------------------------ shortcuts and slices on odd rows
@pytest.mark.parametrize("dt", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("m,c,pad,off,ipad", [(1, 1, 0, 0, 0), (37, 85, 0, 0, 3), (1000, 7, 9, 5, 1), (64, 24, 8, 0, 0), (64, 24, 8, 1, 0), (5, 16, 3, 0, 8), (3, 70001, 0, 0, 0)])
def test_copy_add_of_any_rows(m, c, pad, off, ipad, dt):
    src, base = Mat(m, c, dt, ipad, off, rnd((m, c), 36)), rnd((m, c), 37)
    for data, acc in ((None, 0), (base, 1)):
        out = Mat(m, c, dt, pad, off, data)
        want = src.v.float() + (out.v.float() if acc else 0.0)
        call("plyolo_copy_add", dt, m, c, src.ptr, src.ld, out.ptr, out.ld, acc, hu.stream())
        assert torch.equal(out.v, want.to(out.v.dtype)) and out.untouched()
    call("plyolo_copy_add", dt, m, c, None, 0, out.ptr, out.ld, 0, hu.stream())
    assert not bool(out.v.any()) and out.untouched()


class Net(HipModule):
    """A concatenation of two linear units' outputs with an odd boundary, one part of it read a second time, and a shortcut on odd rows:
    t = [a(x), b(x)];  out = d(c(t)) + a(x) with dropout in front of the shortcut."""

    any_channels = True

    def __init__(self):
        super().__init__()
        self.a = BaseConv(13, 5, 1, 1, bias=True, norm=None, act="silu")
        self.b = BaseConv(13, 11, 1, 1, bias=True, norm=None, act="gelu")
        self.c = BaseConv(16, 9, 1, 1, bias=True, norm=None, act="silu")
        self.d = BaseConv(9, 5, 1, 1, bias=True, norm=None, act=None, drop=0.25)

    def emit(self, g, x):
        a = self.a.emit(g, x)
        t = g.concat([a, self.b.emit(g, x)])
        return self.d.emit(g, self.c.emit(g, t), residual=a)


def net64(m, w, x, keep):
    p = {n: (w[n + ".conv.weight"].flatten(1), w[n + ".conv.bias"]) for n in "abcd"}
    a = act64(x @ p["a"][0].t() + p["a"][1], "silu")
    t = torch.cat([a, act64(x @ p["b"][0].t() + p["b"][1], "gelu")], 1)
    u = act64(t @ p["c"][0].t() + p["c"][1], "silu") @ p["d"][0].t() + p["d"][1]
    return a + keep * u / 0.75


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_shortcuts_and_concatenations_on_odd_rows(dtype):
    torch.manual_seed(38)
    m = Net().to(DEV).train()
    m.compute_dtype = dtype
    x, r = rnd((3, 13, 6, 5), 39, dtype), rnd((3, 5, 6, 5), 40, dtype)
    w = {n: (hu.rnd_bf16(p) if dtype == "bf16" and n.endswith("weight") else p).detach().double().clone().requires_grad_(True) for n, p in m.named_parameters()}
    seed = dropout_state(m).tolist()[0]
    # fp32: chains of three layers of at most 90 rows and 16 channels, sums of mixed sign: (90 + 16 * 3 + 3 * 64) half steps, below 2e-5 of
    # the largest value.  bf16: every stored tensor of the chain (three layers forward, their gradients back) is off by 2^-8 of its own size:
    # 8 of them between the input and a gradient, 8 * 2^-8 of the largest value
    tol = 2e-5 if dtype == "fp32" else 8 * UNIT[0]
    for step in range(2):
        keep = torch.from_numpy(keep_mask(seed, step, 0, 90, 5, 0.25)).to(DEV)
        x64 = rows(x).requires_grad_(True)
        for p in w.values():
            p.grad = None
        y = net64(m, w, x64, keep)
        y.backward(rows(r))
        xi = x.clone().requires_grad_(True)
        m.zero_grad()
        got = m(xi)
        got.backward(r)
        for a, b, what in [(rows(got.detach()), y.detach(), "y"), (rows(xi.grad), x64.grad, "dx")] + [(p.grad, w[n].grad, n) for n, p in m.named_parameters()]:
            assert_close(a, b, tol * float(b.abs().max()), what)


# ------------------------------------------------------------------------------------------------ probabilities that change
def test_a_changed_probability_changes_rate_and_scale():
    """Values between two calls of one shape, as in a schedule: each call follows the value it meets, backward included."""
    m = Dropout(0.5).train()
    m.compute_dtype = "fp32"
    x = torch.ones(2, 64, 32, 32, device=DEV)
    seed = dropout_state(m).tolist()[0]
    for step, p in enumerate((0.5, 0.125, 0.0, 0.75, 1.0, 0.5)):
        m.p = p
        xi = x.clone().requires_grad_(True)
        y = m(xi)
        y.backward(x)
        keep = torch.from_numpy(keep_mask(seed, step, 0, 2048, 64, p)).to(DEV)
        want = keep.double() * (1.0 / (1.0 - p) if p < 1.0 else 0.0)
        assert_close(rows(y.detach()), want, 8 * E32 * want, "y")
        assert torch.equal(xi.grad, y.detach())
    m.p = 0.5
    m.eval()
    with torch.no_grad():
        assert torch.equal(m(x), x)


def test_a_detector_follows_a_changed_probability():
    with open(os.path.join(ROOT, "configs", "model", "yolox", "yolox_test.yaml")) as f:
        cfg = yaml.safe_load(f)
    torch.manual_seed(41)
    m = pl_yolo_amd.build_model(cfg, 3).to(DEV).train()
    m.compute_dtype = "fp32"
    imgs, labels = odet.synthetic_batch(2, 64, 3, num_gt=3, max_gt=8, seed=6)
    unit, losses = m.backbone.stage4[2].conv3, []

    def step():
        m.zero_grad()
        out = m(imgs.to(DEV), labels.to(DEV))
        out["loss"].backward()
        assert all(bool(torch.isfinite(p.grad).all()) for p in m.parameters() if p.grad is not None)
        losses.append(float(out["loss"].detach()))
    state = dropout_state(m)
    for drop, steps in ((0.0, 0), (0.5, 1), (0.0, 1), (0.5, 2)):
        unit.drop = drop
        step()
        assert state.tolist()[1] == steps, (drop, state)
    # batch statistics by atomics: the same arithmetic repeats to fp32 rounding; half the features dropped is far beyond it
    assert abs(losses[2] - losses[0]) <= 1e-5 * abs(losses[0]) < abs(losses[1] - losses[0]) and losses[1] != losses[3]


# ------------------------------------------------------------------------------------------------ whole detectors with group norm
def gn_detector(path, dtype, nc=3):
    with open(os.path.join(ROOT, "configs", "model", path)) as f:
        cfg = yaml.safe_load(f)
    for part in ("backbone", "neck", "head"):
        cfg[part]["norm"] = "gn"
    torch.manual_seed(42)
    m = pl_yolo_amd.build_model(cfg, nc)
    for u in m.modules():      # the units that `norm` does not reach
        if isinstance(u, BaseConv) and isinstance(u.norm, torch.nn.BatchNorm2d):
            u.norm = get_normalization("gn", u.conv.out_channels)
    m = m.to(DEV).train()
    m.compute_dtype = dtype
    return m


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("path", ["yolox/yolox_test.yaml", "yolov7/yolov7_test.yaml"])
def test_a_group_norm_detector_does_not_depend_on_its_batch(path, dtype):
    """The maps of training and of inference are the same bit for bit, and an image's maps do not depend on the others of its batch: fp32 to
    rounding (launches of another batch sum in another order; 1e-3 of the largest value is a thousand times that), where batch statistics
    of these three images move them by their own size."""
    m = gn_detector(path, dtype)
    x = rnd((3, 3, 128, 128), 43, scale=50.0)
    x[1] *= 3.0
    x[2] += 100.0
    with torch.no_grad():
        train = [t.clone() for t in m(x)]
        m.eval()
        for a, b in zip(train, m(x)):
            assert torch.equal(a, b)
        m.train()
        if dtype == "fp32":
            for i in range(3):
                for a, b in zip(train, m(x[i:i + 1])):
                    assert hu.relerr(b[0], a[i]) <= 1e-3


@pytest.mark.parametrize("path", ["yolox/yolox_test.yaml", "yolov7/yolov7_test.yaml"])
def test_group_norm_detector_steps_repeat_on_any_lanes(path, monkeypatch):
    """bf16 training steps with group norm everywhere and dropout in two units: loss and every gradient are the same bit for bit on several
    streams, on one, and again, and so as captured graphs."""
    imgs, labels = odet.synthetic_batch(2, 96, 3, num_gt=3, max_gt=8, seed=77)
    runs = []
    for lanes, graph in (("1", "auto"), ("0", "auto"), ("1", "auto"), ("0", "1"), ("1", "1"), ("0", "0")):
        monkeypatch.setenv("PLYOLO_LANES", lanes)
        monkeypatch.setenv("PLYOLO_GRAPH", graph)
        m = gn_detector(path, "bf16")
        units = [k for k in m.modules() if isinstance(k, BaseConv)]
        units[5].drop, units[-4].drop = 0.25, 0.5
        dropout_state(m).copy_(torch.tensor([12345, 0], device=DEV))
        for _ in range(3):
            m.zero_grad(set_to_none=True)
            loss = m(imgs.to(DEV), labels.to(DEV))["loss"]
            loss.sum().backward()
            runs.append(((lanes, graph), loss.detach().clone(), {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}))
    assert not torch.equal(runs[0][1], runs[1][1])            # another mask each step
    for i in range(3, len(runs)):
        (_, l0, g0), (lanes, l1, g1) = runs[i % 3], runs[i]
        assert torch.equal(l0, l1), (lanes, i)
        off = [n for n in g0 if not torch.equal(g0[n], g1[n])]
        assert set(g0) == set(g1) and len(g0) > 100 and not off, (lanes, i, len(off), off[:8])


# ------------------------------------------------------------------------------------------------ one unit used twice
class Twice(HipModule):
    """a(x) + a(b(x)): the linear unit `a` runs twice in one trace, the second time on a lane of its own, and shares its weights (not its
    bias) with `c`."""

    any_channels = True

    def __init__(self):
        super().__init__()
        self.a = BaseConv(12, 12, 1, 1, bias=True, norm=None, act="silu")
        self.b = BaseConv(12, 12, 1, 1, bias=True, norm=None, act="gelu")
        self.c = BaseConv(12, 12, 1, 1, bias=True, norm=None, act=None)
        self.c.conv.weight = self.a.conv.weight

    def emit(self, g, x):
        y = self.a.emit(g, x)
        with g.on_lane(2):
            t = self.a.emit(g, self.b.emit(g, x))
        return self.c.emit(g, t, residual=y)


@pytest.mark.parametrize("frozen", [None, "weight", "bias"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_gradients_of_a_linear_unit_used_twice_add_up(dtype, frozen):
    torch.manual_seed(44)
    m = Twice().to(DEV).train()
    m.compute_dtype = dtype
    if frozen:
        getattr(m.a.conv, frozen).requires_grad_(False)
    x, r = rnd((2, 12, 9, 7), 45, dtype), rnd((2, 12, 9, 7), 46, dtype)
    w = {n: (hu.rnd_bf16(p) if dtype == "bf16" and n.endswith("weight") else p).detach().double().clone().requires_grad_(True) for n, p in m.named_parameters()}
    x64 = rows(x).requires_grad_(True)

    def unit(t, n, act):
        return act64(t @ w[("a" if n == "c" else n) + ".conv.weight"].view(12, 12).t() + w[n + ".conv.bias"], act)
    y = unit(x64, "a", "silu") + unit(unit(unit(x64, "b", "gelu"), "a", "silu"), "c", "none")
    y.backward(rows(r))
    # as for the network above: 2e-5 of the largest value in fp32, eight stored roundings of it in bf16
    tol = 2e-5 if dtype == "fp32" else 8 * UNIT[0]
    for _ in range(3):
        xi = x.clone().requires_grad_(True)
        m.zero_grad()
        got = m(xi)
        got.backward(r)
        for a, b, what in [(rows(got.detach()), y.detach(), "y"), (rows(xi.grad), x64.grad, "dx")] + \
                [(p.grad, w[n].grad, n) for n, p in m.named_parameters() if p.requires_grad]:
            assert_close(a, b, tol * float(b.abs().max()), what)
    if frozen:
        assert getattr(m.a.conv, frozen).grad is None


# ------------------------------------------------------------------------------------------------ kernels at the ends of their ranges
def test_group_norm_of_more_values_than_a_float_counts():
    """One group of 1.7e10 values.  x is 1 but for its first value, 256: the mean lies 255 away from the origin of the partials, and counts that
    are off by a rounding of fp32 (one part in 1.7e7) make a variance of 255^2 * 6e-8 = 4e-3 out of the true 255^2 / n = 3.8e-6.  A thread
    sums 256 squares of 255 in fp32: each addition is off by at most half a step of the sum, 256 * 256 * 2^-24 = 4e-3 of M2 together, half
    of which reaches rstd (less by eps).  The rest in closed form."""
    c, hw = 1023, 1024 * 16417
    x = torch.ones(hw, c, dtype=torch.bfloat16, device=DEV)
    x[0, 0] = 256.0
    d = GnDesc()
    d.dtype, d.N, d.HW, d.C, d.groups, d.act, d.eps, d.x_ld, d.o_ld, d.r_ld = BF16, 1, hw, c, 1, ACTS["none"], 1e-5, c, c, c
    nws = _lib.lib().plyolo_gn_workspace(C.byref(d))
    ws, st = torch.empty(nws, dtype=torch.uint8, device=DEV), torch.empty(2, device=DEV)
    call("plyolo_gn_act_fwd", C.byref(d), x.data_ptr(), None, None, None, x.data_ptr(), st.data_ptr(), ws.data_ptr(), nws, hu.stream())
    n = float(hw) * c
    mean, var = 1.0 + 255.0 / n, 255.0 ** 2 / n * (1.0 - 1.0 / n)
    rstd = (var + 1e-5) ** -0.5
    assert abs(float(st[0]) - mean) <= 2 * E32 and abs(float(st[1]) - rstd) <= 2e-3 * rstd, (st.tolist(), mean, rstd)
    assert float(x[0, 0]) == float(torch.tensor(255.0 * float(st[1])).bfloat16())
    for i in (1, hw // 2, hw - 1):      # (1 - mean) rstd, a rounding away from 0
        assert float(x[i].float().abs().max()) <= 2 * E32 * rstd


# ------------------------------------------------------------------------------------------------ NaN and infinity through the linear layer
LIN_SIZES = [(5, 24, 40), (300, 85, 179), (3300, 136, 264), (8200, 520, 1032)]      # blocks, cut rows, whole rows, the large tiles


class Linear:
    def __init__(self, dt, m, n, k, act):
        self.dt, self.m, self.n, self.k = dt, m, n, k
        self.x, self.w = Mat(m, k, dt, data=rnd((m, k), 51)), Mat(n, k, dt, data=rnd((n, k), 52, scale=k ** -0.5))
        self.b = rnd((n,), 53)
        d = LinearDesc()
        d.dtype, d.M, d.N, d.K, d.act, d.x_ld, d.w_ld, d.y_ld, d.z_ld = dt, m, n, k, ACTS[act], k, k, n, n
        self.d = d
        self.nws = _lib.lib().plyolo_linear_workspace(C.byref(d), 1)
        self.ws = torch.empty(self.nws, dtype=torch.uint8, device=DEV)

    def fwd(self):
        z, y = Mat(self.m, self.n, self.dt), Mat(self.m, self.n, self.dt)
        call("plyolo_linear_fwd", C.byref(self.d), self.x.ptr, self.w.ptr, self.b.data_ptr(), None, z.ptr, y.ptr, None, 0, hu.stream())
        return y, z

    def bwd(self, dy, z):
        dx, dw, db = Mat(self.m, self.k, self.dt), torch.empty(self.n, self.k, device=DEV), torch.empty(self.n, device=DEV)
        call("plyolo_linear_bwd", C.byref(self.d), dy.ptr, z.ptr if z is not None else None, self.x.ptr, self.w.ptr, dx.ptr, dx.ld, 0, dw.data_ptr(),
             F32, db.data_ptr(), 0, self.ws.data_ptr(), self.nws, hu.stream())
        return dx.v, dw, db


def only(a, b, rows_hit, cols_hit):
    """b differs from a nowhere but in these rows and columns, and is not finite anywhere in them."""
    hit = torch.zeros(a.shape, dtype=torch.bool, device=a.device)
    hit[rows_hit] = True
    hit[..., cols_hit] = True
    return torch.equal(a[~hit], b[~hit]) and not bool(torch.isfinite(b[hit]).any())


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dt", [0, 1], ids=["bf16", "fp32"])
@pytest.mark.parametrize("m,n,k", LIN_SIZES)
def test_linear_keeps_nan_and_infinity_in_their_rows_and_columns(m, n, k, dt, bad):
    """The last row, output and input column (what a tile's ragged end would spread): x[i] reaches y[i] and dw's column, w[o] reaches y's and
    z's column and all of dx, dy[i, o] reaches dx[i], dw[o] and db[o]."""
    t = Linear(dt, m, n, k, "none")
    t.x.v.copy_(t.x.v.sign() * t.x.v.abs().clamp(min=0.01))        # (no zeros: 0 * infinity would be NaN beside the infinities, both not finite)
    dy = Mat(m, n, dt, data=rnd((m, n), 54).sign() * rnd((m, n), 54).abs().clamp(min=0.01))
    (y0, z0), g0 = t.fwd(), t.bwd(dy, None)
    keep = t.x.v.clone()
    t.x.v[-1, -1] = bad
    y1, z1 = t.fwd()
    dx, dw, db = t.bwd(dy, None)
    assert only(y0.v, y1.v, [-1], []) and only(z0.v, z1.v, [-1], [])
    assert torch.equal(dx, g0[0]) and only(g0[1], dw, [], [-1]) and torch.equal(db, g0[2])
    t.x.v.copy_(keep)
    keep = t.w.v.clone()
    t.w.v[-1] = bad
    y1, z1 = t.fwd()
    dx, dw, db = t.bwd(dy, None)
    assert only(y0.v, y1.v, [], [-1]) and only(z0.v, z1.v, [], [-1])
    assert not bool(torch.isfinite(dx).any()) and torch.equal(dw, g0[1]) and torch.equal(db, g0[2])
    t.w.v.copy_(keep)
    dy.v[-1, -1] = bad
    dx, dw, db = t.bwd(dy, None)
    assert only(g0[0], dx, [-1], []) and only(g0[1], dw, [-1], []) and only(g0[2], db, [], [-1])


@pytest.mark.parametrize("act", ["silu", "gelu", "hswish", "lrelu"])
@pytest.mark.parametrize("dt", [0, 1], ids=["bf16", "fp32"])
def test_linear_backward_passes_a_nan_of_z(dt, act):
    t = Linear(dt, 300, 85, 179, act)
    dy = Mat(300, 85, dt, data=rnd((300, 85), 55) + 3.0)
    _, z = t.fwd()
    g0 = t.bwd(dy, z)
    dy.v[7, 84] = float("nan")
    dx, dw, db = t.bwd(dy, z)
    assert only(g0[0], dx, [7], []) and only(g0[1], dw, [84], []) and only(g0[2], db, [], [84])
    dy.v[7, 84] = 1.0
    g0 = t.bwd(dy, z)
    z.v[7, 84] = float("nan")
    dx, dw, db = t.bwd(dy, z)
    if act in ("silu", "gelu"):
        assert only(g0[0], dx, [7], []) and only(g0[1], dw, [84], []) and only(g0[2], db, [], [84])
    else:       # slopes that are chosen by comparisons: a NaN is not above zero (0.1), nor inside (-3, 3) (0)
        assert all(bool(torch.isfinite(v).all()) for v in (dx, dw, db))


def test_relu_clears_nan():
    """The package's relu is u > 0 ? u : 0, in the new operators too: a NaN leaves as 0 (and has slope 0)."""
    t = Linear(1, 20, 8, 16, "relu")
    t.x.v[3] = float("nan")
    y, z = t.fwd()
    assert bool(torch.isnan(z.v[3]).all()) and bool((y.v[3] == 0).all())
    x = rnd((2 * 50, 16), 56)
    x[60, 3] = float("nan")
    d = GnDesc()
    d.dtype, d.N, d.HW, d.C, d.groups, d.act, d.eps, d.x_ld, d.o_ld, d.r_ld = F32, 2, 50, 16, 4, ACTS["relu"], 1e-5, 16, 16, 16
    nws = _lib.lib().plyolo_gn_workspace(C.byref(d))
    ws, st, out = torch.empty(nws, dtype=torch.uint8, device=DEV), torch.empty(2, 4, 2, device=DEV), torch.empty(100, 16, device=DEV)
    call("plyolo_gn_act_fwd", C.byref(d), x.data_ptr(), None, None, None, out.data_ptr(), st.data_ptr(), ws.data_ptr(), nws, hu.stream())
    assert bool(torch.isnan(st[1, 0, 1])) and bool((out[50:, :4] == 0).all()) and bool(torch.isfinite(out).all())


# ------------------------------------------------------------------------------------------------ the rounding of dz
@pytest.mark.parametrize("m,n,k", [(1, 300, 600), (2, 85, 179), (333, 85, 179), (12900, 264, 248), (11600, 520, 1288)])
def test_linear_backward_rounds_dz_once_and_nothing_else(m, n, k):
    """bf16: the products are those of dz rounded to bf16, with fp32 sums: dw in fp32 and db are within the sums' error of that form (db: of
    the unrounded dz), and dx within it before its own rounding.  What the products lose against an unrounded dz is that one rounding."""
    t = Linear(0, m, n, k, "silu")
    dy = Mat(m, n, 0, data=rnd((m, n), 57, scale=0.1))
    _, z = t.fwd()
    dx, dw, db = t.bwd(dy, z)
    u = z.v.double()
    s = 1.0 / (1.0 + torch.exp(-u))
    exact = dy.v.double() * (s * (1.0 + u * (1.0 - s)))
    # the kernel's dz before its rounding is off by 64 E32 |dy| (1 + |z|): a value that close to a border may round to its other side
    edge = 64 * E32 * dy.v.double().abs() * (1.0 + u.abs())
    dz = exact.to(torch.bfloat16).double()
    step = (exact + edge).to(torch.bfloat16).double() - (exact - edge).to(torch.bfloat16).double()
    w, x = t.w.v.double(), t.x.v.double()
    assert_close(dw, dz.t() @ x, step.t() @ x.abs() + (min(m, 4096) + 64) * E32 * (dz.abs().t() @ x.abs()) + 1e-30, "dw")
    want, tol = dz @ w, step @ w.abs() + (n + 4) * E32 * (dz.abs() @ w.abs())
    assert_close(dx, want, tol + UNIT[0] * (want.abs() + tol) + 1e-30, "dx")
    assert_close(db, exact.sum(0), edge.sum(0) + 1100 * E32 * exact.abs().sum(0) + 1e-30, "db")


# ------------------------------------------------------------------------------------------------ what a call returned stays what it was
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("make,c,hw", [(lambda: BaseConv(16, 32, 1, 1, bias=True, norm=None), 16, (1, 1)), (lambda: BaseConv(16, 1, 1, 1, bias=True, norm=None), 16, (3, 4)),
                                       (lambda: BaseConv(1, 8, 1, 1, bias=True, norm=None), 1, (3, 4)), (lambda: Dropout(0.5), 8, (1, 1)),
                                       (lambda: BaseConv(16, 32, 1, 1, norm="gn"), 16, (1, 1))])
def test_outputs_and_gradients_of_a_call_outlive_the_next(make, c, hw, dtype):
    """Maps of one pixel or one channel lie in memory alike channels first and last: what is returned must be a copy all the same."""
    m = make().to(DEV).train()
    m.compute_dtype = dtype
    held = []
    for i in range(3):
        x = rnd((4, c) + hw, 60 + i).requires_grad_(True)
        y = m(x)
        y.backward(rnd(tuple(y.shape), 70 + i))
        held.append((y.detach(), y.detach().clone(), x.grad, x.grad.clone()))
    m.eval()
    with torch.no_grad():
        for i in range(2):
            y = m(rnd((4, c) + hw, 80 + i))
            held.append((y, y.clone(), y, y))
    for y, y_then, dx, dx_then in held:
        assert torch.equal(y, y_then) and torch.equal(dx, dx_then)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_maps_of_one_pixel_outlive_the_next_call(dtype):
    with open(os.path.join(ROOT, "configs", "model", "yolox", "yolox_test.yaml")) as f:
        m = pl_yolo_amd.build_model(yaml.safe_load(f), 3).to(DEV).eval()
    m.compute_dtype = dtype
    with torch.no_grad():
        maps = m(rnd((2, 3, 32, 32), 90, scale=50.0))
        then = [t.clone() for t in maps]
        feats = [rnd((2, 32, 4, 4), 91), rnd((2, 64, 2, 2), 92), rnd((2, 128, 1, 1), 93)]
        own = m.head(feats)
        own_then = [t.clone() for t in own]
        m(rnd((2, 3, 32, 32), 94, scale=50.0))
        m.head([2.0 * t for t in feats])
    assert tuple(maps[2].shape[2:]) == (1, 1)
    assert all(torch.equal(a, b) for a, b in zip(maps + own, then + own_then))


def test_map_gradients_of_one_pixel_outlive_the_next_loss():
    with open(os.path.join(ROOT, "configs", "model", "yolox", "yolox_test.yaml")) as f:
        loss = pl_yolo_amd.build_model(yaml.safe_load(f), 3).to(DEV).train().loss
    labels = torch.zeros(2, 3, 5, device=DEV)
    labels[:, 0] = torch.tensor([1.0, 16.0, 16.0, 12.0, 10.0], device=DEV)

    def grads(seed):
        maps = [1.0 * rnd((2, 8, n, n), seed + n).requires_grad_(True) for n in (4, 2, 1)]
        return torch.autograd.grad(loss(list(maps), labels)["loss"], maps)
    first = grads(95)
    then = [g.clone() for g in first]
    second = grads(105)
    assert all(torch.equal(a, b) for a, b in zip(first, then)) and not torch.equal(first[2], second[2])


# ------------------------------------------------------------------------------------------------ beside BatchNorm units
class Mixed(HipModule):
    """A BatchNorm unit whose output is read by a linear unit (with it as the shortcut), a group-norm unit and a second BatchNorm unit, their
    sum behind dropout read by a third: every kind of unit is the last to write some BatchNorm unit's gradient."""

    def __init__(self, order):
        super().__init__()
        self.a, self.e = BaseConv(16, 32, 3, 1), BaseConv(32, 16, 3, 1)
        self.lin, self.gn, self.c = BaseConv(32, 32, 1, 1, bias=True, norm=None), BaseConv(32, 32, 3, 1, norm="gn"), BaseConv(32, 32, 1, 1)
        self.drop, self.order = Dropout(0.25), order

    def emit(self, g, x):
        t = self.a.emit(g, x)
        out = {}
        for k in self.order:
            out[k] = {"lin": lambda: self.lin.emit(g, t, residual=t), "gn": lambda: self.gn.emit(g, t), "c": lambda: self.c.emit(g, t)}[k]()
        return self.e.emit(g, self.drop.emit(g, self.drop.emit(g, out["lin"], residual=out["gn"]), residual=out["c"]))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("order", [("lin", "gn", "c"), ("c", "lin", "gn"), ("gn", "c", "lin")])
def test_units_beside_batch_norm_units(order, dtype):
    torch.manual_seed(47)
    m = Mixed(order).to(DEV).train()
    m.compute_dtype = dtype
    n, h, w = 4, 24, 20
    x, r = rnd((n, 16, h, w), 48, dtype), rnd((n, 16, h, w), 49, dtype)
    p = {k: (hu.rnd_bf16(v) if dtype == "bf16" and k.endswith("conv.weight") else v).detach().double().clone().requires_grad_(True) for k, v in m.named_parameters()}
    seed = dropout_state(m).tolist()[0]
    keep = [torch.from_numpy(keep_mask(seed, 0, s, n * h * w, 32, 0.25)).to(DEV).view(n, h, w, 32).permute(0, 3, 1, 2) / 0.75 for s in (0, 1)]

    def bn(t, k):
        z = F.conv2d(t, p[k + ".conv.weight"], None, 1, p[k + ".conv.weight"].shape[-1] // 2)
        return act64(F.batch_norm(z, None, None, p[k + ".norm.weight"], p[k + ".norm.bias"], True, 0.0, 1e-3), "silu")
    x64 = x.double().requires_grad_(True)
    t = bn(x64, "a")
    lin = act64(F.conv2d(t, p["lin.conv.weight"], p["lin.conv.bias"]), "silu") + t
    gn = act64(F.group_norm(F.conv2d(t, p["gn.conv.weight"], None, 1, 1), 32, p["gn.norm.weight"], p["gn.norm.bias"], 1e-5), "silu")
    y = bn(keep[1] * (keep[0] * lin + gn) + bn(t, "c"), "e")
    (y * r.double()).sum().backward()
    xi = x.clone().requires_grad_(True)
    got = m(xi)
    (got * r).sum().backward()
    # the bounds of the single units (test_gpu_batchfree_modules.TOL), of the largest value: a lost or doubled contribution is of its order
    f, b = ((2e-2, 6e-2), (2e-5, 5e-4))[TYPES[dtype]]
    assert hu.relerr(got, y) <= 2 * f and hu.relerr(xi.grad, x64.grad) <= b
    for k, v in m.named_parameters():
        e = hu.relerr(v.grad, p[k].grad)
        print(k, e)
        assert e <= b, k


def test_a_group_norm_detector_without_buffers_trains():
    """No BatchNorm, no buffers at all: trainer, EMA and a schedule of dropout probabilities, which leaves one training session behind."""
    from pl_yolo_amd.trainer import Trainer
    m = gn_detector("yolox/yolox_test.yaml", "bf16")
    assert not list(m.buffers())
    imgs, labels = odet.synthetic_batch(2, 64, 3, num_gt=3, max_gt=8, seed=5)
    imgs, labels = imgs.to(DEV), labels.to(DEV)
    tr = Trainer(m, learning_rate=0.005, total_steps=100, ema=True)
    before = m.head.stems[0].norm.weight.detach().clone()
    state = dropout_state(m)
    unit = m.backbone.stage4[2].conv3
    for i in range(4):
        unit.drop = 0.1 * (i + 1)
        assert math.isfinite(float(tr.train_step(imgs, labels)["loss"].detach()))
    assert not torch.equal(before, m.head.stems[0].norm.weight.detach()) and state.tolist()[1] == 4
    assert [k[4] for k in m.runner().sessions] == ["train"]
    m.eval()
    with torch.no_grad():
        assert bool(torch.isfinite(m(imgs, labels)).all())
    assert sorted(k[4] for k in m.runner().sessions) == ["eval", "train"]
