"""-m gpu: group norm, linear layer and dropout where a model meets them: BaseConv(norm="gn"), BaseConv(1x1, bias=True, norm=None),
BaseConv(drop=p), layers.Dropout, and a whole detector with `norm: gn`."""
import copy
import math
import os

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F
import yaml

import hiputil as hu
import pl_yolo_amd
from batchfree import E32, UNIT, act64, assert_close, keep_mask
from conftest import ROOT
from oracle import detector as odet, net as onet
from pl_yolo_amd._lib import PlyoloError
from pl_yolo_amd.layers import BaseConv, Bottleneck, CSPLayer, Dropout, dropout_state

pytestmark = pytest.mark.gpu
DEV = hu.DEV
# relative to the largest value of a tensor; bf16: a handful of roundings of 2^-8 (z, activations, dz) with cancellation in the normalisation,
# as for the width LayerNorm unit; fp32: sums of a few thousand terms
TOL = {"bf16": (2e-2, 6e-2), "fp32": (2e-5, 5e-4)}


def close(got, want, tol, what):
    e = hu.relerr(got, want)
    print("%s %.3g" % (what, e))
    assert e <= tol, (what, e)


def rnd(shape, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV)


def weights(m, dtype):
    return {n: (hu.rnd_bf16(p) if dtype == "bf16" and n.endswith("conv.weight") else p).detach().double().clone().requires_grad_(True) for n, p in m.named_parameters()}


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("act", ["silu", "hswish", None])
@pytest.mark.parametrize("k,s,cin,cout,hw", [(3, 1, 16, 40, (13, 9)), (1, 1, 24, 96, (8, 8)), (3, 2, 32, 64, (14, 10))])
def test_baseconv_group_norm(k, s, cin, cout, hw, act, dtype):
    torch.manual_seed(3)
    m = BaseConv(cin, cout, k, s, norm="gn", act=act).to(DEV).train()
    m.compute_dtype = dtype
    assert isinstance(m.norm, nn.GroupNorm) and m.norm.num_groups == math.gcd(32, cout)
    with torch.no_grad():
        m.norm.weight.uniform_(0.5, 1.5)
        m.norm.bias.uniform_(-0.5, 0.5)
    x = rnd((3, cin) + hw, 5)
    x = hu.rnd_bf16(x) if dtype == "bf16" else x
    r = rnd((3, cout, (hw[0] - 1) // s + 1, (hw[1] - 1) // s + 1), 6)
    w = weights(m, dtype)
    xr = x.double().requires_grad_(True)
    z = F.conv2d(xr, w["conv.weight"], None, s, k // 2)
    if dtype == "bf16":
        # The unit stores z in bf16 and normalises what it stored.  hswish' jumps by 0.5 at u = -3 and 3: a z whose rounding (2^-8 |z|, |u| up
        # to 3 near the jumps: 0.012) carries u across one has half its dout on the other side, which no bound on smooth functions covers.
        # The reference therefore rounds z too (with the identity as the gradient of the rounding, as the unit has it)
        z = z + (hu.rnd_bf16(z.float()).double() - z).detach()
    u = F.group_norm(z, m.norm.num_groups, w["norm.weight"], w["norm.bias"], m.norm.eps)
    y = act64(u, act or "none")
    (y * r.double()).sum().backward()
    xi = x.clone().requires_grad_(True)
    got = m(xi)
    (got * r).sum().backward()
    f, b = TOL[dtype]
    close(got, y, f, "y")
    close(xi.grad, xr.grad, b, "dx")
    for n, p in m.named_parameters():
        close(p.grad, w[n].grad, b, n)
    m.eval()
    with torch.no_grad():
        assert torch.equal(m(x), got)          # the same in inference


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_bottleneck_and_csp_layer_group_norm(dtype):
    """The shortcut is added by the group norm's launch; a CSP layer's same-input pair stays two units."""
    torch.manual_seed(4)
    for m in (Bottleneck(32, 32, True, 1.0, norm="gn"), CSPLayer(32, 64, 1, norm="gn")):
        m = m.to(DEV).train()
        m.compute_dtype = dtype
        x = rnd((2, 32, 12, 12), 7)
        x = hu.rnd_bf16(x) if dtype == "bf16" else x
        w = weights(m, dtype)

        def unit(name, t, k):
            u = F.conv2d(t, w[name + ".conv.weight"], None, 1, k // 2)
            return act64(F.group_norm(u, math.gcd(32, u.shape[1]), w[name + ".norm.weight"], w[name + ".norm.bias"], 1e-5), "silu")

        def bottleneck(t, pre):
            return unit(pre + "conv2", unit(pre + "conv1", t, 1), 3) + t
        xr = x.double().requires_grad_(True)
        if isinstance(m, Bottleneck):
            y = bottleneck(xr, "")
        else:
            y = unit("conv3", torch.cat([bottleneck(unit("conv1", xr, 1), "m.0."), unit("conv2", xr, 1)], 1), 1)
        r = rnd(tuple(y.shape), 8)
        (y * r.double()).sum().backward()
        xi = x.clone().requires_grad_(True)
        got = m(xi)
        (got * r).sum().backward()
        f, b = TOL[dtype]
        close(got, y, f, "y")
        close(xi.grad, xr.grad, b, "dx")
        dead = {id(p) for q in m.modules() if hasattr(q, "dead_parameters") for p in q.dead_parameters()}
        for n, p in m.named_parameters():
            if id(p) not in dead:
                close(p.grad, w[n].grad, b, n)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", None])
@pytest.mark.parametrize("cin,cout,hw,n", [(24, 85, (7, 5), 3), (64, 64, (10, 10), 2), (128, 32, (1, 1), 4)])
def test_baseconv_linear(cin, cout, hw, n, act, dtype):
    torch.manual_seed(5)
    m = BaseConv(cin, cout, 1, 1, bias=True, norm=None, act=act).to(DEV).train()
    m.compute_dtype = dtype
    x = rnd((n, cin) + hw, 9)
    x = hu.rnd_bf16(x) if dtype == "bf16" else x
    w = weights(m, dtype)
    xr = x.double().requires_grad_(True)
    y = act64(F.conv2d(xr, w["conv.weight"], w["conv.bias"]), act or "none")
    r = rnd(tuple(y.shape), 10)
    (y * r.double()).sum().backward()
    xi = x.clone().requires_grad_(True)
    got = m(xi)
    (got * r).sum().backward()
    f, b = (1e-2, 2e-2) if dtype == "bf16" else (2e-5, 5e-5)
    if act == "relu" and dtype == "bf16":
        b = 4e-2        # a pre-activation that rounds to the other side of 0 switches its whole gradient
    close(got, y, f, "y")
    close(xi.grad, xr.grad, b, "dx")
    for name, p in m.named_parameters():
        close(p.grad, w[name].grad, b, name)
    # another step with changed weights: the cast copy follows the masters
    with torch.no_grad():
        m.conv.weight.mul_(-0.5)
        m.conv.bias.add_(1.0)
    y2 = act64(F.conv2d(x.double(), (hu.rnd_bf16(m.conv.weight) if dtype == "bf16" else m.conv.weight).double(), m.conv.bias.double()), act or "none")
    close(m(x), y2, f, "y after an update")
    m.eval()
    with torch.no_grad():
        close(m(x), y2, f, "y in eval mode")


def test_frozen_linear_and_group_norm_parameters():
    torch.manual_seed(6)
    m = nn.ModuleList([BaseConv(16, 16, 1, 1, bias=True, norm=None), BaseConv(16, 16, 3, 1, norm="gn")]).to(DEV).train()
    x = rnd((2, 16, 6, 6), 11).requires_grad_(True)
    for p in (m[0].conv.weight, m[0].conv.bias, m[1].norm.weight, m[1].norm.bias):
        p.requires_grad_(False)
    m[1](m[0](x)).sum().backward()
    assert x.grad is not None and float(x.grad.abs().sum()) > 0 and m[1].conv.weight.grad is not None
    assert all(p.grad is None for p in (m[0].conv.weight, m[0].conv.bias, m[1].norm.weight, m[1].norm.bias))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_dropout_module(dtype):
    torch.manual_seed(7)
    m = Dropout(0.3).train()
    m.compute_dtype = dtype
    x = rnd((2, 24, 5, 7), 12).requires_grad_(True)
    state = dropout_state(m)
    seed, step = state.tolist()
    assert step == 0 and dropout_state(m) is state
    r = rnd((2, 24, 5, 7), 13)
    xr = (hu.rnd_bf16(x.detach()) if dtype == "bf16" else x.detach())
    rr = (hu.rnd_bf16(r) if dtype == "bf16" else r)
    masks = []
    for i in range(3):
        y = m(x)
        (dx,) = torch.autograd.grad((y * r).sum(), x)
        assert state.tolist() == [seed, i + 1]
        keep = torch.from_numpy(keep_mask(seed, i, 0, 70, 24, 0.3)).to(DEV).view(2, 5, 7, 24).permute(0, 3, 1, 2)
        masks.append(keep)
        u = UNIT[0 if dtype == "bf16" else 1]
        for got, src, what in ((y, xr, "y"), (dx, rr, "dx")):
            want = torch.where(keep, src.double() / 0.7, torch.zeros((), dtype=torch.float64, device=DEV))
            assert_close(got, want, (8 * E32 + u) * want.abs(), what)
    assert not torch.equal(masks[0], masks[1])
    # a saved state brings its masks back
    state.copy_(torch.tensor([seed, 1], device=DEV))
    assert torch.equal(m(x) != 0, masks[1] & (xr != 0))
    m.eval()
    with torch.no_grad():
        assert torch.equal(m(x), xr.float())
    assert state.tolist() == [seed, 2]
    # seeds repeat under manual_seed and differ between modules
    torch.manual_seed(7)
    assert dropout_state(Dropout(0.3)).tolist()[0] == seed and dropout_state(Dropout(0.3)).tolist()[0] != seed


class TwoDrops(pl_yolo_amd.layers.HipModule):
    def __init__(self):
        super().__init__()
        self.a = BaseConv(16, 32, 1, 1, bias=True, norm=None, act="silu", drop=0.5)
        self.b = BaseConv(32, 16, 1, 1, bias=True, norm=None, act=None, drop=0.25)

    def emit(self, g, x):
        return self.b.emit(g, self.a.emit(g, x), residual=x)


def test_dropout_inside_units_with_a_shortcut():
    """x + dropout(W2 dropout(silu(W1 x + b1)) + b2): two dropouts of one network have masks of their own (their places), fp32 against
    automatic differentiation with the masks of the definition; in eval mode neither acts."""
    torch.manual_seed(8)
    m = TwoDrops().to(DEV).train()
    m.compute_dtype = "fp32"
    x = rnd((2, 16, 9, 4), 14)
    w = weights(m, "fp32")
    seed = dropout_state(m).tolist()[0]
    r = rnd((2, 16, 9, 4), 15)

    def ref(xr, train):
        rows = xr.permute(0, 2, 3, 1).reshape(72, 16)
        h = act64(rows @ w["a.conv.weight"].view(32, 16).t() + w["a.conv.bias"], "silu")
        if train:
            h = h * torch.from_numpy(keep_mask(seed, 0, 0, 72, 32, 0.5)).to(DEV) * 2.0
        u = h @ w["b.conv.weight"].view(16, 32).t() + w["b.conv.bias"]
        if train:
            u = u * torch.from_numpy(keep_mask(seed, 0, 1, 72, 16, 0.25)).to(DEV) / 0.75
        return (rows + u).view(2, 9, 4, 16).permute(0, 3, 1, 2)
    xr = x.double().requires_grad_(True)
    y = ref(xr, True)
    (y * r.double()).sum().backward()
    xi = x.clone().requires_grad_(True)
    got = m(xi)
    (got * r).sum().backward()
    close(got, y, 2e-6, "y")
    close(xi.grad, xr.grad, 2e-6, "dx")
    for n, p in m.named_parameters():
        close(p.grad, w[n].grad, 1e-5, n)
    m.eval()
    with torch.no_grad():
        close(m(x), ref(x.double(), False), 2e-6, "eval")


# ------------------------------------------------------------------------------------------------ a whole detector
def gn_config():
    with open(os.path.join(ROOT, "configs", "model", "yolox", "yolox_test.yaml")) as f:
        cfg = yaml.safe_load(f)
    for k in ("backbone", "neck", "head"):
        cfg[k]["norm"] = "gn"
    return cfg


def patch_oracle(monkeypatch):
    """The oracle's conv unit with group norm wherever the state carries no running statistics."""
    bn_unit = onet.conv_unit

    def unit(state, prefix, x, stride, training, norm="bn", act="silu", residual=None, groups=1):
        if prefix + ".norm.running_mean" in state:
            return bn_unit(state, prefix, x, stride, training, norm, act, residual, groups)
        w = state[prefix + ".conv.weight"]
        z = onet._q(F.conv2d(x, onet._qw(w), None, stride, w.shape[-1] // 2))      # (_q, _qw: the bf16 pipeline's stores, inside emulate_bf16)
        u = F.group_norm(z, math.gcd(32, w.shape[0]), state[prefix + ".norm.weight"], state[prefix + ".norm.bias"], 1e-5)
        u = onet.activation(u, act)
        return onet._q(u + residual if residual is not None else u)
    monkeypatch.setattr(onet, "conv_unit", unit)


def test_detector_with_group_norm_against_the_oracle(monkeypatch):
    patch_oracle(monkeypatch)
    cfg, nc = gn_config(), 3
    torch.manual_seed(96)
    model = pl_yolo_amd.build_model(cfg, nc)
    state = {k: v.clone() for k, v in model.state_dict().items()}
    imgs, labels = odet.synthetic_batch(2, 64, nc, num_gt=3, max_gt=8, seed=1234)
    ref, ref_grads = odet.train_step_grads({k: v.clone() for k, v in state.items()}, cfg, nc, imgs, labels)
    m = pl_yolo_amd.build_model(cfg, nc)
    m.load_state_dict(state)
    m.compute_dtype = "fp32"
    m = m.to(DEV).train()
    out = m(imgs.to(DEV), labels.to(DEV))
    out["loss"].backward()
    got, want = float(out["loss"].detach()), float(ref["loss"].detach())
    assert abs(got - want) <= 1e-4 * abs(want), (got, want)
    named = dict(m.named_parameters())
    worst = 0.0
    for n, g in ref_grads.items():
        e = hu.relerr(named[n].grad.cpu(), g)
        worst = max(worst, e)
        assert e <= 2e-3, (n, e)
    print("loss %.7g (oracle %.7g), worst gradient %.3g" % (got, want, worst))
    # fuse() leaves group norms alone: only the SPP unit's BatchNorm folds
    m.eval()
    with torch.no_grad():
        e32 = m(imgs.to(DEV), labels.to(DEV)).clone()
        close(m.fuse()(imgs.to(DEV), labels.to(DEV)), e32, 1e-4, "fused")


def test_detector_with_group_norm_in_bf16(monkeypatch):
    """The bf16 training loss against the oracle with the same stores rounded, and a gradient for every live parameter.  (No gradients
    against another arithmetic here: on an untrained toy network the deepest maps normalise 2 x 2 pixels, single channels in the narrow
    layers, and every rounding that differs is divided by a spread near zero.  The units' bf16 gradients are pinned above.)"""
    patch_oracle(monkeypatch)
    cfg, nc = gn_config(), 3
    torch.manual_seed(96)
    model = pl_yolo_amd.build_model(cfg, nc)
    state = {k: v.clone() for k, v in model.state_dict().items()}
    imgs, labels = odet.synthetic_batch(2, 64, nc, num_gt=3, max_gt=8, seed=1234)
    b = pl_yolo_amd.build_model(cfg, nc)
    b.load_state_dict(state)
    b.compute_dtype = "bf16"
    b = b.to(DEV).train()
    with onet.emulate_bf16():
        ref, ref_grads = odet.train_step_grads({k: v.clone() for k, v in state.items()}, cfg, nc, imgs, labels)
    out = b(imgs.to(DEV), labels.to(DEV))
    out["loss"].backward()
    got, want = float(out["loss"].detach()), float(ref["loss"].detach())
    print("loss %.6g (emulating oracle %.6g)" % (got, want))
    assert abs(got - want) <= 1e-2 * abs(want), (got, want)
    named = dict(b.named_parameters())
    assert len(ref_grads) > 100 and all(bool(torch.isfinite(named[n].grad).all()) for n in ref_grads)


def test_detector_with_group_norm_lanes_and_repeats(monkeypatch):
    """bf16 training steps: the multi-stream replay equals the single-stream one bit for bit, and a step repeats."""
    cfg, nc = gn_config(), 3
    imgs, labels = odet.synthetic_batch(2, 96, nc, num_gt=3, max_gt=8, seed=77)
    grads = []
    for lanes in ("1", "0", "1"):
        monkeypatch.setenv("PLYOLO_LANES", lanes)
        torch.manual_seed(96)
        m = pl_yolo_amd.build_model(cfg, nc).to(DEV).train()
        m.compute_dtype = "bf16"
        for _ in range(2):
            m.zero_grad(set_to_none=True)
            m(imgs.to(DEV), labels.to(DEV))["loss"].backward()
        grads.append({n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None})
    assert set(grads[0]) == set(grads[1])
    norms = [n for n in grads[0] if n.endswith("norm.weight")]
    assert len(norms) > 30
    for n in grads[0]:
        a, b, c = (hu.cossim(grads[0][n], grads[i][n]) for i in (0, 1, 2))
        # (the SPP unit keeps BatchNorm, whose statistics are summed by atomics: its neighbours repeat to rounding, not to the bit)
        assert min(b, c) > 0.999, (n, b, c)


def test_detector_with_group_norm_trains():
    from pl_yolo_amd.trainer import Trainer
    cfg, nc = gn_config(), 3
    torch.manual_seed(96)
    m = pl_yolo_amd.build_model(cfg, nc).to(DEV)
    m.compute_dtype = "bf16"
    imgs, labels = odet.synthetic_batch(2, 64, nc, num_gt=3, max_gt=8, seed=5)
    tr = Trainer(m, learning_rate=0.005, total_steps=100, ema=True)
    before = m.backbone.stem.conv.norm.weight.detach().clone()
    for _ in range(3):
        loss = float(tr.train_step(imgs.to(DEV), labels.to(DEV))["loss"].detach())
        assert math.isfinite(loss)
    assert not torch.equal(before, m.backbone.stem.conv.norm.weight.detach())
    assert copy.deepcopy(m) is not m


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_yolov7_with_group_norm(dtype):
    """The other family: every BaseConv takes it, the RepConv blocks keep the BatchNorms their class builds; all parameters get gradients."""
    with open(os.path.join(ROOT, "configs", "model", "yolov7", "yolov7_test.yaml")) as f:
        cfg = yaml.safe_load(f)
    for part in ("backbone", "neck", "head"):
        cfg[part]["norm"] = "gn"
    torch.manual_seed(1)
    m = pl_yolo_amd.build_model(cfg, 3).to(DEV).train()
    m.compute_dtype = dtype
    assert any(isinstance(k, nn.GroupNorm) for k in m.modules())
    imgs, labels = odet.synthetic_batch(2, 64, 3, num_gt=3, max_gt=8, seed=5)
    m(imgs.to(DEV), labels.to(DEV))["loss"].sum().backward()
    for n, p in m.named_parameters():
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()) and float(p.grad.abs().max()) > 0, n


def test_linear_in_a_model_counts_its_operations():
    from pl_yolo_amd import graph as G, utils
    from pl_yolo_amd._lib import BF16
    g = G.Graph(BF16, False, torch.device("cpu"))
    x = g.new_act(1, 8, 8, 32)
    BaseConv(32, 48, 1, 1, bias=True, norm=None).emit(g, x)
    assert [op.macs for op in g.ops if isinstance(op, G.LinearOp)] == [64 * 32 * 48]


def test_refused_compositions():
    with pytest.raises(NotImplementedError):
        BaseConv(8, 8, 3, 1, bias=True, norm=None)
    with pytest.raises(NotImplementedError):
        BaseConv(8, 8, 1, 1, bias=True, norm="gn")
    with pytest.raises(ValueError):
        BaseConv(8, 8, 1, 1, drop=1.5)
    with pytest.raises(ValueError):
        Dropout(-0.1)
    m = BaseConv(16, 16, 3, 1, groups=16, norm="gn").to(DEV).train()
    with pytest.raises(NotImplementedError, match="depthwise"):
        m(torch.zeros(1, 16, 4, 4, device=DEV))
    with pytest.raises(PlyoloError):
        Dropout(0.5)(torch.zeros(1, 8, 4, 4))
