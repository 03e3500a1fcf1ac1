"""Group norm, linear layer and dropout as modules, without a GPU: what a traced session records (nothing runs: plans are only recorded),
which calls are refused, and what a session is keyed by."""
import copy
import os

import pytest
import torch
import torch.nn as nn
import yaml

from conftest import ROOT
from pl_yolo_amd import graph as G
from pl_yolo_amd._lib import PlyoloError, call
from pl_yolo_amd.layers import BaseConv, Dropout, HipModule, get_normalization
from pl_yolo_amd.module_runner import ModuleRunner

CPU = torch.device("cpu")


def trace(module, shape, dtype="bf16", want_grad=True, runner=None):
    """The session of a training call of `module` on an input of this shape: both plans recorded, none run."""
    r = runner or ModuleRunner(module.train())
    return r.session([torch.empty(shape)], False, False, dtype, module.training, want_grad)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("make,cin,cout", [(lambda: BaseConv(179, 85, 1, 1, bias=True, norm=None, act="gelu"), 179, 85),
                                           (lambda: BaseConv(1, 3, 1, 1, bias=True, norm=None, drop=0.5), 1, 3),
                                           (lambda: Dropout(0.25), 85, 85)])
def test_any_channel_count_enters_a_linear_layer_and_a_dropout(make, cin, cout, dtype):
    s = trace(make(), (2, cin, 5, 3), dtype)
    assert [(a.C, a.ld) for a in s.ins] == [(cin, cin)] and [o.C for o in s.outs] == [cout]
    assert s.bwd is not None and all(s.ins[0].storage.ginit)


def test_convolutions_keep_their_channel_vectors():
    for m in (BaseConv(6, 16, 1, 1), BaseConv(6, 16, 3, 1, norm="gn")):
        with pytest.raises(PlyoloError, match="multiple of 8"):
            trace(m, (1, 6, 4, 4))


class Residual(HipModule):
    """x + unit(x)."""

    any_channels = True

    def __init__(self, unit):
        super().__init__()
        self.unit = unit

    def emit(self, g, x):
        return self.unit.emit(g, x, residual=x)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("make", [lambda: BaseConv(85, 85, 1, 1, bias=True, norm=None), lambda: Dropout(0.5),
                                  lambda: BaseConv(85, 85, 1, 1, bias=True, norm=None, drop=0.5)])
def test_a_shortcut_on_rows_of_any_channel_count_records_its_backward(make, dtype):
    s = trace(Residual(make()), (2, 85, 4, 3), dtype)
    assert s.bwd is not None and all(s.ins[0].storage.ginit)


def copy_add(dt=0, M=4, C=5, src=0x10000, i_ld=5, out=0x10000, o_ld=5):
    call("plyolo_copy_add", dt, M, C, src, i_ld, out, o_ld, 0, None)


@pytest.mark.parametrize("kw", [dict(M=0), dict(C=0), dict(i_ld=4), dict(o_ld=4), dict(out=None), dict(src=0x10001), dict(out=0x10001), dict(dt=5)])
def test_copy_add_refuses(kw):
    with pytest.raises(PlyoloError, match="copy_add"):
        copy_add(**kw)


# ------------------------------------------------------------------------------------------------ dropout probabilities
def dropout_ops(s):
    return [op for op in s.g.ops if isinstance(op, G.DropoutOp)]


def test_a_changed_dropout_probability_is_another_session():
    m = nn.Sequential()      # (only holds the units)
    m.a, m.d = BaseConv(16, 16, 1, 1, bias=True, norm=None, drop=0.5), Dropout(0.25)

    class Two(HipModule):
        def __init__(self):
            super().__init__()
            self.a, self.d = m.a, m.d

        def emit(self, g, x):
            return self.d.emit(g, self.a.emit(g, x))
    two = Two().train()
    r = ModuleRunner(two)
    first = trace(two, (1, 16, 4, 4), runner=r)
    assert [op.p for op in dropout_ops(first)] == [0.5, 0.25]
    assert trace(two, (1, 16, 4, 4), runner=r) is first
    two.d.p = 0.1
    second = trace(two, (1, 16, 4, 4), runner=r)
    assert second is not first and [op.p for op in dropout_ops(second)] == [0.5, 0.1]
    two.a.drop = 0.0
    assert [op.p for op in dropout_ops(trace(two, (1, 16, 4, 4), runner=r))] == [0.1]
    two.a.eval()             # as nn.Dropout: a unit in eval mode does not drop, whatever mode its parent is in
    two.a.drop = 0.5
    assert [op.p for op in dropout_ops(trace(two, (1, 16, 4, 4), runner=r))] == [0.1]
    two.train()
    two.d.p = 0.1
    last = trace(two, (1, 16, 4, 4), runner=r)
    two.eval()
    evals = trace(two, (1, 16, 4, 4), want_grad=False, runner=r)
    two.train()
    assert trace(two, (1, 16, 4, 4), runner=r) is last       # (a call in eval mode costs no training session)
    for i in range(1, 9):        # a schedule leaves one session behind, not one a value; those of eval mode stay
        two.d.p = i / 16
        last = trace(two, (1, 16, 4, 4), runner=r)
        assert [op.p for op in dropout_ops(last)] == [0.5, i / 16] and trace(two, (1, 16, 4, 4), runner=r) is last
    assert len(r.sessions) == 2
    two.eval()
    assert trace(two, (1, 16, 4, 4), want_grad=False, runner=r) is evals


def test_detector_sessions_go_by_their_dropout_probabilities():
    import pl_yolo_amd
    from pl_yolo_amd.runner import DetectorRunner
    with open(os.path.join(ROOT, "configs", "model", "yolox", "yolox_test.yaml")) as f:
        m = pl_yolo_amd.build_model(yaml.safe_load(f), 3).train()
    r = DetectorRunner(m)
    r.adopt(CPU)
    before = r.drop_key()
    assert not any(before)
    unit = m.backbone.stage4[2].conv3
    unit.drop = 0.25
    assert r.drop_key() != before
    unit.drop = 0.0
    assert r.drop_key() == before
    unit.drop = 0.25
    m.eval()
    assert not any(r.drop_key())       # nothing is dropped: one session whatever the probabilities


def test_probabilities_set_later_are_checked():
    m = Dropout(0.25).train()
    m.p = 1.5
    with pytest.raises(ValueError, match="between 0 and 1"):
        trace(m, (1, 16, 4, 4))
    u = BaseConv(16, 16, 1, 1, bias=True, norm=None).train()
    u.drop = float("nan")
    with pytest.raises(ValueError, match="between 0 and 1"):
        trace(u, (1, 16, 4, 4))


# ------------------------------------------------------------------------------------------------ where `norm: gn` reaches
def build(path, norm, **more):
    import pl_yolo_amd
    with open(os.path.join(ROOT, "configs", "model", path)) as f:
        cfg = yaml.safe_load(f)
    for part in ("backbone", "neck", "head"):
        cfg[part]["norm"] = norm
    return pl_yolo_amd.build_model(cfg, 3)


def kinds(m, kind):
    return sorted(n for n, k in m.named_modules() if isinstance(k, kind))


YOLOX_FIXED = ["backbone.stage4.1.conv2.norm"] + ["head.stems.%d.norm" % i for i in range(3)]
V7_FIXED = sorted(["backbone.stage%d.0.conv%d.norm" % (s, k) for s in (2, 3, 4) for k in (1, 2)] + ["backbone.stage4.1.conv2.norm"] +
                  ["neck.spp.cv%d.norm" % k for k in range(1, 8)] + ["neck.downsample_conv%d.conv%d.norm" % (d, k) for d in (1, 2) for k in (1, 2)])


@pytest.mark.parametrize("norm,kind", [("gn", nn.GroupNorm), ("ln", nn.LayerNorm)])
@pytest.mark.parametrize("path,fixed", [("yolox/yolox_test.yaml", YOLOX_FIXED), ("yolox/yolox_s.yaml", YOLOX_FIXED), ("yolov7/yolov7_test.yaml", V7_FIXED),
                                        ("yolov7/yolov7.yaml", V7_FIXED)])
def test_norm_reaches_what_the_reference_forwards_it_to(path, fixed, norm, kind):
    """These and no other units keep their BatchNorm whatever `norm` is, as the reference's blocks have it: SPP's second conv and the head's
    stems (network_blocks.py:149, decoupled_head.py:29-31), the 1x1 units of the transitions and the SPP-CSP block (eelan.py:130-131,
    yolov7_neck.py:153-154, network_blocks.py:158-175)."""
    m = build(path, norm)
    assert kinds(m, nn.BatchNorm2d) == fixed
    assert sorted(fixed + kinds(m, kind)) == kinds(build(path, "bn"), nn.BatchNorm2d) and len(kinds(m, kind)) > 30


@pytest.mark.parametrize("path", ["yolox/yolox_test.yaml", "yolov7/yolov7_test.yaml"])
def test_group_norm_in_the_remaining_units(path):
    """The documented way to a network without batch statistics."""
    m = build(path, "gn")
    for u in m.modules():
        if isinstance(u, BaseConv) and isinstance(u.norm, nn.BatchNorm2d):
            u.norm = get_normalization("gn", u.conv.out_channels)
    assert kinds(m, nn.BatchNorm2d) == [] and not list(m.buffers())


def test_repconv_keeps_its_batch_norms():
    from pl_yolo_amd.necks import YOLOv7NECK, RepConv
    m = YOLOv7NECK((1, 1, 1, 1), (32, 64, 64), norm="gn", repconv=True)
    inside = sorted(n for n in kinds(m, nn.BatchNorm2d) if n.split(".")[0] in ("n3", "n4", "n5"))
    assert len(kinds(m, RepConv)) == 3 and inside == sorted(n for k in ("n3", "n4", "n5") for n in
                                                            (k + "." + q for q in kinds(getattr(m, k), nn.BatchNorm2d))) and len(inside) >= 6


# ------------------------------------------------------------------------------------------------ one unit used twice
class Twice(HipModule):
    def __init__(self, a, b):
        super().__init__()
        self.a, self.b = a, b

    def emit(self, g, x):
        return self.b.emit(g, self.a.emit(g, x))


def test_a_group_norm_unit_used_twice_is_refused_in_training():
    """A convolution's weight gradient has one place, which the second use would overwrite."""
    a, b = BaseConv(16, 16, 3, 1, norm="gn"), BaseConv(16, 16, 3, 1, norm="gn")
    assert trace(Twice(a, b), (1, 16, 6, 6)).bwd is not None
    for other in (a, b):
        if other is b:
            b.norm = a.norm                         # the affine pair alone
        with pytest.raises(PlyoloError, match="used twice"):
            trace(Twice(a, other), (1, 16, 6, 6))
        assert trace(Twice(a, other), (1, 16, 6, 6), want_grad=False).bwd is None
    for p in a.parameters():
        p.requires_grad_(False)                     # nothing to overwrite
    assert trace(Twice(a, a), (1, 16, 6, 6)).bwd is not None


def test_a_linear_layer_sharing_its_weights_with_a_convolution_is_refused_in_training():
    a, b = BaseConv(16, 16, 1, 1, bias=True, norm=None), BaseConv(16, 16, 1, 1)
    b.conv.weight = a.conv.weight
    with pytest.raises(PlyoloError, match="used twice"):
        trace(Twice(a, b), (1, 16, 6, 6))


# ------------------------------------------------------------------------------------------------ the dropouts' state
def test_every_rank_draws_its_own_seed(monkeypatch):
    dist, seeds = torch.distributed, []
    for rank in (None, 0, 1, 2, 7):
        torch.manual_seed(9)
        if rank is not None:
            monkeypatch.setattr(dist, "is_initialized", lambda: True)
            monkeypatch.setattr(dist, "get_rank", lambda: rank)
        seed, step = G.rng_state_of(Dropout(0.5), CPU).tolist()
        assert step == 0 and 0 <= seed < 1 << 62
        seeds.append(seed)
    assert seeds[0] == seeds[1] and len(set(seeds[1:])) == 4          # rank 0 draws what a single process draws


def test_a_copy_of_a_module_has_a_state_of_its_own():
    m = BaseConv(16, 16, 1, 1, bias=True, norm=None, drop=0.5).train()
    a = G.rng_state_of(m, CPU)
    r = m.__dict__["_mrunner"] = ModuleRunner(m)
    trace(m, (1, 16, 4, 4), runner=r)
    c = copy.deepcopy(m)
    b = G.rng_state_of(c, CPU)
    assert b is not a and b.data_ptr() != a.data_ptr() and b.tolist() == a.tolist()
    assert c.__dict__.get("_mrunner") is None and c.drop == 0.5
    b[1] = 5
    assert a.tolist()[1] == 0 and G.rng_state_of(m, CPU) is a
