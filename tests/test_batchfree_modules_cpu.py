"""Group norm, linear layer and dropout as modules, without a GPU: what a traced session records (nothing runs: plans are only recorded),
which calls are refused, and what a session is keyed by."""
import os

import pytest
import torch
import torch.nn as nn
import yaml

from conftest import ROOT
from pl_yolo_amd import graph as G
from pl_yolo_amd._lib import PlyoloError, call
from pl_yolo_amd.layers import BaseConv, Dropout, HipModule
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
    two.eval()
    evals = trace(two, (1, 16, 4, 4), want_grad=False, runner=r)
    two.train()
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
