"""Group norm, linear layer and dropout as modules, without a GPU: what a traced session records (nothing runs: plans are only recorded),
which calls are refused, and what a session is keyed by."""
import pytest
import torch

from pl_yolo_amd.layers import BaseConv, Dropout
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
    from pl_yolo_amd._lib import PlyoloError
    for m in (BaseConv(6, 16, 1, 1), BaseConv(6, 16, 3, 1, norm="gn")):
        with pytest.raises(PlyoloError, match="multiple of 8"):
            trace(m, (1, 6, 4, 4))
