"""-m gpu: the batch-free units where their documentation allows more than the shipped models ask for: any channel count, shortcuts on odd
rows, probabilities that change, several streams.

Tolerances: bf16 stored values are off by half a step, 2^-8 relative (UNIT); the linear unit rounds x and W on their way in (the references
here start from the rounded ones), z, dz and its outputs once each."""
import pytest
import torch

import hiputil as hu
from batchfree import E32, UNIT, act64, act_grad64, assert_close, keep_mask
from pl_yolo_amd.layers import BaseConv, Dropout, dropout_state

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
