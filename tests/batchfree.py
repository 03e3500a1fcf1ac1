"""Shared by the tests of the batch-free operators (group norm + activation, linear layer, counter-based dropout): their definitions in
64 bits and row matrices with a pitch, an odd start and guarded surroundings."""
import math

import numpy as np
import torch

ACTS = {"none": 0, "silu": 1, "relu": 2, "lrelu": 3, "hswish": 4, "gelu": 5}
TD = {0: torch.bfloat16, 1: torch.float32}
UNIT = {0: 2.0 ** -8, 1: 2.0 ** -24}      # half a step of the stored type, relative
E32 = 2.0 ** -24                          # half a step of the arithmetic, relative
GUARD = 77.0


class Mat:
    """[m, c] rows at pitch c + pad, starting `off` elements behind a 16-byte boundary, in a buffer that is GUARD everywhere else."""

    def __init__(self, m, c, dt, pad=0, off=0, data=None, device="cuda:0"):
        self.m, self.c, self.ld, self.off = m, c, c + pad, off
        self.buf = torch.full((off + m * self.ld + 64,), GUARD, dtype=TD[dt], device=device)
        self.v = self.buf[off:off + m * self.ld].view(m, self.ld)[:, :c]
        if data is not None:
            self.v.copy_(data)
        self.ptr = self.buf.data_ptr() + off * self.buf.element_size()

    def untouched(self):
        """Nothing outside the rows' c columns was written."""
        b = self.buf.clone()
        b[self.off:self.off + self.m * self.ld].view(self.m, self.ld)[:, :self.c] = GUARD
        return bool((b == GUARD).all())


def act64(u, name):
    if name == "silu":
        return u / (1.0 + torch.exp(-u))
    if name == "relu":
        return u.clamp(min=0.0)
    if name == "lrelu":
        return torch.where(u > 0, u, 0.1 * u)
    if name == "hswish":
        return u * (u + 3.0).clamp(0.0, 6.0) / 6.0
    if name == "gelu":
        return 0.5 * u * (1.0 + torch.erf(u * math.sqrt(0.5)))
    return u


def act_grad64(u, name):
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-u))
        return s * (1.0 + u * (1.0 - s))
    if name == "relu":
        return (u > 0).double()
    if name == "lrelu":
        return torch.where(u > 0, 1.0, 0.1).double()
    if name == "hswish":
        return ((u + 3.0).clamp(0.0, 6.0) + u * ((u > -3) & (u < 3)).double()) / 6.0
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(u * math.sqrt(0.5))) + u * torch.exp(-0.5 * u * u) / math.sqrt(2.0 * math.pi)
    return torch.ones_like(u)


def gn64(x, n, hw, groups, gamma, beta, eps):
    """(xh, u, mean, rstd) of rows x [n*hw, c], all in 64 bits."""
    c = x.shape[1]
    t = x.double().view(n, hw, groups, c // groups)
    mu = t.mean(dim=(1, 3), keepdim=True)
    rs = 1.0 / torch.sqrt(((t - mu) ** 2).mean(dim=(1, 3), keepdim=True) + eps)
    xh = ((t - mu) * rs).reshape(n * hw, c)
    ga = gamma.double() if gamma is not None else torch.ones(c, dtype=torch.float64, device=x.device)
    be = beta.double() if beta is not None else torch.zeros(c, dtype=torch.float64, device=x.device)
    return xh, xh * ga + be, mu.reshape(n, groups), rs.reshape(n, groups)


def gn_bwd64(x, dout, n, hw, groups, gamma, beta, eps, act):
    """(dx, dgamma, dbeta, size) from the formula; size = (sum |du xh|, sum |du|) per channel, what rounding errors scale with."""
    c = x.shape[1]
    xh, u, _, rs = gn64(x, n, hw, groups, gamma, beta, eps)
    ga = gamma.double() if gamma is not None else torch.ones(c, dtype=torch.float64, device=x.device)
    du = dout.double() * act_grad64(u, act)
    v = (du * ga).view(n, hw, groups, -1)
    xg = xh.view(n, hw, groups, -1)
    m1, m2 = v.mean(dim=(1, 3), keepdim=True), (v * xg).mean(dim=(1, 3), keepdim=True)
    dx = (rs.view(n, 1, groups, 1) * (v - m1 - xg * m2)).reshape(n * hw, c)
    return dx, (du * xh).sum(0), du.sum(0), ((du * xh).abs().sum(0), du.abs().sum(0))


M32 = 0xFFFFFFFF


def philox7(ctr, key):
    """Philox4x32 with 7 rounds on Python integers: four counter words, two key words."""
    c, k = list(ctr), list(key)
    for _ in range(7):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & M32, (a >> 32) ^ c[3] ^ k[1], a & M32]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return c


def keep_mask(seed, step, site, m, c, p, first=0):
    """[m, c] truth values of the definition; element index starts at `first`."""
    lo = np.uint64(M32)
    i0, i1 = first // 4, (first + m * c + 3) // 4
    q = np.arange(i0, i1, dtype=np.uint64)
    ctr = [q & lo, q >> np.uint64(32), np.full_like(q, step & M32), np.full_like(q, site)]
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(7):
        a, b = np.uint64(0xD2511F53) * ctr[0], np.uint64(0xCD9E8D57) * ctr[2]
        ctr = [(b >> np.uint64(32)) ^ ctr[1] ^ np.uint64(k0), b & lo, (a >> np.uint64(32)) ^ ctr[3] ^ np.uint64(k1), a & lo]
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    w = np.stack(ctr, axis=1).reshape(-1)[first - 4 * i0:first - 4 * i0 + m * c]
    return (w >> np.uint64(8)).reshape(m, c) >= np.uint64(int(round(float(np.float32(p)) * (1 << 24))))


def assert_close(got, want, tol, what=""):
    """|got - want| <= tol elementwise (tol: tensor or number); prints how much of the tolerance is used."""
    d = (got.double() - want).abs()
    t = tol if torch.is_tensor(tol) else torch.full_like(d, tol)
    bad = ~(d <= t)
    used = float((d / t.clamp(min=1e-300)).max()) if d.numel() else 0.0
    print("%s: %.3f of the tolerance" % (what, used))
    assert not bool(bad.any()), "%s: %d of %d values beyond the tolerance, worst %.3g times" % (what, int(bad.sum()), bad.numel(), used)
