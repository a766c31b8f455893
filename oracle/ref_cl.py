"""Plain 64-bit definitions of the channels-last layers (textboxgan_amd/ops_cl.py), for the tests.  CPU or GPU, no product code."""
import math

import torch

SQRT2 = math.sqrt(2.0)


def pow2(k):
    """2^k in float64, from its bits: a device's pow may be off in the last place"""
    return ((k.long() + 1023) << 52).view(torch.float64)


def pack(x):
    """x [..., C] (any float type) -> (q int8 [rows, 32 nb], e uint8 [rows, nb])."""
    ch = x.shape[-1]
    v = x.reshape(-1, ch).double()
    nb = (ch + 31) // 32
    v = torch.cat([v, v.new_zeros(v.shape[0], nb * 32 - ch)], dim=1).reshape(-1, nb, 32)
    bad = ~torch.isfinite(v).all(dim=2)
    v = torch.where(bad[..., None], 0.0, v)
    m, k = torch.frexp(v.abs().amax(dim=2))          # amax = m 2^k, 1/2 <= m < 1: in the definition's terms 2m, k - 1
    e = (k - 1 - 6 + (128 * m >= 127.5).int()).clamp(-126, 121)
    e = torch.where(m == 0, -126, e)
    q = torch.round(v * pow2(-e)[..., None]).clamp(-127, 127)
    return q.to(torch.int8).reshape(-1, nb * 32), torch.where(bad, 255, e + 127).to(torch.uint8)


def unpack(q, e, shape):
    """the values, float64, in `shape`"""
    s = torch.where(e == 255, math.nan, pow2(e.int() - 127))
    v = (q.double().reshape(*e.shape, 32) * s[..., None]).reshape(q.shape[0], -1)
    return v[:, :shape[-1]].reshape(shape)


def unpack_as(q, e, shape, dtype):
    """the values in `dtype`.  fp16 does not hold 65536 = 64 2^10, to which its own largest values are rounded: a kept value beyond +-65504 that
    may stand for one of the type's (it lies within half a step of them) is the nearest of them"""
    v = unpack(q, e, shape)
    if dtype == torch.float16:
        half = torch.where(e == 255, 0.0, pow2(e.int() - 127) / 2).repeat_interleave(32, dim=1)[:, :shape[-1]].reshape(shape)
        v = torch.where(v.abs() - half <= 65504, v.clamp(-65504, 65504), v)
    return v.to(dtype)


def round_trip(x):
    return unpack(*pack(x), x.shape)


def act(z, name):
    return z if name == "linear" else SQRT2 * torch.where(z > 0, z, 0.2 * z) if name == "lrelu" else z * torch.sigmoid(z)


def dact(z, name):
    if name == "linear":
        return torch.ones_like(z)
    if name == "lrelu":
        return SQRT2 * torch.where(z > 0, 1.0, 0.2).to(z.dtype)
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


def group_norm(x, gamma, beta, groups, name, eps, dy=None, save="input"):
    """dict of y, and with dy: dx, dgamma, dbeta; and the magnitudes `*_amp` that roundings are relative to."""
    n, ch = x.shape[0], x.shape[-1]
    xd = x.double().reshape(n, -1, groups, ch // groups)
    per = lambda v: v.double().reshape(-1, 1, groups, ch // groups)
    ga, be = per(gamma), per(beta)
    mean = xd.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((xd - mean) ** 2).mean(dim=(1, 3), keepdim=True) + eps)
    xh = (xd - mean) * rstd
    z = xh * ga + be
    o = {"y": act(z, name).reshape(x.shape), "y_amp": ((xd.abs() + mean.abs()) * rstd * ga.abs() + be.abs()).reshape(x.shape)}
    if dy is None:
        return o
    if save == "act8":
        c = x.float().reshape(xd.shape) - mean.float()
        q, e = pack(c.reshape(-1, ch))
        kept = unpack(q, e, (q.shape[0], ch)).reshape(xd.shape)
        if name == "lrelu":  # one step back where rounding has crossed the kink
            side = lambda v: v.double() * (rstd * ga) + be > 0
            move = torch.where(side(c) != side(kept), torch.sign(c.double() - kept), 0.0).reshape(-1, ch)
            q[:, :ch] = (q[:, :ch] + move).clamp(-127, 127).to(torch.int8)
            kept = unpack(q, e, (q.shape[0], ch)).reshape(xd.shape)
        o["kept"] = kept.reshape(x.shape)
        xh = kept * rstd
        z = xh * ga + be
    dz = dy.double().reshape(xd.shape) * dact(z, name)
    u = ga * dz
    m = lambda v: v.mean(dim=(1, 3), keepdim=True)
    o["dx"] = (rstd * (u - m(u) - xh * m(u * xh))).reshape(x.shape)
    big = xh.abs() + (0 if save == "act8" else mean.abs() * rstd)
    o["dx_amp"] = (rstd * (u.abs() + m(u.abs()) + big * m((u * big).abs()) + (1 if name == "silu" else 0) * (ga * dy.double().reshape(xd.shape)).abs() * (1 + big * ga.abs()))).reshape(x.shape)
    over = 1 if gamma.dim() == 2 else (0, 1)
    shape = gamma.shape
    o["dgamma"], o["dbeta"] = ((dz * xh).sum(dim=over).reshape(shape), dz.sum(dim=over).reshape(shape))
    wide = dy.double().abs().reshape(xd.shape) * (1.2 if name == "silu" else SQRT2)
    o["dgamma_amp"], o["dbeta_amp"] = ((wide * big * (1 + big * ga.abs())).sum(dim=over).reshape(shape), (wide * (1 + big * ga.abs())).sum(dim=over).reshape(shape))
    return o


def wgrad(x, dy, coef):
    """dw, db, and their magnitudes, from the checkpoint's values x (float64 [rows, cin]) and dy [rows, cout]"""
    d = dy.double().reshape(-1, dy.shape[-1])
    x = x.double().reshape(-1, x.shape[-1])
    return coef * (x.t() @ d), d.sum(dim=0), abs(coef) * (x.abs().t() @ d.abs()), d.abs().sum(dim=0)
