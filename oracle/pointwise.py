"""Group norm over ragged samples, Philox4x32-10 dropout and the 1x1 convolution with its epilogue in float64, with their gradients
written out.  Test infrastructure: torch on the CPU, no kernels."""
import math

import numpy as np
import torch

LEAKY, SILU, GELU = "leaky_relu", "silu", "gelu"


def act(z, activation, leakiness=1.0):
    """(value, slope)"""
    if activation == SILU:
        s = torch.special.expit(z)
        return z * s, s * (1 + z * (1 - s))
    if activation == GELU:
        cdf = torch.erfc(-z * math.sqrt(0.5)) / 2  # (torch's ndtr is within 2^-55 of 1, not of itself)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    slope = torch.where(z > 0, torch.ones_like(z), torch.full_like(z, float(leakiness)))
    return z * slope, slope


def philox(counter, key):
    """uint32 words [..., 4] of counter [..., 4] and key (2 words)"""
    c = [np.asarray(counter)[..., i].astype(np.uint64) for i in range(4)]
    k = [np.uint64(key[0]), np.uint64(key[1])]
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ k[0], b & low, (a >> np.uint64(32)) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low, (k[1] + np.uint64(0xBB67AE85)) & low]
    return np.stack(c, -1).astype(np.uint32)


def keep(seed, offset, rows, planes, p):
    """bool [rows, planes]"""
    seed, offset = int(seed) % 2 ** 64, int(offset) % 2 ** 64
    quads = (planes + 3) // 4
    ctr = np.zeros((rows, quads, 4), np.uint64)
    ctr[..., 0] = np.arange(quads)
    ctr[..., 1] = np.arange(rows)[:, None]
    ctr[..., 2], ctr[..., 3] = offset % 2 ** 32, offset // 2 ** 32
    words = philox(ctr, (seed % 2 ** 32, seed // 2 ** 32)).reshape(rows, quads * 4)[:, :planes]
    return torch.from_numpy(words >= np.uint32(int(p * 2.0 ** 32)))


def group_norm(x, lengths, groups, weight, bias, eps, activation, leakiness, dy=None):
    """x, dy float64 [N, C]; returns dict(y, z, mean, rstd, [dx, dw, db]); mean / rstd per element's sample and group"""
    C = x.size(1)
    w = torch.ones(C, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(C, dtype=torch.float64) if bias is None else bias.double()
    out = {k: torch.zeros_like(x) for k in ("y", "z", "mean", "rstd", "xh", "slope")}
    out.update(dx=torch.zeros_like(x), m1=torch.zeros_like(x), m2=torch.zeros_like(x), dw=torch.zeros_like(w), db=torch.zeros_like(b))
    r = 0
    for n in lengths:
        rows, r = slice(r, r + n), r + n
        if n == 0:
            continue
        g = x[rows].view(n, groups, -1)
        mean = g.mean((0, 2), keepdim=True)
        rstd = ((g - mean) ** 2).mean((0, 2), keepdim=True).add(eps).rsqrt()
        xh = ((g - mean) * rstd).reshape(n, C)
        z = xh * w + b
        out["y"][rows], out["slope"][rows] = act(z, activation, leakiness)
        out["z"][rows], out["xh"][rows] = z, xh
        out["mean"][rows], out["rstd"][rows] = mean.expand_as(g).reshape(n, C), rstd.expand_as(g).reshape(n, C)
        if dy is not None:
            dz = dy[rows] * out["slope"][rows]
            out["dw"] += (dz * xh).sum(0)
            out["db"] += dz.sum(0)
            dn = (dz * w).view(n, groups, -1)
            m1 = dn.mean((0, 2), keepdim=True).expand_as(dn).reshape(n, C)
            m2 = (dn * xh.view_as(dn)).mean((0, 2), keepdim=True).expand_as(dn).reshape(n, C)
            out["m1"][rows], out["m2"][rows] = m1, m2
            out["dx"][rows] = out["rstd"][rows] * (dn.reshape(n, C) - m1 - xh * m2)
    return out


def linear(x, weight, bias, residual, activation, leakiness, mask, p, dy=None):
    """all float64 (mask bool or None); returns dict(y, z, f, [dx, dw, db, dz])"""
    z = x @ weight + (0 if bias is None else bias)
    value, f = act(z, activation, leakiness)
    if mask is not None:
        m = mask.double() / (1 - p)
        value, f = value * m, f * m
    out = dict(y=value + (0 if residual is None else residual), z=z, f=f, value=value)
    if dy is not None:
        dz = dy * f
        out.update(dz=dz, dx=dz @ weight.t(), dw=x.t() @ dz, db=dz.sum(0))
    return out
