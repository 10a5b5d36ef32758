"""The operators around the clipped layers, from their formulas in float64 on the CPU (test infrastructure only)."""
import math

import numpy as np
import torch

from . import dp_oracle as O


def keep_mask(n, p, seed, stream_id, step, offset=0):
    """bool[n]: which elements a dropout call keeps.  32 bits an element: 16 of its group's Philox draw, below them 16 of the
    draw whose group number has bit 63 set; dropped below round(p 2^32)."""
    groups = (n + 7) // 8
    g = np.arange(groups, dtype=np.uint64) + np.uint64(offset)
    key = np.array([seed & 0xFFFFFFFF, ((seed >> 32) & 0xFFFFFFFF) ^ 0x44524F50], dtype=np.uint32)
    halves = []
    for top in (0, 1):
        ctr = np.empty((groups, 4), dtype=np.uint32)
        ctr[:, 0] = (g & np.uint64(0xFFFFFFFF)).astype(np.uint32)
        ctr[:, 1] = (g >> np.uint64(32)).astype(np.uint32) | np.uint32(top << 31)
        ctr[:, 2], ctr[:, 3] = stream_id, step
        w = O.philox4x32_10(ctr, key).astype(np.uint64)
        halves.append(np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], axis=2).reshape(-1)[:n])
    return (halves[0] << np.uint64(16) | halves[1]) >= np.uint64(round(p * 2 ** 32))


def activation(z, name):
    """act(z), act'(z)"""
    if name is None:
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        c = torch.special.ndtr(z)
        return z * c, c + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    h = torch.tanh(k * (z + 0.044715 * z ** 3))
    return z * (1 + h) / 2, (1 + h) / 2 + z * (1 - h * h) / 2 * k * (1 + 3 * 0.044715 * z * z)


def group_norm(x, gamma, beta, G, eps, act=None, keep=None, p=0.0):
    """x [B, T, C] (any float type): (y, mean [B, G], rstd [B, G], xhat, z)"""
    x = x.detach().cpu().double()
    B, T, C = x.shape
    g = x.reshape(B, T, G, C // G)
    mean = g.mean((1, 3))
    rstd = 1 / torch.sqrt((g - mean[:, None, :, None]).square().mean((1, 3)) + eps)
    xhat = ((g - mean[:, None, :, None]) * rstd[:, None, :, None]).reshape(B, T, C)
    z = xhat if gamma is None else xhat * gamma.detach().cpu().double() + beta.detach().cpu().double()
    y = activation(z, act)[0]
    if keep is not None:
        y = torch.where(keep, y / (1 - p) if p < 1 else y, 0.0)
    return y, mean, rstd, xhat, z


def group_norm_backward(dy, gamma, rstd, xhat, z, G, act=None, keep=None, p=0.0):
    """dx and the per-sample (dgamma_b, dbeta_b) [B, C]; with each the sum of the magnitudes of what it is a sum of, which is
    what its rounding errors are relative to."""
    dy = dy.detach().cpu().double()
    B, T, C = dy.shape
    ga = torch.ones(C, dtype=torch.float64) if gamma is None else gamma.detach().cpu().double()
    if keep is not None:
        dy = torch.where(keep, dy / (1 - p) if p < 1 else dy, 0.0)
    gz = dy * activation(z, act)[1]
    by_group = lambda a: a.reshape(B, T, G, C // G)
    spread = lambda a: a[:, None, :, None].expand(B, T, G, C // G).reshape(B, T, C)
    u = gz * ga
    rs = spread(rstd)
    s1, s2 = spread(by_group(u).mean((1, 3))), spread(by_group(u * xhat).mean((1, 3)))
    a1, a2 = spread(by_group(u).abs().mean((1, 3))), spread(by_group(u * xhat).abs().mean((1, 3)))
    dx, dx_mag = rs * (u - s1 - xhat * s2), rs * (u.abs() + a1 + xhat.abs() * a2)
    return {"dx": (dx, dx_mag), "dgamma": ((gz * xhat).sum(1), (gz * xhat).abs().sum(1)), "dbeta": (gz.sum(1), gz.abs().sum(1)), "gz": gz}


def clipped_mean(per_sample, C, clamp, divisor=None):
    """([C] clipped mean, [B] norms) of per-sample gradients [B, C]"""
    norms = per_sample.square().sum(1).sqrt()
    f = torch.from_numpy(O.clip_factor(norms.numpy(), C, clamp))
    return (per_sample * f[:, None]).sum(0) / (divisor or per_sample.shape[0]), norms


def e4m3_blocks(a, down):
    """(the numbers, the scales) that `a` [r, c] stands for in e4m3 with one power-of-two scale for each block of down x 128:
    values float64 (before the scale), scales float64 [ceil(r / down), ceil(c / 128)]."""
    a = a.detach().cpu().double()
    r, c = a.shape
    rb, cb = -(-r // down), -(-c // 128)
    mag = torch.where(torch.isfinite(a), a.abs(), 0.0)
    padded = torch.zeros(rb * down, cb * 128, dtype=torch.float64)
    padded[:r, :c] = mag
    top = padded.view(rb, down, cb, 128).amax((1, 3))
    m, e = torch.frexp(top)
    k = torch.where(top > 0, (e - torch.where(m <= 0.875, 9, 8)).clamp(min=-126), torch.zeros_like(e))
    scale = torch.ldexp(torch.ones_like(top), k)
    v = a / scale.repeat_interleave(down, 0)[:r].repeat_interleave(128, 1)[:, :c]
    # three bits behind the leading one, which does not go below 2^-6; round to nearest even
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v)[1] - 1).clamp(min=-6) - 3)
    return torch.where(torch.isfinite(a), torch.round(v / step) * step, math.nan), scale


def e4m3_stands_for(a, down):
    v, s = e4m3_blocks(a, down)
    return v * s.repeat_interleave(down, 0)[: a.shape[0]].repeat_interleave(128, 1)[:, : a.shape[1]]
