"""Keys whose exact elements lie next to the borders between MXFP4 codes, closer than fp32
tells apart."""

from __future__ import annotations

import math

import torch

from paged_reference import rotate64

# where the nearest code changes, in scales
BORDERS = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
NEAR, APART = 2.0**-28, 2.0**-42  # a directed element's distance from its border, relative


def _pairs(D, rot, interleaved):
    i = torch.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def _blocks(y):
    """Each element's block's largest magnitude, [T, D] as y."""
    return y.abs().unflatten(-1, (-1, 32)).amax(-1).repeat_interleave(32, -1)


def _scale(top):
    part, e = torch.frexp(top)
    return torch.exp2((e - 3 + (part >= 0.875)).double())


def _toward(a, b, target, side, c, s):
    """fp32 (c, s) next to the given ones with a c - b s just past target on its side (1:
    away from 0), and how far past, relative."""
    step = torch.arange(-20, 21, dtype=torch.int32)
    cs = (c.view(torch.int32)[:, None] + step).view(torch.float32)
    ss = (s.view(torch.int32)[:, None] + step).view(torch.float32)
    y = a[:, None, None] * cs.double()[:, :, None] - b[:, None, None] * ss.double()[:, None, :]
    off = (y / target[:, None, None] - 1.0) * side[:, None, None]
    least, at = torch.where(off > APART, off, math.inf).flatten(1).min(1)
    row, n = torch.arange(len(c)), len(step)
    return cs[row, at // n], ss[row, at % n], least


def rotated(T, D, rot, interleaved, norm, dtype, seed):
    """(k [T, 1, D], weight, cos, sin, eps, directed [T, D]): row t's angles are row t's of
    the tables, moved so that one element of a pair lies within NEAR of a border, on
    either side of it; `directed` marks those. Some blocks' largest lie so at 7 / 4 of a
    power of two, where the scale changes."""
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(T, 1, D, generator=g).to(dtype)
    weight = 1 + 0.1 * torch.randn(D, generator=g) if norm else None
    eps = 1e-5
    angle = torch.rand(T, rot // 2, generator=g) * 2 * math.pi
    cos, sin = torch.cos(angle), torch.sin(angle)
    eps64 = float(torch.tensor(eps, dtype=torch.float32))
    plain, _ = rotate64(k, weight, None, None, torch.zeros(T), interleaved, eps64)
    x = plain[:, 0]
    i, j = _pairs(D, rot, interleaved)
    directed = torch.zeros(T, D, dtype=torch.bool)
    rows, pairs = (m.flatten() for m in torch.meshgrid(torch.arange(T), torch.arange(rot // 2),
                                                       indexing="ij"))

    def turned():
        return rotate64(k, weight, cos, sin, torch.arange(T), interleaved, eps64)[0][:, 0]

    def move(goal, allowed):
        """Pairs' first elements to goal [T, rot / 2] where allowed."""
        first, second = x[rows, i[pairs]], x[rows, j[pairs]]
        now = first * cos[rows, pairs].double() - second * sin[rows, pairs].double()
        want = goal[rows, pairs] * torch.sign(now)
        factor = want / now
        c = (cos[rows, pairs].double() * factor).float()
        s = (sin[rows, pairs].double() * factor).float()
        side = torch.where((rows + pairs) % 2 == 0, 1.0, -1.0).double()
        ok = allowed[rows, pairs] & (factor > 0.8) & (factor < 1.25) & \
            (c.abs() > 2.0**-6) & (s.abs() > 2.0**-6) & \
            (first.abs() + second.abs() < 6 * want.abs())
        c2, s2, off = _toward(first, second, want, side, torch.where(ok, c, 0.5),
                              torch.where(ok, s, 0.5))
        ok &= off < NEAR
        cos[rows[ok], pairs[ok]], sin[rows[ok], pairs[ok]] = c2[ok], s2[ok]
        directed[rows[ok], i[pairs[ok]]] = True

    # every third row: the blocks' largest, where they are a pair's first element
    y = turned()
    top = _blocks(y)
    goal = 1.75 * torch.exp2(torch.frexp(top)[1].double() - 1)
    largest = (y.abs() == top)
    move(goal[:, i], largest[:, i] & (torch.arange(T) % 3 == 0)[:, None])
    # the others to the borders next to them. Neither side of a pair may come to lead its
    # block: with 1.25 of slack
    y = turned()
    top = _blocks(y)
    scale = _scale(top)
    a = y.abs() / scale
    goal = BORDERS[(a[..., None] - BORDERS).abs().argmin(-1)] * scale
    free = y.abs() * 1.3 < top
    move(goal[:, i], free[:, i] & free[:, j] & ~directed[:, i] & (goal * 1.3 < top)[:, i])
    return k, weight, cos, sin, eps, directed


def normed(D, dtype):
    """(k [T, 1, D], weight, eps): rows of +-1, so that an element is its weight over
    sqrt(1 + 2^-30): just below a border that fp32 has it on, and from which the nearest
    code is the upper one."""
    g = torch.Generator().manual_seed(D)
    k = torch.where(torch.rand(8, 1, D, generator=g) < 0.5, 1.0, -1.0).to(dtype)
    weight = torch.tensor([0.75, 1.75, 3.5, 0.5, 1.0, 2.0, 3.0, 0.0])[torch.arange(D) % 8]
    top = torch.tensor([6.0, 7.0, 4.0, 7.0])  # (7: just below where the scale changes)
    weight[31::32] = top[:D // 32]
    return k, weight, 2.0**-30
