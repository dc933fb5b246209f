"""Plain 64-bit forms of the serving operators, and the batches they are tested on.

A batch is a list of (new tokens, cache length with them). Its pools hold
finite values only in the slots the lengths cover: every other slot of every
page is NaN, every other table entry garbage, every other page's scale NaN, so
that a kernel which lets any of it through shows it.
"""

from __future__ import annotations

import math

import torch

UNIT = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8,
        torch.float8_e4m3fn: 2.0**-4}  # half a step, relative


def rotate64(x, weight, cos, sin, positions, interleaved, eps):
    """(y, spread) of heads x [T, H, D] at positions [T]: the operator's
    result, and per element |a| + |b| of the pair it came from (what the fp32
    rounding errors of a rotation scale with)."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    spread = y.abs().clone()
    if cos is not None:
        half = cos.shape[1]
        p = positions.long().clamp(0, cos.shape[0] - 1)
        c, s = cos.double()[p][:, None], sin.double()[p][:, None]
        i = torch.arange(half)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        ya, yb = y[..., a].clone(), y[..., b].clone()
        y = y.clone()
        y[..., a], y[..., b] = ya * c - yb * s, yb * c + ya * s
        spread[..., a] = spread[..., b] = ya.abs() + yb.abs()
    return y, spread


def rotate_bound(y, spread, dtype):
    """One rounding to dtype, and the fp32 arithmetic before it: a norm's sum of
    at most 128 squares in an order of 8 + 4 levels, root, quotient and two
    products (under 24 half steps of 2^-24 relative), two products and a sum of
    the rotation (3): 32 of them in all, of the pair's size. Below 2^-14 f16 is
    subnormal: its step is 2^-24 whatever the value, so a rounding is off by up to
    2^-25 however small the value (3.5 2^-24 lies half a step, a seventh of
    itself, from both its neighbours): no fewer than that is asked for."""
    floor = 2.0**-25 if dtype == torch.float16 else 1e-38
    return torch.clamp_min(UNIT[dtype] * y.abs() * (1 + 2.0**-8), floor) + 32 * 2.0**-24 * spread


class Cache:
    """Pools, tables and lengths of a batch [(new, length)], on the CPU."""

    def __init__(self, batch, Hk, D, page, dtype, *, layout="head", seed=0, spare=3, pad=0,
                 extra_pages=0, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.batch, self.Hk, self.D, self.page, self.dtype = batch, Hk, D, page, dtype
        self.fp8 = dtype == torch.float8_e4m3fn
        need = [-(-max(length, 0) // page) for _, length in batch]
        self.pages = sum(need) + spare
        width = max(max(need), 1) + extra_pages
        order = torch.randperm(self.pages, generator=g)
        self.table = torch.empty(len(batch), width, dtype=torch.int32)
        self.table[:] = torch.tensor([-1, 2**31 - 1, -2**31, self.pages])[
            torch.randint(0, 4, self.table.shape, generator=g)]
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n].to(torch.int32)
            at += n
        self.cu = torch.tensor([sum(n for n, _ in batch[:b]) for b in range(len(batch) + 1)],
                               dtype=torch.int32)
        self.tokens = int(self.cu[-1]) + pad
        self.lens = torch.tensor([length for _, length in batch], dtype=torch.int32)
        self.max_len = max(max(length for _, length in batch), 1)
        self.k, self.v = (self._pool(g, layout, scale) for _ in range(2))
        self.k_scales = self.v_scales = None
        if self.fp8:
            self.k_scales, self.v_scales = (
                (1.0 + torch.rand(self.pages, Hk, generator=g)) / 256.0 for _ in range(2))
            unused = torch.ones(self.pages, dtype=torch.bool)
            unused[order[:at]] = False
            self.k_scales[unused] = math.nan
            self.v_scales[unused] = math.nan

    def _pool(self, g, layout, scale):
        """A [pages, Hk, page, D] view, NaN outside the covered slots."""
        shape = (self.pages, self.page, self.Hk, self.D)
        x = torch.randn(shape, generator=g) * scale * (112.0 if self.fp8 else 1.0)
        x = x.clamp(-448, 448) if self.fp8 else x
        used = torch.zeros(shape[:2], dtype=torch.bool)
        for b, (_, length) in enumerate(self.batch):
            for t in range(0, max(length, 0), self.page):
                used[self.table[b, t // self.page].long(), :min(self.page, length - t)] = True
        x = torch.where(used[:, :, None, None], x, math.nan).to(self.dtype)
        if layout == "head":
            return x.permute(0, 2, 1, 3).contiguous()
        return x.permute(0, 2, 1, 3)  # token-major storage

    def values(self, b, which):
        """Sequence b's cached keys or values [Hk, length, D] in 64 bits."""
        pool, scales = (self.k, self.k_scales) if which == "k" else (self.v, self.v_scales)
        n = max(self.batch[b][1], 0)
        ids = self.table[b, :-(-n // self.page)].long()
        x = pool.float()[ids].double()
        if self.fp8:
            x = x * scales.double()[ids][:, :, None, None]
        return x.permute(1, 0, 2, 3).reshape(self.Hk, -1, self.D)[:, :n]

    def to_gpu(self):
        """The device tensors ops take: pools, tables, lengths, scales."""
        def pool(x):
            # .cuda() keeps a dense permuted layout
            return x.cuda()
        kw = {}
        if self.fp8:
            kw = {"k_scales": self.k_scales.cuda(), "v_scales": self.v_scales.cuda()}
        return (pool(self.k), pool(self.v), self.table.cuda(), self.lens.cuda(),
                self.cu.cuda()), kw


def attend64(cache, q, scale=None):
    """(o, lse, bound on |o - kernel's|, bound on |lse - kernel's|) [T, Hq, D] /
    [T, Hq] of q's rows in 64 bits; rows of no sequence are NaN.

    Bounds, with u half a step of q's type. The kernel rounds each probability
    to 16 bits (u), or below 2^-14 in f16 to a step of 2^-24, sums in fp32, and
    rounds the quotient once (u): u A + u |o|, A the attention over |v|. A score
    is a sum of D exact products in fp32: off by at most D 2^-24 of the sum of
    their magnitudes, times the scale; p is off by that much, relative, twice
    (its own and the normaliser's), with 2^-20 for the exponential and the sums.
    """
    T, Hq, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    u, Hk = UNIT[q.dtype], cache.Hk
    group = Hq // Hk
    o = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    lse = torch.full((T, Hq), math.nan, dtype=torch.float64)
    bo, bl = torch.zeros_like(o), torch.zeros_like(lse)
    for b, (n, length) in enumerate(cache.batch):
        r0 = int(cache.cu[b])
        k, v = cache.values(b, "k"), cache.values(b, "v")
        place = length - n + torch.arange(n)
        hide = torch.arange(max(length, 0))[None, :] > place[:, None]
        for h in range(Hq):
            x = q[r0:r0 + n, h].double()
            s = (x @ k[h // group].T * scale).masked_fill(hide, -math.inf)
            size = (x.abs() @ k[h // group].abs().T * scale).masked_fill(hide, 0.0)
            top = s.amax(-1, keepdim=True) if length > 0 else torch.zeros(n, 1).double()
            top = top.clamp_min(-1e300)
            p = torch.exp(s - top)
            total = p.sum(-1, keepdim=True)
            none = total[:, 0] == 0
            vv = v[h // group]
            w = torch.where(none[:, None], 0.0, p / total.clamp_min(1e-300))
            out, spread = w @ vv, w @ vv.abs()
            o[r0:r0 + n, h] = out
            lse[r0:r0 + n, h] = torch.where(none, -math.inf, top[:, 0] + torch.log(total[:, 0]))
            far = D * 2.0**-24 * (size.amax(-1, keepdim=True) if length > 0 else 0.0)
            tiny = length * 2.0**-25 * (vv.abs().amax() if length > 0 else 0.0) \
                if q.dtype == torch.float16 else 0.0
            bo[r0:r0 + n, h] = (u * (1 + 2.0**-6) * (spread + out.abs())
                                + (2 * far + 2.0**-20) * spread + tiny)
            bl[r0:r0 + n, h] = (far[:, 0] if length > 0 else 0.0) + \
                2.0**-20 * (1 + torch.where(none, 0.0, lse[r0:r0 + n, h].abs()))
    return o, lse, bo, bl


def check_attention(cache, q, o, lse, scale=None):
    """The kernel's o and lse (CPU tensors) against attend64's, row by row of
    the sequences; returns the rows of no sequence as a mask."""
    want, wlse, bo, bl = attend64(cache, q, scale)
    stray = torch.isnan(wlse[:, 0])
    got = o.double()
    assert torch.isfinite(got[~stray]).all(), "a value from outside the sequences got through"
    err = ((got - want).abs() - bo)[~stray]
    assert (err <= 0).all(), f"worst excess {err.max().item():.3e}"
    if lse is not None:
        l, wl = lse.double()[~stray], wlse[~stray]
        none = torch.isinf(wl)
        assert torch.equal(l[none], wl[none])
        assert ((l - wl).abs()[~none] <= bl[~stray][~none]).all(), \
            (l - wl).abs()[~none].max().item()
    return stray
