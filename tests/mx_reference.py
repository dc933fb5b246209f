"""MXFP4 pools, and attention with capped, biased or windowed scores, in plain 64-bit
forms, with the batches they are tested on (paged_reference's, MXFP4 pools among them).

A slot that no sequence covers holds codes of 6 under a NaN scale.
"""

from __future__ import annotations

import math

import torch

from paged_reference import UNIT, Cache

VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def scale_bytes(top):
    """The byte of blocks with largest magnitudes top (64 bits, any shape)."""
    part, e = torch.frexp(top.where(torch.isfinite(top), 1.0))
    byte = (e.long() - 1 + 127 - 2 + (part >= 0.875)).clamp(max=252)
    byte = torch.where(top < 2.0**-123, 0, byte)
    return torch.where(torch.isfinite(top), byte, 255)


def nearest(x, byte):
    """Value of the code nearest to x under the scale's byte, halves to the even code."""
    two = torch.exp2(byte.double() - 127.0)
    a = (x / two).abs()
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0)).double()
    y = (torch.round(a / step) * step).clamp_max(6.0) * two * torch.sign(x)
    return torch.where(byte == 0, 0.0, torch.where(byte == 255, math.nan, y))


def encode(x):
    """(codes uint8 [.., D / 2], bytes uint8 [.., D / 32]) of x [.., D] in 64 bits."""
    b = x.double().unflatten(-1, (-1, 32))
    byte = scale_bytes(torch.where(torch.isnan(b), math.inf, b).abs().amax(-1))
    y = nearest(torch.nan_to_num(b, nan=0.0, posinf=0.0, neginf=0.0), byte[..., None])
    two = torch.exp2(byte.double() - 127.0)[..., None]
    a = torch.nan_to_num((y / two).abs())
    code = torch.searchsorted(VALUES, a.contiguous())
    neg = (torch.signbit(b) & (byte != 0)[..., None] & (byte != 255)[..., None])
    code = (code | neg.long() << 3).flatten(-2).to(torch.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, byte.to(torch.uint8)


def decode(codes, byte):
    """64-bit values of codes [.., D / 2] under bytes [.., D / 32]."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    y = VALUES[c & 7] * (1.0 - 2.0 * (c >> 3))
    two = torch.exp2(byte.double() - 127.0)
    two = torch.where(byte == 255, math.nan, two)
    return (y.unflatten(-1, (-1, 32)) * two[..., None]).flatten(-2)


class MxCache(Cache):
    """Cache whose pools are MXFP4."""

    def __init__(self, batch, Hk, D, page, *, layout="head", seed=0, **kw):
        super().__init__(batch, Hk, D, page, torch.float32, layout=layout, seed=seed, **kw)
        self.layout = layout
        for name in ("k", "v"):
            x = getattr(self, name)
            stray = torch.isnan(x)
            codes, byte = encode(torch.where(stray, 1.0, x))
            codes[stray[..., 0::2]] = 0x77
            byte[stray[..., ::32]] = 255
            setattr(self, name, self._lay(codes))
            setattr(self, name + "_scales", self._lay(byte))
        self.dtype = None

    def _lay(self, x):
        if self.layout == "head":
            return x.contiguous()
        return x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)

    def values(self, b, which):
        codes, byte = getattr(self, which), getattr(self, which + "_scales")
        n = max(self.batch[b][1], 0)
        ids = self.table[b, :-(-n // self.page)].long()
        x = decode(codes[ids], byte[ids])
        return x.permute(1, 0, 2, 3).reshape(self.Hk, -1, self.D)[:, :n]

    def to_gpu(self):
        return ((self.k.cuda(), self.v.cuda(), self.table.cuda(), self.lens.cuda(),
                 self.cu.cuda()),
                {"k_scales": self.k_scales.cuda(), "v_scales": self.v_scales.cuda()})


def make_cache(kind, batch, Hk, D, page, **kw):
    """A cache of pools of `kind`: "mx" or a torch dtype."""
    if kind == "mx":
        return MxCache(batch, Hk, D, page, **kw)
    return Cache(batch, Hk, D, page, kind, **kw)


def shaped64(cache, q, *, softcap=None, slopes=None, window=None, scale=None):
    """(o, lse, bound on |o - kernel's|, bound on |lse - kernel's|) of q's rows in 64
    bits; rows of no sequence are NaN.

    Bounds, with u half a step of q's type. A score x is a sum of D exact products in
    fp32 times the scale: off by (D + 2) 2^-24 of the sum of their magnitudes. The cap's
    slope is at most 1, and the score over the cap y has three roundings, 1.5 2^-23 of it.
    Up to |y| = 3/8 the polynomial with its roundings is off by 1.5e-7, 1.3 2^-23 of the
    score: less than 2^-20 in all. Beyond, a score is at least tanh(3/8) = 0.358 of the
    cap, and exponent, v_exp_f32, sum, v_rcp_f32 and the last rounding make at most 2.3
    2^-23 of the cap, 6.3 2^-23 of the score, y's 1.4: again less than 2^-20. A bias is off
    by three roundings of itself, the sum of both by one. So each score has a bound e,
    and with weights w the output is off by at most sum w e (|v| + |o|), the log-sum-exp
    by sum w e; p and V's products as in attend64: rounding to 16 bits (u), in f16 below
    2^-14 to a step of 2^-24, fp32 sums and exponentials 2^-20, the result's rounding u."""
    T, Hq, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    u, group = UNIT[q.dtype], Hq // cache.Hk
    o = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    lse = torch.full((T, Hq), math.nan, dtype=torch.float64)
    bo, bl = torch.zeros_like(o), torch.zeros_like(lse)
    for b, (n, length) in enumerate(cache.batch):
        r0, L = int(cache.cu[b]), max(length, 0)
        k, v = cache.values(b, "k"), cache.values(b, "v")
        place = length - n + torch.arange(n)
        far = (torch.arange(L)[None, :] - place[:, None]).double()
        hide = far > 0
        if window is not None:
            hide |= far <= -window
        for h in range(Hq):
            if L == 0:
                o[r0:r0 + n, h], lse[r0:r0 + n, h] = 0.0, -math.inf
                continue
            x = q[r0:r0 + n, h].double()
            # (hidden keys may hold anything)
            kk, vv = torch.nan_to_num(k[h // group]), v[h // group]
            s = x @ kk.T * scale
            e = (D + 2) * 2.0**-24 * (x.abs() @ kk.abs().T * scale)
            if softcap is not None:
                s = softcap * torch.tanh(s / softcap)
                e = e + 2.0**-20 * s.abs()
            if slopes is not None:
                bias = slopes[h].double() * far
                e = e + 3 * 2.0**-24 * bias.abs() + 2.0**-24 * (s + bias).abs()
                s = s + bias
            s = s.masked_fill(hide, -math.inf)
            top = s.amax(-1, keepdim=True).clamp_min(-1e300)
            p = torch.exp(s - top)
            total = p.sum(-1, keepdim=True)
            none = total[:, 0] == 0
            w = torch.where(none[:, None], 0.0, p / total.clamp_min(1e-300))
            vv = torch.where(torch.isfinite(vv), vv, 0.0)
            out, spread = w @ vv, w @ vv.abs()
            we = w * e
            o[r0:r0 + n, h] = out
            lse[r0:r0 + n, h] = torch.where(none, -math.inf, top[:, 0] + torch.log(total[:, 0]))
            tiny = L * 2.0**-25 * vv.abs().amax() if q.dtype == torch.float16 else 0.0
            bo[r0:r0 + n, h] = (u * (1 + 2.0**-6) * (spread + out.abs()) + 2.0**-20 * spread
                                + we @ vv.abs() + we.sum(-1, keepdim=True) * out.abs() + tiny)
            bl[r0:r0 + n, h] = we.sum(-1) + \
                2.0**-20 * (1 + torch.where(none, 0.0, lse[r0:r0 + n, h].abs()))
    return o, lse, bo, bl


def check_shaped(cache, q, o, lse, **form):
    """The kernel's o and lse (CPU tensors) against shaped64's."""
    want, wlse, bo, bl = shaped64(cache, q, **form)
    stray = torch.isnan(wlse[:, 0])
    got = o.double()
    assert torch.isfinite(got[~stray]).all(), "a value from outside the sequences got through"
    err = ((got - want).abs() - bo)[~stray]
    assert (err <= 0).all(), f"worst excess {err.max().item():.3e}"
    if lse is not None:
        l, wl = lse.double()[~stray], wlse[~stray]
        none = torch.isinf(wl)
        assert torch.equal(l[none], wl[none])
        off = ((l - wl).abs() - bl[~stray])[~none]
        assert (off <= 0).all(), f"worst excess of lse {off.max().item():.3e}"
    return stray
