"""Keys written into MXFP4 pools have the codes and scales of the exact key: directed at the
borders between codes, where fp32 arithmetic, or a rounding of 64-bit results to fp32, takes
the wrong side. The tests without a GPU show that the directed keys tell these apart."""

import math

import pytest
import torch

from mx_keys import APART, BORDERS, NEAR, normed, rotated
from mx_reference import MxCache, decode, encode, nearest, scale_bytes
from paged_reference import rotate64

BF16, F16 = torch.bfloat16, torch.float16

FORMS = [(128, 128, False, True), (128, 64, True, True), (128, 64, False, False),
         (64, 64, False, True), (64, 64, True, False), (64, 40, False, True),
         (128, 128, True, False)]


def _exact(k, weight, cos, sin, interleaved, eps):
    eps = float(torch.tensor(eps, dtype=torch.float32))
    return rotate64(k, weight, cos, sin, torch.arange(len(k)), interleaved, eps)


def _codes32(k, weight, cos, sin, interleaved, eps):
    """Codes and bytes of keys worked out in fp32."""
    y = k.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + torch.tensor(eps)) * weight
    if cos is not None:
        half = cos.shape[1]
        i = torch.arange(half)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        c, s = cos[:len(k), None], sin[:len(k), None]
        ya, yb = y[..., a].clone(), y[..., b].clone()
        y[..., a], y[..., b] = ya * c - yb * s, yb * c + ya * s
    return encode(y)


def _elements(codes):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(-2)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,rot,interleaved,norm", FORMS)
def test_directed_keys_tell_roundings_apart(D, rot, interleaved, norm, dtype):
    k, w, cos, sin, eps, directed = rotated(200, D, rot, interleaved, norm, dtype, D + rot)
    y, spread = _exact(k, w, cos, sin, interleaved, eps)
    codes, byte = encode(y)
    # directed elements lie where they are meant to, farther off than 64-bit arithmetic errs
    # (some ten roundings, 2^-49 of the pair)
    assert directed.sum() > 20 * rot
    scale = torch.exp2(byte.double() - 127).repeat_interleave(32, -1)
    a = (y.abs() / scale)[:, 0][directed]
    near = (a[:, None] / torch.cat((BORDERS, torch.tensor([7.0, 3.5], dtype=torch.float64)))
            - 1).abs().amin(1)
    assert (near < 2 * NEAR).all()
    assert (near * a * scale[:, 0][directed] > 2.0**-45 * spread[:, 0][directed]).all()
    # both mistakes show
    for wrong, wrong_byte in (_codes32(k, w, cos, sin, interleaved, eps), encode(y.float())):
        assert (_elements(wrong) != _elements(codes))[:, 0][directed].double().mean() > 0.1
        assert (wrong_byte != byte).any()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
def test_normed_keys_tell_roundings_apart(D, dtype):
    k, w, eps = normed(D, dtype)
    y, _ = _exact(k, w, None, None, False, eps)
    codes, byte = encode(y)
    for wrong, wrong_byte in (_codes32(k, w, None, None, False, eps), encode(y.float())):
        assert (_elements(wrong) != _elements(codes)).double().mean() > 0.2
        assert (wrong_byte != byte).any()


def _append(k, weight, cos, sin, interleaved, eps):
    """(codes, bytes) [T, Hk, ..] that the pool holds of keys k, token t at place t."""
    from neptune_hip import ops
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    T, Hk, D = k.shape
    cache = MxCache([(T, T)], Hk, D, 64, seed=1)
    (kp, vp, table, lens, cu), scales = cache.to_gpu()
    dev = lambda t: None if t is None else t.cuda()
    ops.kv_append_paged(k.cuda(), k.cuda(), kp, vp, table, lens, cu, cos=dev(cos), sin=dev(sin),
                        k_weight=dev(weight), interleaved=interleaved, eps=eps, **scales)
    torch.cuda.synchronize()
    t = torch.arange(T)
    at = cache.table[0, t // 64].long(), t % 64
    return kp.cpu()[at[0], :, at[1]], scales["k_scales"].cpu()[at[0], :, at[1]]


def _check(codes, byte, y):
    want_codes, want_byte = encode(y)
    assert torch.equal(byte, want_byte)
    assert torch.equal(decode(codes, byte), decode(want_codes, want_byte))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,rot,interleaved,norm", FORMS)
def test_directed_keys(D, rot, interleaved, norm, dtype):
    k, w, cos, sin, eps, _ = rotated(200, D, rot, interleaved, norm, dtype, D + rot)
    y, _ = _exact(k, w, cos, sin, interleaved, eps)
    _check(*_append(k, w, cos, sin, interleaved, eps), y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
def test_normed_keys(D, dtype):
    k, w, eps = normed(D, dtype)
    y, _ = _exact(k, w, None, None, False, eps)
    _check(*_append(k, w, None, None, False, eps), y)
    y, _ = _exact(k, w, None, None, False, 0.0)  # on the borders: halves to the even code
    _check(*_append(k, w, None, None, False, 0.0), y)


@pytest.mark.gpu
@pytest.mark.parametrize("D,rot,interleaved,norm", FORMS)
def test_keys_to_64_bits(D, rot, interleaved, norm):
    """Many ordinary keys: codes and bytes of a value within 2^-48 of the pair's size of the
    exact one (64-bit arithmetic: ten roundings of 2^-53 at most, on either side)."""
    g = torch.Generator().manual_seed(D + rot)
    T, Hk = 1500, 4
    k = torch.randn(T, Hk, D, generator=g).to(BF16)
    w = 1 + 0.1 * torch.randn(D, generator=g) if norm else None
    a = torch.rand(T, rot // 2, generator=g) * 2 * math.pi
    cos, sin = torch.cos(a), torch.sin(a)
    y, spread = _exact(k, w, cos, sin, interleaved, 1e-5)
    codes, byte = _append(k, w, cos, sin, interleaved, 1e-5)
    b, d = y.unflatten(-1, (-1, 32)), 2.0**-48 * spread.unflatten(-1, (-1, 32))
    got = byte.long()
    assert (got >= scale_bytes((b.abs() - d).clamp_min(0).amax(-1))).all()
    assert (got <= scale_bytes((b.abs() + d).amax(-1))).all()
    x = decode(codes, byte).unflatten(-1, (-1, 32))
    assert ((x >= nearest(b - d, got[..., None])) & (x <= nearest(b + d, got[..., None]))).all()
