"""Keys that a norm's mean square takes out of the ordinary on their way into MXFP4 pools:
infinite, NaN, huge, tiny and zero rows, each block as the definition has it."""

import math

import pytest
import torch

from mx_reference import MxCache, encode
from neptune_hip import ops
from paged_reference import rotate64

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _append(k, kw, cos, sin, interleaved, eps):
    """(codes, bytes) [T, Hk, ..] that the pool holds of keys k, token t at place t."""
    T, Hk, D = k.shape
    cache = MxCache([(T, T)], Hk, D, 16, seed=1)
    (kp, vp, table, lens, cu), scales = cache.to_gpu()
    dev = lambda t: None if t is None else t.cuda()
    ops.kv_append_paged(k.cuda(), k.cuda(), kp, vp, table, lens, cu, cos=dev(cos), sin=dev(sin),
                        k_weight=kw.cuda(), interleaved=interleaved, eps=eps, **scales)
    torch.cuda.synchronize()
    t = torch.arange(T)
    at = cache.table[0, t // 16].long(), t % 16
    return kp.cpu()[at[0], :, at[1]], scales["k_scales"].cpu()[at[0], :, at[1]]


def _tables(rows, rot, g):
    if not rot:
        return None, None
    a = torch.rand(rows, rot // 2, generator=g) * 2 * math.pi
    return torch.cos(a), torch.sin(a)


FORMS = [(128, 0, False), (128, 128, False), (128, 64, True), (128, 24, False), (64, 16, False),
         (64, 64, True), (64, 0, False)]


@pytest.mark.parametrize("D,rot,interleaved", FORMS)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_infinite_elements(dtype, D, rot, interleaved):
    """x w / sqrt(inf) is 0 for the finite elements: only the blocks of an infinite one and
    of its partner in the rotation are NaN."""
    g = torch.Generator().manual_seed(D + rot)
    T, Hk = 20, 3
    k = torch.randn(T, Hk, D, generator=g).to(dtype)
    at = {(2, 0): [0], (3, 1): [D - 1], (5, 2): [5], (9, 0): [37, 38]}
    for (t, h), elements in at.items():
        for i, e in enumerate(elements):
            k[t, h, e] = -math.inf if i or t == 3 else math.inf
    k[11, 1, 7] = math.nan  # the mean with it: the whole row
    kw = 1 + 0.1 * torch.randn(D, generator=g)
    codes, byte = _append(k, kw, *_tables(T, rot, g), interleaved, 1e-5)
    half = rot // 2
    for t in range(T):
        for h in range(Hk):
            got_c, got_b = codes[t, h].view(-1, 16), byte[t, h]
            if (t, h) == (11, 1):
                assert (got_b == 255).all()
            elif (t, h) not in at:
                assert ((got_b > 0) & (got_b < 255)).all()
            else:
                bad = set()
                for e in at[t, h]:
                    partner = e
                    if e < rot:
                        partner = e ^ 1 if interleaved else e + half if e < half else e - half
                    bad |= {e // 32, partner // 32}
                for block in range(D // 32):
                    if block in bad:
                        assert got_b[block] == 255
                    else:
                        assert got_b[block] == 0 and not got_c[block].any()


@pytest.mark.parametrize("D,rot,interleaved", FORMS)
def test_rows_of_any_size(D, rot, interleaved):
    """Rows whose squares pass fp32's range above and below, normed to ordinary keys: the
    nearest codes to them; a zero row is zeros."""
    g = torch.Generator().manual_seed(D + rot)
    T, Hk = 18, 2
    k = torch.randn(T, Hk, D, generator=g)
    for t, size in enumerate((1e30, 1e25, 3e37, 1e-25, 1e-30, 1e-37)):
        k[t] *= size
    k[7] = 0.0
    k = k.to(BF16)
    kw = 1 + 0.1 * torch.randn(D, generator=g)
    cos, sin = _tables(T, rot, g)
    for eps in (0.0, 2e-38):
        rows = torch.arange(T) if eps else torch.arange(T)[torch.arange(T) != 7]
        codes, byte = _append(k[rows], kw, cos, sin, interleaved, eps)
        y, _ = rotate64(k[rows], kw, cos, sin, torch.arange(len(rows)), interleaved,
                        float(torch.tensor(eps, dtype=torch.float32)))
        want_codes, want_byte = encode(y)
        assert torch.equal(byte, want_byte)
        assert torch.equal(codes, want_codes)
