"""Caps of attention_paged far from ordinary scores."""

import math

import pytest
import torch

from neptune_hip import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


@pytest.mark.parametrize("cap,scale", [(60, 72), (60, 74), (50, 65), (40, 54), (60, 68), (0, 10),
                                       (-50, -42), (30, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_largest_score_wins(dtype, cap, scale):
    """Scores of 2^-4 of the cap and, of one key, twice that. Where the difference is large the
    row is that key's value, and where it is small the mean of all."""
    n, L, D = 100, 900, 128
    x = 2.0**(cap - 4 - scale)  # a product: 2^-8 or less of q's and k's elements
    half = 2.0**((cap - 4 - scale) // 2)
    rest = x / half
    assert half * rest == x and rest >= 2.0**-14 and half >= 2.0**-14
    q = torch.zeros(n, 2, D, dtype=dtype)
    q[:, :, 3] = half
    k = torch.zeros(L, D)
    k[:, 3] = rest
    k[130, 3] = 2 * rest
    g = torch.Generator().manual_seed(1)
    v = torch.randn(L, D, generator=g).to(dtype)
    pages = -(-L // 64)
    pool = torch.zeros(2, pages * 64, D, dtype=dtype)
    pool[0, :L], pool[1, :L] = k.to(dtype), v
    pool = pool.view(2, pages, 1, 64, D).cuda()
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    o, lse = ops.attention_paged(
        q.cuda(), pool[0], pool[1], table, torch.tensor([L], dtype=torch.int32, device="cuda"),
        torch.tensor([0, n], dtype=torch.int32, device="cuda"), return_lse=True, scale=2.0**scale,
        softcap=2.0**cap)
    torch.cuda.synchronize()
    low, high = (2.0**cap * math.tanh(y) for y in (2.0**-4, 2.0**-3))
    seen = L - n + torch.arange(n) + 1
    if cap >= 30:
        assert torch.equal(o.cpu(), v[130].expand(n, 2, D))
        want = torch.full((n,), high, dtype=torch.float64)
    else:
        w = math.exp(high - low)
        mean = (v.double().cumsum(0)[seen - 1] + (w - 1) * v[130].double()) / (seen - 1 + w)[:, None]
        # P's and the result's rounding (half steps of 2^-8 and 2^-11), fp32 sums
        u = torch.finfo(dtype).eps / 2
        spread = (v.double().abs().cumsum(0)[seen - 1] + w * v[130].double().abs()) / seen[:, None]
        assert ((o.cpu().double() - mean[:, None]).abs() <=
                (2.5 * u + 2.0**-18) * spread[:, None] + L * 2.0**-25).all()
        want = low + torch.log(seen - 1 + w)
    # scores: 2^-20 of themselves; log, exp and sums 2^-20
    assert ((lse.cpu().double() - want[:, None]).abs() <=
            2.0**-19 * want[:, None].abs() + 2.0**-20).all()
