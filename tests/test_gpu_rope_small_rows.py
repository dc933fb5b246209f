"""Norm of rows so small that their mean square is a subnormal float."""

import pytest
import torch

from neptune_hip import ops
from paged_reference import Cache, rotate64, rotate_bound

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _rows(shape, exponent, dtype):
    """Whole numbers up to 8, times 2^exponent: with exponent >= -71 their squares' sum
    and its 128th part are exact floats, subnormal or not, so that only the root and the
    products round."""
    g = torch.Generator().manual_seed(-exponent)
    x = torch.randint(-8, 9, shape, generator=g).double() * 2.0**exponent
    x[..., 0] = 2.0**exponent  # no row of zeros
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("eps", [0.0, 2.0**-140, 2.0**-128])
@pytest.mark.parametrize("exponent", [-71, -69, -66, -64, -62, -60])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_norm(D, exponent, eps, dtype):
    q, k = _rows((2, 3, 5, D), exponent, dtype), _rows((2, 1, 5, D), exponent, dtype)
    g = torch.Generator().manual_seed(1)
    a = torch.rand(10, D // 2, generator=g, dtype=torch.float64) * 6.28
    cos, sin = torch.cos(a).float(), torch.sin(a).float()
    pos = torch.arange(5, dtype=torch.int32).repeat(2, 1)
    w = 1 + torch.rand(D, generator=g)
    got = ops.qk_norm_rope(q.cuda(), k.cuda(), cos.cuda(), sin.cuda(), pos.cuda(),
                           q_weight=w.cuda(), k_weight=w.cuda(), eps=eps)
    for x, y in ((q, got[0].cpu()), (k, got[1].cpu())):
        H = x.shape[1]
        rows = x.permute(0, 2, 1, 3).reshape(10, H, D)
        want, spread = rotate64(rows, w, cos, sin, pos.reshape(-1), False, eps)
        err = (y.permute(0, 2, 1, 3).reshape(10, H, D).double() - want).abs()
        assert (err <= rotate_bound(want, spread, dtype)).all()


def test_keys_on_their_way_into_the_cache():
    cache = Cache([(4, 4), (3, 20)], 2, 64, 16, BF16)
    k, w = _rows((7, 2, 64), -66, BF16), torch.ones(64)
    (kp, vp, table, lens, cu), _ = cache.to_gpu()
    ops.kv_append_paged(k.cuda(), k.cuda(), kp, vp, table, lens, cu, k_weight=w.cuda(), eps=0.0)
    want, spread = rotate64(k, w, None, None, None, False, 0.0)
    cache.k = kp.cpu()
    got = torch.cat([cache.values(0, "k"), cache.values(1, "k")[:, 17:]], 1).permute(1, 0, 2)
    assert ((got - want).abs() <= rotate_bound(want, spread, BF16)).all()
