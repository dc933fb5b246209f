"""ops.qk_norm_rope against a 64-bit form."""

import pytest
import torch

from neptune_hip import ops
from paged_reference import rotate64, rotate_bound

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _tables(rows, rot, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(rows, rot // 2, generator=g, dtype=torch.float64) * 6.28
    return torch.cos(a).float(), torch.sin(a).float()


def _check(x, got, weight, cos, sin, positions, interleaved, eps=1e-6):
    """x, got [B, H, S, D] CPU tensors; positions [B, S]."""
    B, H, S, D = x.shape
    rows = x.permute(0, 2, 1, 3).reshape(B * S, H, D)
    y, spread = rotate64(rows, weight, cos, sin, positions.reshape(-1), interleaved, eps)
    err = (got.permute(0, 2, 1, 3).reshape(B * S, H, D).double() - y).abs()
    over = err - rotate_bound(y, spread, x.dtype)
    assert (over <= 0).all(), f"worst excess {over.max().item():.3e}"


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("B,Hq,Hk,S,D,rot", [
    (1, 1, 1, 1, 64, 64), (3, 8, 2, 1, 128, 128), (2, 5, 3, 77, 64, 32), (1, 32, 8, 130, 128, 128),
    (2, 4, 4, 33, 32, 32), (1, 7, 1, 19, 128, 48), (2, 3, 2, 9, 32, 8), (5, 28, 7, 3, 128, 64)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", ["none", "both", "k"])
def test_shapes(dtype, B, Hq, Hk, S, D, rot, interleaved, norm):
    g = torch.Generator().manual_seed(B + 10 * S + D)
    q = torch.randn(B, S, Hq, D, generator=g).to(dtype).transpose(1, 2)
    k = (3 * torch.randn(B, Hk, S, D, generator=g)).to(dtype)
    qw = 1 + torch.rand(D, generator=g) if norm == "both" else None
    kw = 1 - torch.rand(D, generator=g) if norm != "none" else None
    cos, sin = _tables(100, rot)
    pos = torch.randint(0, 100, (B, S), generator=g, dtype=torch.int32)
    qo, ko = ops.qk_norm_rope(q.cuda(), k.cuda(), cos.cuda(), sin.cuda(), pos.cuda(),
                              q_weight=None if qw is None else qw.cuda(),
                              k_weight=None if kw is None else kw.cuda(),
                              interleaved=interleaved)
    assert qo.is_contiguous() and ko.is_contiguous()
    _check(q, qo.cpu(), qw, cos, sin, pos, interleaved)
    _check(k, ko.cpu(), kw, cos, sin, pos, interleaved)


def test_in_place_in_a_fused_projection():
    """q and k as slices of one [B, S, heads, D] buffer, rewritten in place;
    the value heads between and behind them stay."""
    g = torch.Generator().manual_seed(5)
    fused = torch.randn(2, 50, 12, 128, generator=g).to(BF16)
    cos, sin = _tables(64, 128)
    pos = torch.arange(50, dtype=torch.int32).repeat(2, 1)
    w = torch.ones(128)
    dev = fused.cuda()
    q, k = dev[:, :, :6].transpose(1, 2), dev[:, :, 8:10].transpose(1, 2)
    qo, ko = ops.qk_norm_rope(q, k, cos.cuda(), sin.cuda(), pos.cuda(), q_weight=w.cuda(),
                              out=(q, k))
    assert qo is q and ko is k
    got = dev.cpu()
    _check(fused[:, :, :6].transpose(1, 2), got[:, :, :6].transpose(1, 2), w, cos, sin, pos, False)
    _check(fused[:, :, 8:10].transpose(1, 2), got[:, :, 8:10].transpose(1, 2), None, cos, sin, pos,
           False)
    for at in (slice(6, 8), slice(10, 12)):
        assert torch.equal(got[:, :, at], fused[:, :, at])


def test_positions_outside_the_tables_are_clamped():
    q = torch.ones(1, 2, 4, 64, dtype=BF16, device="cuda")
    k = torch.ones(1, 1, 4, 64, dtype=BF16, device="cuda")
    cos, sin = _tables(10, 64)
    far = torch.tensor([[-2**31, -1, 10, 2**31 - 1]], dtype=torch.int32)
    near = torch.tensor([[0, 0, 9, 9]], dtype=torch.int32)
    a = ops.qk_norm_rope(q, k, cos.cuda(), sin.cuda(), far.cuda())
    b = ops.qk_norm_rope(q, k, cos.cuda(), sin.cuda(), near.cuda())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_zero_rows_and_eps():
    q = torch.zeros(1, 2, 3, 128, dtype=F16, device="cuda")
    k = torch.full((1, 1, 3, 128), 2.0**-24, dtype=F16, device="cuda")  # subnormal
    cos, sin = _tables(4, 128)
    pos = torch.zeros(1, 3, dtype=torch.int32)
    w = torch.ones(128)
    qo, ko = ops.qk_norm_rope(q, k, cos.cuda(), sin.cuda(), pos.cuda(), q_weight=w.cuda(),
                              k_weight=w.cuda(), eps=1e-12)
    assert (qo == 0).all()
    _check(k.cpu(), ko.cpu(), w, cos, sin, pos, False, eps=1e-12)
