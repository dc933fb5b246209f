"""E4M3 codes of ops.kv_append_paged are those of the fp32 quotient x / scale: exact
ties go to the even code, scales of any size count as they are."""

import pytest
import torch

from neptune_hip import ops

pytestmark = pytest.mark.gpu

F16, BF16, FP8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _codes(x, scales):
    """(key codes, value codes) as floats of rows x [T, Hk, 64], each a sequence of one
    token with a page of its own under scales [T, Hk]."""
    T, Hk, D = x.shape
    kp, vp = (torch.zeros(T, Hk, 16, D, dtype=FP8, device="cuda") for _ in range(2))
    table = torch.arange(T, dtype=torch.int32, device="cuda")[:, None]
    lens = torch.ones(T, dtype=torch.int32, device="cuda")
    s = scales.cuda()
    ops.kv_append_paged(x.cuda(), x.cuda(), kp, vp, table, lens, k_scales=s, v_scales=s)
    return tuple(p[:, :, 0].cpu().float() for p in (kp, vp))


def _check(x, scales):
    want = (x.float() / scales[..., None]).clamp(-448.0, 448.0)  # (keeps NaN)
    want = torch.where(scales[..., None] == 0, 0.0, want).to(FP8).float()
    for got in _codes(x, scales):
        same = (got == want) | (torch.isnan(got) & torch.isnan(want))
        bad = (~same).nonzero()
        assert same.all(), (len(bad), [(x[tuple(i)].item(), scales[tuple(i[:2])].item(),
                                        got[tuple(i)].item(), want[tuple(i)].item())
                                       for i in bad[:3]])


@pytest.mark.parametrize("dtype,odd", [(BF16, (1, 3, 5, 7)), (F16, (1, 3, 5, 7, 11, 21, 43, 63))],
                         ids=str)
def test_ties_go_to_the_even_code(dtype, odd):
    """x = scale times the middle of two codes, all of them exact: 5 bits times at most
    3 (bf16) or 6 (f16). 1.3671875 over 0.0546875 is 25, between 24 and 26."""
    middles = [m * 2.0**e for e in range(-10, 4) for m in range(17, 32, 2)]
    middles += [(n + 0.5) * 2.0**-9 for n in range(8)]  # of subnormal codes
    middles = [m for m in middles if 2.0**-12 < m < 448]
    row = torch.tensor(middles + [-m for m in middles], dtype=torch.float64)
    row = torch.cat([row, row.new_zeros(-len(row) % 64)]).view(-1, 1, 64)
    for k in odd:
        for e in (-8, -7, -3, 0):
            scale = k * 2.0**e
            x = (row * scale).to(dtype)
            keep = x.double() == row * scale  # f16 runs out of exponents below
            x = torch.where(keep, x, 0)
            _check(x, torch.full(x.shape[:2], scale))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
def test_random_values(dtype):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(4000, 3, 64, generator=g).to(dtype)
    for scales in (3.5 + torch.rand(4000, 3, generator=g)) / 448, \
            torch.randint(1, 200, (4000, 3), generator=g) / 128.0, \
            -torch.rand(4000, 3, generator=g).to(BF16).float():
        _check(x, scales)


def test_scales_of_any_size():
    """Down to subnormal floats, whose reciprocals pass the largest, and up to the
    largest; zero, infinite and NaN."""
    g = torch.Generator().manual_seed(4)
    e = torch.arange(-148, 128).double()
    scales = (2.0**e * (1 + torch.rand(len(e), generator=g).double())).float()
    scales = torch.cat([scales, torch.tensor([0.0, float("inf"), float("nan"), 2.0**-149,
                                              3.4028234e38])])[:, None]
    # values up to twice the largest code, as far as bf16 holds them
    x = (scales.double().clamp(0, 3e38)[..., None] * torch.randn(len(scales), 1, 64, generator=g)
         .double() * 300).clamp(-3.3e38, 3.3e38)
    x[-5:] = torch.randn(5, 1, 64, generator=g).double()
    x[:, 0, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")]).double()
    _check(x.to(BF16), scales)


@pytest.mark.parametrize("scale", [0.0123, -3.7, 2.0**-64, 2.0**64])
def test_values_of_any_size(scale):
    """Powers of two and their neighbours, from the smallest to the largest."""
    e = torch.arange(-133, 128).double()
    row = torch.cat([2.0**e, 2.0**e * 1.375, -2.0**e * 1.9921875]).clamp(-3.38e38, 3.38e38)
    row = torch.cat([row, row.new_zeros(-len(row) % 64)]).view(-1, 1, 64).to(BF16)
    _check(row, torch.full(row.shape[:2], scale))
