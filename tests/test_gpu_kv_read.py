"""ops.kv_read_paged: pools of every kind as rows of every type, rows without a slot,
rows of no sequence, whole sequences, strided outputs."""

import math

import pytest
import torch

from mx_reference import make_cache
from neptune_hip import ops
from paged_reference import UNIT

pytestmark = pytest.mark.gpu

F32, BF16, F16, FP8 = torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _want(cache, which):
    """64-bit rows [T, Hk, D]; NaN where a row is of no sequence."""
    out = torch.full((cache.tokens, cache.Hk, cache.D), math.nan, dtype=torch.float64)
    for b, (n, length) in enumerate(cache.batch):
        x = cache.values(b, which).transpose(0, 1)
        for i in range(n):
            t = length - n + i
            out[int(cache.cu[b]) + i] = x[t] if t >= 0 else 0.0
    return out


BATCHES = {
    "rows": [(1, 1), (3, 50), (0, 40), (17, 17), (70, 200), (5, 0), (6, 2)],
    "whole": [(100, 100), (33, 33), (0, 0), (1, 1)],
    "many": [(1 + b % 3, 5 + 7 * b % 90) for b in range(90)],
}


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind", ["mx", BF16, F16, FP8], ids=str)
@pytest.mark.parametrize("dtype,layout,page,strided", [
    (F32, "head", 16, False), (BF16, "token", 48, True), (F16, "head", 1, False),
    (None, "token", 64, False)])
def test_read(batch, D, kind, dtype, layout, page, strided):
    Hk = 3
    cache = make_cache(kind, BATCHES[batch], Hk, D, page, layout=layout, seed=D + page, pad=3)
    (kp, vp, table, lens, cu), scales = cache.to_gpu()
    want_dtype = dtype or (BF16 if kind in ("mx", FP8) else kind)
    if strided:  # keys and values side by side
        both = torch.full((cache.tokens, 2 * Hk + 1, D), 7.0, dtype=dtype).cuda()
        out = both[:, :Hk], both[:, Hk + 1:]
    else:
        out = tuple(torch.full((cache.tokens, Hk, D), 7.0, dtype=want_dtype).cuda()
                    for _ in range(2))
    got = ops.kv_read_paged(kp, vp, table, lens, cu, dtype=dtype, out=out, **scales)
    torch.cuda.synchronize()
    assert got[0] is out[0] and got[1] is out[1]
    for which, y in zip("kv", got):
        want = _want(cache, which)
        y = y.cpu().double()
        stray = torch.isnan(want[:, 0, 0])
        assert (y[stray] == 7.0).all(), "rows of no sequence stay as they were"
        y, want = y[~stray], want[~stray]
        if kind == "mx" or kind == want_dtype:
            # codes of N(0, 1) fit every type: exactly
            assert torch.equal(y, want)
        else:
            # one rounding of the product to fp32, one to the type; f16 below 2^-14 has
            # steps of 2^-24
            u = UNIT[want_dtype] * (1 + 2.0**-6) + 2.0**-24
            assert ((y - want).abs() <= u * want.abs() + (2.0**-25 if want_dtype == F16 else 0)).all()
    if strided:
        assert (both[:, Hk] == 7.0).all()


@pytest.mark.parametrize("kind", ["mx", BF16, FP8], ids=str)
def test_rows_without_a_slot_are_zeros(kind):
    cache = make_cache(kind, [(8, 40), (4, 60)], 2, 64, 16, seed=5)
    cache.table[0, 2] = -1            # places 32 .. 39
    cache.table[1, 3] = cache.pages   # places 48 .. 59
    cache.lens[1] = 200               # past the table's row
    (kp, vp, table, lens, cu), scales = cache.to_gpu()
    k, v = ops.kv_read_paged(kp, vp, table, lens, cu, tokens=12, **scales)
    torch.cuda.synchronize()
    assert not k[:12].any() and not v[:12].any()


def test_last_tokens_without_cu_seqlens():
    cache = make_cache("mx", [(1, 1), (1, 17), (1, 40)], 2, 128, 16, seed=3)
    (kp, vp, table, lens, _), scales = cache.to_gpu()
    k, v = ops.kv_read_paged(kp, vp, table, lens, dtype=F32, **scales)
    torch.cuda.synchronize()
    for which, y in (("k", k), ("v", v)):
        assert torch.equal(y.cpu().double(), _want(cache, which))


def test_special_codes():
    """NaN scales, and scales whose products pass the type: as fp32 rounds them."""
    cache = make_cache("mx", [(4, 4)], 1, 64, 16, seed=6)
    page = int(cache.table[0, 0])
    cache.k[page, 0, :4] = 0x7f  # 6, and -6 in the high half
    cache.k_scales[page, 0, 0] = torch.tensor([255, 127])
    cache.k_scales[page, 0, 1] = torch.tensor([141, 103])   # 2^14, 2^-24
    cache.k_scales[page, 0, 2] = torch.tensor([252, 2])     # 2^125, 2^-125
    (kp, vp, table, lens, cu), scales = cache.to_gpu()
    for dtype in (F32, BF16, F16):
        k, _ = ops.kv_read_paged(kp, vp, table, lens, cu, tokens=4, dtype=dtype, **scales)
        torch.cuda.synchronize()
        k = k[:, 0].cpu()
        assert torch.isnan(k[0, :32]).all() and (k[0, 32:].abs() == 6).all()
        for row, (a, b) in ((1, (14, -24)), (2, (125, -125))):
            want = torch.tensor([-6.0 * 2.0**a, -6.0 * 2.0**b], dtype=torch.float64).to(dtype)
            assert k[row, 0] == want[0] and k[row, 32] == want[1]
