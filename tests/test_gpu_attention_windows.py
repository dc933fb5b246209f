"""Windows of attention_paged where they hide nothing, though its windowed kernels run, and
E4M3 codes and scales that are NaN in front of a window."""

import math

import pytest
import torch

from mx_reference import check_shaped, make_cache, shaped64
from neptune_hip import ops

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _run(cache, dtype, Hq, most, **form):
    g = torch.Generator().manual_seed(7)
    q = torch.randn(cache.tokens, Hq, cache.D, generator=g).to(dtype)
    args, scales = cache.to_gpu()
    o, lse = ops.attention_paged(q.cuda(), *args, return_lse=True, max_seq_len=most, **form,
                                 **scales)
    torch.cuda.synchronize()
    return q, o.cpu(), lse.cpu()


@pytest.mark.parametrize("batch", [[(40, 400), (1, 300)], [(3, 390), (200, 200), (0, 50), (1, 1)]],
                         ids=["chunk", "prompt"])
@pytest.mark.parametrize("kind,dtype,D", [(BF16, BF16, 128), (F16, F16, 64), (FP8, BF16, 128),
                                          (FP8, BF16, 64), ("mx", BF16, 128), ("mx", F16, 64)],
                         ids=str)
@pytest.mark.parametrize("window", [400, 401, 2047])
def test_windows_past_every_row(batch, kind, dtype, D, window):
    """max_seq_len above the window: the host keeps it, and no row is as long."""
    cache = make_cache(kind, batch, 2, D, 64, seed=9, extra_pages=30)
    q, o, lse = _run(cache, dtype, 8, 2048, window=window)
    check_shaped(cache, q, o, lse)


@pytest.mark.parametrize("n,length", [(150, 300), (3, 300), (12, 700), (60, 2300)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("form", [{}, dict(softcap=20.0)], ids=str)
def test_nan_codes_in_front_of_a_window(n, length, D, form):
    """A NaN code of V reaches the rows whose window holds it, that element alone."""
    cache, clean = (make_cache(FP8, [(n, length)], 2, D, 64, seed=4) for _ in range(2))
    window = 40
    t = length - n - 20
    codes = cache.v.view(torch.uint8)
    at = int(cache.table[0, t // 64]), 1, t % 64
    codes[at][0], codes[at][D - 1] = 0x7f, 0xff
    q, o, lse = _run(cache, BF16, 8, length, window=window, **form)
    want, wlse, bo, bl = shaped64(clean, q, window=window, **form)
    sees = length - n + torch.arange(n) < t + window
    assert sees.any()
    hit = torch.zeros(n, 8, D, dtype=torch.bool)
    hit[sees, 4:, 0] = hit[sees, 4:, D - 1] = True
    assert torch.isnan(o[hit]).all()
    assert (((o.double() - want).abs() - bo)[~hit] <= 0).all()
    assert ((lse.double() - wlse).abs() <= bl).all()


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("n,length", [(150, 512), (3, 512), (40, 2304)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale", [math.nan, math.inf, -1.0, 0.0])
def test_scales_of_pages_in_front_of_a_window(scale, n, length, D, page):
    """The scales of pages that lie wholly in front of every row's window are no matter:
    the window begins with a page, in the middle of a tile's key block or at its start."""
    cache, clean = (make_cache(FP8, [(n, length)], 2, D, page, seed=4) for _ in range(2))
    window = (length - n) % page + 1 + page  # the first row's begins where a page does
    first = length - n - window + 1
    assert first % page == 0
    for p in range(first // page):
        for s in (cache.k_scales, cache.v_scales):
            s[int(cache.table[0, p])] = scale
    q, o, lse = _run(cache, BF16, 8, length, window=window)
    want, wlse, bo, bl = shaped64(clean, q, window=window)
    assert ((o.double() - want).abs() <= bo).all()
    assert ((lse.double() - wlse).abs() <= bl).all()


@pytest.mark.parametrize("n", [150, 3])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("which", ["k", "v"])
def test_a_nan_scale_that_some_rows_see(which, D, n):
    """A page under a NaN scale, one key head's: the rows whose window reaches it are NaN,
    the others as without it."""
    length, page, window = 512, 64, 100
    cache, clean = (make_cache(FP8, [(n, length)], 2, D, page, seed=4) for _ in range(2))
    p = (length - n - 50) // page
    getattr(cache, which + "_scales")[int(cache.table[0, p]), 1] = math.nan
    q, o, lse = _run(cache, BF16, 8, length, window=window)
    want, wlse, bo, bl = shaped64(clean, q, window=window)
    place = length - n + torch.arange(n)
    sees = (place >= p * page) & (place < (p + 1) * page - 1 + window)
    hit = torch.zeros(n, 8, dtype=torch.bool)
    hit[sees, 4:] = True
    assert hit.any()
    assert torch.isnan(o[hit]).all()
    assert ((o.double() - want).abs() <= bo)[~hit].all()
    bad = hit if which == "k" else torch.zeros_like(hit)
    assert torch.isnan(lse[bad]).all()
    assert ((lse.double() - wlse).abs() <= bl)[~bad].all()
