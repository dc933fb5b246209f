"""attention_paged over scores of 2^24 to 2^60: a row is the mean of the keys that share its
largest score, whatever a step of fp32 is there."""

import math

import pytest
import torch

from mx_reference import encode, make_cache
from neptune_hip import ops
from paged_reference import UNIT

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _cache(kind, batch, D, size, g):
    """A cache whose keys are 0 but for element 3, a quarter, half or all of `size`."""
    cache = make_cache(kind, batch, 2, D, 16 if size > 2.0**20 else 64, seed=3)
    k = torch.zeros(cache.pages, 2, cache.page, D)
    k[..., 3] = size * torch.exp2(-torch.randint(0, 3, k.shape[:3], generator=g).float())
    if kind == "mx":
        cache.k, cache.k_scales = encode(k)
    elif kind == FP8:
        cache.k = (k / size).to(FP8)
        cache.k_scales = torch.full((cache.pages, 2), size)
    else:
        cache.k = k.to(kind)
    return cache


BATCHES = {"tokens": [(1, 1), (1, 70), (4, 300), (1, 2500)],
           "chunks": [(90, 300), (40, 40), (150, 2100)], "guessed": [(7, 900), (8, 8)]}


@pytest.mark.parametrize("form", [{}, dict(window=80), dict(softcap=True)], ids=str)
@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind,dtype,power", [
    (BF16, BF16, 12), (BF16, BF16, 16), (BF16, BF16, 30), (F16, F16, 12), (F16, F16, 14),
    (FP8, BF16, 16), (FP8, BF16, 30), ("mx", BF16, 12), ("mx", BF16, 16), ("mx", BF16, 30),
    ("mx", F16, 13), ("mx", F16, 14)], ids=str)
def test_rows_are_their_largest_scores(kind, dtype, power, D, batch, form):
    g = torch.Generator().manual_seed(power + D)
    Hq, size, window = 8, 2.0**power, form.get("window")
    cap = None
    if form.get("softcap"):  # above all scores, so that those that differ still do
        cap = 2.0**min(2 * power + 4, 60)
        size = 2.0**min(power, 28)
        form = dict(softcap=cap)
    cache = _cache(kind, BATCHES[batch], D, size, g)
    q = torch.zeros(cache.tokens, Hq, D)
    q[..., 3] = size * (1 + torch.randint(0, 8, q.shape[:2], generator=g) / 8.0)
    q[..., 3] *= torch.where(torch.rand(q.shape[:2], generator=g) < 0.3, -1.0, 1.0)
    q = q.to(dtype)
    args, scales = cache.to_gpu()
    o, lse = ops.attention_paged(q.cuda(), *args, return_lse=True, max_seq_len=cache.max_len,
                                 scale=1.0, **form, **scales)
    torch.cuda.synchronize()
    o, lse, u = o.cpu().double(), lse.cpu().double(), UNIT[dtype]
    for b, (n, length) in enumerate(cache.batch):
        r0 = int(cache.cu[b])
        k, v = cache.values(b, "k"), cache.values(b, "v")
        place = length - n + torch.arange(n)
        far = torch.arange(length)[None, :] - place[:, None]
        hide = far > 0 if window is None else (far > 0) | (far <= -window)
        for h in range(Hq):
            s = q[r0:r0 + n, h].double() @ k[h // 4].T  # exact, in fp32 too
            if cap is not None:
                s = cap * torch.tanh(s / cap)
            s = s.masked_fill(hide, -math.inf)
            top = s.amax(-1, keepdim=True)
            p = torch.exp(s - top)
            total = p.sum(-1)
            w = p / total[:, None]
            want, spread = w @ v[h // 4], w @ v[h // 4].abs()
            # P's and the result's rounding, fp32 sums and exponentials; f16 below 2^-14. The
            # scores themselves have a rounding: scores that differ at all differ by far more
            bound = u * (1 + 2.0**-6) * (spread + want.abs()) + 2.0**-20 * spread
            if dtype == F16:
                bound += length * 2.0**-25 * v[h // 4].abs().amax()
            assert ((o[r0:r0 + n, h] - want).abs() <= bound).all()
            wl = top[:, 0] + torch.log(total)
            # the score times log2(e) and back: three roundings, and log2(e)'s own; a cap's
            # polynomial, 2^-20
            assert ((lse[r0:r0 + n, h] - wl).abs() <= 2.0**-19 * wl.abs() + 2.0**-18).all()
