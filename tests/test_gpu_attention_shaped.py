"""ops.attention_paged over MXFP4 pools, and with capped, biased or windowed scores over
pools of every kind, against 64-bit forms."""

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


def _q(cache, Hq, dtype, seed=7, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(cache.tokens, Hq, cache.D, generator=g) * scale).to(dtype)


def _run(cache, q, *, scale=None, softcap=None, slopes=None, window=None, out=None):
    args, scales = cache.to_gpu()
    out = torch.full(q.shape, 7.0, dtype=q.dtype).cuda() if out is None else out
    o, lse = ops.attention_paged(q.cuda(), *args, return_lse=True, max_seq_len=cache.max_len,
                                 out=out, scale=scale, softcap=softcap, window=window,
                                 slopes=None if slopes is None else slopes.cuda(), **scales)
    torch.cuda.synchronize()
    return o.cpu(), lse.cpu()


BATCHES = {
    "one": [(1, 1)],
    "tokens": [(1, 5), (1, 64), (1, 300), (1, 1000), (1, 0)],
    "guessed": [(4, 700), (3, 33), (8, 8), (0, 50), (2, 1)],
    "chunks": [(200, 500), (1, 900), (33, 33), (70, 1100)],
    "long": [(3, 5000)],
    "prompt": [(300, 300)],
}


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("D,page,layout,dtype,heads", [
    (128, 64, "head", BF16, (8, 2)), (128, 16, "token", F16, (4, 4)),
    (64, 48, "head", F16, (12, 3)), (64, 256, "token", BF16, (7, 1)),
    (128, 96, "head", BF16, (28, 4))])
def test_mx(batch, D, page, layout, dtype, heads):
    Hq, Hk = heads
    cache = make_cache("mx", BATCHES[batch], Hk, D, page, layout=layout, seed=D + page, pad=2)
    q = _q(cache, Hq, dtype)
    o, lse = _run(cache, q)
    stray = check_shaped(cache, q, o, lse)
    assert (o[stray] == 7.0).all(), "rows of no sequence stay as they were"


FORMS = {
    "cap": dict(softcap=30.0),
    "tight cap": dict(softcap=1.5),
    "slopes": dict(slopes=True),
    "window": dict(window=100),
    "window of one": dict(window=1),
    "window of a page": dict(window=64),
    "all": dict(softcap=20.0, slopes=True, window=333),
}


def _form(form, Hq):
    form = dict(form)
    if form.get("slopes"):
        # both signs, and none
        form["slopes"] = torch.exp2(-8.0 * (torch.arange(Hq) + 1) / Hq) * \
            torch.tensor([1.0, -0.02, 0.0])[torch.arange(Hq) % 3]
    return form


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("batch", ["tokens", "guessed", "chunks", "long"])
@pytest.mark.parametrize("kind,D,page,dtype,heads", [
    (BF16, 128, 64, BF16, (8, 2)), (F16, 64, 16, F16, (4, 4)), (F16, 128, 32, F16, (6, 1)),
    (BF16, 64, 64, BF16, (8, 8)), (FP8, 128, 64, BF16, (8, 2)), (FP8, 64, 16, BF16, (12, 3)),
    ("mx", 128, 64, BF16, (8, 2)), ("mx", 64, 48, F16, (12, 3))], ids=str)
def test_shaped(form, batch, kind, D, page, dtype, heads):
    Hq, Hk = heads
    cache = make_cache(kind, BATCHES[batch], Hk, D, page, seed=D + page)
    form = _form(FORMS[form], Hq)
    q = _q(cache, Hq, dtype)
    o, lse = _run(cache, q, **form)
    check_shaped(cache, q, o, lse, **form)


@pytest.mark.parametrize("kind", [BF16, FP8, "mx"], ids=str)
def test_large_scores_under_a_cap(kind):
    """Scores far past the cap: both of its forms, in one block."""
    cache = make_cache(kind, [(40, 400), (1, 500)], 2, 128, 64, seed=9)
    q = _q(cache, 8, BF16, scale=12.0)
    q[::2] *= 0.01
    o, lse = _run(cache, q, softcap=5.0, scale=0.3)
    check_shaped(cache, q, o, lse, softcap=5.0, scale=0.3)


@pytest.mark.parametrize("kind", [BF16, FP8, "mx"], ids=str)
@pytest.mark.parametrize("window", [400, 401, 10**6])
def test_window_that_hides_nothing(kind, window):
    cache = make_cache(kind, [(40, 400), (1, 300)], 2, 64, 64, seed=9)
    q = _q(cache, 8, BF16)
    o, lse = _run(cache, q)
    ow, lsew = _run(cache, q, window=window)
    assert torch.equal(o, ow) and torch.equal(lse, lsew)


@pytest.mark.parametrize("n,length,page", [(150, 300, 16), (12, 100, 64), (40, 2500, 64)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("form", [{}, dict(window=30), dict(softcap=20.0)], ids=str)
@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_blocks_behind_a_row(which, form, D, n, length, page):
    """NaN blocks reach the rows that see them, whole (K) or their elements (V), and no
    others."""
    cache = make_cache("mx", [(n, length)], 2, D, page, seed=D)
    clean = make_cache("mx", [(n, length)], 2, D, page, seed=D)
    t = length - n + 5  # seen by row 5 and later ones, of head 1
    scales = getattr(cache, which + "_scales")
    scales[int(cache.table[0, t // page]), 1, t % page, 1] = 255
    q = _q(cache, 8, BF16)
    o, lse = _run(cache, q, **form)
    want, wlse, bo, bl = shaped64(clean, q, **form)
    place = length - n + torch.arange(n)
    sees = (place >= t) & (place < t + form.get("window", 10**9))
    hit = torch.zeros(n, 8, D, dtype=torch.bool)
    hit[sees, 4:, slice(None) if which == "k" else slice(32, 64)] = True
    assert torch.isnan(o[hit]).all()
    err = (o.double() - want).abs() - bo
    assert (err[~hit] <= 0).all()
    if which == "v":
        assert ((lse.double() - wlse).abs() <= bl).all()


@pytest.mark.parametrize("kind", [BF16, F16], ids=str)
@pytest.mark.parametrize("n,length", [(150, 300), (3, 300)])
def test_infinities_outside_a_window(kind, n, length):
    """Infinities and NaN of V in front of a row's window do not reach it."""
    cache = make_cache(kind, [(n, length)], 2, 128, 64, seed=4)
    clean = make_cache(kind, [(n, length)], 2, 128, 64, seed=4)
    window, t = 40, length - n - 20
    at = int(cache.table[0, t // 64]), 1, t % 64
    cache.v[at[0], at[1], at[2], 0], cache.v[at[0], at[1], at[2], 1] = math.inf, math.nan
    q = _q(cache, 8, kind)
    o, _ = _run(cache, q, window=window)
    want, _, bo, _ = shaped64(clean, q, window=window)
    place = length - n + torch.arange(n)
    sees = place < t + window
    assert sees.any()
    hit = torch.zeros(n, 8, 128, dtype=torch.bool)
    hit[sees, 4:, :2] = True
    assert (o[sees][:, 4:, 0] == math.inf).all() and torch.isnan(o[sees][:, 4:, 1]).all()
    assert (((o.double() - want).abs() - bo)[~hit] <= 0).all()


def test_every_row_has_its_own_mask():
    """One key head over many query heads, odd group, window within a tile's rows."""
    cache = make_cache(BF16, [(100, 257)], 1, 128, 16, seed=11)
    q = _q(cache, 5, BF16)
    for window in (2, 17, 128, 200):
        o, lse = _run(cache, q, window=window)
        check_shaped(cache, q, o, lse, window=window)


@pytest.mark.parametrize("form", ["cap", "slopes", "window of a page", "all"])
@pytest.mark.parametrize("kind,D", [(BF16, 128), (FP8, 128), (FP8, 64), ("mx", 128), ("mx", 64)],
                         ids=str)
def test_tables_longer_than_a_wave(kind, D, form):
    """Chunks over more pages than a wave holds entries of, read from the end back."""
    cache = make_cache(kind, [(200, 2500), (40, 2100)], 2, D, 16, seed=D)
    q = _q(cache, 8, BF16)
    form = _form(FORMS[form], 8)
    o, lse = _run(cache, q, **form)
    check_shaped(cache, q, o, lse, **form)


@pytest.mark.parametrize("D", [64, 128])
def test_long_chains_of_single_tokens(D):
    """Tiles enough that no keys are cut: each wave goes over more pages than it holds
    table entries of."""
    cache = make_cache("mx", [(1, 4500 + 37 * b) for b in range(8)], 64, D, 16, seed=D)
    q = _q(cache, 64, BF16)
    o, lse = _run(cache, q)
    check_shaped(cache, q, o, lse)


@pytest.mark.parametrize("form", [{}, dict(softcap=5.0)], ids=str)
@pytest.mark.parametrize("batch,heads", [
    ([(211, 1203), (293, 2421), (0, 2600), (139, 2150), (316, 2616)], (64, 64)),
    ([(40, 1600 + 61 * i) for i in range(16)], (64, 32))], ids=["5", "16"])
def test_order_of_sequences_changes_nothing(batch, heads, form):
    """Long chains over MXFP4 pools start with the sequences of long items: outputs are
    those of the sequences in the order of their lengths, to the bit."""
    Hq, Hk = heads
    cache = make_cache("mx", batch, Hk, 128, 64, seed=5)
    q = _q(cache, Hq, BF16)
    (k, v, table, lens, cu), scales = cache.to_gpu()
    ends = cu.tolist()
    come = range(len(batch))
    results = []
    for order in (sorted(come, key=lambda b: -batch[b][1]), list(come), list(come)[::-1],
                  sorted(come, key=lambda b: batch[b][1] % 7)):
        rows = torch.cat([torch.arange(ends[b], ends[b + 1]) for b in order])
        new = [0]
        for b in order:
            new.append(new[-1] + batch[b][0])
        at = torch.tensor(order).cuda()
        o, lse = ops.attention_paged(
            q[rows].cuda(), k, v, table[at].contiguous(), lens[at].contiguous(),
            torch.tensor(new, dtype=torch.int32).cuda(), return_lse=True,
            max_seq_len=cache.max_len, **form, **scales)
        back = rows.argsort()
        results.append((o.cpu()[back], lse.cpu()[back]))
    for o, lse in results[1:]:
        assert torch.equal(o, results[0][0]) and torch.equal(lse, results[0][1])
    assert torch.isfinite(results[0][0]).all() and torch.isfinite(results[0][1]).all()
