"""ops.kv_append_paged: what lands in the pages, and what stays as it was."""

import math

import pytest
import torch

from neptune_hip import ops
from paged_reference import UNIT, Cache, rotate64, rotate_bound

pytestmark = pytest.mark.gpu

F16, BF16, FP8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _bits(x):
    return x.contiguous().view(torch.uint8 if x.element_size() == 1 else torch.int16)


def _tables(rows, rot, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(rows, rot // 2, generator=g, dtype=torch.float64) * 6.28
    return torch.cos(a).float(), torch.sin(a).float()


def _slots(cache):
    """(row, sequence, place, page or -1) of every row of the sequences."""
    out = []
    for b, (n, length) in enumerate(cache.batch):
        for i in range(n):
            t = length - n + i
            page = -1
            if t >= 0 and t // cache.page < cache.table.shape[1]:
                page = int(cache.table[b, t // cache.page])
                page = page if 0 <= page < cache.pages else -1
            out.append((int(cache.cu[b]) + i, b, t, page))
    return out


def _append(cache, Hq, dtype, *, rot=0, interleaved=False, norm=False, fused=False, cu=True,
            out=None, values=1.0):
    """Runs the call and checks every slot of both pools and every row of q."""
    g = torch.Generator().manual_seed(21)
    T, Hk, D = cache.tokens, cache.Hk, cache.D
    if fused:
        buf = torch.randn(T, Hq + 2 * Hk, D, generator=g).to(dtype)
        q, k, v = buf[:, :Hq], buf[:, Hq:Hq + Hk], buf[:, Hq + Hk:]
        dev = buf.cuda()
        dq, dk, dv = dev[:, :Hq], dev[:, Hq:Hq + Hk], dev[:, Hq + Hk:]
    else:
        q, k, v = ((values * torch.randn(T, h, D, generator=g)).to(dtype) for h in (Hq, Hk, Hk))
        dq, dk, dv = q.cuda(), k.cuda(), v.cuda()
    qw, kw = ((1 + torch.rand(D, generator=g), 1 - torch.rand(D, generator=g)) if norm
              else (None, None))
    cos, sin = _tables(max(cache.max_len, 1), rot) if rot else (None, None)

    def dev_of(x):
        return None if x is None else x.cuda()

    (kp, vp, table, lens, cud), scales = cache.to_gpu()
    if out == "in_place":
        out = dq
    r = ops.kv_append_paged(dk, dv, kp, vp, table, lens, cud if cu else None,
                            q=dq if Hq else None, cos=dev_of(cos), sin=dev_of(sin),
                            interleaved=interleaved, q_weight=dev_of(qw) if Hq else None,
                            k_weight=dev_of(kw), out=out, **scales)
    torch.cuda.synchronize()
    kgot, vgot = kp.cpu(), vp.cpu()
    slots = _slots(cache)
    places = torch.zeros(T, dtype=torch.long)
    for row, _, t, _ in slots:
        places[row] = t
    wk, sk = rotate64(k, kw, cos, sin, places, interleaved, 1e-6)
    written = torch.zeros(cache.pages, cache.page, dtype=torch.bool)
    for row, _, t, page in slots:
        if page < 0:
            continue
        written[page, t % cache.page] = True
        for got, want, spread, sc in ((kgot, wk[row], sk[row], cache.k_scales),
                                      (vgot, v[row].double(), v[row].double().abs(),
                                       cache.v_scales)):
            x = got[page, :, t % cache.page]
            if cache.fp8:
                s = sc[page].double()[:, None]
                y = (want / s).clamp(-448, 448)
                # one rounding to a code, by half a step (2^-10 below the
                # smallest normal), of a value that fp32 has 32 half steps off
                bound = torch.maximum(UNIT[FP8] * y.abs(), torch.tensor(2.0**-10)) \
                    + 34 * 2.0**-24 * spread / s
            else:
                y, bound = want, rotate_bound(want, spread, dtype)
            assert ((x.double() - y).abs() <= bound).all(), (row, page)
    for got, before in ((kgot, cache.k), (vgot, cache.v)):
        keep = ~written[:, None, :, None].expand(got.shape)
        assert torch.equal(_bits(got)[keep], _bits(before)[keep]), "a slot of no row was written"
    if Hq:
        wq, sq = rotate64(q, qw, cos, sin, places, interleaved, 1e-6)
        rows = [row for row, *_ in slots]
        err = (r.cpu().double() - wq).abs() - rotate_bound(wq, sq, dtype)
        assert (err[rows] <= 0).all()
    else:
        assert r is None
    return r


BATCHES = [
    ("single_tokens", [(1, 1), (1, 64), (1, 65), (1, 130)]),
    ("prompts", [(70, 70), (1, 1), (129, 129)]),
    ("chunks", [(40, 100), (0, 30), (17, 60), (0, 0), (3, 3)]),
    ("negative_places", [(4, 2), (3, -5), (2, 40)]),
]


@pytest.mark.parametrize("name,batch", BATCHES, ids=[b[0] for b in BATCHES])
@pytest.mark.parametrize("Hq,Hk,D,page,dtype,kv,layout,rot,interleaved,norm", [
    (8, 2, 128, 64, BF16, BF16, "head", 128, False, True),
    (0, 3, 64, 16, F16, F16, "token", 32, True, False),
    (4, 4, 64, 1, BF16, BF16, "head", 0, False, True),
    (7, 1, 128, 33, BF16, FP8, "token", 64, False, False),
    (28, 7, 64, 32, F16, FP8, "head", 64, True, True),
], ids=str)
def test_shapes(name, batch, Hq, Hk, D, page, dtype, kv, layout, rot, interleaved, norm):
    cache = Cache(batch, Hk, D, page, kv, layout=layout, seed=6)
    _append(cache, Hq, dtype, rot=rot, interleaved=interleaved, norm=norm)


@pytest.mark.parametrize("n", [63, 64, 65, 150])
def test_many_sequences(n):
    cache = Cache([((i * 7) % 4, 5 + (i * 13) % 40) for i in range(n)], 2, 64, 16, BF16)
    _append(cache, 4, BF16, rot=64)


@pytest.mark.parametrize("n", [700, 4096, 4097])
def test_sequences_by_the_thousand(n):
    """More than a lane has one of, and than 64 lanes have 64 of; most of them empty
    in long runs, some with several tokens."""
    g = torch.Generator().manual_seed(n)
    new = torch.randint(0, 4, (n,), generator=g) * (torch.rand(n, generator=g) < 0.2)
    new[n // 3:n // 2] = 0
    new[0] = new[-1] = 1
    cache = Cache([(int(x), int(x) + i % 20) for i, x in enumerate(new)], 1, 64, 16, BF16)
    _append(cache, 2, BF16, rot=64)


def test_many_tokens():
    """Enough groups for the form that takes several heads a group."""
    cache = Cache([(1100, 1100), (700, 950)], 4, 64, 64, BF16)
    _append(cache, 6, BF16, rot=64, norm=True)


def test_fused_projection_in_place():
    cache = Cache([(9, 9), (3, 80)], 2, 128, 64, BF16)
    _append(cache, 8, BF16, rot=128, norm=True, fused=True, out="in_place")


def test_without_cu_seqlens():
    _append(Cache([(1, 5), (1, 64), (1, 0), (1, 200)], 2, 128, 64, BF16), 4, BF16, rot=128,
            cu=False)


def test_rows_without_a_slot():
    """Table entries outside the pool, places past the table, rows behind the
    last sequence: nothing is stored, and the rows behind keep q's output."""
    cache = Cache([(30, 100), (5, 20), (6, 6)], 2, 64, 16, BF16, pad=5, spare=4)
    cache.table[0, 5] = cache.pages      # tokens 80 .. 95
    cache.table[2, 0] = -1
    cache.lens[1] = 16 * cache.table.shape[1] + 2  # the last 2 of 5 rows are past the table
    cache.batch = [(30, 100), (5, 16 * cache.table.shape[1] + 2), (6, 6)]
    out = torch.full((cache.tokens, 4, 64), 55.0, dtype=BF16, device="cuda")
    r = _append(cache, 4, BF16, out=out)
    assert (r[-5:] == 55.0).all()


def test_codes():
    """Saturation, zeros, NaN, infinities and pages of scale 0 in E4M3 pools."""
    cache = Cache([(4, 4), (4, 4)], 1, 64, 16, FP8, spare=0)
    cache.k_scales[:] = cache.v_scales[:] = 0.5
    cache.k_scales[cache.table[1, 0]] = 0.0
    x = torch.zeros(8, 1, 64, dtype=BF16)
    x[:, 0, :8] = torch.tensor([1e30, -1e30, math.inf, -math.inf, 240.0, -0.0, 2.0**-11, math.nan])
    (kp, vp, table, lens, cu), scales = cache.to_gpu()
    ops.kv_append_paged(x.cuda(), x.cuda(), kp, vp, table, lens, cu, **scales)
    k, v = kp.cpu(), vp.cpu()
    want = torch.tensor([448.0, -448.0, 448.0, -448.0, 480.0, 0.0, 2.0**-9 / 2, math.nan])
    want[4], want[6] = 448.0, 0.0  # 480 saturates, half the smallest code ties to zero
    page = int(cache.table[0, 0])
    for got in (k[page, 0, 0, :8].float(), v[int(cache.table[1, 0]), 0, 3, :8].float()):
        assert torch.equal(got[:7], want[:7]) and math.isnan(got[7])
    assert (k[int(cache.table[1, 0]), 0, :4].float() == 0).all()
