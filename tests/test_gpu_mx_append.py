"""ops.kv_append_paged into MXFP4 pools: bytes and codes against the definition in 64
bits, slots of no row untouched, blocks out of the ordinary, places without a slot."""

import math

import pytest
import torch

from mx_reference import MxCache, decode, encode, nearest, scale_bytes
from neptune_hip import ops
from paged_reference import rotate64, rotate_bound

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _tables(rows, rot, g):
    a = torch.rand(rows, rot // 2, generator=g) * 2 * math.pi
    return torch.cos(a), torch.sin(a)


def _noise(cache, g):
    """Every byte of the pools anything, so that what is not written shows."""
    for name in ("k", "v", "k_scales", "v_scales"):
        x = getattr(cache, name)
        setattr(cache, name, cache._lay(torch.randint(0, 256, x.shape, generator=g)
                                        .to(torch.uint8)))


def _slots(cache):
    """(row, page, place) of every row that has a slot."""
    out = []
    for b, (n, length) in enumerate(cache.batch):
        for i in range(n):
            t = length - n + i
            if t < 0 or t // cache.page >= cache.table.shape[1]:
                continue
            page = int(cache.table[b, t // cache.page])
            if 0 <= page < cache.pages:
                out.append((int(cache.cu[b]) + i, page, t % cache.page, t))
    return out


def _within(codes, byte, x, slack):
    """Bytes and codes are those of some value within `slack` of x (64 bits)."""
    b, d = x.unflatten(-1, (-1, 32)), slack.unflatten(-1, (-1, 32))
    lo = scale_bytes((b.abs() - d).clamp_min(0).amax(-1))
    hi = scale_bytes((b.abs() + d).amax(-1))
    byte64 = byte.long()
    assert ((byte64 >= lo) & (byte64 <= hi)).all()
    got = decode(codes, byte).unflatten(-1, (-1, 32))
    at = byte64[..., None]
    assert ((got >= nearest(b - d, at)) & (got <= nearest(b + d, at))).all()


BATCHES = {
    "step": [(1, 1), (1, 64), (1, 65), (1, 200)],
    "ragged": [(1, 1), (3, 50), (0, 40), (17, 17), (130, 200), (5, 0), (6, 2)],
    "many": [(1 + b % 3, 5 + 7 * b % 90) for b in range(90)],
}


@pytest.mark.parametrize("batch", BATCHES)
@pytest.mark.parametrize("D,rot,interleaved", [
    (128, 128, False), (128, 24, False), (128, 64, True), (128, 0, False), (64, 64, False),
    (64, 40, False), (64, 64, True), (64, 8, False)])
@pytest.mark.parametrize("dtype,layout,page,norm", [
    (BF16, "head", 64, True), (F16, "token", 48, False), (BF16, "token", 1, False),
    (F16, "head", 16, True)])
def test_append(batch, D, rot, interleaved, dtype, layout, page, norm):
    g = torch.Generator().manual_seed(D + rot + page)
    cache = MxCache(BATCHES[batch], 3, D, page, layout=layout, seed=1, pad=4)
    _noise(cache, g)
    T, Hq, Hk = cache.tokens, 7, 3
    q, k, v = (torch.randn(T, h, D, generator=g).to(dtype) for h in (Hq, Hk, Hk))
    cos, sin = _tables(cache.max_len, rot, g) if rot else (None, None)
    qw, kw = ((1 + 0.1 * torch.randn(D, generator=g) for _ in range(2)) if norm else (None, None))
    dev = lambda t: None if t is None else t.cuda()
    (kp, vp, table, lens, cu), scales = cache.to_gpu()
    out = torch.full((T, Hq, D), 7.0, dtype=dtype).cuda()
    got = ops.kv_append_paged(k.cuda(), v.cuda(), kp, vp, table, lens, cu, q=q.cuda(),
                              cos=dev(cos), sin=dev(sin), interleaved=interleaved,
                              q_weight=dev(qw), k_weight=dev(kw), eps=1e-5, out=out, **scales)
    torch.cuda.synchronize()
    assert got is out
    slots = _slots(cache)
    row, page_, place, t = (torch.tensor(x) for x in zip(*slots))
    # queries: rows of the sequences, whether or not their keys have a slot
    pos = torch.cat([length - n + torch.arange(n) for n, length in cache.batch])
    seen = len(pos)
    y, spread = rotate64(q[:seen], qw, cos, sin, pos, interleaved, 1e-5)
    assert ((out[:seen].cpu().double() - y).abs() <= rotate_bound(y, spread, dtype)).all()
    assert (out[seen:] == 7.0).all(), "rows of no sequence stay as they were"
    # keys
    y, spread = rotate64(k[row], kw, cos, sin, t, interleaved, 1e-5)
    slack = 32 * 2.0**-24 * spread if norm or rot else torch.zeros_like(y)
    kp, vp, ks, vs = (x.cpu() for x in (kp, vp, scales["k_scales"], scales["v_scales"]))
    _within(kp[page_, :, place], ks[page_, :, place], y, slack)
    # values: every bit
    codes, byte = encode(v[row].double())
    assert torch.equal(vs[page_, :, place], byte)
    assert torch.equal(vp[page_, :, place], codes)
    # the rest of the pools
    for now, then in ((kp, cache.k), (vp, cache.v), (ks, cache.k_scales), (vs, cache.v_scales)):
        same = (now == then).all(-1)
        same[page_, :, place] = True
        assert same.all(), "a slot of no row was written"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_blocks_out_of_the_ordinary(dtype, D):
    """Ties, zeros, tiny and huge blocks, infinities and NaN: as the definition says,
    and a NaN block leaves its neighbours alone."""
    g = torch.Generator().manual_seed(D)
    T, Hk = 24, 2
    v = torch.randn(T, Hk, D, generator=g)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -5.0, 6.5, 0.0])
    v[0] = ties.repeat(D)[:D]
    v[1] = 0.0
    v[2] = -0.0
    v[3] *= 2.0**-122 if dtype == BF16 else 2.0**-20
    v[4] *= 2.0**-126 if dtype == BF16 else 2.0**-24
    v[5] *= 3e37 if dtype == BF16 else 2e4
    v[6, 0, 1], v[7, 1, D - 1], v[8, 0, 33] = math.inf, -math.inf, math.nan
    v[9] = 7.0
    v[10] = torch.where(torch.arange(D) % 2 == 0, 6.96875, -1e-3)
    v = v.to(dtype)
    if dtype == BF16:
        v[11] = torch.finfo(BF16).max
    cache = MxCache([(T, T)], Hk, D, 16, seed=2)
    (kp, vp, table, lens, cu), scales = cache.to_gpu()
    assert ops.kv_append_paged(v.cuda(), v.cuda(), kp, vp, table, lens, cu, **scales) is None
    torch.cuda.synchronize()
    codes, byte = encode(v.double())
    t = torch.arange(T)
    at = cache.table[0, t // 16].long(), t % 16
    for pool, scale in ((kp, scales["k_scales"]), (vp, scales["v_scales"])):
        assert torch.equal(scale.cpu()[at[0], :, at[1]], byte)
        assert torch.equal(decode(pool.cpu()[at[0], :, at[1]], byte).nan_to_num(9e9),
                           decode(codes, byte).nan_to_num(9e9))
    assert byte[6, 0, 0] == byte[8, 0, 1] == 255 and byte[6, 1, 0] != 255


def test_without_cu_seqlens_and_torch_types():
    """One token a sequence; pools of torch's own four-bit and scale types."""
    cache = MxCache([(1, 1), (1, 17), (1, 40)], 2, 128, 16, seed=3)
    (kp, vp, table, lens, _), scales = cache.to_gpu()
    k = torch.randn(3, 2, 128).to(BF16)
    kp4, vp4 = (x.view(torch.float4_e2m1fn_x2) for x in (kp, vp))
    kw = {n: s.view(torch.float8_e8m0fnu) for n, s in scales.items()}
    ops.kv_append_paged(k.cuda(), k.cuda(), kp4, vp4, table, lens, **kw)
    torch.cuda.synchronize()
    codes, byte = encode(k.double())
    for b, (_, length) in enumerate(cache.batch):
        page, place = int(table[b, (length - 1) // 16]), (length - 1) % 16
        assert torch.equal(kp.cpu()[page, :, place], codes[b])
        assert torch.equal(scales["v_scales"].cpu()[page, :, place], byte[b])


def test_scales_beside_codes_in_one_buffer():
    """Codes and scales of a slot as neighbours: views of one allocation."""
    Hk, D, page, pages = 2, 128, 16, 4
    both = torch.zeros(pages, Hk, page, 160, dtype=torch.uint8).cuda()
    kp, vp = both[..., :64], both[..., 64:128]
    ks, vs = both[..., 128:132], both[..., 132:136]
    k, v = (torch.randn(40, Hk, D).to(BF16) for _ in range(2))
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32).cuda()
    lens = torch.tensor([40], dtype=torch.int32).cuda()
    cu = torch.tensor([0, 40], dtype=torch.int32).cuda()
    ops.kv_append_paged(k.cuda(), v.cuda(), kp, vp, table, lens, cu, k_scales=ks, v_scales=vs)
    kr, vr = ops.kv_read_paged(kp, vp, table, lens, cu, tokens=40, dtype=torch.float32,
                               k_scales=ks, v_scales=vs)
    torch.cuda.synchronize()
    for x, r in ((k, kr), (v, vr)):
        assert torch.equal(r.cpu().double(), decode(*encode(x.double())))
    assert not both[..., 136:].any() and not both[1].any()
