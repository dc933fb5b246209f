"""ops.attention_paged where a page's scale or a token's value is out of the
ordinary: E4M3 scales of zero, negative, tiny and NaN, infinities in V that a row
does see, and batches of many more sequences than tokens."""

import pytest
import torch

from neptune_hip import ops
from paged_reference import Cache, attend64, check_attention

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
INF = float("inf")


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _q(cache, Hq, dtype, seed=7):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(cache.tokens, Hq, cache.D, generator=g).to(dtype)


def _run(cache, q):
    args, scales = cache.to_gpu()
    o, lse = ops.attention_paged(q.cuda(), *args, return_lse=True, max_seq_len=cache.max_len,
                                 **scales)
    torch.cuda.synchronize()
    return o.cpu(), lse.cpu()


BATCHES = [[(200, 500)], [(3, 300)], [(33, 33), (1, 90)], [(40, 2500)], [(2, 3000)]]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("batch", BATCHES, ids=str)
def test_scales_of_any_kind(batch, page, D):
    """Zero, negative and tiny scales of K and of V, each page and head its own."""
    cache = Cache(batch, 2, D, page, FP8, seed=D + page)
    g = torch.Generator().manual_seed(page)
    odd = torch.tensor([0.0, -1.0 / 256, 2.0**-140, 1.0 / 256])
    used = ~torch.isnan(cache.k_scales[:, 0])
    for scales in (cache.k_scales, cache.v_scales):
        pick = odd[torch.randint(0, 4, scales.shape, generator=g)]
        scales[used] = pick[used]
    q = _q(cache, 8, BF16)
    o, lse = _run(cache, q)
    want, wlse, bo, bl = attend64(cache, q)
    # Where every scale of V that a row sees is 2^-140, its probabilities times it lie
    # below bf16's normal numbers: rounding one is then off by half a subnormal step,
    # 2^-134, times a code of at most 448, and there are as many as keys; so is the
    # result's rounding. attend64's bounds are relative and have no such floor.
    floor = (cache.max_len * 448 + 1) * 2.0**-134
    assert ((o.double() - want).abs() <= bo + floor).all()
    none = torch.isinf(wlse)
    assert torch.equal(lse.double()[none], wlse[none])
    assert ((lse.double() - wlse).abs() <= bl)[~none].all()


@pytest.mark.parametrize("bad", [float("nan"), INF, -INF, 0.0, -1.0])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,length,page", [(150, 300, 16), (150, 300, 64), (12, 100, 16),
                                           (40, 2500, 64)])
def test_scales_of_pages_behind_a_row(n, length, page, D, bad):
    """The scales of pages that a row does not see do not reach it."""
    cache = Cache([(n, length)], 2, D, page, FP8, seed=D)
    clean = Cache([(n, length)], 2, D, page, FP8, seed=D)
    first = (length - n + 5) // page + 1  # the first page that row 5 does not see
    for index in range(first, -(-length // page)):
        cache.k_scales[int(cache.table[0, index])] = bad
        cache.v_scales[int(cache.table[0, index])] = bad
    q = _q(cache, 8, BF16)
    o, lse = _run(cache, q)
    seen = length - n + torch.arange(n) >= first * page
    want, wlse, bo, bl = attend64(clean, q)
    assert ((o.double() - want).abs() <= bo)[~seen].all()
    assert ((lse.double() - wlse).abs() <= bl)[~seen].all()
    if bad != bad:
        assert torch.isnan(o[seen]).all()


@pytest.mark.parametrize("dtype", [BF16, F16], ids=str)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,length", [(1, 1), (1, 33), (1, 3000), (1, 64), (1, 95), (2, 45),
                                      (50, 130)])
@pytest.mark.parametrize("Hq", [2, 8])
def test_infinities_that_a_row_sees(Hq, n, length, D, dtype):
    """In the last token's value: its element is infinite, the others are not."""
    cache = Cache([(n, length)], 2, D, 16, dtype, seed=length)
    page = int(cache.table[0, (length - 1) // 16])
    cache.v[page, 0, (length - 1) % 16, 3] = INF
    cache.v[page, 1, (length - 1) % 16, D - 2] = -INF
    q = _q(cache, Hq, dtype)
    o, lse = _run(cache, q)
    clean = Cache([(n, length)], 2, D, 16, dtype, seed=length)
    want, wlse, bo, bl = attend64(clean, q)
    got = o.double()
    for h, d, x in ((0, 3, INF), (1, D - 2, -INF)):
        heads = slice(h * (Hq // 2), (h + 1) * (Hq // 2))
        assert (got[n - 1, heads, d] == x).all()
        got[n - 1, heads, d] = want[n - 1, heads, d]
    assert ((got - want).abs() <= bo).all()
    assert ((lse.double() - wlse).abs() <= bl).all()


def test_many_sequences_without_tokens():
    """Sequences with nothing new, thousands of them, cost no work-groups."""
    batch = [(0, 40)] * 3000 + [(2, 1500)] + [(0, 0)] * 3000 + [(1, 700)]
    small = Cache([(2, 1500), (1, 700)], 2, 64, 16, BF16, seed=3)
    width = small.table.shape[1]
    table = torch.zeros(len(batch), width, dtype=torch.int32)
    table[3000], table[-1] = small.table[0], small.table[1]
    cu = torch.zeros(len(batch) + 1, dtype=torch.int32)
    cu[3001:] = 2
    cu[-1] = 3
    lens = torch.tensor([length for _, length in batch], dtype=torch.int32)
    q = _q(small, 8, BF16)
    o, lse = ops.attention_paged(q.cuda(), small.k.cuda(), small.v.cuda(), table.cuda(),
                                 lens.cuda(), cu.cuda(), return_lse=True, max_seq_len=1500)
    check_attention(small, q, o.cpu(), lse.cpu())


@pytest.mark.parametrize("n,D", [(1, 64), (1, 128), (9, 128), (40, 64), (40, 128)])
def test_scales_cost_no_rounding_of_their_own(n, D):
    """E4M3 rows whose keys' weight lies on one key come out rounded once: half a step of
    bf16, 2^-9 of the next power of two above, so 2^-8 of the value at most, and 2^-12 of
    that for the fp32 products. A second rounding, of the probability with the scale,
    would be off by as much again."""
    cache = Cache([(n, n)], 2, D, 16, FP8, seed=n)
    used = ~torch.isnan(cache.k_scales[:, 0])
    cache.v_scales[used] = 1.03 / 128.0  # between two steps of bf16
    cache.k = torch.full_like(cache.k.float(), 0.0).to(FP8)
    for t in range(n):  # key t points along its own direction
        page, place = int(cache.table[0, t // 16]), t % 16
        row = torch.zeros(D)
        row[t] = 448.0
        cache.k[page, :, place] = row.to(FP8)
    cache.k_scales[used] = 1.0
    q = torch.zeros(n, 8, D)
    for t in range(n):
        q[t, :, t] = 8.0  # a row's score of its own key passes all others by hundreds
    o, _ = _run(cache, q.to(BF16))
    want = cache.values(0, "v").permute(1, 0, 2).repeat_interleave(4, dim=1)
    assert ((o.double() - want).abs() <= 2.0**-8 * (1 + 2.0**-12) * want.abs()).all()
    step = torch.exp2(torch.floor(torch.log2(want.abs().clamp_min(1e-30))) - 8)  # half a step
    assert ((o.double() - want).abs() <= step * (1 + 2.0**-10)).all()


@pytest.mark.parametrize("Hk", [257, 512, 513, 700])
def test_more_kv_heads_than_work_groups(Hk):
    """Heads by the hundred fill the GPU: no keys are cut from 513 on."""
    cache = Cache([(1, 600), (3, 530)], Hk, 64, 16, BF16, seed=2)
    q = _q(cache, Hk, BF16)
    check_attention(cache, q, *_run(cache, q))
    need = ops.attention_paged_workspace_bytes(4, 2, Hk, Hk, 64, 600)
    assert (need == 0) == (Hk > 512)


def test_overlapping_sequences_stay_within_the_buffers():
    """cu_seqlens that run back name rows twice, more than the launch has room for:
    nothing outside the outputs and the workspace is touched, and the call ends."""
    cache = Cache([(64, 900)], 2, 64, 16, BF16, seed=6)
    q = _q(cache, 8, BF16)
    B = 40
    cu = torch.tensor([0, 64] * (B // 2) + [64], dtype=torch.int32)
    lens = torch.full((B,), 900, dtype=torch.int32)
    table = cache.table[:1].repeat(B, 1)
    need = ops.attention_paged_workspace_bytes(64, B, 8, 2, 64, 900)
    guard = 1 << 16
    ws = torch.full((need + 2 * guard,), 77, dtype=torch.uint8, device="cuda")
    out = torch.full((64 + 64, 8, 64), 5.0, dtype=BF16, device="cuda")
    ops.attention_paged(q.cuda(), cache.k.cuda(), cache.v.cuda(), table.cuda(), lens.cuda(),
                        cu.cuda(), max_seq_len=900, out=out[32:96],
                        workspace=ws[guard:guard + need])
    torch.cuda.synchronize()
    assert (out[:32] == 5.0).all() and (out[96:] == 5.0).all()
    assert (ws[:guard] == 77).all() and (ws[guard + need:] == 77).all()
