"""ops.attention_paged against a 64-bit form: head layouts, types, pages, lengths.

Chunks of every size from none to several tiles over caches from nothing to
thousands of tokens; the pools hold NaN wherever no token lies.
"""

import pytest
import torch

from neptune_hip import ops
from paged_reference import Cache, check_attention

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _q(cache, Hq, dtype, seed=7, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(cache.tokens, Hq, cache.D, generator=g) * scale).to(dtype)


def _run(cache, q, **kw):
    args, scales = cache.to_gpu()
    kw.setdefault("max_seq_len", cache.max_len)
    r = ops.attention_paged(q.cuda(), *args, return_lse=True, **scales, **kw)
    torch.cuda.synchronize()
    return r[0].cpu(), r[1].cpu()


SHAPES = [
    # (new, length) of each sequence
    ("one", [(1, 1)]),
    ("single_tokens", [(1, 1), (1, 2), (1, 63), (1, 64), (1, 65), (1, 130)]),
    ("block_edges", [(63, 63), (64, 64), (65, 65), (1, 64), (2, 65)]),
    ("empty_ones", [(0, 0), (3, 3), (0, 50), (5, 20), (0, 0)]),
    # places below zero: rows that see nothing, wholly and in part
    ("negative_places", [(4, 2), (1, 0), (3, -5), (140, 100), (2, 7)]),
    ("chunks", [(37, 200), (130, 131), (1, 300), (33, 33)]),
    ("tiles", [(300, 420), (257, 257)]),
]


@pytest.mark.parametrize("name,batch", SHAPES, ids=[s[0] for s in SHAPES])
@pytest.mark.parametrize("Hq,Hk,D,page,qt,kt,layout", [
    (8, 2, 128, 64, BF16, BF16, "head"),
    (4, 4, 64, 48, F16, F16, "token"),
    (10, 2, 64, 16, BF16, BF16, "head"),
    (16, 1, 128, 16, F16, F16, "token"),
    (8, 2, 128, 32, BF16, FP8, "head"),
    (6, 2, 64, 16, BF16, FP8, "token"),
    (8, 8, 128, 112, BF16, FP8, "token"),
], ids=str)
def test_shapes(name, batch, Hq, Hk, D, page, qt, kt, layout):
    cache = Cache(batch, Hk, D, page, kt, layout=layout, seed=3)
    q = _q(cache, Hq, qt)
    o, lse = _run(cache, q)
    check_attention(cache, q, o, lse)


@pytest.mark.parametrize("qt,kt,D,page", [(BF16, BF16, 128, 64), (F16, F16, 64, 16),
                                          (BF16, FP8, 128, 16), (BF16, FP8, 64, 64),
                                          (BF16, BF16, 128, 272)])
@pytest.mark.parametrize("batch", [
    [(1, 5000)], [(3, 2900), (1, 450), (40, 3333)], [(1, 4097), (150, 1500)],
    [(1, 200 + 37 * i) for i in range(12)]], ids=["single", "mixed", "long_and_chunk", "twelve"])
def test_split_keys(batch, qt, kt, D, page):
    """Lengths at which the keys are cut, beside ones where they are not."""
    cache = Cache(batch, 2, D, page, kt, seed=11)
    assert ops.attention_paged_workspace_bytes(cache.tokens, len(batch), 8, 2, D, cache.max_len,
                                               dtype=qt, fp8=kt == FP8) > 0
    q = _q(cache, 8, qt)
    o, lse = _run(cache, q)
    check_attention(cache, q, o, lse)


def test_long_tables_of_small_pages():
    """More pages than a window of the block table holds, many times over."""
    for kt in (BF16, FP8):
        cache = Cache([(2, 9000), (70, 3001)], 1, 128, 16, kt, seed=5)
        q = _q(cache, 4, BF16)
        o, lse = _run(cache, q)
        check_attention(cache, q, o, lse)


@pytest.mark.parametrize("D,kt", [(64, BF16), (128, BF16), (64, FP8), (128, FP8)], ids=str)
@pytest.mark.parametrize("new", [2, 40])
def test_whole_chains_over_small_pages(new, D, kt):
    """A chain of thousands of keys in one work-group, window after window of
    the block table: beside a prompt so large that no keys are cut."""
    cache = Cache([(new, 4501), (8700, 8700)], 1, D, 16, kt, seed=6)
    q = _q(cache, 16, BF16)
    o, lse = _run(cache, q)
    cache.batch = [(new, 4501)]
    check_attention(cache, q[:new], o[:new], lse[:new])


@pytest.mark.parametrize("new", [1, 3, 8, 9, 31, 32, 33, 40])
@pytest.mark.parametrize("D,qt,kt", [(64, F16, F16), (128, BF16, BF16), (64, BF16, FP8),
                                     (128, BF16, FP8)], ids=str)
def test_few_rows(new, D, qt, kt):
    """Tiles around the 32 rows of the narrow form, whole and cut, and a chunk's
    last few rows."""
    for group, batch in ((1, [(new, new + 7), (new, 100), (new, 31), (new, 2000)]),
                         (4, [(new, new), (new, 777)]), (1, [(128 + new, 500)])):
        cache = Cache(batch, 2, D, 32, kt, seed=new)
        q = _q(cache, 2 * group, qt)
        o, lse = _run(cache, q)
        check_attention(cache, q, o, lse)


@pytest.mark.parametrize("n", [63, 64, 65, 200])
def test_many_sequences(n):
    """Around and past a wave's 64 sequences, some with no new token."""
    batch = [((i * 7) % 5, 20 + (i * 13) % 90) for i in range(n)]
    batch[n // 2] = (3, 1500)
    cache = Cache(batch, 2, 64, 32, BF16, seed=n)
    q = _q(cache, 4, BF16)
    o, lse = _run(cache, q)
    check_attention(cache, q, o, lse)


def test_rows_behind_the_last_sequence_stay():
    for batch in ([(5, 40), (9, 9)], [(5, 4000), (9, 700)]):  # whole and split keys
        cache = Cache(batch, 2, 128, 64, BF16, pad=6)
        q = _q(cache, 8, BF16)
        out = torch.full((cache.tokens, 8, 128), 77.0, dtype=BF16, device="cuda")
        o, lse = _run(cache, q, out=out)
        stray = check_attention(cache, q, o, lse)
        assert stray.sum() == 6 and (o[stray] == 77.0).all()


def test_without_cu_seqlens():
    cache = Cache([(1, 90), (1, 1), (1, 700)], 2, 128, 64, BF16)
    q = _q(cache, 8, BF16)
    args, _ = cache.to_gpu()
    a = ops.attention_paged(q.cuda(), *args[:4], max_seq_len=700)
    b = ops.attention_paged(q.cuda(), *args, max_seq_len=700)
    assert torch.equal(a, b)


def test_single_tokens_agree_with_decode():
    """One new token per sequence is decode_paged's call."""
    cache = Cache([(1, 300), (1, 64), (1, 1), (1, 2222)], 2, 128, 64, BF16, seed=9)
    q = _q(cache, 8, BF16)
    o, lse = _run(cache, q)
    check_attention(cache, q, o, lse)
    args, _ = cache.to_gpu()
    o2, lse2 = ops.decode_paged(q.cuda(), args[0], args[1], args[2].clamp(0, cache.pages - 1),
                                args[3], max_seq_len=cache.max_len, return_lse=True)
    check_attention(cache, q, o2.cpu(), lse2.cpu())


def test_strided_queries_and_outputs():
    """q and o as slices of fused [tokens, heads, D] buffers; K and V pools of
    different strides."""
    cache = Cache([(40, 100), (3, 500)], 2, 128, 32, BF16, seed=2)
    g = torch.Generator().manual_seed(1)
    fused = torch.randn(cache.tokens, 8 + 4, 128, generator=g).to(BF16).cuda()
    q = fused[:, 2:10]
    out = torch.zeros(cache.tokens, 12, 136, dtype=BF16, device="cuda")[:, 1:9, :128]
    (k, v, *rest), _ = cache.to_gpu()
    v = v.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)  # token-major beside head-major
    o, lse = ops.attention_paged(q, k, v, *rest, out=out, return_lse=True)
    assert o.data_ptr() == out.data_ptr()
    check_attention(cache, q.cpu(), o.cpu(), lse.cpu())


@pytest.mark.parametrize("D,qt,kt", [(64, F16, F16), (128, BF16, BF16), (64, BF16, FP8),
                                     (128, BF16, FP8)], ids=str)
@pytest.mark.parametrize("n,length", [(5, 5), (8, 200), (60, 100), (200, 333), (3, 2500)])
def test_masked_places_may_hold_anything(n, length, D, qt, kt):
    """Infinities and NaN in the keys and values of late tokens: rows before them
    are as if they were not there, rows that see them show them."""
    cache = Cache([(n, length)], 2, D, 32, kt, seed=n)
    at = length - 1 - n // 3  # the first token that holds any
    bad = [float("inf"), float("-inf"), float("nan")]
    page, place = int(cache.table[0, at // 32]), at % 32
    where = {}
    for i, x in enumerate(bad):
        x = float("nan") if kt == FP8 else x
        cache.v[page, 0, place, 7 * i + 3] = x
        where[7 * i + 3] = x
    last = int(cache.table[0, (length - 1) // 32])
    cache.k[last, 1, (length - 1) % 32, 5] = float("nan")  # the last row sees it: NaN all along
    q = _q(cache, 4, qt)
    o, lse = _run(cache, q)
    seen = length - n + torch.arange(n) >= at
    clean = Cache([(n, length)], 2, D, 32, kt, seed=n)  # the same without them
    clean_o, clean_lse = _run(clean, q)
    assert torch.equal(o[~seen], clean_o[~seen])
    assert torch.equal(lse[:n - 1], clean_lse[:n - 1])
    rows = seen.nonzero()[:, 0][:-1]  # all but the last
    for d in range(D):
        for h in (0, 1):
            got = o[rows, h, d].float()
            if d in where:
                want = torch.full_like(got, where[d])
                assert torch.equal(torch.isnan(got), torch.isnan(want))
                assert torch.equal(got[~torch.isnan(got)], want[~torch.isnan(want)])
            else:
                assert torch.isfinite(got).all()
    assert torch.isnan(o[n - 1, 2:]).all() and torch.isnan(lse[n - 1, 2:]).all()


def test_scale_and_large_scores():
    """Scores of hundreds: one key takes all of a row's weight."""
    cache = Cache([(50, 400), (2, 900)], 2, 128, 64, BF16, seed=4)
    q = _q(cache, 4, BF16, scale=6.0)
    o, lse = _run(cache, q, scale=0.5)
    check_attention(cache, q, o, lse, scale=0.5)


def test_max_seq_len_is_only_a_bound():
    cache = Cache([(7, 300), (1, 1000)], 2, 128, 64, BF16, extra_pages=40)
    q = _q(cache, 8, BF16)
    o, lse = _run(cache, q, max_seq_len=None)
    check_attention(cache, q, o, lse)
    # longer sequences are cut to it: the last rows see its tokens
    args, _ = cache.to_gpu()
    cut = Cache([(7, 300), (1, 640)], 2, 128, 64, BF16, extra_pages=40)
    cut.k, cut.v, cut.table = cache.k, cache.v, cache.table
    o, lse = ops.attention_paged(q.cuda(), *args, max_seq_len=640, return_lse=True)
    check_attention(cut, q, o.cpu(), lse.cpu())


def test_pools_past_32_bit_offsets():
    """Pages whose bytes begin past 2^32 from the pool's start."""
    pages, Hk, page, D = 70000, 1, 256, 128  # 4.6 GB a pool
    k = torch.zeros(pages, Hk, page, D, dtype=BF16, device="cuda")
    v = torch.zeros_like(k)
    cache = Cache([(20, 700), (1, 1300)], Hk, D, page, BF16, seed=8, spare=0)
    far = pages - 1 - torch.arange(cache.pages)
    k[far.cuda()], v[far.cuda()] = cache.k.cuda(), cache.v.cuda()
    table = torch.where((cache.table >= 0) & (cache.table < cache.pages),
                        pages - 1 - cache.table, cache.table)
    q = _q(cache, 4, BF16)
    o, lse = ops.attention_paged(q.cuda(), k, v, table.cuda(), cache.lens.cuda(), cache.cu.cuda(),
                                 max_seq_len=cache.max_len, return_lse=True)
    check_attention(cache, q, o.cpu(), lse.cpu())
