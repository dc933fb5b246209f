"""The serving operators at the ends of what they take: offsets past 32 bits, groups of
heads larger than a tile, and the rotation captured and on another stream."""

import pytest
import torch

from neptune_hip import ops
from paged_reference import Cache, check_attention, rotate64, rotate_bound

pytestmark = pytest.mark.gpu

F16, BF16, FP8 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _tables(rows, rot, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(rows, rot // 2, generator=g, dtype=torch.float64) * 6.28
    return torch.cos(a).float(), torch.sin(a).float()


def test_rotation_past_32_bit_offsets():
    """Tokens 64 KB apart: the last ones begin past 2^32 bytes, in and out."""
    T, row = 70000, 1 << 15
    buf = torch.zeros(T, row, dtype=BF16, device="cuda")  # 4.6 GB
    x = buf[:, :3 * 64].view(T, 3, 64)
    far = torch.tensor([0, 1, 32767, 32768, 65535, 65536, T - 1])
    g = torch.Generator().manual_seed(2)
    rows = torch.randn(len(far), 3, 64, generator=g).to(BF16)
    x[far.cuda()] = rows.cuda()
    cos, sin = _tables(100, 64)
    pos = (torch.arange(T) % 100).to(torch.int32)
    q, k = x[:, :2].transpose(0, 1)[None], x[:, 2:].transpose(0, 1)[None]
    ops.qk_norm_rope(q, k, cos.cuda(), sin.cuda(), pos[None].cuda(), out=(q, k))
    want, spread = rotate64(rows, None, cos, sin, pos[far], False, 1e-6)
    assert ((x[far.cuda()].cpu().double() - want).abs() <= rotate_bound(want, spread, BF16)).all()


@pytest.mark.parametrize("kv", [BF16, FP8], ids=str)
def test_append_past_32_bit_offsets(kv):
    """Pages, and rows of k and v, that begin past 2^32 bytes."""
    page, D = 64, 128
    pages = (1 << 32) // (page * D * (1 if kv == FP8 else 2)) + 1000
    pool = [torch.zeros(pages, 1, page, D, dtype=kv, device="cuda") for _ in range(2)]
    T, row = 70000, 1 << 15
    k = torch.zeros(T, row, dtype=BF16, device="cuda")[:, :D].view(T, 1, D)
    g = torch.Generator().manual_seed(3)
    rows = torch.randn(200, 1, D, generator=g).to(BF16)
    k[T - 200:] = rows.cuda()
    # one sequence of no new tokens before, then 100 + 100 at the end
    cu = torch.tensor([0, T - 200, T - 100, T], dtype=torch.int32, device="cuda")
    lens = torch.tensor([-1 << 30, 100, 130], dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 0, 0], [pages - 1, pages - 3, -1], [5, pages - 2, pages - 999]],
                         dtype=torch.int32)
    scales = {}
    if kv == FP8:
        s = torch.full((pages, 1), 1.0 / 64, device="cuda")
        scales = dict(k_scales=s, v_scales=s)
    ops.kv_append_paged(k, k, *pool, table.cuda(), lens, cu, **scales)
    for x in pool:
        for b, (first, r0) in enumerate(((0, 0), (30, 100)), start=1):
            t = first + torch.arange(100)
            ids = table[b, t // page].long()
            got = x[ids.cuda(), 0, (t % page).cuda()].cpu()
            want = rows[r0:r0 + 100, 0]
            if kv == FP8:
                want = (want.float() * 64).clamp(-448, 448).to(FP8)
            assert torch.equal(got.float(), want.float())
        assert (x[0].float() == 0).all()


@pytest.mark.parametrize("D,qt,kt", [(64, F16, F16), (128, BF16, BF16), (128, BF16, FP8)], ids=str)
@pytest.mark.parametrize("Hq,batch", [(64, [(1, 40), (3, 700)]), (129, [(1, 65), (2, 64)]),
                                      (300, [(1, 1500), (4, 90)])])
def test_groups_larger_than_a_tile(Hq, batch, D, qt, kt):
    """A token's rows over several tiles of 128, or most of one."""
    cache = Cache(batch, 1, D, 32, kt, seed=Hq)
    g = torch.Generator().manual_seed(1)
    q = torch.randn(cache.tokens, Hq, D, generator=g).to(qt)
    args, scales = cache.to_gpu()
    o, lse = ops.attention_paged(q.cuda(), *args, return_lse=True, max_seq_len=cache.max_len,
                                 **scales)
    check_attention(cache, q, o.cpu(), lse.cpu())


def test_rotation_captured_and_on_another_stream():
    g = torch.Generator().manual_seed(4)
    q, k = (torch.zeros(2, h, 9, 128, dtype=BF16, device="cuda") for h in (8, 2))
    cos, sin = (t.cuda() for t in _tables(50, 128))
    pos = torch.zeros(2, 9, dtype=torch.int32, device="cuda")
    w = torch.rand(128, generator=g).cuda()
    call = lambda **kw: ops.qk_norm_rope(q, k, cos, sin, pos, q_weight=w, k_weight=w, **kw)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = call()
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=g))
        k.copy_(torch.randn(k.shape, generator=g))
        pos.copy_(torch.randint(0, 50, pos.shape, generator=g, dtype=torch.int32))
        graph.replay()
        got = [t.clone() for t in outs]
        torch.cuda.synchronize()
        want = call()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            other = call()
        stream.synchronize()
        for a, b, c in zip(got, want, other):
            assert torch.equal(a, b) and torch.equal(a, c)
