"""The paged-cache operators together, as a serving engine runs them: append
with norm and rotation, then attention, chunk by chunk and token by token;
captured in graphs, on streams, from threads."""

import threading

import pytest
import torch

from neptune_hip import _abi, ops
from paged_reference import Cache, check_attention, rotate64, rotate_bound

pytestmark = pytest.mark.gpu

BF16, F16, FP8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


def _tables(rows, rot):
    i = torch.arange(rot // 2, dtype=torch.float64)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-2 * i / rot)[None]
    return torch.cos(a).float(), torch.sin(a).float()


class Engine:
    """Pools, table and tables of a few sequences whose tokens are known from
    the start: x[b] = (q, k, v) [length, heads, D]."""

    def __init__(self, lengths, Hq, Hk, D, page, dtype, kv, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.Hq, self.Hk, self.D, self.page = lengths, Hq, Hk, D, page
        self.x = [[torch.randn(n, h, D, generator=g).to(dtype) for h in (Hq, Hk, Hk)]
                  for n in lengths]
        self.w = [1 + 0.1 * torch.randn(D, generator=g) for _ in range(2)]
        self.cos, self.sin = _tables(max(lengths), D)
        # a cache of the whole lengths gives the tables; its pools start as NaN
        self.cache = Cache([(n, n) for n in lengths], Hk, D, page, kv, seed=seed)
        self.cache.k.fill_(float("nan"))
        self.cache.v.fill_(float("nan"))
        (self.k, self.v, self.table, _, _), self.scales = self.cache.to_gpu()
        self.dev = dict(cos=self.cos.cuda(), sin=self.sin.cuda(), q_weight=self.w[0].cuda(),
                        k_weight=self.w[1].cuda())

    def batch(self, spans):
        """(q, k, v, lens, cu) on the device of tokens start .. end - 1 of each
        sequence."""
        q, k, v = (torch.cat([x[i][s:e] for x, (s, e) in zip(self.x, spans)]).cuda()
                   for i in range(3))
        lens = torch.tensor([e for _, e in spans], dtype=torch.int32)
        cu = torch.tensor([0] + [e - s for s, e in spans], dtype=torch.int32).cumsum(0)
        return q, k, v, lens.cuda(), cu.to(torch.int32).cuda()

    def step(self, spans):
        q, k, v, lens, cu = self.batch(spans)
        qr = ops.kv_append_paged(k, v, self.k, self.v, self.table, lens, cu, q=q, **self.dev,
                                 **self.scales)
        o, lse = ops.attention_paged(qr, self.k, self.v, self.table, lens, cu, return_lse=True,
                                     max_seq_len=max(self.lengths), **self.scales)
        return qr, o, lse

    def view(self, spans):
        """The cache as it is now, with these new tokens, for check_attention."""
        c = self.cache
        c.k, c.v = self.k.cpu(), self.v.cpu()
        c.batch = [(e - s, e) for s, e in spans]
        c.cu = torch.tensor([0] + [e - s for s, e in spans]).cumsum(0).to(torch.int32)
        return c


@pytest.mark.parametrize("Hq,Hk,D,page,dtype,kv", [
    (8, 2, 128, 64, BF16, BF16), (4, 4, 64, 16, F16, F16), (8, 2, 128, 32, BF16, FP8)], ids=str)
def test_chunks_then_tokens(Hq, Hk, D, page, dtype, kv):
    e = Engine([300, 41, 555], Hq, Hk, D, page, dtype, kv)
    at = [0, 0, 0]
    for new in ([200, 0, 3], [97, 40, 500], [1, 1, 1], [2, 0, 7], [0, 0, 44]):
        spans = [(a, a + n) for a, n in zip(at, new)]
        qr, o, lse = e.step(spans)
        at = [s[1] for s in spans]
        # queries: norm and rotation at their places
        for i, (s, t) in enumerate(spans):
            r0 = sum(b - a for a, b in spans[:i])
            want, spread = rotate64(e.x[i][0][s:t], e.w[0], e.cos, e.sin, torch.arange(s, t), False,
                                    1e-6)
            err = (qr[r0:r0 + t - s].cpu().double() - want).abs()
            assert (err <= rotate_bound(want, spread, dtype)).all()
        # attention over what the cache now holds
        check_attention(e.view(spans), qr.cpu(), o.cpu(), lse.cpu())
    assert at == e.lengths
    if kv != FP8:  # the cache holds every key, rotated, and every value
        c = e.view([(0, n) for n in e.lengths])
        for b, n in enumerate(e.lengths):
            want, spread = rotate64(e.x[b][1], e.w[1], e.cos, e.sin, torch.arange(n), False, 1e-6)
            err = (c.values(b, "k").permute(1, 0, 2) - want).abs()
            assert (err <= rotate_bound(want, spread, dtype)).all()
            assert torch.equal(c.values(b, "v").permute(1, 0, 2), e.x[b][2].double())


def test_a_prompt_agrees_with_contiguous_attention():
    """qk_norm_rope + attention over [B, H, S, D] and append + attention_paged
    are one layer's prompt both ways."""
    e = Engine([257, 257], 8, 2, 128, 64, BF16, BF16)
    spans = [(0, 257)] * 2
    qr, o, _ = e.step(spans)
    q, k, v = (torch.stack([x[i] for x in e.x]).cuda().transpose(1, 2) for i in range(3))
    pos = torch.arange(257, dtype=torch.int32, device="cuda").repeat(2, 1)
    q2, k2 = ops.qk_norm_rope(q, k, e.dev["cos"], e.dev["sin"], pos, q_weight=e.dev["q_weight"],
                              k_weight=e.dev["k_weight"])
    assert torch.equal(q2.transpose(1, 2).reshape(514, 8, 128), qr)
    o2 = ops.attention(q2, k2, v, causal=True)
    # both within the bound of the same 64-bit attention
    o2 = o2.transpose(1, 2).reshape(514, 8, 128)
    check_attention(e.view(spans), qr.cpu(), o2.cpu(), None)
    check_attention(e.view(spans), qr.cpu(), o.cpu(), None)


def test_decode_paged_reads_what_append_wrote():
    for kv in (BF16, FP8):
        e = Engine([130, 700], 8, 2, 128, 64, BF16, kv)
        e.step([(0, 129), (0, 699)])
        spans = [(129, 130), (699, 700)]
        qr, o, lse = e.step(spans)
        table = e.table.clamp(0, e.cache.pages - 1)
        o2, lse2 = ops.decode_paged(qr, e.k, e.v, table, torch.tensor([130, 700], dtype=torch.int32,
                                    device="cuda"), max_seq_len=700, return_lse=True, **e.scales)
        check_attention(e.view(spans), qr.cpu(), o.cpu(), lse.cpu())
        check_attention(e.view(spans), qr.cpu(), o2.cpu(), lse2.cpu())


class Static:
    """A step's buffers for capture: 24 rows at most over 3 sequences, cut
    keys."""

    def __init__(self, e):
        self.e = e
        self.q = torch.zeros(24, e.Hq, e.D, dtype=BF16, device="cuda")
        self.k, self.v = (torch.zeros(24, e.Hk, e.D, dtype=BF16, device="cuda") for _ in range(2))
        self.lens = torch.zeros(3, dtype=torch.int32, device="cuda")
        self.cu = torch.zeros(4, dtype=torch.int32, device="cuda")
        need = ops.attention_paged_workspace_bytes(24, 3, e.Hq, e.Hk, e.D, max(e.lengths),
                                                   fp8=bool(e.scales))
        assert need > 0
        self.workspace = torch.empty(need, dtype=torch.uint8, device="cuda")

    def load(self, spans):
        q, k, v, lens, cu = self.e.batch(spans)
        for dst, src in ((self.q, q), (self.k, k), (self.v, v)):
            dst.zero_()
            dst[:src.shape[0]].copy_(src)
        self.lens.copy_(lens)
        self.cu.copy_(cu)

    def run(self, out, qr, workspace):
        e = self.e
        ops.kv_append_paged(self.k, self.v, e.k, e.v, e.table, self.lens, self.cu, q=self.q,
                            out=qr, **e.dev, **e.scales)
        return ops.attention_paged(qr, e.k, e.v, e.table, self.lens, self.cu, out=out,
                                   return_lse=True, max_seq_len=max(e.lengths),
                                   workspace=workspace, **e.scales)


@pytest.mark.parametrize("kv", [BF16, FP8], ids=str)
def test_graphs_that_share_a_workspace(kv):
    """Two captured steps with one workspace, replayed in turn with new tokens,
    lengths and paddings; eager steps and synchronizations in between. Every
    replay equals the eager step on the same cache bit for bit."""
    e = Engine([900, 64, 2500], 8, 2, 128, 64, BF16, kv)
    e.step([(0, 800), (0, 20), (0, 2400)])
    s = Static(e)
    outs, qrs = ([torch.full((24, 8, 128), -7.0, dtype=BF16, device="cuda") for _ in range(2)]
                 for _ in range(2))
    s.load([(800, 801), (20, 21), (2400, 2401)])
    s.run(outs[0], qrs[0], s.workspace)  # first call, eager
    torch.cuda.synchronize()
    graphs, lses = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            lses.append(s.run(outs[i], qrs[i], s.workspace)[1])
        graphs.append(g)
    at = [801, 21, 2401]
    for n, new in enumerate(([1, 1, 1], [5, 0, 9], [0, 7, 16], [1, 1, 1], [8, 8, 8])):
        spans = [(a, a + k) for a, k in zip(at, new)]
        at = [t for _, t in spans]
        s.load(spans)
        i, rows = n % 2, sum(new)
        outs[i].fill_(-7.0)
        qrs[i].fill_(0.5)
        graphs[i].replay()
        got, lse = outs[i].clone(), lses[i].clone()
        torch.cuda.synchronize()
        out, qr = torch.full_like(outs[i], -7.0), torch.full_like(qrs[i], 0.5)
        want, wlse = s.run(out, qr, None)
        assert torch.equal(got, want) and torch.equal(lse[:rows], wlse[:rows])
        assert (got[rows:] == -7.0).all() and torch.equal(qrs[i], qr)
        check_attention(e.view(spans), qr[:rows].cpu(), got[:rows].cpu(), lse[:rows].cpu())


def _thread_work(e, spans, stream):
    with torch.cuda.stream(stream):
        r = [e.step(s) for s in spans]
    stream.synchronize()
    return r


def test_threads_on_own_streams():
    """Three engines at once, each from its own thread and stream, give what
    they give one after another."""
    spans = [[(0, 150), (0, 600)], [(150, 151), (600, 601)], [(151, 170), (601, 602)]]
    kinds = [(BF16, BF16), (F16, F16), (BF16, FP8)]

    def engines():
        return [Engine([170, 602], 8, 2, 128, 64, d, kv, seed=i)
                for i, (d, kv) in enumerate(kinds)]

    torch.cuda.synchronize()
    want = [_thread_work(e, spans, torch.cuda.Stream()) for e in engines()]
    es, got = engines(), [None] * 3
    torch.cuda.synchronize()

    def run(i):
        got[i] = _thread_work(es[i], spans, torch.cuda.Stream())

    threads = [threading.Thread(target=run, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    for w, g in zip(want, got):
        for a, b in zip(w, g):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_callers_workspace():
    e = Engine([3000], 8, 2, 128, 64, BF16, BF16)
    e.step([(0, 2999)])
    q, k, v, lens, cu = e.batch([(2999, 3000)])
    qr = ops.kv_append_paged(k, v, e.k, e.v, e.table, lens, cu, q=q, **e.dev)
    need = ops.attention_paged_workspace_bytes(1, 1, 8, 2, 128, 3000)
    assert need > 0
    args = (qr, e.k, e.v, e.table, lens, cu)
    want = ops.attention_paged(*args, max_seq_len=3000)
    for fill in (0, 255):  # it needs no clearing
        ws = torch.full((need + 512,), fill, dtype=torch.uint8, device="cuda")
        assert torch.equal(ops.attention_paged(*args, max_seq_len=3000, workspace=ws[:need]), want)
        assert (ws[need:] == fill).all(), "bytes behind the workspace were written"
    with pytest.raises(_abi.NeptuneWorkspaceTooSmall):
        ops.attention_paged(*args, max_seq_len=3000, workspace=ws[:need - 1])
    with pytest.raises(_abi.NeptuneUnsupported, match="aligned"):
        ops.attention_paged(*args, max_seq_len=3000, workspace=ws[8:need + 8])
    with pytest.raises(ValueError, match="device tensors"):
        ops.attention_paged(*args, max_seq_len=3000, workspace=torch.empty(need))


def test_bad_tables_and_lengths_stay_in_bounds():
    """cu_seqlens that go back or past the rows, lengths past the table, tables
    of garbage: results are meaningless, memory outside the tensors is not
    touched (rows around them keep their values)."""
    e = Engine([200, 200], 8, 2, 128, 64, BF16, BF16)
    e.step([(0, 200), (0, 200)])
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.ones(40, 8, 128, dtype=BF16, device="cuda")
    k = torch.ones(40, 2, 128, dtype=BF16, device="cuda")
    guard = torch.full((60, 8, 128), 3.0, dtype=BF16, device="cuda")
    pools = [torch.full((e.cache.pages + 2, 2, 64, 128), 5.0, dtype=BF16, device="cuda")
             for _ in range(2)]
    for cu, lens in (([0, 30, 20], [200, 200]), ([-5, 100, 2**30], [200, 2**31 - 1]),
                     ([0, 20, 40], [-2**31, 10**6]), ([40, 0, 40], [2**30, 5])):
        cu, lens = torch.tensor(cu, **i32), torch.tensor(lens, **i32)
        for table in (e.table, torch.full_like(e.table, 2**31 - 1), torch.full_like(e.table, -9)):
            inner = [p[1:-1] for p in pools]
            out = guard[10:50]
            ops.kv_append_paged(k, k, *inner, table, lens, cu, q=q, out=out, cos=e.dev["cos"],
                                sin=e.dev["sin"])
            ops.attention_paged(q, *inner, table, lens, cu, out=out)
            torch.cuda.synchronize()
            assert (guard[:10] == 3.0).all() and (guard[50:] == 3.0).all()
            assert all((p[0] == 5.0).all() and (p[-1] == 5.0).all() for p in pools)
