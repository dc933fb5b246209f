"""A serving step over a 4-bit cache as an engine takes it: new tokens quantised into
their pages, attention over them with capped, biased and windowed scores, the cache read
back; eager, captured, on other streams, from several threads, past 32-bit offsets, with
tables and lengths of garbage."""

import threading

import pytest
import torch

from mx_reference import MxCache, check_shaped, decode, encode, make_cache, shaped64
from neptune_hip import ops

pytestmark = pytest.mark.gpu

BF16, F16, U8 = torch.bfloat16, torch.float16, torch.uint8


@pytest.fixture(autouse=True)
def _needs_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")


class Engine:
    """Sequences of up to `lengths` tokens over MXFP4 pools of garbage."""

    def __init__(self, lengths, Hq, Hk, D, page, dtype, seed=0, layout="head", **form):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.Hq, self.Hk, self.D, self.page, self.dtype = lengths, Hq, Hk, D, page, dtype
        self.form = form
        # the table and an all-covered cache's shape
        self.cache = MxCache([(0, n) for n in lengths], Hk, D, page, layout=layout, seed=seed)
        for name in ("k", "v", "k_scales", "v_scales"):
            x = getattr(self.cache, name)
            setattr(self.cache, name, self.cache._lay(torch.randint(0, 256, x.shape, generator=g)
                                                      .to(U8)))
        (self.k, self.v, self.table, _, _), self.scales = self.cache.to_gpu()
        T = max(lengths)
        self.rows = [tuple(torch.randn(n, h, D, generator=g).to(dtype) for h in (Hq, Hk, Hk))
                     for n in lengths]
        a = torch.rand(T, D // 2, generator=g) * 6.28
        self.dev = dict(cos=torch.cos(a).cuda(), sin=torch.sin(a).cuda(),
                        q_weight=(1 + 0.1 * torch.randn(D, generator=g)).cuda(),
                        k_weight=(1 + 0.1 * torch.randn(D, generator=g)).cuda())

    def batch(self, spans):
        """q, k, v of the tokens spans[b] = (from, to), lengths and cu_seqlens."""
        q, k, v = (torch.cat([r[i][a:b] for r, (a, b) in zip(self.rows, spans)]).cuda()
                   for i in range(3))
        lens = torch.tensor([b for _, b in spans], dtype=torch.int32, device="cuda")
        cu = torch.tensor([0] + [b - a for a, b in spans], dtype=torch.int32, device="cuda")
        return q, k, v, lens, cu.cumsum(0).to(torch.int32)

    def step(self, spans):
        q, k, v, lens, cu = self.batch(spans)
        qr = ops.kv_append_paged(k, v, self.k, self.v, self.table, lens, cu, q=q, **self.dev,
                                 **self.scales)
        o, lse = ops.attention_paged(qr, self.k, self.v, self.table, lens, cu, return_lse=True,
                                     max_seq_len=max(self.lengths), **self.device_form(),
                                     **self.scales)
        return qr, o, lse

    def device_form(self):
        return {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in self.form.items()}

    def view(self, spans):
        """The cache as the GPU holds it, for 64-bit attention of spans."""
        torch.cuda.synchronize()
        c = self.cache
        c.batch = [(b - a, b) for a, b in spans]
        n = [b - a for a, b in spans]
        c.cu = torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32)
        c.tokens = sum(n)
        c.k, c.v = self.k.cpu(), self.v.cpu()
        c.k_scales, c.v_scales = (self.scales[x].cpu() for x in ("k_scales", "v_scales"))
        return c


def _slopes(Hq):
    return torch.exp2(-8.0 * (torch.arange(Hq) + 1) / Hq)


FORMS = [{}, dict(softcap=30.0), dict(window=90), dict(slopes=True, softcap=20.0, window=700)]


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("Hq,Hk,D,page,dtype,layout", [
    (8, 2, 128, 64, BF16, "head"), (12, 3, 64, 48, F16, "token"), (5, 5, 128, 16, F16, "head")])
def test_prompts_then_tokens(Hq, Hk, D, page, dtype, layout, form):
    if form.get("slopes"):
        form = dict(form, slopes=_slopes(Hq))
    e = Engine([140, 1100, 33], Hq, Hk, D, page, dtype, seed=D + page, layout=layout, **form)
    at = [0, 0, 0]
    for new in ([100, 900, 0], [1, 1, 30], [20, 150, 1], [1, 1, 1], [0, 4, 0]):
        spans = [(a, a + n) for a, n in zip(at, new)]
        at = [b for _, b in spans]
        qr, o, lse = e.step(spans)
        cache = e.view(spans)
        check_shaped(cache, qr.cpu(), o.cpu(), lse.cpu(), **form)
    # the cache read back, whole sequences and as the last step wrote it: what the codes
    # stand for, and for values what their own quantisation gives
    lens = torch.tensor(at, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0] + at, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
    k, v = ops.kv_read_paged(e.k, e.v, e.table, lens, cu, tokens=sum(at), dtype=torch.float32,
                             **e.scales)
    torch.cuda.synchronize()
    r0 = 0
    for b, n in enumerate(at):
        assert torch.equal(k[r0:r0 + n].cpu().double(), cache.values(b, "k").transpose(0, 1)[:n])
        assert torch.equal(v[r0:r0 + n].cpu().double(), decode(*encode(e.rows[b][2][:n].double())))
        r0 += n


def test_attention_over_what_is_read_back():
    """The prompt's rows read back through contiguous attention equal attention over the
    pages: both see the cache's values."""
    e = Engine([300], 8, 2, 128, 64, BF16)
    qr, o, _ = e.step([(0, 300)])
    lens = torch.tensor([300], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    k, v = ops.kv_read_paged(e.k, e.v, e.table, lens, cu, tokens=300, **e.scales)
    flat = ops.attention(qr.transpose(0, 1)[None], k.transpose(0, 1)[None], v.transpose(0, 1)[None],
                         causal=True)[0].transpose(0, 1)
    cache = e.view([(0, 300)])
    check_shaped(cache, qr.cpu(), flat.cpu(), None)
    check_shaped(cache, qr.cpu(), o.cpu(), None)


class Static:
    """A step's buffers for capture: 24 rows at most over 3 sequences, cut keys."""

    def __init__(self, e):
        self.e = e
        self.q = torch.zeros(24, e.Hq, e.D, dtype=e.dtype, device="cuda")
        self.k, self.v = (torch.zeros(24, e.Hk, e.D, dtype=e.dtype, device="cuda") for _ in range(2))
        self.lens = torch.zeros(3, dtype=torch.int32, device="cuda")
        self.cu = torch.zeros(4, dtype=torch.int32, device="cuda")
        self.form = e.device_form()
        need = ops.attention_paged_workspace_bytes(24, 3, e.Hq, e.Hk, e.D, max(e.lengths))
        assert need > 0
        self.workspace = torch.empty(need, dtype=U8, device="cuda")

    def load(self, spans):
        q, k, v, lens, cu = self.e.batch(spans)
        for dst, src in ((self.q, q), (self.k, k), (self.v, v)):
            dst.zero_()
            dst[:src.shape[0]].copy_(src)
        self.lens.copy_(lens)
        self.cu.copy_(cu)

    def run(self, out, qr, rows, workspace):
        e = self.e
        ops.kv_append_paged(self.k, self.v, e.k, e.v, e.table, self.lens, self.cu, q=self.q,
                            out=qr, **e.dev, **e.scales)
        ops.kv_read_paged(e.k, e.v, e.table, self.lens, self.cu, out=rows, **e.scales)
        return ops.attention_paged(qr, e.k, e.v, e.table, self.lens, self.cu, out=out,
                                   return_lse=True, max_seq_len=max(e.lengths),
                                   workspace=workspace, **self.form, **e.scales)


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_graphs_that_share_a_workspace(form):
    """Two captured steps with one workspace, replayed in turn with new tokens, lengths
    and paddings; eager steps and synchronizations in between. Every replay equals the
    eager step on the same cache bit for bit."""
    if form.get("slopes"):
        form = dict(form, slopes=_slopes(8))
    e = Engine([900, 64, 2500], 8, 2, 128, 64, BF16, **form)
    e.step([(0, 800), (0, 20), (0, 2400)])
    s = Static(e)

    def buffers():
        return (torch.full((24, 8, 128), -7.0, dtype=BF16, device="cuda"),
                torch.full((24, 8, 128), 0.5, dtype=BF16, device="cuda"),
                tuple(torch.full((24, 2, 128), 0.25, device="cuda") for _ in range(2)))

    sets = [buffers() for _ in range(2)]
    s.load([(800, 801), (20, 21), (2400, 2401)])
    s.run(*sets[0], s.workspace)  # first call, eager
    torch.cuda.synchronize()
    graphs, lses = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            lses.append(s.run(*sets[i], s.workspace)[1])
        graphs.append(g)
    at = [801, 21, 2401]
    for n, new in enumerate(([1, 1, 1], [5, 0, 9], [0, 7, 16], [1, 1, 1], [8, 8, 8])):
        spans = [(a, a + k) for a, k in zip(at, new)]
        at = [t for _, t in spans]
        s.load(spans)
        i, rows = n % 2, sum(new)
        for x, y in zip((*sets[i][:2], *sets[i][2]), (*buffers()[:2], *buffers()[2])):
            x.copy_(y)
        graphs[i].replay()
        got = [t.clone() for t in (*sets[i][:2], *sets[i][2])]
        lse = lses[i].clone()
        torch.cuda.synchronize()
        fresh = buffers()
        _, wlse = s.run(*fresh, None)
        for a, b in zip(got, (*fresh[:2], *fresh[2])):
            assert torch.equal(a, b)
        assert torch.equal(lse[:rows], wlse[:rows])
        assert (got[0][rows:] == -7.0).all() and (got[2][rows:] == 0.25).all()
        check_shaped(e.view(spans), got[1][:rows].cpu(), got[0][:rows].cpu(), lse[:rows].cpu(),
                     **form)


def test_threads_on_own_streams():
    """Engines at once, each from its own thread and stream, give what they give one
    after another."""
    spans = [[(0, 150), (0, 600)], [(150, 151), (600, 601)], [(151, 170), (601, 602)]]
    kinds = [(BF16, {}), (F16, dict(softcap=20.0)), (BF16, dict(window=100))]

    def engines():
        return [Engine([170, 602], 8, 2, 128, 64, d, seed=i, **f) for i, (d, f) in enumerate(kinds)]

    def work(e, stream):
        with torch.cuda.stream(stream):
            r = [e.step(s) for s in spans]
        stream.synchronize()
        return r

    torch.cuda.synchronize()
    want = [work(e, torch.cuda.Stream()) for e in engines()]
    es, got = engines(), [None] * 3
    torch.cuda.synchronize()

    def run(i):
        got[i] = work(es[i], torch.cuda.Stream())

    threads = [threading.Thread(target=run, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    for w, g in zip(want, got):
        for a, b in zip(w, g):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_the_same_twice():
    """Cut keys are joined in an order of their own: the same bits every time."""
    e = Engine([3000, 500], 8, 2, 128, 64, BF16, softcap=30.0)
    e.step([(0, 2990), (0, 499)])
    a = e.step([(2990, 2995), (499, 500)])
    for _ in range(5):
        b = e.step([(2990, 2995), (499, 500)])
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_past_32_bit_offsets():
    """Pages of codes and of scales that begin past 2^32 bytes of their pools."""
    page, D = 64, 128
    pages = (1 << 32) // (page * D // 2) + 1000
    codes = [torch.zeros(pages, 1, page, D // 2, dtype=U8, device="cuda") for _ in range(2)]
    # scales a page every 8 KiB
    scales = [torch.zeros(pages, 8192, dtype=U8, device="cuda")[:, :4 * page].view(pages, 1, page, 4)
              for _ in range(2)]
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(150, 1, D, generator=g).to(BF16) for _ in range(2))
    q = torch.randn(150, 4, D, generator=g).to(BF16)
    table = torch.tensor([[pages - 1, pages - 999, pages - 3]], dtype=torch.int32)
    lens = torch.tensor([150], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 150], dtype=torch.int32, device="cuda")
    kw = dict(k_scales=scales[0], v_scales=scales[1])
    args = (*codes, table.cuda(), lens, cu)
    ops.kv_append_paged(k.cuda(), v.cuda(), *args, **kw)
    kr, vr = ops.kv_read_paged(*args, tokens=150, dtype=torch.float32, **kw)
    o = ops.attention_paged(q.cuda(), *args, **kw)
    one = ops.attention_paged(q[-1:].cuda(), *codes, table.cuda(), lens, **kw)
    torch.cuda.synchronize()
    for x, r in ((k, kr), (v, vr)):
        assert torch.equal(r.cpu().double(), decode(*encode(x.double())))
    small = MxCache([(150, 150)], 1, D, page, seed=1)
    ids = small.table[0, :3].long()
    t = torch.arange(150)
    for name, x in (("k", k), ("v", v)):
        c, s = encode(x.double())
        getattr(small, name)[ids[t // page], 0, t % page] = c[:, 0]
        getattr(small, name + "_scales")[ids[t // page], 0, t % page] = s[:, 0]
    check_shaped(small, q, o.cpu(), None)
    want, _, bo, _ = shaped64(small, q)
    assert ((one.cpu().double()[0] - want[-1]).abs() <= bo[-1]).all()
    assert not codes[0][0].any() and not codes[0][pages - 2].any()


def test_bad_tables_and_lengths_stay_in_bounds():
    """cu_seqlens that go back or past the rows, lengths past the table, tables of
    garbage: results are meaningless, memory outside the tensors is not touched (rows
    around them keep their values)."""
    e = Engine([200, 200], 8, 2, 128, 64, BF16)
    e.step([(0, 200), (0, 200)])
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.ones(40, 8, 128, dtype=BF16, device="cuda")
    k = torch.ones(40, 2, 128, dtype=BF16, device="cuda")
    guard = torch.full((60, 8, 128), 3.0, dtype=BF16, device="cuda")
    rows = torch.full((60, 2, 2, 128), 3.0, dtype=BF16, device="cuda")
    pages = e.cache.pages
    pools = [torch.full((pages + 2, 2, 64, w), 5, dtype=U8, device="cuda") for w in (64, 64, 4, 4)]
    slopes = torch.full((8,), 0.5, device="cuda")
    for cu, lens in (([0, 30, 20], [200, 200]), ([-5, 100, 2**30], [200, 2**31 - 1]),
                     ([0, 20, 40], [-2**31, 10**6]), ([40, 0, 40], [2**30, 5])):
        cu, lens = torch.tensor(cu, **i32), torch.tensor(lens, **i32)
        for table in (e.table, torch.full_like(e.table, 2**31 - 1), torch.full_like(e.table, -9)):
            inner = [p[1:-1] for p in pools]
            out = guard[10:50]
            kw = dict(k_scales=inner[2], v_scales=inner[3])
            ops.kv_append_paged(k, k, *inner[:2], table, lens, cu, q=q, out=out, cos=e.dev["cos"],
                                sin=e.dev["sin"], **kw)
            ops.kv_read_paged(*inner[:2], table, lens, cu, out=(rows[10:50, 0], rows[10:50, 1]), **kw)
            for form in ({}, dict(softcap=20.0, slopes=slopes, window=50)):
                ops.attention_paged(q, *inner[:2], table, lens, cu, out=out, **form, **kw)
            torch.cuda.synchronize()
            for x in (guard, rows):
                assert (x[:10] == 3.0).all() and (x[50:] == 3.0).all()
            assert all((p[0] == 5).all() and (p[-1] == 5).all() for p in pools)


@pytest.mark.parametrize("kind", ["mx", BF16], ids=str)
def test_many_sequences(kind):
    """More sequences than a wave has lanes, most of one new token."""
    batch = [(1 + 3 * (b % 17 == 0), 1 + 7 * b % 300) for b in range(150)]
    batch = [(min(n, length), length) for n, length in batch]
    cache = make_cache(kind, batch, 2, 64, 16, seed=8)
    q = torch.randn(cache.tokens, 8, 64, generator=torch.Generator().manual_seed(1)).to(BF16)
    args, scales = cache.to_gpu()
    for form in ({}, dict(window=64, softcap=10.0)):
        o, lse = ops.attention_paged(q.cuda(), *args, return_lse=True, max_seq_len=cache.max_len,
                                     **form, **scales)
        torch.cuda.synchronize()
        check_shaped(cache, q, o.cpu(), lse.cpu(), **form)


@pytest.mark.parametrize("group", [3, 16, 17, 31, 33, 200])
def test_groups(group):
    """Query heads of a key head around the forms' 16 and 32 rows, and past a tile."""
    cache = make_cache("mx", [(1, 300), (2, 90), (3, 1000)], 1, 128, 32, seed=group)
    q = torch.randn(cache.tokens, group, 128, generator=torch.Generator().manual_seed(1)).to(F16)
    args, scales = cache.to_gpu()
    slopes = _slopes(group)
    for form in ({}, dict(softcap=15.0, slopes=slopes)):
        dev = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in form.items()}
        o, lse = ops.attention_paged(q.cuda(), *args, return_lse=True, max_seq_len=cache.max_len,
                                     **dev, **scales)
        torch.cuda.synchronize()
        check_shaped(cache, q, o.cpu(), lse.cpu(), **form)
