"""Cases of the serving step around a paged KV cache, and what they compute.

Three operators of neptune_hip.ops, as one transformer layer of a serving
engine calls them between its projections:

* rope     qk_norm_rope: RMS norm of each query and key head with the position
           rotation in the same pass (f32, f16, bf16; half-split or
           interleaved pairs; the whole head or a part of it rotated);
* append   kv_append_paged: the new tokens' keys and values into their pages,
           keys normalised and rotated on the way, queries with them (bf16 and
           f16 pools, E4M3 pools with one scale per page and head);
* attend   attention_paged: a ragged batch of new tokens, one to thousands for
           each sequence, over the paged cache that holds them already.

Activations are N(0, 1), as projections after a norm give; norm weights are
1 + 0.1 N(0, 1); pages lie in the pool in random order.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
           "fp8": torch.float8_e4m3fn}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2, "fp8": 1}
_EPS = 1e-6


def _ops():
    package = str(Path(__file__).resolve().parents[1] / "mlir-toy_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from neptune_hip import ops
    return ops


def _rope(name, dtype, B, S, Hq, Hk, D, rot, interleaved, norm, first):
    return dict(name=name, kind="rope", dtype=dtype, B=B, S=S, Hq=Hq, Hk=Hk, D=D, rot=rot,
                interleaved=interleaved, norm=norm, first=first)


def _append(name, dtype, kv, B, new, old, lens, Hq, Hk, D, page, layout, rot, interleaved, norm):
    return dict(name=name, kind="append", dtype=dtype, kv=kv, B=B, new=new, old=old, lens=lens,
                Hq=Hq, Hk=Hk, D=D, page=page, layout=layout, rot=rot, interleaved=interleaved,
                norm=norm)


def _attend(name, dtype, kv, B, new, old, lens, Hq, Hk, D, page, layout, lse):
    return dict(name=name, kind="attend", dtype=dtype, kv=kv, B=B, new=new, old=old, lens=lens,
                Hq=Hq, Hk=Hk, D=D, page=page, layout=layout, lse=lse)


def listed():
    return [
        # the smallest call: one generated token for each of a batch of users
        _rope("rope_step", "bf16", 16, 1, 32, 8, 128, 128, False, True, 2000),
        # a batch of whole prompts before attention over contiguous K and V
        _rope("rope_prompts", "bf16", 4, 4096, 32, 8, 128, 128, False, True, 0),
        # an evaluation in fp32: odd length, a part of a small head rotated
        _rope("rope_f32_part", "f32", 2, 1500, 12, 12, 64, 32, True, False, 0),
        # a decode step's cache write: one token for each sequence
        _append("append_step", "bf16", "bf16", 32, 1, 1000, "even", 32, 8, 128, 64, "head", 128,
                False, True),
        # prompts of uneven lengths entering a token-major cache
        _append("append_prompts", "bf16", "bf16", 5, 3001, 0, "ragged", 32, 8, 128, 64, "token",
                128, False, False),
        # chunks behind a shared prefix entering an E4M3 cache
        _append("append_fp8", "bf16", "fp8", 8, 250, 900, "ragged", 32, 8, 128, 32, "head", 64,
                True, True),
        # one user generating over a long document
        _attend("attend_one_long", "bf16", "bf16", 1, 1, 32767, "even", 32, 8, 128, 64, "head",
                False),
        # a batch that checks a few guessed tokens at a time
        _attend("attend_guessed", "bf16", "bf16", 16, 4, 8000, "ragged", 32, 8, 128, 64, "head",
                True),
        # the largest: whole prompts at the benchmark's lengths, just appended
        _attend("attend_prompts", "bf16", "bf16", 4, 4096, 0, "even", 32, 8, 128, 64, "head", True),
        # a chunk of one long prompt over what is cached of it
        _attend("attend_chunk", "bf16", "bf16", 1, 1000, 30000, "even", 32, 8, 128, 64, "token",
                False),
        # an engine's mixed batch over an E4M3 cache: one prompt's chunk beside
        # sequences that generate
        _attend("attend_fp8_mixed", "bf16", "fp8", 8, 500, 8000, "mixed", 32, 8, 128, 64, "head",
                False),
        # a small f16 model: head_dim 64, small pages, odd lengths
        _attend("attend_f16_d64", "f16", "f16", 6, 130, 1500, "ragged", 16, 4, 64, 48, "head",
                True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = ((32, 8), (32, 32), (32, 4), (16, 4), (16, 16), (12, 12), (8, 1), (8, 8), (4, 2), (28, 7))


def draw(rng):
    kind = rng.choice(("rope", "append", "attend", "attend"))
    Hq, Hk = rng.choice(_HEADS)
    D = rng.choice((64, 128, 128))
    if kind == "rope":
        B = _log_int(rng, 1, 32)
        S = _log_int(rng, 1, min(4096, 16384 // B))
        if rng.random() < 0.25:
            S = 1
        dtype = rng.choice(("f32", "f16", "bf16", "bf16"))
        if dtype == "f32":
            D = rng.choice((32, 64, 128))
            S = max(1, S // 2)
        rot = rng.choice((D, D, D // 2))
        return dict(kind=kind, dtype=dtype, B=B, S=S, Hq=Hq, Hk=Hk, D=D, rot=rot,
                    interleaved=rng.random() < 0.3, norm=rng.random() < 0.6,
                    first=rng.randrange(0, 30000))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    kv = "fp8" if dtype == "bf16" and rng.random() < 0.35 else dtype
    layout = rng.choice(("head", "head", "token"))
    if kind == "append":
        B = _log_int(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 1, min(4096, 16000 // B))
        return dict(kind=kind, dtype=dtype, kv=kv, B=B, new=new, old=rng.randrange(0, 1000),
                    lens=rng.choice(("even", "ragged", "mixed")), Hq=Hq, Hk=Hk, D=D,
                    page=rng.choice((16, 32, 64, 64, 96, 128)), layout=layout,
                    rot=rng.choice((D, D, D // 2)), interleaved=rng.random() < 0.3,
                    norm=rng.random() < 0.5)
    B = _log_int(rng, 1, 32)
    new = _log_int(rng, 1, min(3000, 16000 // B))
    if rng.random() < 0.25:
        new = rng.randrange(1, 9)
    # the rectangle of every sequence's longest chunk and cache stays under the
    # prompts' of the listed cases
    most = min(32000, 1_100_000_000 // (B * Hq * new), 300_000 // B)
    old = _log_int(rng, 1, max(most - new, 1)) - 1 if most > new else 0
    return dict(kind=kind, dtype=dtype, kv=kv, B=B, new=new, old=old,
                lens=rng.choice(("even", "ragged", "ragged", "mixed")), Hq=Hq, Hk=Hk, D=D,
                page=rng.choice((16, 32, 48, 64, 64, 128, 256)), layout=layout,
                lse=rng.random() < 0.5)


def _lengths(case):
    """(new tokens, cache length with them) of each sequence, by the case
    alone. even: all alike; ragged: new between a part and all of case["new"],
    old between an eighth and all of case["old"]; mixed: every sequence but one
    in eight has a single new token."""
    B, new, old = case["B"], case["new"], case["old"]
    if case["lens"] == "even":
        return [new] * B, [old + new] * B
    rng = random.Random(f"{B} {new} {old} {case['Hq']} {case['page']}")
    if case["lens"] == "mixed":
        n = [new if b % 8 == 0 else 1 for b in range(B)]
    else:
        n = [rng.randint(max(1, new // 4), new) for _ in range(B)]
    o = [rng.randint(old // 8, old) for _ in range(B)]
    o[rng.randrange(B)] = old
    return n, [a + b for a, b in zip(n, o)]


def _tables(positions, rot):
    """cos and sin [positions, rot / 2] of the usual angles, base 10000."""
    i = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    p = torch.arange(positions, dtype=torch.float64, device="cuda")
    a = p[:, None] * torch.exp(-math.log(10000.0) * 2.0 * i / rot)[None, :]
    return torch.cos(a).float(), torch.sin(a).float()


def _pool(values, dtype, layout):
    """A pool's [pages, Hk, page, D] view of values(shape), stored head-major
    or token-major."""
    if layout == "token":
        return values("token").to(dtype).permute(0, 2, 1, 3)
    return values("head").to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    dtype = _DTYPES[case["dtype"]]
    Hq, Hk, D = case["Hq"], case["Hk"], case["D"]
    s = dict(case)
    if case["kind"] != "attend":
        s["q_weight"] = 1 + 0.1 * randn(D) if case["norm"] else None
        s["k_weight"] = 1 + 0.1 * randn(D) if case["norm"] else None
    if case["kind"] == "rope":
        B, S = case["B"], case["S"]
        s["cos"], s["sin"] = _tables(case["first"] + S, case["rot"])
        # as a projection leaves them: token by token, all heads of one together
        s["q"] = randn(B, S, Hq, D).to(dtype).transpose(1, 2)
        s["k"] = randn(B, S, Hk, D).to(dtype).transpose(1, 2)
        s["positions"] = (case["first"] + torch.arange(S, device="cuda", dtype=torch.int32)
                          ).repeat(B, 1)
        return s
    new, lens = _lengths(case)
    B, T, page = case["B"], sum(new), case["page"]
    pages = [-(-n // page) for n in lens]
    order = torch.randperm(sum(pages), generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(B, max(pages), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    s["block_table"] = table
    s["cu_seqlens"] = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32,
                                   device="cuda")
    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["max_seq_len"], s["max_new"] = max(lens), max(new)

    def values(layout):
        shape = (at, page, Hk, D) if layout == "token" else (at, Hk, page, D)
        x = randn(*shape)
        # the codes of N(0, 1) under scales of an absolute maximum near 4
        return (x * 112.0).clamp_(-448.0, 448.0) if case["kv"] == "fp8" else x

    s["k_pages"] = _pool(values, _DTYPES[case["kv"]], case["layout"])
    s["v_pages"] = _pool(values, _DTYPES[case["kv"]], case["layout"])
    s["k_scales"] = s["v_scales"] = None
    if case["kv"] == "fp8":
        s["k_scales"], s["v_scales"] = ((3.5 + torch.rand((at, Hk), generator=g, device="cuda"))
                                        / 448.0 for _ in range(2))
    s["q"] = randn(T, Hq, D).to(dtype)
    if case["kind"] == "append":
        s["cos"], s["sin"] = _tables(max(lens), case["rot"])
        s["k"], s["v"] = (randn(T, Hk, D).to(dtype) for _ in range(2))
    return s


def _rotated(x, weight, cos, sin, interleaved):
    """x [.., heads, D] normalised (with a weight) and rotated by cos, sin
    [.., 1, rot / 2], in fp32."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight
    half = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _rope_plain(s):
    p = s["positions"].long()
    cos, sin = s["cos"][p][:, None], s["sin"][p][:, None]
    return tuple(_rotated(s[x], s[x + "_weight"], cos, sin, s["interleaved"])
                 .to(s[x].dtype).contiguous() for x in ("q", "k"))


def _rows(s):
    """Sequence and position of every new row, the rows counted from the end
    of its sequence."""
    cu, lens = s["cu_seqlens"].long(), s["seq_lens"].long()
    row = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    return b, lens[b] - cu[1:][b] + row


def _append_plain(s):
    b, t = _rows(s)
    page = s["block_table"].long()[b, t // s["page"]]
    cos, sin = s["cos"][t][:, None], s["sin"][t][:, None]
    q = _rotated(s["q"], s["q_weight"], cos, sin, s["interleaved"]).to(s["q"].dtype)
    k = _rotated(s["k"], s["k_weight"], cos, sin, s["interleaved"])
    v = s["v"].float()
    if s["kv"] == "fp8":
        k = (k / s["k_scales"][page][..., None]).clamp(-448.0, 448.0)
        v = (v / s["v_scales"][page][..., None]).clamp(-448.0, 448.0)
        s["k_pages"].view(torch.uint8)[page, :, t % s["page"]] = \
            k.to(torch.float8_e4m3fn).view(torch.uint8)
        s["v_pages"].view(torch.uint8)[page, :, t % s["page"]] = \
            v.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        s["k_pages"][page, :, t % s["page"]] = k.to(s["k_pages"].dtype)
        s["v_pages"][page, :, t % s["page"]] = v.to(s["v_pages"].dtype)
    return q, s["k_pages"], s["v_pages"]


def _cached(s, name, page, place):
    """The tokens at (page, place) [B, L] of a pool as fp32 [B, Hk, L, D]."""
    pool = s[name + "_pages"]
    if s["kv"] == "fp8":
        x = pool.view(torch.uint8)[page, :, place].view(torch.float8_e4m3fn).float()
        x = x * s[name + "_scales"][page][..., None]
    else:
        x = pool[page, :, place].float()
    return x.permute(0, 2, 1, 3).contiguous()


def _attend_plain(s):
    Hq, Hk, D, new, L = s["Hq"], s["Hk"], s["D"], s["max_new"], s["max_seq_len"]
    group = Hq // Hk
    cu, lens = s["cu_seqlens"].long(), s["seq_lens"].long()
    B, n = lens.shape[0], cu[1:] - cu[:-1]
    key = torch.arange(L, device="cuda")
    i = torch.arange(new, device="cuda")
    # a sequence's tokens, those behind its end read from its last one
    token = torch.minimum(key[None, :], lens[:, None] - 1)
    page = s["block_table"].long().gather(1, token // s["page"])
    k, v = (_cached(s, name, page, token % s["page"]) for name in ("k", "v"))
    row = cu[:-1, None] + torch.minimum(i[None, :], n[:, None] - 1)
    q = s["q"][row].float().view(B, new, Hk, group, D).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q.reshape(B, Hk, group * new, D) * (1.0 / math.sqrt(D)), k.transpose(2, 3))
    seen = key <= (lens - n)[:, None, None] + i[None, :, None]
    x = x.view(B, Hk, group, new, L).masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hk, group * new, L), v).view(B, Hk, group, new, D) / total
    b, t = _rows(s)
    i = t - (lens - n)[b]
    o = o.permute(0, 3, 1, 2, 4)[b, i].reshape(-1, Hq, D).to(s["q"].dtype)
    if not s["lse"]:
        return o
    return o, (top + torch.log(total)).squeeze(-1).permute(0, 3, 1, 2)[b, i].reshape(-1, Hq)


def run(s):
    if own:
        ops = _ops()
        if s["kind"] == "rope":
            return ops.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["positions"],
                                    q_weight=s["q_weight"], k_weight=s["k_weight"], eps=_EPS,
                                    interleaved=s["interleaved"])
        if s["kind"] == "append":
            q = ops.kv_append_paged(s["k"], s["v"], s["k_pages"], s["v_pages"], s["block_table"],
                                    s["seq_lens"], s["cu_seqlens"], q=s["q"], cos=s["cos"],
                                    sin=s["sin"], interleaved=s["interleaved"],
                                    q_weight=s["q_weight"], k_weight=s["k_weight"], eps=_EPS,
                                    k_scales=s["k_scales"], v_scales=s["v_scales"])
            return q, s["k_pages"], s["v_pages"]
        return ops.attention_paged(s["q"], s["k_pages"], s["v_pages"], s["block_table"],
                                   s["seq_lens"], s["cu_seqlens"], max_seq_len=s["max_seq_len"],
                                   return_lse=s["lse"], k_scales=s["k_scales"],
                                   v_scales=s["v_scales"])
    if s["kind"] == "rope":
        return _rope_plain(s)
    if s["kind"] == "append":
        return _append_plain(s)
    return _attend_plain(s)


def work(case):
    Hq, Hk, D, w = case["Hq"], case["Hk"], case["D"], _BYTES[case["dtype"]]
    norm = 4 * D if case.get("norm") else 0  # operations of a head's norm
    if case["kind"] == "rope":
        rows = case["B"] * case["S"]
        table = case["S"] * case["rot"] * 4  # cos and sin of each position
        return {"bytes": 2 * rows * (Hq + Hk) * D * w + table + rows * 4,
                "flops": rows * (Hq + Hk) * (3 * case["rot"] + norm)}
    new, lens = _lengths(case)
    T, wk = sum(new), _BYTES[case["kv"]]
    tables = sum(-(-n // case["page"]) for n in lens) * 4 + case["B"] * 8
    if case["kind"] == "append":
        positions = set()
        for n, m in zip(new, lens):
            positions.update(range(m - n, m))
        return {"bytes": T * D * (2 * Hq * w + 2 * Hk * (w + wk)) + len(positions) * case["rot"] * 4
                + tables, "flops": T * (Hq + Hk) * (3 * case["rot"] + norm)}
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, lens))
    scales = 8 * Hk * sum(-(-m // case["page"]) for m in lens) if wk == 1 else 0
    return {"bytes": 2 * sum(lens) * Hk * D * wk + 2 * T * Hq * D * w + (T * Hq * 4 if case["lse"] else 0)
            + tables + scales, "flops": 4 * D * Hq * pairs}


def _exact_turn(x, weight, cos, sin, interleaved):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + _EPS) * weight.double()
    c, s = cos.double(), sin.double()
    half = c.shape[-1]
    first = torch.arange(half, device="cuda") * (2 if interleaved else 1)
    second = first + (1 if interleaved else half)
    z = torch.complex(x[..., first], x[..., second]) * torch.complex(c, s)
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        p = s["positions"][0].long()
        return tuple(_exact_turn(s[x], s[x + "_weight"], s["cos"][p], s["sin"][p],
                                 s["interleaved"]) for x in ("q", "k"))
    new, lens = _lengths(case)
    starts = [sum(new[:b]) for b in range(len(new))]
    if case["kind"] == "append":
        pools = [s["k_pages"].double(), s["v_pages"].double()]
        q = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, (at, n, m) in enumerate(zip(starts, new, lens)):
            t = torch.arange(m - n, m, device="cuda")
            page, place = s["block_table"][b, t // case["page"]].long(), t % case["page"]
            c, z = s["cos"][t][:, None], s["sin"][t][:, None]
            q[at:at + n] = _exact_turn(s["q"][at:at + n], s["q_weight"], c, z, s["interleaved"])
            rows = [_exact_turn(s["k"][at:at + n], s["k_weight"], c, z, s["interleaved"]),
                    s["v"][at:at + n].double()]
            for pool, x, name in zip(pools, rows, ("k_scales", "v_scales")):
                if case["kv"] == "fp8":
                    x = (x / s[name].double()[page][..., None]).clamp(-448, 448)
                pool[page, :, place] = x
        return q, pools[0], pools[1]
    Hq, Hk, D, page = case["Hq"], case["Hk"], case["D"], case["page"]
    group = Hq // Hk
    o = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for b, (at, n, m) in enumerate(zip(starts, new, lens)):
        ids = s["block_table"][b, :-(-m // page)].long()
        hide = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
        for h in range(Hk):
            k, v = (pool[:, h].view(torch.uint8)[ids].view(pool.dtype).double()
                    if case["kv"] == "fp8" else pool[:, h][ids].double()
                    for pool in (s["k_pages"], s["v_pages"]))
            if case["kv"] == "fp8":
                k = k * s["k_scales"].double()[ids, h][:, None, None]
                v = v * s["v_scales"].double()[ids, h][:, None, None]
            k, v = k.reshape(-1, D)[:m], v.reshape(-1, D)[:m]
            for j in range(group):
                x = s["q"][at:at + n, h * group + j].double() @ k.T / math.sqrt(D)
                x = x.masked_fill(hide, -math.inf)
                total = torch.logsumexp(x, -1)
                o[at:at + n, h * group + j] = torch.exp(x - total[:, None]) @ v
                lse[at:at + n, h * group + j] = total
    return (o, lse) if case["lse"] else o
