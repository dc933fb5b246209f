"""Cases of a serving step over a 4-bit paged cache, and what they compute.

What neptune_hip.ops does for a cache of MXFP4 pools (E2M1 codes, two to a byte,
under one E8M0 scale for 32 elements of a head row), and for scores that are not
plain products:

* append   kv_append_paged: the new tokens' keys and values quantised as they are
           written, keys normalised and rotated on the way, queries with them; the
           rows are then read back (kv_read_paged), so that what the cache holds
           comes out as the values it stands for;
* read     kv_read_paged: cached tokens back as rows, of MXFP4 and E4M3 pools;
* attend   attention_paged over MXFP4 pools, one to thousands of new tokens a
           sequence;
* scores   attention_paged with scores capped by a tanh, with a bias that grows
           with the distance, within a sliding window; over 16-bit, E4M3 and MXFP4
           pools.

Activations are N(0, 1), as projections after a norm give; norm weights are
1 + 0.1 N(0, 1); pages lie in the pool in random order; cached tokens are quantised
N(0, 1).
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4.0, "f16": 2.0, "bf16": 2.0, "fp8": 1.0, "mx": 17.0 / 32.0}
_EPS = 1e-6
_BLOCK = 32


def _ops():
    package = str(Path(__file__).resolve().parents[1] / "mlir-toy_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from neptune_hip import ops
    return ops


def _append(name, dtype, B, new, old, lens, Hq, Hk, D, page, layout, rot, interleaved, norm):
    return dict(name=name, kind="append", dtype=dtype, kv="mx", B=B, new=new, old=old, lens=lens,
                Hq=Hq, Hk=Hk, D=D, page=page, layout=layout, rot=rot, interleaved=interleaved,
                norm=norm)


def _read(name, dtype, kv, B, new, old, lens, Hk, D, page, layout):
    return dict(name=name, kind="read", dtype=dtype, kv=kv, B=B, new=new, old=old, lens=lens,
                Hq=Hk, Hk=Hk, D=D, page=page, layout=layout)


def _attend(name, dtype, kv, B, new, old, lens, Hq, Hk, D, page, layout, lse, cap=0.0,
            slopes=False, window=0):
    return dict(name=name, kind="attend", dtype=dtype, kv=kv, B=B, new=new, old=old, lens=lens,
                Hq=Hq, Hk=Hk, D=D, page=page, layout=layout, lse=lse, cap=cap, slopes=slopes,
                window=window)


def listed():
    return [
        # the smallest: a decode step's cache write, one token for each sequence
        _append("append_step", "bf16", 32, 1, 1000, "even", 32, 8, 128, 64, "head", 128, False,
                True),
        # prompts of uneven lengths entering a token-major cache
        _append("append_prompts", "bf16", 5, 3001, 0, "ragged", 32, 8, 128, 64, "token", 128,
                False, False),
        # chunks of a small f16 model, a part of each head rotated
        _append("append_f16_d64", "f16", 8, 250, 900, "ragged", 16, 4, 64, 48, "head", 32, True,
                True),
        # one sequence's cached prefix as rows, for attention over contiguous keys
        _read("read_prefix", "bf16", "mx", 1, 2000, 0, "even", 8, 128, 64, "head"),
        # a batch of long sequences leaving the cache
        _read("read_batch", "bf16", "mx", 16, 8000, 0, "ragged", 8, 128, 64, "head"),
        # one user generating over a long document
        _attend("attend_one_long", "bf16", "mx", 1, 1, 32767, "even", 32, 8, 128, 64, "head",
                False),
        # a batch of users generating
        _attend("attend_step", "bf16", "mx", 32, 1, 8000, "ragged", 32, 8, 128, 64, "head", False),
        # an engine's mixed batch of a small f16 model: a prompt's chunk beside
        # sequences that generate, odd pages
        _attend("attend_f16_mixed", "f16", "mx", 8, 500, 8000, "mixed", 16, 4, 64, 48, "token",
                True),
        # the largest: whole prompts at the benchmark's lengths, just appended
        _attend("attend_prompts", "bf16", "mx", 4, 4096, 0, "even", 32, 8, 128, 64, "head", True),
        # a few guessed tokens at a time, capped scores within a window
        _attend("scores_guessed", "bf16", "bf16", 16, 4, 8000, "ragged", 32, 8, 128, 64, "head",
                True, cap=50.0, window=4096),
        # a chunk of one long prompt, a bias by distance, a key head for each query head
        _attend("scores_biased_chunk", "f16", "f16", 1, 1000, 12000, "even", 16, 16, 128, 64,
                "token", False, slopes=True),
        # chunks over a 4-bit cache, capped
        _attend("scores_capped_mx", "bf16", "mx", 4, 700, 5000, "ragged", 32, 8, 128, 64, "head",
                False, cap=30.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = ((32, 8), (32, 32), (32, 4), (16, 4), (16, 16), (12, 12), (8, 1), (8, 8), (4, 2), (28, 7))


def draw(rng):
    kind = rng.choice(("append", "read", "attend", "attend", "scores", "scores"))
    Hq, Hk = rng.choice(_HEADS)
    D = rng.choice((64, 128, 128))
    page = rng.choice((16, 32, 48, 64, 64, 96, 128, 256))
    layout = rng.choice(("head", "head", "token"))
    lens = rng.choice(("even", "ragged", "ragged", "mixed"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    if kind == "append":
        B = _log_int(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log_int(rng, 1, min(4096, 16000 // B))
        return dict(kind=kind, dtype=dtype, kv="mx", B=B, new=new, old=rng.randrange(0, 1000),
                    lens=lens, Hq=Hq, Hk=Hk, D=D, page=page, layout=layout,
                    rot=rng.choice((D, D, D // 2, 24)), interleaved=rng.random() < 0.3,
                    norm=rng.random() < 0.5)
    if kind == "read":
        B = _log_int(rng, 1, 64)
        new = _log_int(rng, 1, min(16000, 500_000 // (B * Hk)))
        return dict(kind=kind, dtype=rng.choice(("bf16", "f16", "f32")),
                    kv=rng.choice(("mx", "mx", "fp8")), B=B, new=new, old=rng.randrange(0, 300),
                    lens=lens, Hq=Hk, Hk=Hk, D=D, page=page, layout=layout)
    B = _log_int(rng, 1, 32)
    new = _log_int(rng, 1, min(3000, 16000 // B))
    if rng.random() < 0.3:
        new = rng.randrange(1, 9)
    # the rectangle of every sequence's longest chunk and cache stays under the
    # prompts' of the listed cases
    most = min(32000, 1_100_000_000 // (B * Hq * new), 300_000 // B)
    old = _log_int(rng, 1, max(most - new, 1)) - 1 if most > new else 0
    case = dict(kind="attend", dtype=dtype, kv="mx", B=B, new=new, old=old, lens=lens, Hq=Hq,
                Hk=Hk, D=D, page=page, layout=layout, lse=rng.random() < 0.5, cap=0.0,
                slopes=False, window=0)
    if kind == "scores":
        case["kv"] = rng.choice((dtype, dtype, "mx", "fp8" if dtype == "bf16" else "mx"))
        form = rng.randrange(1, 8)  # a cap, slopes, a window, or several of them
        case["cap"] = rng.choice((20.0, 30.0, 50.0)) if form & 1 else 0.0
        case["slopes"] = form & 2 != 0
        case["window"] = _log_int(rng, 1, 6000) if form & 4 else 0
    return case


def _lengths(case):
    """(new tokens, cache length with them) of each sequence, by the case
    alone. even: all alike; ragged: new between a part and all of case["new"],
    old between an eighth and all of case["old"]; mixed: every sequence but one
    in eight has a single new token."""
    B, new, old = case["B"], case["new"], case["old"]
    if case["lens"] == "even":
        return [new] * B, [old + new] * B
    rng = random.Random(f"{B} {new} {old} {case['Hk']} {case['page']}")
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


def _quantised(x):
    """x [.., D] in 32 or 64 bits as (codes uint8 [.., D / 2], scales uint8 [.., D / 32]). A
    block's scale is 2^(e - 2), e the exponent of its largest magnitude rounded to two
    significant bits, so that what passes 6 scales passes it by a sixth at most."""
    b = x.unflatten(-1, (-1, _BLOCK))
    top = b.abs().amax(-1).float()
    e = ((top.view(torch.int32) + 0x200000) >> 23) - 2
    none = top < 2.0 ** -123
    e = torch.where(none, torch.zeros_like(e), e)
    # times 2^(127 - e), in two steps that are both ordinary numbers
    half = (127 - e) >> 1
    rest = 127 - e - half
    y = b * _two_to(half)[..., None] * _two_to(rest)[..., None]
    a = y.abs()
    code = torch.zeros(a.shape, dtype=torch.uint8, device=x.device)
    # nearest, halves to the even code
    for edge, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False),
                     (3.5, True), (5.0, False)):
        code += (a >= edge) if up else (a > edge)
    code |= (y < 0).to(torch.uint8) << 3
    code = torch.where(none[..., None], torch.zeros_like(code), code).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, e.to(torch.uint8)


def _two_to(e):
    """2^e as float32 for integers e in -126 .. 127."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _dequantised(codes, scales):
    """fp32 values of codes [.., D / 2] under scales [.., D / 32]."""
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=codes.device)
    x = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1).flatten(-2)
    two = _two_to(scales.to(torch.int32).clamp_min(1) - 127)
    return (x.unflatten(-1, (-1, _BLOCK)) * two[..., None]).flatten(-2)


def _pool(x, layout):
    """x [pages, page, Hk, ..] as a [pages, Hk, page, ..] view, stored head-major or
    token-major."""
    x = x.permute(0, 2, 1, 3)
    return x if layout == "token" else x.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    dtype, kv = _DTYPES[case["dtype"]], case["kv"]
    Hq, Hk, D, page = case["Hq"], case["Hk"], case["D"], case["page"]
    s = dict(case)
    new, lens = _lengths(case)
    B, T = case["B"], sum(new)
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
    s["tokens"], s["max_seq_len"], s["max_new"] = T, max(lens), max(new)
    for name in ("k", "v"):
        x = randn(at, page, Hk, D)
        if kv == "mx":
            codes, scales = _quantised(x)
            s[name + "_pages"] = _pool(codes, case["layout"])
            s[name + "_scales"] = _pool(scales, case["layout"])
        elif kv == "fp8":
            # the codes of N(0, 1) under scales of an absolute maximum near 4
            s[name + "_pages"] = _pool((x * 112.0).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn),
                                       case["layout"])
            s[name + "_scales"] = (3.5 + torch.rand((at, Hk), generator=g, device="cuda")) / 448.0
        else:
            s[name + "_pages"] = _pool(x.to(dtype), case["layout"])
            s[name + "_scales"] = None
    if case["kind"] == "append":
        s["q_weight"] = 1 + 0.1 * randn(D) if case["norm"] else None
        s["k_weight"] = 1 + 0.1 * randn(D) if case["norm"] else None
        s["cos"], s["sin"] = _tables(max(lens), case["rot"])
        s["k"], s["v"] = (randn(T, Hk, D).to(dtype) for _ in range(2))
    if case["kind"] != "read":
        s["q"] = randn(T, Hq, D).to(dtype)
    if case["kind"] == "attend":
        # slopes 2^(-8 (h + 1) / heads)
        h = torch.arange(Hq, device="cuda")
        s["slopes"] = torch.exp2(-8.0 * (h + 1) / Hq).float() if case["slopes"] else None
    return s


def _rotated(x, weight, cos, sin, interleaved):
    """x [.., heads, D] in 32 or 64 bits normalised (with a weight) and rotated by
    cos, sin [.., 1, rot / 2]."""
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


def _rows(s):
    """Sequence and position of every new row, the rows counted from the end
    of its sequence."""
    cu, lens = s["cu_seqlens"].long(), s["seq_lens"].long()
    row = torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    return b, lens[b] - cu[1:][b] + row


def _held(s, name, page, place):
    """The tokens at (page, place) of a pool as fp32 [.., Hk, D]."""
    pool, scales = s[name + "_pages"], s[name + "_scales"]
    if s["kv"] == "mx":
        return _dequantised(pool[page, :, place], scales[page, :, place])
    if s["kv"] == "fp8":
        x = pool.view(torch.uint8)[page, :, place].view(torch.float8_e4m3fn).float()
        return x * scales[page][..., None]
    return pool[page, :, place].float()


def _read_plain(s, dtype):
    b, t = _rows(s)
    page = s["block_table"].long()[b, t // s["page"]]
    return tuple(_held(s, name, page, t % s["page"]).to(dtype) for name in ("k", "v"))


def _append_plain(s):
    b, t = _rows(s)
    page = s["block_table"].long()[b, t // s["page"]]
    cos, sin = s["cos"][t][:, None], s["sin"][t][:, None]
    q = _rotated(s["q"].float(), s["q_weight"], cos, sin, s["interleaved"]).to(s["q"].dtype)
    # in 64 bits: a key next to the border of two codes goes to the nearer one
    k = _rotated(s["k"].double(), s["k_weight"], cos, sin, s["interleaved"])
    for name, x in (("k", k), ("v", s["v"].float())):
        codes, scales = _quantised(x)
        s[name + "_pages"][page, :, t % s["page"]] = codes
        s[name + "_scales"][page, :, t % s["page"]] = scales
    return (q,) + _read_plain(s, torch.bfloat16)


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
    k, v = (_held(s, name, page, token % s["page"]).permute(0, 2, 1, 3).contiguous()
            for name in ("k", "v"))
    row = cu[:-1, None] + torch.minimum(i[None, :], n[:, None] - 1)
    q = s["q"][row].float().view(B, new, Hk, group, D).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q.reshape(B, Hk, group * new, D) * (1.0 / math.sqrt(D)),
                     k.transpose(2, 3).contiguous())
    x = x.view(B, Hk, group, new, L)
    if s["cap"]:
        x = x.div_(s["cap"]).tanh_().mul_(s["cap"])
    place = (lens - n)[:, None, None] + i[None, :, None]  # [B, new, 1]
    if s["slopes"] is not None:
        far = (key - place).float()  # [B, new, L]
        for h in range(Hq):
            x[:, h // group, h % group] += s["slopes"][h] * far
    seen = key <= place
    if s["window"]:
        seen &= key > place - s["window"]
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
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
    if not own:
        if s["kind"] == "read":
            return _read_plain(s, _DTYPES[s["dtype"]])
        return _append_plain(s) if s["kind"] == "append" else _attend_plain(s)
    ops = _ops()
    pools = (s["k_pages"], s["v_pages"], s["block_table"], s["seq_lens"], s["cu_seqlens"])
    scales = dict(k_scales=s["k_scales"], v_scales=s["v_scales"])
    if s["kind"] == "attend":
        return ops.attention_paged(s["q"], *pools, max_seq_len=s["max_seq_len"],
                                   return_lse=s["lse"], softcap=s["cap"] or None,
                                   slopes=s["slopes"], window=s["window"] or None, **scales)
    if s["kind"] == "read":
        return ops.kv_read_paged(*pools, tokens=s["tokens"], dtype=_DTYPES[s["dtype"]], **scales)
    q = ops.kv_append_paged(s["k"], s["v"], *pools, q=s["q"], cos=s["cos"], sin=s["sin"],
                            interleaved=s["interleaved"], q_weight=s["q_weight"],
                            k_weight=s["k_weight"], eps=_EPS, **scales)
    # (bf16 holds whatever the codes stand for)
    return (q,) + ops.kv_read_paged(*pools, tokens=s["tokens"], dtype=torch.bfloat16, **scales)


def work(case):
    Hq, Hk, D, w = case["Hq"], case["Hk"], case["D"], _BYTES[case["dtype"]]
    new, lens = _lengths(case)
    T, wk = sum(new), _BYTES[case["kv"]]
    tables = sum(-(-n // case["page"]) for n in lens) * 4 + case["B"] * 8
    if case["kind"] == "read":
        return {"bytes": int(2 * T * Hk * D * (wk + w)) + tables, "flops": 2 * T * Hk * D}
    if case["kind"] == "append":
        norm = 4 * D if case["norm"] else 0  # operations of a head's norm
        positions = set()
        for n, m in zip(new, lens):
            positions.update(range(m - n, m))
        # q, k and v in, q out, codes out and in again, the rows read back out
        return {"bytes": int(T * D * (2 * Hq * w + 2 * Hk * (2 * w + 2 * wk)))
                + len(positions) * case["rot"] * 4 + tables,
                "flops": T * (Hq + Hk) * (3 * case["rot"] + norm) + 8 * T * Hk * D}
    window = case["window"] or 1 << 40
    pairs = sum(_pairs(m - n, m, window) for n, m in zip(new, lens))
    keys = sum(min(m, n + window - 1) for n, m in zip(new, lens))
    return {"bytes": int(2 * keys * Hk * D * wk) + int(2 * T * Hq * D * w)
            + (T * Hq * 4 if case["lse"] else 0) + tables, "flops": 4 * D * Hq * pairs}


def _pairs(first, end, window):
    """Pairs of rows at places first .. end - 1 with the keys they see."""
    def upto(p):  # sum of min(i + 1, window) over i < p
        few = min(p, window)
        return few * (few + 1) // 2 + (p - few) * window
    return upto(end) - upto(first)


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


def _exact_code(x):
    """What MXFP4 holds of x [.., D], in 64 bits: multiples of the step of each
    magnitude's binade, halves to the even one."""
    b = x.unflatten(-1, (-1, _BLOCK))
    part, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    two = torch.exp2(e.double() - 3.0 + (part >= 0.875))
    a = (b / two).abs()
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    y = (torch.round(a / step) * step).clamp_max(6.0) * two
    return torch.where(b < 0, -y, y).flatten(-2)


def _exact_values(case, s, name, ids, h):
    """Head h of the pages `ids` of a pool in 64 bits [tokens, D]."""
    x = s[name + "_pages"][:, h]
    if case["kv"] == "mx":
        x = x[ids].reshape(-1, case["D"] // 2).to(torch.int64)
        y = torch.empty(x.shape[0], case["D"], dtype=torch.float64, device="cuda")
        for odd in (0, 1):
            c = x >> 4 if odd else x & 15
            e, m = c >> 1 & 3, c & 1
            # exponent 0: m / 2; else (1 + m / 2) 2^(e - 1)
            v = torch.where(e == 0, 0.5 * m, torch.ldexp(1.0 + 0.5 * m.double(), e - 1))
            y[:, odd::2] = torch.where(c >= 8, -v, v)
        two = s[name + "_scales"][:, h][ids].reshape(-1, case["D"] // _BLOCK).double() - 127.0
        return y * torch.exp2(two).repeat_interleave(_BLOCK, -1)
    if case["kv"] == "fp8":
        y = x.view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
        y = y * s[name + "_scales"].double()[ids, h][:, None, None]
    else:
        y = x[ids].double()
    return y.reshape(-1, case["D"])


def exact(case, seed):
    s = prepare(case, seed)
    new, lens = _lengths(case)
    starts = [sum(new[:b]) for b in range(len(new))]
    Hq, Hk, D, page = case["Hq"], case["Hk"], case["D"], case["page"]
    if case["kind"] == "append":
        q, k = (torch.empty(s[x].shape, dtype=torch.float64, device="cuda") for x in ("q", "k"))
        for at, n, m in zip(starts, new, lens):
            c, z = s["cos"][m - n:m, None], s["sin"][m - n:m, None]
            for x, out in (("q", q), ("k", k)):
                out[at:at + n] = _exact_turn(s[x][at:at + n], s[x + "_weight"], c, z,
                                             s["interleaved"])
        return q, _exact_code(k), _exact_code(s["v"].double())
    if case["kind"] == "read":
        out = [torch.empty(sum(new), Hk, D, dtype=torch.float64, device="cuda") for _ in range(2)]
        for b, (at, n, m) in enumerate(zip(starts, new, lens)):
            ids = s["block_table"][b, :-(-m // page)].long()
            for h in range(Hk):
                for x, name in zip(out, ("k", "v")):
                    x[at:at + n, h] = _exact_values(case, s, name, ids, h)[m - n:m]
        return tuple(out)
    group = Hq // Hk
    o = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for b, (at, n, m) in enumerate(zip(starts, new, lens)):
        ids = s["block_table"][b, :-(-m // page)].long()
        hide = torch.ones(n, m, dtype=torch.bool, device="cuda").triu(m - n + 1)
        if case["window"]:
            hide |= torch.ones(n, m, dtype=torch.bool, device="cuda").tril(m - n - case["window"])
        key = torch.arange(m, dtype=torch.float64, device="cuda")
        far = key[None, :] - key[m - n:, None]
        for h in range(Hk):
            k, v = (_exact_values(case, s, name, ids, h)[:m] for name in ("k", "v"))
            for j in range(group):
                head = h * group + j
                x = s["q"][at:at + n, head].double() @ k.T / math.sqrt(D)
                if case["cap"]:
                    x = case["cap"] * torch.tanh(x / case["cap"])
                if case["slopes"]:
                    x = x + s["slopes"][head].double() * far
                x = x.masked_fill(hide, -math.inf)
                total = torch.logsumexp(x, -1)
                o[at:at + n, head] = torch.exp(x - total[:, None]) @ v
                lse[at:at + n, head] = total
    return (o, lse) if case["lse"] else o
