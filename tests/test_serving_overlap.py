"""CPU tests of which outputs qk_norm_rope, kv_append_paged and attention_paged
take beside their inputs: heads side by side in one buffer, but no shared byte;
and of tensors that are one row expanded. Refusals come before any HIP call."""

import ctypes
import random

import pytest
import torch

from neptune_hip import _abi, ops

INVALID, UNSUPPORTED, NO_DEVICE = (_abi.ERR_INVALID_ARGUMENT, _abi.ERR_UNSUPPORTED,
                                   _abi.ERR_NO_DEVICE)
FAR = 1 << 44
bf16, f32, i32 = torch.bfloat16, torch.float32, torch.int32


@pytest.fixture(scope="module")
def lib():
    lib = _abi.load_library()
    if lib.neptune_device_count() > 0:
        pytest.skip("a HIP device is visible; the no-device path is not reachable")
    return lib


def _rope(lib, sizes, D, q, k, qo, ko):
    """Each tensor (address, strides); sizes (B, Hq, Hk, S)."""
    d = _abi.RopeDesc()
    d.batch, d.heads_q, d.heads_kv, d.seq = sizes
    d.head_dim, d.rot_dim, d.table_len, d.dtype, d.eps = D, D, 100, _abi.DTYPE_BF16, 1e-6
    for name, t in (("q", q), ("k", k), ("qo", qo), ("ko", ko)):
        getattr(d, name + "_stride")[:] = t[1]
    return lib.neptune_qk_norm_rope(
        ctypes.byref(d), q[0], k[0], None, None, 90 * FAR, 91 * FAR, 92 * FAR, qo[0], ko[0], None)


def _bytes(t, sizes, D):
    (p, st), (B, H, S) = t, sizes
    return {p + 2 * (b * st[0] + h * st[1] + s * st[2]) + x
            for b in range(B) for h in range(H) for s in range(S) for x in range(0, 2 * D, 16)}


def test_rope_takes_what_shares_no_byte(lib):
    """Against the sets of bytes, 16 at a time, of random small tensors."""
    rng, D, seen = random.Random(5), 32, {INVALID: 0, NO_DEVICE: 0}
    for _ in range(1500):
        B, Hq, Hk, S = (rng.choice((1, 2, 3)) for _ in range(4))
        row = rng.choice((D, D + 8, (Hq + Hk) * D, 2 * D))
        order = rng.sample(range(3), 3)

        def strides(heads):
            st, run = [0, 0, 0], row
            for axis in order:  # innermost first
                st[axis] = run
                run *= (B, Hq + Hk, S)[axis] if rng.random() < 0.8 else heads
            return tuple(st)

        common = strides(Hq)
        one = lambda base, heads: (base + 16 * rng.choice((0, 4, 4 * Hq, 8, 12, 1, Hq * row // 8,
                                                           rng.randrange(200))),
                                   common if rng.random() < 0.8 else strides(heads))
        q, k = one(FAR, Hq), one(FAR, Hk)
        qo = q if rng.random() < 0.5 else one(rng.choice((FAR, 2 * FAR)), Hq)
        ko = k if rng.random() < 0.5 else one(rng.choice((FAR, 2 * FAR)), Hk)
        sets = {id(t): _bytes(t, (B, n, S), D) for t, n in ((q, Hq), (k, Hk), (qo, Hq), (ko, Hk))}
        same = lambda a, b, n: a[0] == b[0] and all(
            x == y for x, y, m in zip(a[1], b[1], (B, n, S)) if m > 1)
        bad = bool(sets[id(qo)] & sets[id(ko)] or sets[id(qo)] & sets[id(k)] or
                   sets[id(ko)] & sets[id(q)])
        bad = bad or (not same(qo, q, Hq) and bool(sets[id(qo)] & sets[id(q)]))
        bad = bad or (not same(ko, k, Hk) and bool(sets[id(ko)] & sets[id(k)]))
        want = INVALID if bad else NO_DEVICE
        got = _rope(lib, (B, Hq, Hk, S), D, q, k, qo, ko)
        assert got == want, ((B, Hq, Hk, S), q, k, qo, ko)
        seen[want] += 1
    assert min(seen.values()) > 300


def test_rope_large_and_tangled(lib):
    B, Hq, Hk, S, D = 64, 32, 8, 32768, 128
    row = (Hq + 2 * Hk) * D
    st = (S * row, D, row)
    q, k = (FAR, st), (FAR + 2 * Hq * D, st)
    assert _rope(lib, (B, Hq, Hk, S), D, q, k, q, k) == NO_DEVICE
    moved = (FAR + 2 * (Hq - 1) * D, st)  # q's last head
    assert _rope(lib, (B, Hq, Hk, S), D, q, moved, q, moved) == INVALID
    # strides that take thousands of tries count as sharing
    odd = (FAR + 16, (8 * 1000003, 8 * 999983, 8 * 1000033))
    assert _rope(lib, (64, 64, 64, 64), D, (FAR, (8 * 1000211, 8 * 999979, 8 * 1000099)), k,
                 odd, (2 * FAR, (0, 0, 0))) == INVALID


def _append(lib, kp, vp, q=None, k=None, v=None, qo=None, tokens=10, fp8=False, batch=3,
            cu=True):
    """Pools (address, strides); q, k, v, qo (address, strides) or apart."""
    d = _abi.AppendDesc()
    d.tokens, d.batch, d.heads_q, d.heads_kv, d.head_dim = tokens, batch, 8, 2, 128
    d.dtype, d.kv_dtype = _abi.DTYPE_BF16, _abi.DTYPE_FP8_E4M3 if fp8 else _abi.DTYPE_BF16
    for name, t in (("q", q), ("k", k), ("v", v), ("qo", qo)):
        if t:
            getattr(d, name + "_stride")[:] = t[1]
    at = [t[0] if t else (20 + i) * FAR for i, t in enumerate((k, v, q, qo))]
    p = _abi.PagedKvDesc()
    p.num_pages, p.page_size, p.max_pages = 1000, 16, 32
    p.k_stride[:], p.v_stride[:] = kp[1], vp[1]
    far = [(40 + i) * FAR for i in range(5)]
    far[1] = far[1] if cu else None
    return lib.neptune_kv_append_paged(
        ctypes.byref(d), ctypes.byref(p), *at[:3], None, None, None, None, *far[:3], kp[0], vp[0],
        *far[3:], at[3], None)


def test_append_pools_share_no_byte(lib):
    page, Hk, D = 16, 2, 128
    dense = (Hk * page * D, page * D, D)
    assert _append(lib, (FAR, dense), (FAR, dense)) == INVALID
    assert _append(lib, (FAR, dense), (FAR + 2 * 999 * Hk * page * D, dense)) == INVALID
    assert _append(lib, (FAR, dense), (FAR + 2 * 1000 * Hk * page * D, dense)) == NO_DEVICE
    # K and V of a page, of a head, of a token side by side
    for st, off in (((2 * Hk * page * D, page * D, D), Hk * page * D),
                    ((2 * Hk * page * D, 2 * page * D, D), page * D),
                    ((2 * Hk * page * D, 2 * page * D, 2 * D), D),
                    ((2 * Hk * page * D, D, 2 * Hk * D), Hk * D)):
        assert _append(lib, (FAR, st), (FAR + 2 * off, st)) == NO_DEVICE
        assert _append(lib, (FAR, st), (FAR + off, st), fp8=True) == NO_DEVICE
        assert _append(lib, (FAR, st), (FAR + 2 * off - 16, st)) == INVALID


def test_append_in_one_projection(lib):
    dense, other = (4096, 2048, 128), (7 * FAR, (4096, 2048, 128))
    st = (12 * 128, 128)
    q, k, v = ((FAR + 2 * 128 * h, st) for h in (0, 8, 10))
    assert _append(lib, (6 * FAR, dense), other, q, k, v, q) == NO_DEVICE
    assert _append(lib, (6 * FAR, dense), other, q, k, v, v) == INVALID
    over = (FAR + 2 * 128 * 7, st)  # q's last head is k's first
    assert _append(lib, (6 * FAR, dense), other, q, over, v, q) == INVALID
    assert _append(lib, (6 * FAR, dense), other, q, k, over, q) == INVALID


def meta(*shape, dtype=bf16):
    return torch.empty(shape, dtype=dtype, device="meta")


def test_expanded_rows_are_refused():
    """All strides zero would read as contiguous, far past the row."""
    row = lambda *shape: meta(128).expand(*shape)
    cache = dict(k_pages=meta(20, 2, 64, 128), v_pages=meta(20, 2, 64, 128),
                 block_table=meta(3, 8, dtype=i32), seq_lens=meta(3, dtype=i32),
                 cu_seqlens=meta(4, dtype=i32))
    rope = dict(cos=meta(100, 64, dtype=f32), sin=meta(100, 64, dtype=f32),
                positions=meta(2, 5, dtype=i32))
    for call in (
            lambda: ops.qk_norm_rope(row(2, 8, 5, 128), meta(2, 2, 5, 128), **rope),
            lambda: ops.qk_norm_rope(meta(2, 8, 5, 128), row(2, 2, 5, 128), **rope),
            lambda: ops.kv_append_paged(row(10, 2, 128), meta(10, 2, 128), **cache),
            lambda: ops.kv_append_paged(meta(10, 2, 128), row(10, 2, 128), **cache),
            lambda: ops.kv_append_paged(meta(10, 2, 128), meta(10, 2, 128), q=row(10, 8, 128),
                                        **cache),
            lambda: ops.attention_paged(row(10, 8, 128), **cache)):
        with pytest.raises(ValueError, match="one row expanded"):
            call()


@pytest.mark.parametrize("scale", [0.0, 1e-60])
def test_a_scale_of_zero_is_not_the_default(scale):
    with pytest.raises(ValueError, match="scale"):
        ops.attention_paged(meta(10, 8, 128), meta(20, 2, 64, 128), meta(20, 2, 64, 128),
                            meta(3, 8, dtype=i32), meta(3, dtype=i32), meta(4, dtype=i32),
                            scale=scale)


def test_batch_bound():
    """Every work-group looks through all sequences: a launch takes 65536."""
    w = ops.attention_paged_workspace_bytes
    assert w(1, 1 << 16, 8, 2, 128, 2000) >= 0
    with pytest.raises(_abi.NeptuneUnsupported, match="too large"):
        w(1, (1 << 16) + 1, 8, 2, 128, 2000)


def test_append_batch_bound(lib):
    """With cu_seqlens likewise; one token per sequence needs no search."""
    pools = (6 * FAR, (4096, 2048, 128)), (7 * FAR, (4096, 2048, 128))
    assert _append(lib, *pools, batch=1 << 16) == NO_DEVICE
    assert _append(lib, *pools, batch=(1 << 16) + 1) == UNSUPPORTED
    many = (1 << 16) + 1
    assert _append(lib, *pools, batch=many, tokens=many, cu=False) == NO_DEVICE
