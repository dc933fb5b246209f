"""CPU tests of what MXFP4 pools, kv_read_paged and shaped scores refuse: the torch
front (meta tensors, no GPU) and the C-ABI, whose refusals come before any HIP call,
and the layout of their descriptors."""

import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

from neptune_hip import _abi, ops

ROOT = Path(__file__).resolve().parents[1]
bf16, f16, f32, u8, i32 = torch.bfloat16, torch.float16, torch.float32, torch.uint8, torch.int32
INVALID, UNSUPPORTED, SMALL, NO_DEVICE = (_abi.ERR_INVALID_ARGUMENT, _abi.ERR_UNSUPPORTED,
                                          _abi.ERR_WORKSPACE_TOO_SMALL, _abi.ERR_NO_DEVICE)


def meta(*shape, dtype=bf16):
    return torch.empty(shape, dtype=dtype, device="meta")


def _pools(D=128, dtype=u8, scale=u8, layout="head"):
    def lay(width, t):
        if layout == "head":
            return meta(20, 2, 64, width, dtype=t)
        return meta(20, 64, 2, width, dtype=t).permute(0, 2, 1, 3)
    return dict(k_pages=lay(D // 2, dtype), v_pages=lay(D // 2, dtype),
                k_scales=lay(D // 32, scale), v_scales=lay(D // 32, scale),
                block_table=meta(3, 8, dtype=i32), seq_lens=meta(3, dtype=i32),
                cu_seqlens=meta(4, dtype=i32))


def _append(**kw):
    a = dict(k=meta(10, 2, 128), v=meta(10, 2, 128), q=meta(10, 8, 128), **_pools())
    a.update(kw)
    return ops.kv_append_paged(**a)


def _attend(**kw):
    a = dict(q=meta(10, 8, 128), **_pools())
    a.update(kw)
    return ops.attention_paged(**a)


def _read(**kw):
    a = dict(tokens=10, **_pools())
    a.update(kw)
    return ops.kv_read_paged(**a)


@pytest.mark.parametrize("call", [_append, _attend, _read])
@pytest.mark.parametrize("kw,match", [
    ({}, "device tensors"), (_pools(layout="token"), "device tensors"),
    (_pools(scale=torch.float8_e8m0fnu), "device tensors"),
    (_pools(dtype=torch.float4_e2m1fn_x2, scale=torch.float8_e8m0fnu), "device tensors"),
    (dict(k_scales=meta(20, 2, 64, 2, dtype=u8)), "k_scales"),
    (dict(v_scales=meta(20, 64, 2, 4, dtype=u8)), "v_scales"),
    (dict(v_scales=meta(20, 2, dtype=f32)), "v_scales"),
    (dict(v_scales=None), "v_scales"),
    (dict(k_scales=meta(20, 2, 4, 64, dtype=u8).transpose(2, 3)), "k_scales"),
    (dict(v_pages=meta(20, 2, 64, 64, dtype=torch.float8_e4m3fn)), "pools must be"),
    (dict(v_pages=meta(20, 2, 64, 32, dtype=u8)), "matching"),
    (dict(k_pages=meta(20, 2, 64, 64, dtype=u8).transpose(1, 2), v_pages=meta(20, 64, 2, 64, dtype=u8)),
     "k_scales"),
])
def test_pools_front(call, kw, match):
    with pytest.raises(ValueError, match=match):
        call(**kw)


@pytest.mark.parametrize("kw,match", [
    (dict(q=meta(10, 8, 64)), "q is"), (dict(k=meta(10, 2, 64), v=meta(10, 2, 64)), "k is"),
    (dict(k=meta(10, 2, 128, dtype=f32), v=meta(10, 2, 128, dtype=f32)), "float16 or bfloat16"),
])
def test_append_front(kw, match):
    with pytest.raises(ValueError, match=match):
        _append(**kw)


@pytest.mark.parametrize("kw,match", [
    (dict(softcap=0.0), "softcap"), (dict(softcap=-1.0), "softcap"),
    (dict(softcap=math.nan), "softcap"), (dict(window=0), "window"), (dict(window=-5), "window"),
    (dict(slopes=meta(2, dtype=f32)), "slopes"), (dict(slopes=meta(8)), "slopes"),
    (dict(slopes=meta(16, dtype=f32)[::2]), "slopes"),
    (dict(softcap=30.0, window=7, slopes=meta(8, dtype=f32)), "device tensors"),
    (dict(scale=0.0), "scale"),
])
def test_scores_front(kw, match):
    with pytest.raises(ValueError, match=match):
        _attend(**kw)


@pytest.mark.parametrize("kw,match", [
    (dict(tokens=None), "tokens"), (dict(dtype=torch.float64), "dtype"),
    (dict(out=meta(10, 2, 128)), "pair"), (dict(out=(meta(10, 2, 128), None)), "pair"),
    (dict(out=(meta(10, 2, 128), meta(10, 2, 64))), "v_out is"),
    (dict(out=(meta(10, 2, 128), meta(10, 2, 128)), dtype=f16), "k_out is"),
    (dict(out=(meta(9, 2, 128), meta(9, 2, 128))), "k_out is"),
    (dict(cu_seqlens=None), "one new token"),
    (dict(k_scales=None, v_scales=None), "k_scales"),  # then E4M3 codes
])
def test_read_front(kw, match):
    with pytest.raises(ValueError, match=match):
        _read(**kw)


def test_other_pools_take_no_bytes_of_scales():
    pool = meta(20, 2, 64, 128)
    scales = meta(20, 2, 64, 4, dtype=u8)
    with pytest.raises(ValueError, match="E4M3 pools only"):
        _attend(k_pages=pool, v_pages=pool, k_scales=scales, v_scales=scales)


# ---- C-ABI -----------------------------------------------------------------

FAR = 1 << 44  # placeholder addresses, far apart: no call here gets past validation


def _ptr(i):
    return (i + 1) * FAR


@pytest.fixture(scope="module")
def lib():
    return _abi.load_library()


def _set(desc, kw):
    for k, v in kw.items():
        if k.endswith("stride"):
            getattr(desc, k)[:] = v
        else:
            setattr(desc, k, v)
    return desc


def _pages(**kw):
    p = _abi.PagedKvDesc()
    p.num_pages, p.page_size, p.max_pages = 64, 64, 32
    p.k_stride[:] = p.v_stride[:] = (2 * 64 * 64, 64 * 64, 64)
    return _set(p, kw)


def _mx(**kw):
    m = _abi.MxDesc()
    m.k_stride[:] = m.v_stride[:] = (2 * 64 * 4, 64 * 4, 4)
    return _set(m, kw)


def _ref(desc):
    return None if desc is None else ctypes.byref(desc)


def _append_call(lib, pages=None, mx=None, ptrs=None, **kw):
    d = _abi.AppendDesc()
    d.tokens, d.batch, d.heads_q, d.heads_kv, d.head_dim = 10, 3, 8, 2, 128
    d.rot_dim, d.table_len = 32, 100
    d.dtype, d.kv_dtype = _abi.DTYPE_BF16, _abi.DTYPE_MXFP4
    p = [_ptr(i) for i in range(15)]
    # 0 k, 1 v, 2 q, 3 qw, 4 kw, 5 cos, 6 sin, 7 table, 8 cu, 9 lens, 10 kp, 11 vp, 12 ks, 13 vs, 14 qo
    for i, v in (ptrs or {}).items():
        p[i] = v
    return lib.neptune_kv_append_paged_mx(
        ctypes.byref(_set(d, kw)), _ref(_pages(**(pages or {}))),
        None if mx == "none" else _ref(_mx(**(mx or {}))), *p, None)


def _attend_call(lib, pages=None, mx=None, score=None, ptrs=None, ws=1 << 30, **kw):
    d = _abi.AttnPagedDesc()
    d.tokens, d.batch, d.heads_q, d.heads_kv, d.head_dim, d.seq_kv = 10, 3, 8, 2, 128, 2000
    d.dtype, d.kv_dtype = _abi.DTYPE_BF16, _abi.DTYPE_MXFP4
    p = [_ptr(i) for i in range(12)]
    # 0 q, 1 kp, 2 vp, 3 ks, 4 vs, 5 slopes, 6 table, 7 cu, 8 lens, 9 o, 10 lse, 11 workspace
    for i, v in (ptrs or {}).items():
        p[i] = v
    sc = None
    if score is not None:
        sc = _set(_abi.ScoreDesc(), score)
    return lib.neptune_attn_paged_ext(
        ctypes.byref(_set(d, kw)), _ref(_pages(**(pages or {}))),
        None if mx == "none" else _ref(_mx(**(mx or {}))), _ref(sc), *p, ws, None)


def _read_call(lib, pages=None, mx=None, ptrs=None, **kw):
    d = _abi.KvReadDesc()
    d.tokens, d.batch, d.heads_kv, d.head_dim = 10, 3, 2, 128
    d.dtype, d.kv_dtype = _abi.DTYPE_F32, _abi.DTYPE_MXFP4
    p = [_ptr(i) for i in range(9)]
    # 0 kp, 1 vp, 2 ks, 3 vs, 4 table, 5 cu, 6 lens, 7 ko, 8 vo
    for i, v in (ptrs or {}).items():
        p[i] = v
    return lib.neptune_kv_read_paged(
        ctypes.byref(_set(d, kw)), _ref(_pages(**(pages or {}))),
        None if mx == "none" else _ref(_mx(**(mx or {}))), *p, None)


# pools of MXFP4, whatever the entry point
SHARED = [
    (dict(tokens=0), INVALID), (dict(batch=-1), INVALID), (dict(heads_kv=0), INVALID),
    (dict(head_dim=96), UNSUPPORTED), (dict(head_dim=48), UNSUPPORTED),
    (dict(mx="none"), INVALID), (dict(mx=dict(k_stride=(512, 256, 0))), INVALID),
    (dict(mx=dict(v_stride=(512, 256, 6))), UNSUPPORTED),
    (dict(mx=dict(v_stride=(1 << 62, 256, 4))), UNSUPPORTED),
    (dict(pages=dict(num_pages=0)), INVALID), (dict(pages=dict(k_stride=(0, 4096, 64))), INVALID),
    (dict(pages=dict(v_stride=(8192, 4096, 72))), UNSUPPORTED),
    (dict(pages=dict(num_pages=1 << 31, k_stride=(16, 4096, 64), v_stride=(16, 4096, 64))),
     UNSUPPORTED),
]


def _check(status, got, lib):
    assert got == status and lib.neptune_last_error()


def _reachable(lib, status):
    if status == NO_DEVICE and lib.neptune_device_count() > 0:
        pytest.skip("a HIP device is visible; the no-device path is not reachable")


@pytest.mark.parametrize("kw,status", SHARED + [
    (dict(dtype=_abi.DTYPE_F32), UNSUPPORTED), (dict(kv_dtype=_abi.DTYPE_BF16), UNSUPPORTED),
    (dict(kv_dtype=_abi.DTYPE_FP8_E4M3), UNSUPPORTED),
    (dict(ptrs={12: None}), INVALID), (dict(ptrs={13: None}), INVALID),
    (dict(ptrs={12: _ptr(12) + 2}), UNSUPPORTED), (dict(ptrs={10: None}), INVALID),
    (dict(ptrs={10: _ptr(10) + 8}), UNSUPPORTED),
    (dict(ptrs={13: _ptr(12) + 8}), INVALID),          # the scales' pools over each other
    (dict(ptrs={12: _ptr(10) + 64}), INVALID),         # scales over codes
    (dict(ptrs={13: _ptr(1)}), INVALID),               # scales over v
    (dict(ptrs={14: _ptr(12)}), INVALID),              # qo over scales
    (dict(ptrs={8: None}), INVALID), (dict(rot_dim=12), UNSUPPORTED), (dict(rot_dim=132), INVALID),
    (dict(tokens=1 << 31), UNSUPPORTED),
    ({}, NO_DEVICE), (dict(ptrs={14: _ptr(2)}), NO_DEVICE), (dict(dtype=_abi.DTYPE_F16), NO_DEVICE),
    (dict(head_dim=64, pages=dict(k_stride=(4096, 2048, 32), v_stride=(4096, 2048, 32)),
          mx=dict(k_stride=(256, 128, 2), v_stride=(256, 128, 2)), ptrs={12: _ptr(12) + 2}),
     NO_DEVICE),
    (dict(pages=dict(page_size=1)), NO_DEVICE),
    # codes and scales of a slot side by side in one buffer share no byte
    (dict(pages=dict(k_stride=(20480, 10240, 160), v_stride=(20480, 10240, 160)),
          mx=dict(k_stride=(20480, 10240, 160), v_stride=(20480, 10240, 160)),
          ptrs={11: _ptr(10) + 64, 12: _ptr(10) + 128, 13: _ptr(10) + 132}), NO_DEVICE),
    (dict(pages=dict(k_stride=(20480, 10240, 160), v_stride=(20480, 10240, 160)),
          mx=dict(k_stride=(20480, 10240, 160), v_stride=(20480, 10240, 160)),
          ptrs={11: _ptr(10) + 64, 12: _ptr(10) + 128, 13: _ptr(10) + 128}), INVALID),
])
def test_append_abi(lib, kw, status):
    _reachable(lib, status)
    _check(status, _append_call(lib, **kw), lib)


@pytest.mark.parametrize("kw,status", SHARED + [
    (dict(heads_q=9), INVALID), (dict(dtype=_abi.DTYPE_F32), UNSUPPORTED),
    (dict(kv_dtype=_abi.DTYPE_F16), UNSUPPORTED),
    (dict(dtype=_abi.DTYPE_F16, kv_dtype=_abi.DTYPE_FP8_E4M3), UNSUPPORTED),
    (dict(score=dict(softcap=-1.0)), INVALID), (dict(score=dict(softcap=math.nan)), INVALID),
    (dict(score=dict(softcap=math.inf)), INVALID), (dict(score=dict(softcap=1e-30)), UNSUPPORTED),
    (dict(score=dict(softcap=1e30)), UNSUPPORTED), (dict(score=dict(window=-1)), INVALID),
    (dict(pages=dict(page_size=24, max_pages=100)), UNSUPPORTED),
    (dict(pages=dict(max_pages=31)), INVALID),
    (dict(pages=dict(k_stride=(1 << 31, 4096, 64))), UNSUPPORTED),   # pages 2 GiB apart
    (dict(pages=dict(v_stride=(64, 1 << 36, 1 << 25))), UNSUPPORTED),  # tokens over 2 GiB
    (dict(mx=dict(k_stride=(1 << 31, 256, 4))), UNSUPPORTED),
    (dict(mx=dict(v_stride=(4, 1 << 36, 1 << 25))), UNSUPPORTED),
    (dict(ptrs={3: None}), INVALID), (dict(ptrs={4: _ptr(4) + 1}), UNSUPPORTED),
    (dict(ptrs={9: _ptr(0)}), INVALID), (dict(ptrs={9: _ptr(3)}), INVALID),
    (dict(ptrs={9: _ptr(4) + 1024}), INVALID), (dict(ptrs={11: None}), SMALL), (dict(ws=16), SMALL),
    ({}, NO_DEVICE), (dict(ptrs={5: None}), NO_DEVICE), (dict(dtype=_abi.DTYPE_F16), NO_DEVICE),
    (dict(score=dict(softcap=30.0, window=100)), NO_DEVICE),
    (dict(score=dict(window=1 << 40)), NO_DEVICE),
    (dict(mx=dict(k_stride=(8, 1 << 33, 4)), pages=dict(k_stride=(4096, 1 << 35, 64))), NO_DEVICE),
])
def test_attend_abi(lib, kw, status):
    _reachable(lib, status)
    _check(status, _attend_call(lib, **kw), lib)


@pytest.mark.parametrize("kw,status", [
    (dict(), NO_DEVICE), (dict(kv_dtype=_abi.DTYPE_F16), UNSUPPORTED),
    (dict(kv_dtype=_abi.DTYPE_FP8_E4M3), NO_DEVICE),
    (dict(kv_dtype=_abi.DTYPE_FP8_E4M3, ptrs={4: None}), INVALID),
])
def test_attend_abi_other_pools(lib, kw, status):
    """The extended entry point over 16-bit and E4M3 pools: no MXFP4 descriptor."""
    _reachable(lib, status)
    pages = dict(k_stride=(2 * 64 * 128, 64 * 128, 128), v_stride=(2 * 64 * 128, 64 * 128, 128))
    got = _attend_call(lib, **{**dict(kv_dtype=_abi.DTYPE_BF16, mx="none", pages=pages), **kw})
    _check(status, got, lib)


@pytest.mark.parametrize("kw,status", SHARED + [
    (dict(dtype=_abi.DTYPE_FP8_E4M3), UNSUPPORTED), (dict(kv_dtype=_abi.DTYPE_F32), UNSUPPORTED),
    (dict(ptrs={0: None}), INVALID), (dict(ptrs={2: None}), INVALID), (dict(ptrs={4: None}), INVALID),
    (dict(ptrs={5: None}), INVALID), (dict(ptrs={6: None}), INVALID), (dict(ptrs={7: None}), INVALID),
    (dict(ptrs={8: _ptr(7) + 16}), INVALID), (dict(ptrs={7: _ptr(0)}), INVALID),
    (dict(ptrs={8: _ptr(3)}), INVALID), (dict(ptrs={8: _ptr(8) + 4}), UNSUPPORTED),
    (dict(ko_stride=(256, 0)), INVALID), (dict(vo_stride=(258, 128)), UNSUPPORTED),
    (dict(tokens=1 << 31), UNSUPPORTED), (dict(batch=1 << 17), UNSUPPORTED),
    (dict(kv_dtype=_abi.DTYPE_FP8_E4M3, mx="none", ptrs={8: _ptr(2)},
          pages=dict(k_stride=(16384, 8192, 128), v_stride=(16384, 8192, 128))), INVALID),
    ({}, NO_DEVICE), (dict(dtype=_abi.DTYPE_F16), NO_DEVICE), (dict(pages=dict(page_size=1)), NO_DEVICE),
    (dict(tokens=3, ptrs={5: None}), NO_DEVICE),
    # keys and values side by side
    (dict(ko_stride=(512, 128), vo_stride=(512, 128), ptrs={8: _ptr(7) + 1024}), NO_DEVICE),
    (dict(kv_dtype=_abi.DTYPE_BF16, mx="none", ptrs={2: None, 3: None},
          pages=dict(k_stride=(16384, 8192, 128), v_stride=(16384, 8192, 128))), NO_DEVICE),
])
def test_read_abi(lib, kw, status):
    _reachable(lib, status)
    _check(status, _read_call(lib, **kw), lib)


def test_plain_entry_points_refuse_mxfp4(lib):
    d = _abi.AttnPagedDesc()
    d.tokens, d.batch, d.heads_q, d.heads_kv, d.head_dim, d.seq_kv = 10, 3, 8, 2, 128, 2000
    d.dtype, d.kv_dtype = _abi.DTYPE_BF16, _abi.DTYPE_MXFP4
    p = [_ptr(i) for i in range(11)]
    assert lib.neptune_attn_paged(ctypes.byref(d), _ref(_pages()), *p, 1 << 30, None) == UNSUPPORTED
    a = _abi.AppendDesc()
    a.tokens, a.batch, a.heads_q, a.heads_kv, a.head_dim = 10, 3, 8, 2, 128
    a.dtype, a.kv_dtype = _abi.DTYPE_BF16, _abi.DTYPE_MXFP4
    p = [_ptr(i) for i in range(15)]
    assert lib.neptune_kv_append_paged(ctypes.byref(a), _ref(_pages()), *p, None) == UNSUPPORTED
    c = _abi.DecodeDesc()
    c.batch, c.heads_q, c.heads_kv, c.seq_kv, c.head_dim = 3, 8, 2, 2000, 128
    c.q_dtype, c.kv_dtype = _abi.DTYPE_BF16, _abi.DTYPE_MXFP4
    n = ctypes.c_size_t()
    assert lib.neptune_decode_workspace_bytes(ctypes.byref(c), ctypes.byref(n)) == UNSUPPORTED


def test_workspace_is_that_of_other_pools(lib):
    sizes = []
    for kv in (_abi.DTYPE_BF16, _abi.DTYPE_MXFP4):
        d = _abi.AttnPagedDesc()
        d.tokens, d.batch, d.heads_q, d.heads_kv, d.head_dim, d.seq_kv = 4, 2, 32, 8, 128, 9000
        d.dtype, d.kv_dtype = _abi.DTYPE_BF16, kv
        n = ctypes.c_size_t()
        assert lib.neptune_attn_paged_workspace_bytes(ctypes.byref(d), ctypes.byref(n)) == _abi.OK
        sizes.append(n.value)
    assert sizes[0] == sizes[1] > 0


def test_null_descriptors(lib):
    assert lib.neptune_kv_append_paged_mx(None, None, None, *[FAR] * 15, None) == INVALID
    assert lib.neptune_kv_read_paged(None, None, None, *[FAR] * 9, None) == INVALID
    assert lib.neptune_attn_paged_ext(None, None, None, None, *[FAR] * 12, 0, None) == INVALID
    d = _abi.KvReadDesc(10, 3, 2, 128, (0, 0), (0, 0), _abi.DTYPE_F32, _abi.DTYPE_MXFP4)
    assert lib.neptune_kv_read_paged(ctypes.byref(d), None, None, *[FAR] * 9, None) == INVALID


def test_descriptors_match_the_c_header(tmp_path):
    pairs = [("neptune_mx_desc", _abi.MxDesc), ("neptune_kv_read_desc", _abi.KvReadDesc),
             ("neptune_score_desc", _abi.ScoreDesc)]
    lines = [f'printf("%zu\\n", offsetof({c}, {f}));' for c, cls in pairs for f, _ in cls._fields_]
    lines += [f'printf("%zu\\n", sizeof({c}));' for c, _ in pairs]
    src = tmp_path / "layout.c"
    src.write_text("#include <stddef.h>\n#include <stdio.h>\n#include \"neptune_hip.h\"\n"
                   "int main(void) {" + "\n".join(lines) + "return 0; }")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", "-I", str(ROOT / "include"), str(src), "-o", str(exe)],
                   check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True,
                                          text=True).stdout.split()]
    want = [getattr(cls, f).offset for _, cls in pairs for f, _ in cls._fields_]
    assert got == want + [ctypes.sizeof(cls) for _, cls in pairs]
